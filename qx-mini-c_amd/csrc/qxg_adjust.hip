// Penalties, biases, temperature and grammar mask on logits, with the best tokens (qxg_adjust_logits).
#include "qxg_dev.h"
#include "qxg_ops.h"

namespace {
constexpr int PER = QXS_SLICE / 256;    // tokens a thread
constexpr uint32_t HAS_BIAS = 0x40000000u, SEEN = 0x80000000u;

// Order of a logit as an unsigned number, 0 (never picked) for -inf and NaN; -0 as +0.  A key is that
// over ~token: larger first, then the lower token; no two are alike.
DEV uint32_t rank_of(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
DEV uint64_t key_of(uint32_t rank, uint32_t v) { return rank ? (uint64_t)rank << 32 | (uint32_t)~v : 0; }
DEV float key_value(uint64_t k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
// The n-th largest of the wave's 64 keys (unlike ones but for 0), found a bit at a time: 0 when fewer are
// not 0.  The token bits are searched only where several keys share the n-th's rank.
DEV uint64_t wave_nth(uint64_t k, uint32_t n) {
    const uint32_t hi = (uint32_t)(k >> 32), lo = (uint32_t)k;
    uint32_t th = 0;
#pragma unroll
    for (int b = 31; b >= 0; --b)
        if ((uint32_t)__popcll(__ballot(hi >= (th | 1u << b))) >= n) th |= 1u << b;
    if (th == 0) return 0;
    const uint32_t above = (uint32_t)__popcll(__ballot(hi > th));
    const bool at = hi == th;
    uint32_t tl = 0;
    if (above + (uint32_t)__popcll(__ballot(at)) == n) {
        uint32_t low = at ? lo : ~0u;   // the smallest of those
#pragma unroll
        for (int o = 32; o; o >>= 1) low = min(low, (uint32_t)__shfl_xor((int)low, o));
        tl = low;
    } else {
        for (int b = 31; b >= 0; --b)
            if (above + (uint32_t)__popcll(__ballot(at && lo >= (tl | 1u << b))) >= n) tl |= 1u << b;
    }
    return (uint64_t)th << 32 | tl;
}
// (maximum, sum of exp(x - maximum)) of two sets; NaN in the sum stays
DEV float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    return make_float2(m, a.y * (a.x == m ? 1.0f : __builtin_amdgcn_exp2f((a.x - m) * 1.4426950408889634f)) +
                              b.y * (b.x == m ? 1.0f : __builtin_amdgcn_exp2f((b.x - m) * 1.4426950408889634f)));
}
DEV float2 wave_join(float2 v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = join(v, make_float2(__shfl_xor(v.x, o), __shfl_xor(v.y, o)));
    return v;
}
DEV float lse_of(float2 v) { return v.y != v.y ? NAN : fabsf(v.x) == INFINITY ? v.x : v.x + logf(v.y); }

// N values of 16 bytes
template <typename T> struct Pack { T v[16 / sizeof(T)]; };
}  // namespace

// A workgroup takes QXS_SLICE tokens of a row, 16 bytes of it a thread and step.  It reads the row's
// whole history and bias list and keeps those of its tokens in LDS (counts by integer atomics, biases
// summed in list order by the first entry of each token), so the dense pass reads and writes each
// logit once.  The best tokens are taken wave by wave: the n-th largest of the 64 lanes' largest bounds the
// wave's n-th largest from below and at most n lanes reach it, so at most 16 n keys are
// left, which are ranked by counting.
template <typename T>
__global__ __launch_bounds__(256) void qxs_slice(QxsArgs A) {
    constexpr int N = 16 / sizeof(T), STEPS = PER / N;
    __shared__ union {
        struct { uint32_t count[QXS_SLICE]; float bias[QXS_SLICE]; } s;   // count: SEEN, HAS_BIAS, occurrences behind the prompt
        uint64_t keys[4][16 * QXG_MAX_TOPN];
    } u;
    __shared__ uint32_t s_ids[1024];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const uint32_t r = blockIdx.y, v0 = blockIdx.x * QXS_SLICE, V = A.a.vocab;
    const T *in = (const T *)A.a.logits + r * A.a.logits_row + v0;
    T *out = (T *)A.a.out + r * A.a.out_row + v0;
    const uint32_t here = min(QXS_SLICE, V - v0);   // tokens of the slice
    const bool wide_in = (uintptr_t)in % 16 == 0, wide_out = (uintptr_t)out % 16 == 0;
    float x[PER];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t t = (s * 256 + tid) * N;
        if (wide_in && t + N <= here) {
            const Pack<T> p = __builtin_bit_cast(Pack<T>, *reinterpret_cast<const uint4 *>(in + t));
#pragma unroll
            for (int j = 0; j < N; ++j) x[s * N + j] = (float)p.v[j];
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) x[s * N + j] = t + j < here ? (float)in[t + j] : -INFINITY;
        }
    }
    const float rep = A.a.penalties ? A.a.penalties[3 * r] : 1.0f, freq = A.a.penalties ? A.a.penalties[3 * r + 1] : 0.0f,
                pres = A.a.penalties ? A.a.penalties[3 * r + 2] : 0.0f, temp = A.a.temperature ? A.a.temperature[r] : 1.0f;
    const uint32_t mrow = A.a.mask_rows ? A.a.mask_rows[r] : r;
    const uint32_t *mask = A.a.mask && mrow < A.a.masks ? A.a.mask + (uint64_t)mrow * A.words : nullptr;
    uint32_t open[STEPS];   // the mask bits of the thread's tokens, from bit 0
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t t = (s * 256 + tid) * N;
        open[s] = mask && t < here ? mask[(v0 + t) >> 5] >> (t & 31) : ~0u;
    }
    const bool sparse = A.a.history || A.a.bias_ids;
    if (sparse) {
#pragma unroll
        for (int i = 0; i < PER / 4; ++i) reinterpret_cast<uint4 *>(u.s.count)[i * 256 + tid] = make_uint4(0, 0, 0, 0);
        for (uint32_t i = tid; i < A.a.biases; i += 256) s_ids[i] = A.a.bias_ids[(uint64_t)r * A.a.biases + i];
        __syncthreads();
        if (A.a.history) {
            const uint32_t n = A.a.history_lens ? min(A.a.history_lens[r], A.a.history_slots) : A.a.history_slots;
            const uint32_t prompt = A.a.prompt_lens ? A.a.prompt_lens[r] : 0u;
            const uint32_t *hist = A.a.history + r * A.a.history_row;
            for (uint32_t i0 = tid; i0 < n; i0 += 8 * 256) {
                uint32_t t[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) t[k] = i0 + 256 * k < n ? hist[i0 + 256 * k] - v0 : ~0u;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (t[k] < here) {
                        atomicOr(&u.s.count[t[k]], SEEN);
                        if (i0 + 256 * k >= prompt) atomicAdd(&u.s.count[t[k]], 1u);
                    }
            }
        }
        for (uint32_t i = tid; i < A.a.biases; i += 256) {
            const uint32_t v = s_ids[i];
            if (v - v0 >= here) continue;
            bool first = true;
            for (uint32_t j = 0; j < i; ++j) first = first && s_ids[j] != v;
            if (!first) continue;
            const float *val = A.a.bias_values + (uint64_t)r * A.a.biases;
            float sum = val[i];
            for (uint32_t j = i + 1; j < A.a.biases; ++j)
                if (s_ids[j] == v) sum += val[j];
            u.s.bias[v - v0] = sum;
            atomicOr(&u.s.count[v - v0], HAS_BIAS);
        }
        __syncthreads();
    }
    float m = -INFINITY;
    bool nan = false;
    uint32_t best = 0, at = 0;   // the thread's largest, by rank (the first of equal ones is the lower token)
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t t = (s * 256 + tid) * N;
        Pack<T> p;
#pragma unroll
        for (int j4 = 0; j4 < N; j4 += 4) {
            uint4 c4 = make_uint4(0, 0, 0, 0);
            if (sparse) c4 = *reinterpret_cast<const uint4 *>(&u.s.count[t + j4]);
            const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = j4 + k;
                float y = x[s * N + j];
                if (c[k]) {
                    if (c[k] & SEEN) y = y > 0.0f ? y / rep : y * rep;
                    const uint32_t made = c[k] & 0x3fffffffu;
                    if (made) {
                        y -= freq * (float)made;
                        y -= pres;
                    }
                    if (c[k] & HAS_BIAS) y += u.s.bias[t + j];
                }
                y /= temp;
                if (!((open[s] >> j) & 1) || t + j >= here) y = -INFINITY;
                x[s * N + j] = y;
                p.v[j] = (T)y;
                m = fmaxf(m, y);
                nan = nan || y != y;
                const uint32_t k32 = rank_of(y);
                if (k32 > best) { best = k32; at = t + j; }
            }
        }
        if (wide_out && t + N <= here) *reinterpret_cast<uint4 *>(out + t) = __builtin_bit_cast(uint4, p);
        else
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (t + j < here) out[t + j] = p.v[j];
    }
    const uint32_t list = blockIdx.x * 4 + wave;   // one of the row's lists of n keys
    if (A.a.lse) {
        float sum = 0.0f;
        if (m > -INFINITY) {
#pragma unroll
            for (int i = 0; i < PER; ++i) sum += x[i] == m ? 1.0f : __builtin_amdgcn_exp2f((x[i] - m) * 1.4426950408889634f);
        }
        const float2 ms = wave_join(make_float2(m, nan ? NAN : sum));
        if (lane == 0) A.ms[((uint64_t)r * A.slices) * 4 + list] = ms;
    }
    const uint32_t n = A.a.top_n;
    if (!n) return;
    const uint64_t least = wave_nth(key_of(best, v0 + at), n);
    __syncthreads();   // the counts are read: their space takes the keys
    uint64_t *keys = u.keys[wave];
    uint32_t have = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint64_t k = key_of(rank_of(x[i]), v0 + ((i / N) * 256 + tid) * N + i % N);
        const bool f = k && k >= least;
        const uint64_t b = __ballot(f);
        if (f) keys[have + __popcll(b & ((1ull << lane) - 1ull))] = k;
        have += (uint32_t)__popcll(b);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint64_t *to = A.keys + ((uint64_t)r * A.slices * 4 + list) * n;
    for (uint32_t i = lane; i < have; i += 64) {
        const uint64_t k = keys[i];
        uint32_t above = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < have; ++j) above += keys[j] > k;
        if (above < n) to[above] = k;
    }
    if (have < n && lane >= have && lane < n) to[lane] = 0;
}

// The lists of a row joined: a workgroup a row.  The n-th largest of 64 strips' largest keys bounds the n-th of
// all from below; the keys that reach it are ranked by counting.
template <typename T>
__global__ __launch_bounds__(256) void qxs_join(QxsArgs A) {
    constexpr uint32_t ROOM = 4096;
    __shared__ uint64_t s_key[ROOM], s_best[4][64];
    __shared__ float2 s_ms[4];
    __shared__ uint32_t s_have;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const uint32_t r = blockIdx.x, lists = A.slices * 4, n = A.a.top_n;
    const uint64_t *keys = A.keys + (uint64_t)r * lists * n;
    if (tid == 0) s_have = 0;
    if (A.a.lse) {
        float2 ms = make_float2(-INFINITY, 0.0f);
        for (uint32_t i = tid; i < lists; i += 256) ms = join(ms, A.ms[(uint64_t)r * lists + i]);
        ms = wave_join(ms);
        if (lane == 0) s_ms[wave] = ms;
    }
    uint64_t best = 0;   // of the lists of strip tid % 64: each list's first key is its largest
    if (n)
        for (uint32_t i = tid; i < lists; i += 256) best = umax64(best, keys[(uint64_t)i * n]);
    s_best[wave][lane] = best;
    __syncthreads();
    if (A.a.lse && tid == 0) A.a.lse[r] = lse_of(join(join(s_ms[0], s_ms[1]), join(s_ms[2], s_ms[3])));
    if (!n) return;
    best = umax64(umax64(s_best[0][lane], s_best[1][lane]), umax64(s_best[2][lane], s_best[3][lane]));
    const uint64_t least = wave_nth(best, n);
    for (uint32_t i = tid; i < lists * n; i += 256) {
        const uint64_t k = keys[i];
        if (k && k >= least) {
            const uint32_t at = atomicAdd(&s_have, 1u);
            if (at < ROOM) s_key[at] = k;
        }
    }
    __syncthreads();
    const uint32_t have = s_have;
    auto put = [&](uint32_t at, uint64_t k) {
        const uint32_t v = ~(uint32_t)k;
        float x = k ? key_value(k) : -INFINITY;
        if (k && x == 0.0f) x = copysignf(0.0f, (float)((const T *)A.a.out)[r * A.a.out_row + v]);   // (the key has no -0)
        A.a.top_ids[(uint64_t)r * n + at] = k ? v : QXG_NO_TOKEN;
        if (A.a.top_logits) A.a.top_logits[(uint64_t)r * n + at] = x;
    };
    if (have <= ROOM) {
        for (uint32_t i = tid; i < have; i += 256) {
            const uint64_t k = s_key[i];
            uint32_t above = 0;
#pragma unroll 4
            for (uint32_t j = 0; j < have; ++j) above += s_key[j] > k;
            if (above < n) put(above, k);
        }
        if (tid >= have && tid < n) put(tid, 0);
        return;
    }
    // (a strip of very many lists, all of them large: one pick after the other)
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < n; ++k) {
        uint64_t b = 0;
        for (uint32_t i = tid; i < lists * n; i += 256) {
            const uint64_t y = keys[i];
            b = y < last ? umax64(b, y) : b;
        }
        b = wave_max_u64(b);
        __syncthreads();
        if (lane == 0) s_best[0][wave] = b;
        __syncthreads();
        last = umax64(umax64(s_best[0][0], s_best[0][1]), umax64(s_best[0][2], s_best[0][3]));
        if (tid == 0) put(k, last);
    }
}

namespace {
template <typename T> void launch(const QxsArgs &A, hipStream_t s) {
    hipLaunchKernelGGL(qxs_slice<T>, dim3(A.slices, A.a.rows), dim3(256), 0, s, A);
    if (A.a.lse || A.a.top_n) hipLaunchKernelGGL(qxs_join<T>, dim3(A.a.rows), dim3(256), 0, s, A);
}
}  // namespace

void qxs_launch(const QxsArgs &A, hipStream_t s) {
    if (A.a.type == QXG_TYPE_F32) launch<float>(A, s);
    else if (A.a.type == QXG_TYPE_F16) launch<_Float16>(A, s);
    else launch<__bf16>(A, s);
}
