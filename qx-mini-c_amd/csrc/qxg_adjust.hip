// Penalties, biases, temperature and grammar mask on logits, with the best tokens (qxg_adjust_logits).
#include "qxg_dev.h"
#include "qxg_ops.h"

namespace {
// of a token in LDS: occurrences behind the prompt, the index of its first bias entry, whether it has one, and
// whether it is anywhere in the history
constexpr uint32_t COUNT = (1u << 20) - 1, BIAS_SHIFT = 20, HAS_BIAS = 0x40000000u, SEEN = 0x80000000u;
static_assert(QXS_HISTORY <= COUNT && QXS_BIASES <= 1u << (30 - BIAS_SHIFT), "the fields of a token's word");

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
// A bound that exactly n of the wave's 64 keys reach (hi: their ranks, lo(): their other bits, unlike but where the
// rank is 0), found a bit at a time until it is one; 0 when fewer than n are not 0.  The low bits are asked for
// only where several keys share the n-th's rank.
template <typename F> DEV uint64_t wave_nth(uint32_t hi, uint32_t n, F lo) {
    uint32_t th = 0, tl = 0;
    for (int b = 31; b >= 0; --b) {
        const uint32_t c = (uint32_t)__popcll(__ballot(hi >= (th | 1u << b)));
        if (c >= n) th |= 1u << b;
        if (c == n) return (uint64_t)th << 32;
    }
    if (th == 0) return 0;
    const uint32_t above = (uint32_t)__popcll(__ballot(hi > th)), low = lo();
    const bool at = hi == th;
    for (int b = 31; b >= 0; --b)
        if (above + (uint32_t)__popcll(__ballot(at && low >= (tl | 1u << b))) >= n) tl |= 1u << b;
    return (uint64_t)th << 32 | tl;
}
// (maximum, sum of exp(x - maximum)) of two sets; NaN in the sum stays
DEV float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    return make_float2(m, a.y * (a.x == m ? 1.0f : __builtin_amdgcn_exp2f((a.x - m) * 1.4426950408889634f)) +
                              b.y * (b.x == m ? 1.0f : __builtin_amdgcn_exp2f((b.x - m) * 1.4426950408889634f)));
}
DEV float lse_of(float2 v) { return v.y != v.y ? NAN : fabsf(v.x) == INFINITY ? v.x : v.x + logf(v.y); }

// the larger ones of numbers and quiet NaN
DEV float max_of(float a, float b, float c) {
    float m;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
    return m;
}
// the largest of the wave's values (numbers), and the sum of them
DEV float wave_most(float v) {
    v = fmaxf(v, dppf<DPP_XOR1>(v)); v = fmaxf(v, dppf<DPP_XOR2>(v)); v = fmaxf(v, dppf<DPP_ROR4>(v)); v = fmaxf(v, dppf<DPP_ROR8>(v));
    return fmaxf(fmaxf(rdlanef(v, 0), rdlanef(v, 16)), fmaxf(rdlanef(v, 32), rdlanef(v, 48)));
}
DEV float wave_total(float v) {
    v += dppf<DPP_XOR1>(v); v += dppf<DPP_XOR2>(v); v += dppf<DPP_ROR4>(v); v += dppf<DPP_ROR8>(v);
    return (rdlanef(v, 0) + rdlanef(v, 16)) + (rdlanef(v, 32) + rdlanef(v, 48));
}

DEV float2 wave_join(float2 v) {
    const float m = wave_most(v.x);
    return make_float2(m, wave_total(v.y * (v.x == m ? 1.0f : __builtin_amdgcn_exp2f((v.x - m) * 1.4426950408889634f))));
}

// N values of 16 bytes
template <typename T> struct Pack { T v[16 / sizeof(T)]; };
}  // namespace

// A workgroup takes a slice of a row, 16 bytes of it a thread and step.  It reads the row's whole history
// and bias list and keeps those of its tokens in LDS (counts by integer atomics, biases summed in list
// order by the first entry of each token), so the dense pass reads and writes each logit once.  The best
// tokens: a bound that n of a wave's 64 lanes' largest reach bounds the wave's n-th largest from below, and
// so the slice's; at most n lanes of a wave reach the slice's, so at most PER n of its keys do, about n / 2 of most
// rows.  Only of more than n are the n largest taken, by counting.
// A workgroup's chain of latencies bounds it, not the bytes: 64 rows of 151936 f32 logits with 4000 tokens of
// history each, best 32: 30 us (78 MB read and written, 15.5 us at the rate of a copy).  Of a workgroup's 12 us,
// 5 are the first loads, 1 the history's counts, 3 the dense pass, 3 the best tokens; 6, 7 or 8 workgroups a CU
// are alike, and so are divisions and products with corrected reciprocals.  One row: 6.7 us.
template <typename T, int STEPS>
__global__ __launch_bounds__(256) void qxs_slice(QxsArgs A) {
    constexpr int N = 16 / sizeof(T), PER = N * STEPS, EARLY = 16;
    constexpr uint32_t SLICE = 256 * PER;
    __shared__ union {
        uint32_t token[SLICE];
        uint64_t keys[4][PER * QXG_MAX_TOPN];
    } u;
    extern __shared__ uint32_t s_ids[];   // [biases], then their values
    float *s_sum = reinterpret_cast<float *>(s_ids + A.a.biases);
    __shared__ uint64_t s_least[4];
    __shared__ uint32_t s_twice;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const uint32_t r = blockIdx.y, v0 = blockIdx.x * SLICE, V = A.a.vocab;
    const T *in = (const T *)A.a.logits + r * A.a.logits_row + v0;
    T *out = (T *)A.a.out + r * A.a.out_row + v0;
    const uint32_t here = min(SLICE, V - v0);   // tokens of the slice
    const bool wide_in = (uintptr_t)in % 16 == 0, wide_out = (uintptr_t)out % 16 == 0;
    // Everything that needs nothing else is loaded at once, whether it turns out to be used or not (absent
    // arrays: the workspace's first words): one after the other, the loads' latencies were half of the time.
    const float *none = reinterpret_cast<const float *>(A.ms);
    const float *pen = A.a.penalties ? A.a.penalties + 3 * r : none, *tem = A.a.temperature ? A.a.temperature + r : none;
    const uint32_t *lens = A.a.history_lens ? A.a.history_lens + r : (const uint32_t *)none,
                   *made = A.a.prompt_lens ? A.a.prompt_lens + r : (const uint32_t *)none,
                   *rows = A.a.mask_rows ? A.a.mask_rows + r : (const uint32_t *)none;
    float rep = pen[0], freq = pen[1], pres = pen[2], temp = tem[0];
    uint32_t entries = lens[0], prompt = made[0], mrow = rows[0];
    const uint32_t slots = A.a.history ? A.a.history_slots : 0u;
    const uint32_t *hist = A.a.history + r * A.a.history_row;
    uint32_t early[EARLY];   // the history's first entries
#pragma unroll
    for (int k = 0; k < EARLY; ++k) early[k] = tid + 256 * k < slots ? hist[tid + 256 * k] : QXG_NO_TOKEN;
    float x[PER];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t t = (s * 256 + tid) * N;
        if (wide_in && t + N <= here) {
            const Pack<T> p = __builtin_bit_cast(Pack<T>, *reinterpret_cast<const nt4 *>(in + t));
#pragma unroll
            for (int j = 0; j < N; ++j) x[s * N + j] = (float)p.v[j];
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) x[s * N + j] = t + j < here ? (float)in[t + j] : -INFINITY;
        }
    }
    const bool sparse = slots || A.a.biases;
    if (sparse) {
        if (tid == 0) s_twice = 0;
#pragma unroll
        for (int i = 0; i < PER / 4; ++i) reinterpret_cast<nt4 *>(u.token)[i * 256 + tid] = nt4{0, 0, 0, 0};
        for (uint32_t i = tid; i < A.a.biases; i += 256) {
            s_ids[i] = A.a.bias_ids[(uint64_t)r * A.a.biases + i];
            s_sum[i] = A.a.bias_values[(uint64_t)r * A.a.biases + i];
        }
    }
    mrow = A.a.mask_rows ? mrow : r;
    const uint32_t *mask = A.a.mask && mrow < A.a.masks ? A.a.mask + (uint64_t)mrow * A.words : nullptr;
    uint32_t open[STEPS];   // the mask bits of the thread's tokens, from bit 0; 0 behind the vocabulary
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t t = (s * 256 + tid) * N, left = here > t ? here - t : 0u;
        open[s] = (mask && left ? mask[(v0 + t) >> 5] >> (t & 31) : ~0u) & (left < N ? (1u << left) - 1u : ~0u);
    }
    if (!A.a.penalties) { rep = 1.0f; freq = pres = 0.0f; }
    if (!A.a.temperature) temp = 1.0f;
    entries = A.a.history_lens ? min(entries, slots) : slots;
    prompt = A.a.prompt_lens ? prompt : 0u;
    if (sparse) {
        __syncthreads();
        auto note = [&](uint32_t i, uint32_t v) {
            if (v - v0 >= here || i >= entries) return;
            atomicOr(&u.token[v - v0], SEEN);
            if (i >= prompt) atomicAdd(&u.token[v - v0], 1u);
        };
#pragma unroll
        for (int k = 0; k < EARLY; ++k) note(tid + 256 * k, early[k]);
        for (uint32_t i = tid + 256 * EARLY; i < entries; i += 256) note(i, hist[i]);
        constexpr int EACH = QXS_BIASES / 256;
#pragma unroll
        for (int k = 0; k < EACH; ++k) {
            const uint32_t i = tid + 256 * k, v = i < A.a.biases ? s_ids[i] : QXG_NO_TOKEN;
            if (v - v0 < here && (atomicOr(&u.token[v - v0], HAS_BIAS | i << BIAS_SHIFT) & HAS_BIAS)) s_twice = 1;
        }
        if (A.a.biases) __syncthreads();
        if (A.a.biases && s_twice) {   // (uniform) a token of several entries: its first one takes the sum, in order
            float sum[EACH];
            bool first[EACH];
#pragma unroll
            for (int k = 0; k < EACH; ++k) {
                const uint32_t i = tid + 256 * k, v = i < A.a.biases ? s_ids[i] : QXG_NO_TOKEN;
                first[k] = v - v0 < here;
                if (!first[k]) continue;
                for (uint32_t j = 0; j < i; ++j) first[k] = first[k] && s_ids[j] != v;
                if (!first[k]) continue;
                sum[k] = s_sum[i];
                for (uint32_t j = i + 1; j < A.a.biases; ++j)
                    if (s_ids[j] == v) sum[k] += s_sum[j];
                u.token[v - v0] = (u.token[v - v0] & ~((QXS_BIASES - 1) << BIAS_SHIFT)) | i << BIAS_SHIFT;
            }
            __syncthreads();   // every entry's own value is read
#pragma unroll
            for (int k = 0; k < EACH; ++k)
                if (first[k]) s_sum[tid + 256 * k] = sum[k];
        }
        __syncthreads();
    }
    float m = -INFINITY;   // the thread's largest
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const uint32_t t = (s * 256 + tid) * N;
        Pack<T> p;
#pragma unroll
        for (int j4 = 0; j4 < N; j4 += 4) {
            nt4 c4 = {0, 0, 0, 0};
            if (sparse) c4 = *reinterpret_cast<const nt4 *>(&u.token[t + j4]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = j4 + k;
                const uint32_t c = c4[k];
                float y = x[s * N + j];
                if (c) {
                    if (c & SEEN) y = y > 0.0f ? y / rep : y * rep;
                    if (c & COUNT) {
                        y -= freq * (float)(c & COUNT);
                        y -= pres;
                    }
                    if (c & HAS_BIAS) y += s_sum[(c >> BIAS_SHIFT) & (QXS_BIASES - 1)];
                }
                y /= temp;
                const uint32_t is = (uint32_t)__builtin_amdgcn_sbfe((int)open[s], j, 1);   // all bits of it
                y = __uint_as_float((is & __float_as_uint(y)) | (~is & 0xff800000u));
                x[s * N + j] = y;
                p.v[j] = (T)y;
            }
            // (the division has made every NaN a quiet one)
            m = max_of(max_of(m, x[s * N + j4], x[s * N + j4 + 1]), x[s * N + j4 + 2], x[s * N + j4 + 3]);
        }
        if (wide_out && t + N <= here) *reinterpret_cast<nt4 *>(out + t) = __builtin_bit_cast(nt4, p);
        else
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (t + j < here) out[t + j] = p.v[j];
    }
    const uint64_t list = (uint64_t)r * A.slices * 4 + blockIdx.x * 4 + wave;
    if (A.a.lse) {
        const float most = wave_most(m);
        float sum = 0.0f;
        if (fabsf(most) < INFINITY) {
#pragma unroll
            for (int i = 0; i < PER; ++i) sum += __builtin_amdgcn_exp2f((x[i] - most) * 1.4426950408889634f);
            sum = wave_total(sum);
        } else {   // an infinite maximum is the result, but for NaN
            bool nan = false;
#pragma unroll
            for (int i = 0; i < PER; ++i) nan = nan || x[i] != x[i];
            sum = __ballot(nan) ? NAN : most > 0.0f ? 1.0f : 0.0f;
        }
        const float2 ms = make_float2(most, sum);
        if (lane == 0) A.ms[list] = ms;
    }
    const uint32_t n = A.a.top_n;
    if (!n) return;
    uint64_t least = wave_nth(rank_of(m), n, [&] {   // (of equal ones the lower token counts more)
        uint32_t at = 0;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i) at = x[i] == m ? ((i / N) * 256 + tid) * N + i % N : at;
        return ~(v0 + at);
    });
    if (lane == 0) s_least[wave] = least;
    __syncthreads();   // (also: the tokens' words are read, their space takes the keys)
    least = umax64(umax64(s_least[0], s_least[1]), umax64(s_least[2], s_least[3]));
    const float low = least ? key_value(least) : -INFINITY;
    uint64_t *keys = u.keys[wave];
    uint32_t have = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (__ballot(x[i] >= low) == 0) continue;
        const uint64_t k = key_of(rank_of(x[i]), v0 + ((i / N) * 256 + tid) * N + i % N);
        const bool f = k && k >= least;
        const uint64_t b = __ballot(f);
        if (f) keys[have + __popcll(b & ((1ull << lane) - 1ull))] = k;
        have += (uint32_t)__popcll(b);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint64_t *to = A.keys + list * n;
    if (have <= n) {
        if (lane < n) to[lane] = lane < have ? keys[lane] : 0;
        return;
    }
    for (uint32_t i = lane; i < have; i += 64) {
        const uint64_t k = keys[i];
        uint32_t above = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < have; ++j) above += keys[j] > k;
        if (above < n) to[above] = k;
    }
}

// The lists of a row joined: a workgroup a row.  The n-th largest of 64 strips' largest keys (strip: every
// 64th key) bounds the n-th of all from below; the keys that reach it are ranked by counting.
// (One row 4 .. 6 us, 64 rows of 38 slices 9.5 us: loads, one search, one count, each a latency.)
template <typename T>
__global__ __launch_bounds__(1024) void qxs_join(QxsArgs A) {
    constexpr uint32_t ROOM = 4096;
    constexpr int HELD = 8;   // keys a thread holds; those behind are read twice
    __shared__ uint64_t s_key[ROOM], s_best[16][64];
    __shared__ float2 s_ms[16];
    __shared__ uint32_t s_have;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const uint32_t r = blockIdx.x, lists = A.slices * 4, n = A.a.top_n, total = lists * n;
    const uint64_t *keys = A.keys + (uint64_t)r * total;
    uint64_t k[HELD], best = 0;   // of strip tid % 64
#pragma unroll
    for (int j = 0; j < HELD; ++j) k[j] = tid + 1024u * j < total ? keys[tid + 1024 * j] : 0;
    if (tid == 0) s_have = 0;
    if (A.a.lse) {
        float2 ms = make_float2(-INFINITY, 0.0f);
        for (uint32_t i = tid; i < lists; i += 1024) ms = join(ms, A.ms[(uint64_t)r * lists + i]);
        ms = wave_join(ms);
        if (lane == 0) s_ms[wave] = ms;
    }
#pragma unroll
    for (int j = 0; j < HELD; ++j) best = umax64(best, k[j]);
    for (uint32_t i = tid + 1024 * HELD; i < total; i += 1024) best = umax64(best, keys[i]);
    s_best[wave][lane] = best;
    __syncthreads();
    if (A.a.lse && wave == 0) {
        const float2 ms = wave_join(lane < 16 ? s_ms[lane] : make_float2(-INFINITY, 0.0f));
        if (lane == 0) A.a.lse[r] = lse_of(ms);
    }
    if (!n) return;
#pragma unroll
    for (int w = 0; w < 16; ++w) best = umax64(best, s_best[w][lane]);
    const uint64_t least = wave_nth((uint32_t)(best >> 32), n, [&] { return (uint32_t)best; });
    auto offer = [&](uint64_t key) {
        if (key && key >= least) {
            const uint32_t at = atomicAdd(&s_have, 1u);
            if (at < ROOM) s_key[at] = key;
        }
    };
#pragma unroll
    for (int j = 0; j < HELD; ++j) offer(k[j]);
    for (uint32_t i = tid + 1024 * HELD; i < total; i += 1024) offer(keys[i]);
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
        for (uint32_t i = tid >> 3; i < have; i += 128) {   // 8 threads a key
            const uint64_t k = s_key[i];
            uint32_t above = 0;
#pragma unroll 4
            for (uint32_t j = tid & 7; j < have; j += 8) above += s_key[j] > k;
            above += (uint32_t)dppi<DPP_XOR1>((int)above); above += (uint32_t)dppi<DPP_XOR2>((int)above);
            above += (uint32_t)dppi<DPP_HALF_MIRROR>((int)above);
            if ((tid & 7) == 0 && above < n) put(above, k);
        }
        if (tid >= have && tid < n) put(tid, 0);
        return;
    }
    // (a strip of very many lists, all of them large: one pick after the other)
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < n; ++k) {
        uint64_t b = 0;
        for (uint32_t i = tid; i < total; i += 1024) {
            const uint64_t y = keys[i];
            b = y < last ? umax64(b, y) : b;
        }
        b = wave_max_u64(b);
        __syncthreads();
        if (lane == 0) s_best[0][wave] = b;
        __syncthreads();
        last = wave_max_u64(s_best[0][lane & 15]);
        if (tid == 0) put(k, last);
    }
}

namespace {
template <typename T> hipError_t launch(const QxsArgs &A, hipStream_t s) {
    constexpr int STEPS = QXS_SLICE * sizeof(T) / 4096;
    auto *kernel = A.small ? qxs_slice<T, 1> : qxs_slice<T, STEPS>;
    const hipError_t e = qxg_launch(kernel, dim3(A.slices, A.a.rows), dim3(256), A.a.biases * 8, s, A);
    return e != hipSuccess || !(A.a.lse || A.a.top_n) ? e : qxg_launch(qxs_join<T>, dim3(A.a.rows), dim3(1024), 0, s, A);
}
}  // namespace

hipError_t qxs_launch(const QxsArgs &A, hipStream_t s) {
    if (A.a.type == QXG_TYPE_F32) return launch<float>(A, s);
    if (A.a.type == QXG_TYPE_F16) return launch<_Float16>(A, s);
    return launch<__bf16>(A, s);
}
