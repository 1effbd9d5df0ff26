// Penalties, biases, temperature and grammar mask on logits, with the best tokens (qxg_adjust_logits).
#include "qxg_dev.h"
#include "qxg_ops.h"

namespace {
// key of token v with logit x: larger first, then the lower token; 0 (never picked) for -inf and NaN
DEV uint64_t pick_key(float x, uint32_t v) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);   // (-0 ranks as +0)
    return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~v;
}
DEV float key_value(uint64_t k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
// the largest of the block's 256 keys, in every thread
DEV uint64_t block_best(uint64_t k, uint64_t *s) {
    k = wave_max_u64(k);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = k;
    __syncthreads();
    return umax64(umax64(s[0], s[1]), umax64(s[2], s[3]));
}
// (maximum, sum of exp(x - maximum)) of two sets
DEV float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    if (m == -INFINITY) return make_float2(m, a.y + b.y);   // (a sum is 0 or NaN here)
    return make_float2(m, a.y * (a.x == m ? 1.0f : expf(a.x - m)) + b.y * (b.x == m ? 1.0f : expf(b.x - m)));
}
DEV float2 block_join(float2 v, float2 *s) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = join(v, make_float2(__shfl_xor(v.x, o), __shfl_xor(v.y, o)));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return join(join(s[0], s[1]), join(s[2], s[3]));
}
DEV float lse_of(float2 v) { return v.x == INFINITY ? (v.y == v.y ? INFINITY : NAN) : v.x == -INFINITY ? (v.y == v.y ? -INFINITY : NAN) : v.x + logf(v.y); }
}  // namespace

// A workgroup takes QXS_SLICE tokens of a row.  It reads the row's whole history and bias list and
// keeps those of its tokens in LDS (counts by integer atomics, biases summed in list order by the
// first entry of each token), so the dense pass reads and writes each logit once.
template <typename T>
__global__ __launch_bounds__(256) void qxs_slice(QxsArgs A) {
    constexpr int PER = QXS_SLICE / 256;
    __shared__ uint32_t s_count[QXS_SLICE];   // bit 31: seen; below: occurrences behind the prompt
    __shared__ float s_bias[QXS_SLICE];
    __shared__ uint8_t s_has[QXS_SLICE];
    __shared__ uint64_t s_key[4];
    __shared__ float2 s_ms[4];
    const int tid = threadIdx.x;
    const uint32_t r = blockIdx.y, v0 = blockIdx.x * QXS_SLICE, V = A.a.vocab;
    for (int i = tid; i < (int)QXS_SLICE; i += 256) { s_count[i] = 0; s_has[i] = 0; }
    __syncthreads();
    if (A.a.history) {
        const uint32_t n = A.a.history_lens ? min(A.a.history_lens[r], A.a.history_slots) : A.a.history_slots;
        const uint32_t prompt = A.a.prompt_lens ? A.a.prompt_lens[r] : 0u;
        const uint32_t *hist = A.a.history + r * A.a.history_row;
        for (uint32_t i = tid; i < n; i += 256) {
            const uint32_t v = hist[i];
            if (v >= V || v - v0 >= QXS_SLICE) continue;
            atomicOr(&s_count[v - v0], 0x80000000u);
            if (i >= prompt) atomicAdd(&s_count[v - v0], 1u);
        }
    }
    if (A.a.bias_ids) {
        const uint32_t *ids = A.a.bias_ids + (uint64_t)r * A.a.biases;
        const float *val = A.a.bias_values + (uint64_t)r * A.a.biases;
        for (uint32_t i = tid; i < A.a.biases; i += 256) {
            const uint32_t v = ids[i];
            if (v >= V || v - v0 >= QXS_SLICE) continue;
            bool first = true;
            for (uint32_t j = 0; j < i; ++j) first = first && ids[j] != v;
            if (!first) continue;
            float sum = val[i];
            for (uint32_t j = i + 1; j < A.a.biases; ++j) if (ids[j] == v) sum += val[j];
            s_bias[v - v0] = sum;
            s_has[v - v0] = 1;
        }
    }
    __syncthreads();
    const float rep = A.a.penalties ? A.a.penalties[3 * r] : 1.0f, freq = A.a.penalties ? A.a.penalties[3 * r + 1] : 0.0f,
                pres = A.a.penalties ? A.a.penalties[3 * r + 2] : 0.0f, temp = A.a.temperature ? A.a.temperature[r] : 1.0f;
    const uint32_t mrow = A.a.mask_rows ? A.a.mask_rows[r] : r;
    const uint32_t *mask = A.a.mask && mrow < A.a.masks ? A.a.mask + (uint64_t)mrow * A.words : nullptr;
    const T *in = (const T *)A.a.logits + r * A.a.logits_row;
    T *out = (T *)A.a.out + r * A.a.out_row;
    uint64_t key[PER];
    float2 ms = make_float2(-INFINITY, 0.0f);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
        const uint32_t t = u * 256 + tid, v = v0 + t;
        key[u] = 0;
        if (v >= V) continue;
        float x = (float)in[v];
        const uint32_t c = s_count[t];
        if (c) {
            x = x > 0.0f ? x / rep : x * rep;
            if (c & 0x7fffffffu) {
                x -= freq * (float)(c & 0x7fffffffu);
                x -= pres;
            }
        }
        if (s_has[t]) x += s_bias[t];
        x /= temp;
        if (mask && !((mask[v >> 5] >> (v & 31)) & 1)) x = -INFINITY;
        out[v] = (T)x;
        key[u] = pick_key(x, v);
        ms = join(ms, x == x ? make_float2(x, x == -INFINITY ? 0.0f : 1.0f) : make_float2(-INFINITY, NAN));
    }
    if (A.a.lse) {
        ms = block_join(ms, s_ms);
        if (tid == 0) A.ms[(uint64_t)r * A.slices + blockIdx.x] = ms;
    }
    for (uint32_t k = 0; k < A.a.top_n; ++k) {
        uint64_t best = 0;
#pragma unroll
        for (int u = 0; u < PER; ++u) best = umax64(best, key[u]);
        best = block_best(best, s_key);
        if (tid == 0) A.keys[((uint64_t)r * A.slices + blockIdx.x) * A.a.top_n + k] = best;
#pragma unroll
        for (int u = 0; u < PER; ++u) key[u] = key[u] == best ? 0 : key[u];
    }
}

// The slices of a row joined: a workgroup a row.
template <typename T>
__global__ __launch_bounds__(256) void qxs_join(QxsArgs A) {
    __shared__ uint64_t s_key[4];
    __shared__ float2 s_ms[4];
    const int tid = threadIdx.x;
    const uint32_t r = blockIdx.x, n = A.slices * A.a.top_n;
    if (A.a.lse) {
        float2 ms = make_float2(-INFINITY, 0.0f);
        for (uint32_t i = tid; i < A.slices; i += 256) ms = join(ms, A.ms[(uint64_t)r * A.slices + i]);
        ms = block_join(ms, s_ms);
        if (tid == 0) A.a.lse[r] = lse_of(ms);
    }
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < A.a.top_n; ++k) {   // the largest below the last one picked
        uint64_t best = 0;
        for (uint32_t i = tid; i < n; i += 256) {
            const uint64_t x = A.keys[(uint64_t)r * n + i];
            best = x < last ? umax64(best, x) : best;
        }
        best = last = block_best(best, s_key);
        if (tid == 0) {
            const uint32_t v = ~(uint32_t)best;
            float x = best ? key_value(best) : -INFINITY;
            if (best && x == 0.0f) x = copysignf(0.0f, (float)((const T *)A.a.out)[r * A.a.out_row + v]);   // (the key has no -0)
            A.a.top_ids[(uint64_t)r * A.a.top_n + k] = best ? v : QXG_NO_TOKEN;
            if (A.a.top_logits) A.a.top_logits[(uint64_t)r * A.a.top_n + k] = x;
        }
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
