// Eviction from a KV cache by accumulated attention weight (qxg_kv_select, qxg_kv_compact).
#include "qxg_dev.h"
#include "qxg_ops.h"

namespace {
// Weights as unsigned keys in their order; NaN as -inf, -0 as +0
DEV uint32_t weight_key(float w) {
    const uint32_t u = __float_as_uint(w == w ? w + 0.0f : -INFINITY);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// exclusive prefix of a flag count over the block's 1024 threads (16 waves), and the total
DEV uint32_t block_rank(bool f, uint32_t *s_w, uint32_t &total) {
    const uint64_t m = __ballot(f);
    const int wave = wave_id(), lane = threadIdx.x & 63;
    __syncthreads();
    if (lane == 0) s_w[wave] = __popcll(m);
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int w = 0; w < 16; ++w) {
        before += w < wave ? s_w[w] : 0u;
        all += s_w[w];
    }
    total = all;
    return before + __popcll(m & ((1ull << lane) - 1ull));
}
}  // namespace

// A workgroup a group.  The smallest key that is kept is found a byte at a time from the top (a
// histogram of the keys that share the bytes found so far), then the positions are listed in order.
extern "C" __global__ __launch_bounds__(1024) void qxe_select(qxg_kv_select_args A) {
    __shared__ uint32_t s_hist[16][256], s_w[16], s_key, s_need;
    const int tid = threadIdx.x;
    const uint32_t g = blockIdx.x, len = min(A.lens[g], A.positions), kept = min(len, A.budget);
    uint32_t *keep = A.keep + g * A.keep_group;
    const float *acc = A.account + g * A.account_group;
    if (tid == 0) A.kept[g] = kept;
    if (len <= A.budget) {
        for (uint32_t p = tid; p < len; p += 1024) keep[p] = p;
        return;
    }
    const uint32_t lo = A.sinks, hi = len - A.recent;
    uint32_t need = A.budget - A.sinks - A.recent, key = 0;
    if (need) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 16 * 256; i += 1024) (&s_hist[0][0])[i] = 0;
            __syncthreads();
            for (uint32_t p = lo + tid; p < hi; p += 1024) {
                const uint32_t k = weight_key(acc[p]);
                if (shift == 24 || (k >> (shift + 8)) == (key >> (shift + 8))) atomicAdd(&s_hist[tid >> 6][(k >> shift) & 255], 1u);
            }
            __syncthreads();
            if (tid < 256) {
                uint32_t n = 0;
                for (int w = 0; w < 16; ++w) n += s_hist[w][tid];
                s_hist[0][tid] = n;
            }
            __syncthreads();
            if (tid == 0) {
                int d = 255;
                while (s_hist[0][d] < need) need -= s_hist[0][d--];
                s_key = key | (uint32_t)d << shift;
                s_need = need;
            }
            __syncthreads();
            key = s_key;
            need = s_need;
            __syncthreads();
        }
    } else {
        key = ~0u;   // none of the middle
    }
    uint32_t at = 0, equal = 0;
    for (uint32_t p0 = 0; p0 < len; p0 += 1024) {
        const uint32_t p = p0 + tid;
        const bool mid = p >= lo && p < hi;
        const uint32_t k = mid ? weight_key(acc[p]) : 0u;
        uint32_t eqs, ns;
        const uint32_t er = block_rank(mid && k == key, s_w, eqs);
        const bool f = p < len && (!mid || k > key || (k == key && equal + er < need));
        const uint32_t r = block_rank(f, s_w, ns);
        if (f) keep[at + r] = p;
        at += ns;
        equal += eqs;
    }
}

// Rows moved in place.  A workgroup takes a strip of 128 bytes of a group's K or V rows (or its scales
// and account) and goes through the list in order, 256 rows at a time: all are read before any is
// written, and no later row's source lies below what an earlier step writes.
extern "C" __global__ __launch_bounds__(256) void qxe_compact(qxg_kv_compact_args A) {
    const int tid = threadIdx.x;
    const uint32_t g = blockIdx.y, strips = (A.row_bytes + 127) / 128;
    const uint32_t n = min(A.kept[g * A.kept_group], min(A.slots, A.positions - A.first));
    const uint32_t *keep = A.keep + g * A.keep_group;
    constexpr int U = 8;
    if (blockIdx.x < 2 * strips) {
        const uint32_t strip = blockIdx.x >> 1, byte = strip * 128 + (tid & 7) * 16;
        uint8_t *base = (uint8_t *)(blockIdx.x & 1 ? A.v : A.k) + g * A.kv_group + byte;
        const bool in = byte < A.row_bytes;
        for (uint32_t i0 = 0; i0 < n; i0 += 32 * U) {
            uint4 x[U];
            bool ok[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t i = i0 + 32 * u + (tid >> 3), p = i < n ? keep[i] : ~0u;
                ok[u] = in && p < A.positions && p != A.first + i;
                if (ok[u]) x[u] = *reinterpret_cast<const uint4 *>(base + p * A.kv_row);
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (ok[u]) *reinterpret_cast<uint4 *>(base + (A.first + i0 + 32 * u + (tid >> 3)) * A.kv_row) = x[u];
            __syncthreads();
        }
    } else {
        float *ks = A.kscale + g * A.scale_group, *vs = A.vscale + g * A.scale_group;
        for (uint32_t i0 = 0; i0 < n; i0 += 256) {
            const uint32_t i = i0 + tid, p = i < n ? keep[i] : ~0u;
            const bool ok = p < A.positions;
            const float a = ok ? ks[p] : 0.0f, b = ok ? vs[p] : 0.0f;
            if (ok && A.account) A.account_out[g * A.account_out_group + A.first + i] = A.account[g * A.account_group + p];
            __syncthreads();
            if (ok) {
                ks[A.first + i] = a;
                vs[A.first + i] = b;
            }
            __syncthreads();
        }
    }
}

void qxe_launch_select(const qxg_kv_select_args &a, hipStream_t s) {
    hipLaunchKernelGGL(qxe_select, dim3(a.groups), dim3(1024), 0, s, a);
}
void qxe_launch_compact(const qxg_kv_compact_args &a, hipStream_t s) {
    hipLaunchKernelGGL(qxe_compact, dim3(2 * ((a.row_bytes + 127) / 128) + 1, a.groups), dim3(256), 0, s, a);
}
