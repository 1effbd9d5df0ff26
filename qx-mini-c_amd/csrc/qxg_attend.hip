// Tree attention over an INT8 cache (qxg_tree_attention) and the account of attention weights.
//
// Mathematics.  s = dot * ks[pos] * scale with dot = q . code.  The codes are exact in fp16; q is
// scaled by a power of two into [2^13, 2^14) and taken as fp16 (16-bit q: exact) or hi + lo (f32 q:
// 22 bits), so the matrix cores' f32 sums are those of f32 products.  The softmax runs in base 2 in
// one pass with a running maximum and denominator a column; weights times vs[pos] go into the second
// product as fp16 (hi + lo for f32) under a power-of-two scale of the column in the chunk.
//
// Tiles.  v_mfma_f32_32x32x16_f16, rows positions, columns (node, q head of the kv head).  Lane half h
// of A and B holds dims (D / 2) h + 8 s + j of k-step s, so a lane's K codes are D / 2 consecutive
// bytes of its row.  Result register r of lane l is position 8 (r / 4) + 4 (l / 32) + r % 4, column
// l % 32: the k layout of the second product's B operand, so weights never leave their lane.
#include "qxg_pf.h"
#include "qxg_ops.h"

namespace {
template <typename T> DEV void load8(const T *p, float (&v)[8]);
template <> DEV void load8(const float *p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> DEV void load8(const _Float16 *p, float (&v)[8]) {
    const h8v a = __builtin_bit_cast(h8v, *reinterpret_cast<const uint4 *>(p));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
}
template <> DEV void load8(const __bf16 *p, float (&v)[8]) {
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <typename T> DEV void store4(T *p, float4 v) {
    T t[4] = {(T)v.x, (T)v.y, (T)v.z, (T)v.w};
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4 *>(p) = v;
    else *reinterpret_cast<uint2 *>(p) = __builtin_bit_cast(uint2, t);
}

struct Seq { uint32_t len, count; };   // of sequence b, clamped to the arrays
DEV Seq sequence(const QxaArgs &A, uint32_t b) {
    Seq s;
    s.count = min(A.a.counts ? A.a.counts[b] : A.a.nodes, min(A.a.nodes, A.a.positions));
    s.len = min(A.a.lens[b], A.a.positions - s.count);
    return s;
}
// The positions from p0 on that the node sees, as bits: the cached ones, then the mask's nodes
DEV uint32_t visible(const QxaArgs &A, const Seq &q, uint32_t b, uint32_t node, uint32_t p0) {
    uint32_t bits, end = q.len + q.count;
    if (A.a.mask) {
        const uint32_t *row = A.a.mask + ((uint64_t)b * A.a.nodes + node) * A.words;
        if (p0 >= q.len) {
            const uint32_t j = p0 - q.len, w = j >> 5;
            const uint64_t two = (w < A.words ? row[w] : 0u) | (uint64_t)(w + 1 < A.words ? row[w + 1] : 0u) << 32;
            bits = (uint32_t)(two >> (j & 31));
        } else {
            const uint32_t cached = q.len - p0;
            bits = cached < 32 ? (row[0] << cached) | ((1u << cached) - 1u) : ~0u;
        }
    } else {
        bits = ~0u;
        end = q.len + min(node + 1, q.count);
    }
    const uint32_t left = end > p0 ? end - p0 : 0u;
    return left < 32 ? bits & ((1u << left) - 1u) : bits;
}
// the mask's bit of register r in lane half h
DEV bool seen(uint32_t bits, int r, int h) { return (bits >> (8 * (r >> 2) + 4 * h + (r & 3))) & 1; }

template <int D> struct KRow { uint4 k[D / 32]; };
template <int D> DEV KRow<D> load_k(const QxaArgs &A, uint32_t b, uint32_t g, uint32_t pos, int h) {
    KRow<D> x;
    const uint4 *row = reinterpret_cast<const uint4 *>(A.a.k + b * A.a.kv_batch + pos * A.a.kv_row + g * D + (D / 2) * h);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) x.k[i] = row[i];
    return x;
}
template <int D> DEV uint4 k_step(const KRow<D> &x, int s) {
    const uint4 w = x.k[s >> 1];
    return s & 1 ? i8x8_to_f16(w.z, w.w) : i8x8_to_f16(w.x, w.y);
}
}  // namespace

// A workgroup takes a tile of columns of one kv head and a run of 32-position chunks; its 4 waves take
// every fourth chunk, each with its own running maximum, denominator and context, merged at the end.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void qxa_tree(QxaArgs A) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int KS = D / 16, DT = D / 32, NP = SPLIT ? 2 : 1;
    __shared__ uint4 s_q[KS * NP * 64];
    __shared__ float s_sf[32], s_ks[4][32], s_vs[4][32], s_m[2][32], s_den[2][32];
    __shared__ union { uint32_t vt[4][D * 9]; float acc[2][32][D + 1]; } u;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), col = lane & 31, h = lane >> 5;
    const uint32_t g = blockIdx.x / A.tiles, tile = blockIdx.x % A.tiles, b = blockIdx.z;
    const Seq q = sequence(A, b);
    const uint32_t c = tile * 32 + col, node = min(c / A.group, A.a.nodes - 1), head = g * A.group + c % A.group;
    const bool used = c < A.columns && node < q.count;
    if (tile * 32 / A.group >= q.count) return;   // the whole tile is behind count
    const uint32_t total = q.len + q.count, nchunk = (total + 31) / 32;
    const uint32_t c_lo = (uint64_t)nchunk * blockIdx.y / A.splits, c_hi = (uint64_t)nchunk * (blockIdx.y + 1) / A.splits;
    {   // q fragments: a thread takes D / 8 dims of a column
        const int qc = tid >> 3, seg = tid & 7;
        const uint32_t cc = tile * 32 + qc, n = cc / A.group;
        const bool ok = cc < A.columns && n < q.count;
        const T *row = (const T *)A.a.q + b * A.a.q_batch + (uint64_t)(ok ? n : 0) * A.a.q_node +
                       (g * A.group + (ok ? cc % A.group : 0)) * D + seg * (D / 8);
        float v[D / 64][8], mx = 0.0f;
        bool fin = true;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
            load8(row + 8 * i, v[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) { fin = fin && isfinite(v[i][j]); mx = fmaxf(mx, fabsf(v[i][j])); }
        }
        mx = fin ? mx : INFINITY;
        mx = fmaxf(mx, dppf<DPP_XOR1>(mx)); mx = fmaxf(mx, dppf<DPP_XOR2>(mx)); mx = fmaxf(mx, dppf<DPP_HALF_MIRROR>(mx));
        const bool bad = !(mx < INFINITY);   // a q that is not finite makes its row NaN
        const float sc = pow2_scale(bad ? 0.0f : mx, 14);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = bad || !ok ? 0.0f : v[i][j];
            uint4 hi, lo;
            split8(v[i], sc, hi, lo);
            const int at = seg * (D / 64) + i, s = at % KS, l = qc + 32 * (at / KS);
            s_q[(s * NP) * 64 + l] = hi;
            if (SPLIT) s_q[(s * NP + 1) * 64 + l] = lo;
        }
        if (seg == 0) s_sf[qc] = bad ? NAN : A.scale2 / sc;
    }
    __syncthreads();
    const float sf = s_sf[col];
    float m = -INFINITY, den = 0.0f;
    f16x acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = zero16();
    uint32_t *vt = u.vt[wave];
#pragma unroll 1
    for (uint32_t ci = c_lo + wave; ci < c_hi; ci += 4) {
        const uint32_t pb = ci * 32, pk = min(pb + col, total - 1);   // (rows past the last read it again)
        const KRow<D> kr = load_k<D>(A, b, g, pk, h);
        if (lane < 32) {
            s_ks[wave][lane] = A.a.kscale[b * A.a.scale_batch + pk];
            s_vs[wave][lane] = A.a.vscale[b * A.a.scale_batch + pk];
        }
        // V transposed: 4 positions x 4 dims of bytes a lane and step
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const int bq = lane + 64 * i, pq = bq & 7, dq = bq >> 3;
            uint32_t w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                w[r] = *reinterpret_cast<const uint32_t *>(A.a.v + b * A.a.kv_batch + min(pb + 4 * pq + r, total - 1) * A.a.kv_row + g * D + 4 * dq);
            const uint32_t a0 = perm(w[1], w[0], 0x05010400u), a1 = perm(w[3], w[2], 0x05010400u);
            const uint32_t a2 = perm(w[1], w[0], 0x07030602u), a3 = perm(w[3], w[2], 0x07030602u);
            vt[(4 * dq + 0) * 9 + pq] = perm(a1, a0, 0x05040100u);
            vt[(4 * dq + 1) * 9 + pq] = perm(a1, a0, 0x07060302u);
            vt[(4 * dq + 2) * 9 + pq] = perm(a3, a2, 0x05040100u);
            vt[(4 * dq + 3) * 9 + pq] = perm(a3, a2, 0x07060302u);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        f16x sh = zero16(), sl = zero16();
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint4 kf = k_step<D>(kr, s);
            sh = mfma(kf, s_q[(s * NP) * 64 + lane], sh);
            if (SPLIT) sl = mfma(kf, s_q[(s * NP + 1) * 64 + lane], sl);
        }
        const bool edge = pb + 32 > q.len;   // the chunk holds nodes
        const uint32_t bits = edge ? visible(A, q, b, node, pb) : ~0u;
        float sc[16], e[16], pv[16], cmax = -INFINITY, pmx = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float k = s_ks[wave][8 * (r >> 2) + 4 * h + (r & 3)];
            sc[r] = (SPLIT ? sh[r] + sl[r] : sh[r]) * k * sf;
            if (edge) sc[r] = seen(bits, r, h) ? sc[r] : -INFINITY;
            cmax = fmaxf(cmax, sc[r]);
        }
        cmax = fmaxf(cmax, __shfl_xor(cmax, 32));
        if (__ballot(cmax > m + 8.0f) != 0) {
            const float mn = fmaxf(m, cmax), alpha = m == mn ? 1.0f : exp2_fast(m - mn);
            m = mn;
            den *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= alpha;
        }
        const float mm = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            e[r] = exp2_fast(sc[r] - mm);
            pv[r] = e[r] * s_vs[wave][8 * (r >> 2) + 4 * h + (r & 3)];
            if (edge) pv[r] = seen(bits, r, h) ? pv[r] : 0.0f;
            den += e[r];
            pmx = fmaxf(pmx, fabsf(pv[r]));
        }
        pmx = fmaxf(pmx, __shfl_xor(pmx, 32));
        const float psc = pow2_scale(pmx, 15), pinv = 1.0f / psc;
        uint4 phi[2], plo[2];
        split8(pv, psc, phi[0], plo[0]);
        split8(pv + 8, psc, phi[1], plo[1]);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            f16x x = zero16();
            const uint32_t *row = vt + (32 * d + col) * 9;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint4 vf = i8x8_to_f16(row[4 * s + h], row[4 * s + 2 + h]);
                x = mfma(vf, phi[s], x);
                if (SPLIT) x = mfma(vf, plo[s], x);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] = fmaf(x[r], pinv, acc[d][r]);
        }
    }
    // merge the 4 waves: 2 + 3 into 0 + 1, then 1 into 0
    den += __shfl_xor(den, 32);
    __syncthreads();
#pragma unroll 1
    for (int nw = 2; nw; nw >>= 1) {
        if (wave >= nw && wave < 2 * nw) {
            const int slot = wave - nw;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) u.acc[slot][col][32 * d + 8 * (r >> 2) + 4 * h + (r & 3)] = acc[d][r];
            if (h == 0) { s_m[slot][col] = m; s_den[slot][col] = den; }
        }
        __syncthreads();
        if (wave < nw) {
            const float mo = s_m[wave][col], mn = fmaxf(m, mo);
            const float fa = m == mn ? 1.0f : exp2_fast(m - mn), fb = mo == mn ? 1.0f : exp2_fast(mo - mn);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    acc[d][r] = acc[d][r] * fa + u.acc[wave][col][32 * d + 8 * (r >> 2) + 4 * h + (r & 3)] * fb;
            den = den * fa + s_den[wave][col] * fb;
            m = mn;
        }
        __syncthreads();
    }
    if (wave == 0 && used) {
        const uint64_t row = ((uint64_t)b * A.a.nodes + node) * A.a.heads + head;
        if (A.splits == 1) {
            const float inv = den == 0.0f ? 0.0f : 1.0f / den;
            T *out = (T *)A.a.out + b * A.a.out_batch + node * A.a.out_node + head * D;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    store4(out + 32 * d + 8 * k + 4 * h,
                           make_float4(acc[d][4 * k] * inv, acc[d][4 * k + 1] * inv, acc[d][4 * k + 2] * inv, acc[d][4 * k + 3] * inv));
            if (h == 0 && A.lse) A.lse[row] = den == 0.0f ? -INFINITY : (m + __log2f(den)) * 0.69314718055994531f;
        } else {
            const uint64_t at = (uint64_t)blockIdx.y * A.a.batch * A.a.nodes * A.a.heads + row;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    store4(A.part + at * D + 32 * d + 8 * k + 4 * h,
                           make_float4(acc[d][4 * k], acc[d][4 * k + 1], acc[d][4 * k + 2], acc[d][4 * k + 3]));
            if (h == 0) A.md[at] = make_float2(m, den);
        }
    }
}

// The splits of a row joined: a wave a row, splits in order.
template <typename T, int D>
__global__ __launch_bounds__(256) void qxa_join(QxaArgs A) {
    const uint64_t rows = (uint64_t)A.a.batch * A.a.nodes * A.a.heads, row = blockIdx.x * 4ull + wave_id();
    if (row >= rows) return;
    const int lane = threadIdx.x & 63;
    const uint32_t head = row % A.a.heads, node = row / A.a.heads % A.a.nodes, b = row / A.a.heads / A.a.nodes;
    if (node >= sequence(A, b).count) return;
    float m = -INFINITY, den = 0.0f, v[D / 64] = {};
    for (uint32_t z = 0; z < A.splits; ++z) m = fmaxf(m, A.md[z * rows + row].x);
    for (uint32_t z = 0; z < A.splits; ++z) {
        const uint64_t at = z * rows + row;
        const float2 s = A.md[at];
        const float f = s.x == m ? 1.0f : exp2_fast(s.x - m);
        den = fmaf(f, s.y, den);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) v[i] = fmaf(f, A.part[at * D + 64 * i + lane], v[i]);
    }
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
    T *out = (T *)A.a.out + b * A.a.out_batch + node * A.a.out_node + head * D;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) out[64 * i + lane] = (T)(v[i] * inv);
    if (lane == 0 && A.lse) A.lse[row] = den == 0.0f ? -INFINITY : (m + __log2f(den)) * 0.69314718055994531f;
}

// account[p] = decay * account[p] + sum over nodes and heads of 2^(s - lse).  A workgroup takes 32
// positions; its waves take every fourth (kv head, tile), compute the scores again and keep, per lane,
// its column's sums of the 16 positions that its registers hold; lanes and waves are added up in a
// fixed order, so no two workgroups add to one position.
template <typename T, int D>
__global__ __launch_bounds__(256) void qxa_account(QxaArgs A) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int KS = D / 16;
    __shared__ float s_sum[4][32];
    const int lane = threadIdx.x & 63, wave = wave_id(), col = lane & 31, h = lane >> 5;
    const uint32_t b = blockIdx.y;
    const Seq q = sequence(A, b);
    const uint32_t total = q.len + q.count, nchunk = (total + 31) / 32;
    for (uint32_t ci = blockIdx.x; ci < nchunk; ci += gridDim.x) {
        const uint32_t pb = ci * 32, pk = min(pb + col, total - 1);
        const bool edge = pb + 32 > q.len;
        float ks[16], sum[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            ks[r] = A.a.kscale[b * A.a.scale_batch + min(pb + 8 * (r >> 2) + 4 * h + (r & 3), total - 1)];
            sum[r] = 0.0f;
        }
        for (uint32_t pair = wave; pair < A.a.kv_heads * A.tiles; pair += 4) {
            const uint32_t g = pair / A.tiles, c = pair % A.tiles * 32 + col, node = min(c / A.group, A.a.nodes - 1);
            if (pair % A.tiles * 32 / A.group >= q.count) continue;
            const bool used = c < A.columns && node < q.count;
            const uint32_t head = g * A.group + (used ? c % A.group : 0);
            const KRow<D> kr = load_k<D>(A, b, g, pk, h);
            const T *row = (const T *)A.a.q + b * A.a.q_batch + (used ? node : 0) * A.a.q_node + head * D + (D / 2) * h;
            float v[KS][8], mx = 0.0f;
            bool fin = true;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                load8(row + 8 * s, v[s]);
#pragma unroll
                for (int j = 0; j < 8; ++j) { fin = fin && isfinite(v[s][j]); mx = fmaxf(mx, fabsf(v[s][j])); }
            }
            mx = fin ? mx : INFINITY;
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const bool bad = !(mx < INFINITY);
            const float psc = pow2_scale(bad ? 0.0f : mx, 14), sf = bad ? NAN : A.scale2 / psc;
            f16x sh = zero16(), sl = zero16();
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint4 kf = k_step<D>(kr, s);
                uint4 hi, lo;
                split8(v[s], bad ? 0.0f : psc, hi, lo);
                sh = mfma(kf, hi, sh);
                if (SPLIT) sl = mfma(kf, lo, sl);
            }
            const float l = used ? A.lse[((uint64_t)b * A.a.nodes + node) * A.a.heads + head] : -INFINITY;
            const float l2 = l * 1.4426950408889634f;
            const uint32_t bits = l == -INFINITY ? 0u : edge ? visible(A, q, b, node, pb) : ~0u;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float sc = (SPLIT ? sh[r] + sl[r] : sh[r]) * ks[r] * sf;
                sum[r] += seen(bits, r, h) ? exp2_fast(sc - l2) : 0.0f;
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
#pragma unroll
            for (int o = 16; o; o >>= 1) sum[r] += __shfl_xor(sum[r], o);
            if (col == 0) s_sum[wave][8 * (r >> 2) + 4 * h + (r & 3)] = sum[r];
        }
        __syncthreads();
        const uint32_t p = pb + threadIdx.x;
        if (threadIdx.x < 32 && p < total) {
            float *at = A.a.account + b * A.a.account_batch + p;
            const int t = threadIdx.x;
            *at = *at * A.a.decay + ((s_sum[0][t] + s_sum[1][t]) + (s_sum[2][t] + s_sum[3][t]));
        }
        __syncthreads();
    }
}

namespace {
template <typename T, int D> void launch(const QxaArgs &A, hipStream_t s) {
    const uint64_t rows = (uint64_t)A.a.batch * A.a.nodes * A.a.heads;
    hipLaunchKernelGGL((qxa_tree<T, D>), dim3(A.a.kv_heads * A.tiles, A.splits, A.a.batch), dim3(256), 0, s, A);
    if (A.splits > 1) hipLaunchKernelGGL((qxa_join<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, A);
    if (A.a.account) {
        const uint32_t chunks = (uint32_t)std::min<uint64_t>(65535, ((uint64_t)A.a.max_len + A.a.nodes + 31) / 32);
        hipLaunchKernelGGL((qxa_account<T, D>), dim3(chunks, A.a.batch), dim3(256), 0, s, A);
    }
}
}  // namespace

void qxa_launch(const QxaArgs &A, hipStream_t s) {
    if (A.a.type == QXG_TYPE_F32) A.a.dim == 64 ? launch<float, 64>(A, s) : launch<float, 128>(A, s);
    else if (A.a.type == QXG_TYPE_F16) A.a.dim == 64 ? launch<_Float16, 64>(A, s) : launch<_Float16, 128>(A, s);
    else A.a.dim == 64 ? launch<__bf16, 64>(A, s) : launch<__bf16, 128>(A, s);
}
