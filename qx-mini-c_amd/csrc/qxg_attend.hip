// Tree attention over an INT8 cache (qxg_tree_attention) and the account of attention weights.
//
// Mathematics.  s = dot * ks[pos] * scale with dot = q . code.  The codes are exact in fp16; q is
// scaled by a power of two into [2^13, 2^14) and taken as fp16 (16-bit q: exact) or hi + lo (f32 q:
// 22 bits), so the matrix cores' f32 sums are those of f32 products.  The softmax runs in base 2 in
// one pass: a column keeps a reference M, the sum of e = 2^(s - M) and the context, the sum of e vs[pos] v.
// M follows the running maximum to within 2^8 and is shifted by a power of two that keeps e vs, which enters
// the second product as fp16 hi + lo, in fp16's range; it cancels in the end.  (hi alone, 11 bits, put even BF16
// results off by up to 2^-10 of their terms' size, which shows where terms cancel; lo costs 4 x 1 nodes over 30000 positions
// 1 us of 58, 8 x 13 over 2900 nothing that shows.)
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
// The splits of a sequence: their number and where they start among all sequences' (the states in part and md
// lie in that order).  About A.splits for the whole batch, shared out by the sequences' chunks of 32
// positions, so that a split is about as long in each; up to twice as many where nodes are not in use, so that
// there are as many workgroups all the same; beyond 64 sequences as many for each.
struct Splits { uint32_t count, first; };
DEV bool shared_out(const QxaArgs &A) { return A.a.batch <= 64 && A.splits > 1; }
// running sum over the wave's lanes
DEV uint32_t wave_running(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xf, 0xf, true);   // row_shr:1, 2, 4, 8
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xf, 0xf, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, false);   // row_bcast:15 into rows 1 and 3
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, false);   // row_bcast:31 into rows 2 and 3
    return v;
}
DEV float wave_sum(float v) {   // of all lanes, in a fixed order
    v += dppf<DPP_XOR1>(v); v += dppf<DPP_XOR2>(v); v += dppf<DPP_ROR4>(v); v += dppf<DPP_ROR8>(v);
    return (rdlanef(v, 0) + rdlanef(v, 16)) + (rdlanef(v, 32) + rdlanef(v, 48));
}
DEV uint32_t chunks_of(const Seq &q) { return max(1u, (q.len + q.count + 31) / 32); }
DEV Splits lane_splits(const QxaArgs &A) {   // of sequence `lane`
    const uint32_t lane = threadIdx.x & 63;
    uint32_t chunks = 0;
    float all = 0.0f, busy = 0.0f;   // (shares need not be exact, only the same in every workgroup)
    if (lane < A.a.batch) {
        const Seq q = sequence(A, lane);
        chunks = chunks_of(q);
        all = (float)chunks;
        busy = all * (float)((q.count * A.group + A.wg_columns - 1) / A.wg_columns);   // times workgroups with nodes in use
    }
    all = wave_sum(all);
    busy = wave_sum(busy);
    const float share = (float)chunks * (float)A.splits * fminf((float)A.wgs / busy, 2.0f / all);
    const uint32_t n = lane < A.a.batch ? min(chunks, max(1u, (uint32_t)share)) : 0u;
    return {n, wave_running(n) - n};
}
DEV Splits splits_of(const QxaArgs &A, uint32_t b) {
    if (!shared_out(A)) return {A.splits, b * A.splits};
    if (A.a.batch == 1) return {min(chunks_of(sequence(A, 0)), A.splits), 0};
    const Splits s = lane_splits(A);
    return {(uint32_t)__builtin_amdgcn_readlane((int)s.count, (int)b), (uint32_t)__builtin_amdgcn_readlane((int)s.first, (int)b)};
}
// The workgroup's sequence and split: of all sequences' splits in order, or by the grid.  count 0: none
struct Job { uint32_t b, z; Splits s; };
DEV Job job_of(const QxaArgs &A) {
    Job j{blockIdx.z, blockIdx.y, {A.splits, blockIdx.z * A.splits}};
    if (A.a.batch == 1 && A.splits > 1) {
        j = {0, blockIdx.y, splits_of(A, 0)};
        if (j.z >= j.s.count) j.s.count = 0;
    } else if (shared_out(A)) {
        const Splits s = lane_splits(A);
        const uint64_t mine = __ballot(s.count && s.first <= blockIdx.y);
        j.b = 63u - (uint32_t)__builtin_clzll(mine);   // (the first sequence's start at 0)
        j.s.count = (uint32_t)__builtin_amdgcn_readlane((int)s.count, (int)j.b);
        j.s.first = (uint32_t)__builtin_amdgcn_readlane((int)s.first, (int)j.b);
        j.z = blockIdx.y - j.s.first;
        if (j.z >= j.s.count) j.s.count = 0;
    }
    return j;
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
// the mask's bit of register r, of bits >> 4 h in lane half h
DEV bool seen(uint32_t w, int r) { return w & (1u << (8 * (r >> 2) + (r & 3))); }

// What turns dot * kscale into base-2 scores, of a q scaled by sc.  Not 0, with which -inf in a masked place would become
// NaN (so small a factor, of dots below 2^28, leaves all scores as good as 0 anyway).
DEV float score_factor(const QxaArgs &A, float sc, bool bad) {   // bad: a q that is not finite, which makes its row NaN
    return bad ? NAN : fmaxf(A.scale2 / sc, 0x1p-126f);
}

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

namespace {
// A column's softmax state.  Both halves of a wave hold their columns' m, c, M, most and limit; den is each lane's own
// sum.  m (the maximum, rounded, as of the last time that it grew by 8) and c (M's shift) are whole numbers, M = m - c, so
// that moving M and scaling what has been summed by the power of two that belongs to it agree exactly.  Where f32 has no room
// for that (m from FAR on), e is 2^((s - m) + c) instead of 2^(s - M), with s rounded as m is: with M alone, equal scores
// weighed differently from 2^24 on.
constexpr float FAR = 4194304.0f;
template <int D> struct State {
    // most: the largest |e vs| so far.  limit: what it may reach before M has to move; 0 where m has grown, so that the next
    // weights place it anew (else values far smaller than those before them, which outweigh them, lost bits:
    // V scales smaller by 10^6, scores higher by 2^80: 8e-5 off, by 10^9: 8e-2).
    float m = -INFINITY, M = -INFINITY, den = 0.0f, most = 0.0f, limit = 0.0f, c = 0.0f;
    bool far = false;   // one of the wave's columns is
    f16x acc[D / 32];
    DEV State() {
#pragma unroll
        for (int d = 0; d < D / 32; ++d) acc[d] = zero16();
    }
    DEV void rescale(float f) {
        den *= f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] *= f;
    }
    DEV void close() {   // before it is joined with others: M holds the shift or there is none
        if (!far) return;
        rescale(exp2_fast(-c));
        M = m;
    }
};
DEV float max_of_halves(float v) {   // of lanes l and l ^ 32
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
DEV float max16(const float (&v)[16]) {   // (as a tree: a dependent instruction waits twice as long as another)
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = fmaxf(fmaxf(v[4 * i], v[4 * i + 1]), fmaxf(v[4 * i + 2], v[4 * i + 3]));
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
template <typename T> constexpr bool two_halves_q = sizeof(T) == 4;

// v = hi + lo (+ 2^-22 of it), a conversion for two values and one mixed-precision fma a remainder (its factor is
// hidden, or it becomes a conversion back and a subtraction)
typedef float f2v __attribute__((ext_vector_type(2)));
DEV void split_pairs(const float *v, uint4 &hi, uint4 &lo) {
    float minus = -1.0f;
    asm("" : "+s"(minus));
    uint32_t a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f2v x = {v[2 * i], v[2 * i + 1]};
        const h2v h = __builtin_convertvector(x, h2v);
        a[i] = __builtin_bit_cast(uint32_t, h);
        const h2v l = {(_Float16)fmaf((float)h[0], minus, x[0]), (_Float16)fmaf((float)h[1], minus, x[1])};
        b[i] = __builtin_bit_cast(uint32_t, l);
    }
    hi = make_uint4(a[0], a[1], a[2], a[3]);
    lo = make_uint4(b[0], b[1], b[2], b[3]);
}

// A chunk's scores into weights, in steps.  bits: the chunk's positions that the column sees (edge: not all of them,
// for some column; each of the two uses opens the word anew, or the tests of its bits move into every chunk).
//
// Of the scores (still to be multiplied by sf): the mask, and the maximum, which moves M where it has grown by 8.
template <int D>
DEV void reference(State<D> &S, float sf, bool edge, uint32_t bits, int h, float (&s)[16]) {
    if (edge) {
        uint32_t w = bits >> (4 * h);
        asm volatile("" : "+v"(w));
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = seen(w, r) ? s[r] : -INFINITY;
    }
    const float cmax = max_of_halves(max16(s)) * sf;   // (sf > 0, or NaN)
    if (__ballot(cmax > S.m + 8.0f) != 0) {   // (whole wave)
        const bool grow = cmax > S.m + 8.0f;
        const float mn = rintf(cmax);
        const float f = !grow || S.m == -INFINITY ? 1.0f : exp2_fast(S.m - mn);
        S.rescale(f);
        S.most *= f;
        if (grow) {
            S.M = mn - S.c;
            S.m = mn;
            S.limit = 0.0f;
        }
        S.far = S.far || __ballot(grow && fabsf(mn) >= FAR) != 0;
    }
}
// The weights as the second product's operands phi and plo, M moved where they leave fp16's range
template <int D>
DEV void operands(State<D> &S, float den, float sf, bool edge, uint32_t bits, int h, float (&p)[16], uint4 (&phi)[2], uint4 (&plo)[2]) {
    if (edge) {   // (a masked position's scales do not count, whatever they are; fma(-inf, NaN) is NaN)
        uint32_t w = bits >> (4 * h);
        asm volatile("" : "+v"(w));
        if (sf != sf && bits == 0) den = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = seen(w, r) ? p[r] : 0.0f;
    }
    S.den += den;
    float a[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) a[r] = fabsf(p[r]);
    const float pmx = max_of_halves(max16(a));
    S.most = fmaxf(S.most, pmx);
    if (__ballot(pmx > S.limit) != 0) {   // the first weights after m has grown, or one beyond fp16
        const bool move = pmx > S.limit && pmx < INFINITY;
        // the largest so far to [2^6, 2^7), but e itself (up to 2^8 times the shift) stays far inside f32; a
        // larger one, where that has kept it from there, moves M again
        int k = (int)(__float_as_uint(pow2_scale(S.most, 7)) >> 23) - 127;
        k = move ? max(min(k, 96 - (int)S.c), -126) : 0;
        const float f = __uint_as_float((uint32_t)(127 + k) << 23);
        S.most *= f;
        if (move) {
            S.c += (float)k;
            S.M = S.m - S.c;
            S.limit = S.most < 64.0f ? S.most : 32768.0f;
        }
        S.rescale(f);
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] *= f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) split_pairs(p + 8 * i, phi[i], plo[i]);
}
// all of a chunk at once; its scores to keep, if there is one
template <int D>
DEV void weigh(State<D> &S, const f16x &dot, float sf, const float *ks, const float *vs, bool edge, uint32_t bits, int h, uint4 (&phi)[2],
               uint4 (&plo)[2], f4x *keep = nullptr) {
    float s[16], p[16], den[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f4x k4 = *reinterpret_cast<const f4x *>(ks + 8 * j + 4 * h);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * j + r] = dot[4 * j + r] * k4[r];
    }
    reference<D>(S, sf, edge, bits, h, s);
    if (keep) {
#pragma unroll
        for (int r = 0; r < 16; ++r) keep[r / 4][r % 4] = s[r];
    }
    const float M = S.M == -INFINITY ? 0.0f : S.M;
    if (!S.far) {
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = fmaf(s[r], sf, -M);
    } else {
        const bool far = S.m != -INFINITY && fabsf(S.m) >= FAR;
#pragma unroll
        for (int r = 0; r < 16; ++r) p[r] = far ? (s[r] * sf - S.m) + S.c : fmaf(s[r], sf, -M);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f4x v4 = *reinterpret_cast<const f4x *>(vs + 8 * j + 4 * h);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float e = exp2_fast(p[4 * j + r]);
            den[r] += e;
            p[4 * j + r] = e * v4[r];
        }
    }
    operands<D>(S, (den[0] + den[1]) + (den[2] + den[3]), sf, edge, bits, h, p, phi, plo);
}
// column c of kv head g
struct Column { uint32_t node, head; bool used; };
DEV Column column(const QxaArgs &A, const Seq &q, uint32_t g, uint32_t c) {
    const uint32_t node = min(c / A.group, A.a.nodes - 1);
    return {node, g * A.group + c % A.group, c < A.columns && node < q.count};
}
// A row's sums: lse, and for the account what makes weights of scores, as they were summed (weights by lse, in f32, were 10^-4
// off for scores around 1000).
DEV void finish_row(const QxaArgs &A, float M, float den, uint64_t row) {
    if (A.a.lse) A.a.lse[row] = den == 0.0f ? -INFINITY : (M + __log2f(den)) * 0.69314718055994531f;
    if (A.norm) A.norm[row] = den == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(M, 1.0f / den);
}
// a column's sums, or with several splits the state's part
DEV void finish_sums(const QxaArgs &A, float M, float den, bool whole, uint64_t row, uint64_t state) {
    if (!whole) A.md[state] = make_float2(M, den);
    else finish_row(A, M, den, row);
}
// a column's result: out, or with several splits its state
template <typename T, int D>
DEV void finish_column(const QxaArgs &A, const State<D> &S, float den, const Job &job, uint32_t node, uint32_t head, int h) {
    const uint32_t b = job.b;
    const uint64_t row = ((uint64_t)b * A.a.nodes + node) * A.a.heads + head;
    if (A.splits == 1) {
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
        T *out = (T *)A.a.out + b * A.a.out_batch + node * A.a.out_node + head * D;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                store4(out + 32 * d + 8 * k + 4 * h, make_float4(S.acc[d][4 * k] * inv, S.acc[d][4 * k + 1] * inv,
                                                                 S.acc[d][4 * k + 2] * inv, S.acc[d][4 * k + 3] * inv));
        if (h == 0) finish_sums(A, S.M, den, true, row, 0);
    } else {
        const uint64_t at = (uint64_t)(job.s.first + job.z) * A.a.nodes * A.a.heads + node * A.a.heads + head;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                store4(A.part + at * D + 32 * d + 8 * k + 4 * h,
                       make_float4(S.acc[d][4 * k], S.acc[d][4 * k + 1], S.acc[d][4 * k + 2], S.acc[d][4 * k + 3]));
        if (h == 0) finish_sums(A, S.M, den, false, row, at);
    }
}
}  // namespace

// Few columns, or little work.  A workgroup takes a tile of columns of one kv head and a run of
// 32-position chunks; its 4 waves take every fourth chunk, each with a state of its own, merged at the end.  The
// next chunk's rows are on their way while one is worked on.  The cache's bytes bound it (single BF16 tokens over 4 x
// 30000 positions of 8 kv heads, 247 MB: 62 us, 4.0 TB/s where a copy has 5.1; over 14000 to 30000 each, 176 MB, 50 us, 59
// where scores are kept, KEEP), or with few of them the chain of latencies: 8.5 us for a token over 37 positions, 12.8 for 16
// nodes of 32 heads over 1500 (splits of a chunk a wave), 27 for 64 nodes over 4032, where issue counts as well.
template <typename T, int D, bool KEEP>
__global__ __launch_bounds__(256, 2) void qxa_tree(QxaArgs A) {
    constexpr bool SPLIT = two_halves_q<T>;
    constexpr int KS = D / 16, DT = D / 32, NP = SPLIT ? 2 : 1;
    __shared__ uint4 s_q[KS * NP * 64];
    __shared__ float s_sf[32];
    __shared__ __align__(16) float s_ks[4][32], s_vs[4][32];
    __shared__ float s_m[2][32], s_den[2][32];
    __shared__ union { uint32_t vt[4][D * 9]; float acc[2][32][D + 1]; } u;
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), col = lane & 31, h = lane >> 5;
    const uint32_t g = blockIdx.x / A.tiles, tile = blockIdx.x % A.tiles;
    struct { KRow<D> k; uint32_t v[4 * DT]; float ks, vs; } nx;
    auto load = [&](uint32_t b, uint32_t ci) {   // (rows past the array's last read it again; those behind the nodes are masked)
        const uint32_t pb = ci * 32, last = A.a.positions - 1, pk = min(pb + col, last);
        nx.k = load_k<D>(A, b, g, pk, h);
        nx.ks = A.a.kscale[b * A.a.scale_batch + pk];
        nx.vs = A.a.vscale[b * A.a.scale_batch + pk];
#pragma unroll
        for (int i = 0; i < DT; ++i) {   // 4 positions x 4 dims of bytes a lane and step
            const int bq = lane + 64 * i, dq = bq % (D / 4), pq = bq / (D / 4);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                nx.v[4 * i + r] = *reinterpret_cast<const uint32_t *>(A.a.v + b * A.a.kv_batch + min(pb + 4 * pq + r, last) * A.a.kv_row + g * D + 4 * dq);
        }
    };
    const int qc = tid >> 3, seg = tid & 7;   // q: a thread takes D / 8 dims of a column
    const uint32_t qcc = tile * 32 + qc;
    float qv[D / 64][8];
    auto load_q = [&](uint32_t b) {
        const T *row = (const T *)A.a.q + b * A.a.q_batch + (uint64_t)(qcc < A.columns ? qcc / A.group : 0) * A.a.q_node +
                       (g * A.group + (qcc < A.columns ? qcc % A.group : 0)) * D + seg * (D / 8);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) load8(row + 8 * i, qv[i]);
    };
    // Where the sequence needs no lengths to be known, q (and the first chunk, if the split starts at 0) need not wait
    // for them (0.6 us of a small call).
    const bool known = !shared_out(A) || A.a.batch == 1;
    if (known) load_q(blockIdx.z);
    if (A.splits == 1) load(blockIdx.z, wave);
    const Job job = job_of(A);
    const uint32_t b = job.b;
    const Seq q = sequence(A, b);
    const uint32_t c = tile * 32 + col, node = min(c / A.group, A.a.nodes - 1), head = g * A.group + c % A.group;
    const bool used = c < A.columns && node < q.count;
    if (job.s.count == 0 || tile * 32 / A.group >= q.count) return;   // the whole tile is behind count
    const uint32_t total = q.len + q.count, nchunk = (total + 31) / 32;
    const uint32_t c_lo = (uint64_t)nchunk * job.z / job.s.count, c_hi = (uint64_t)nchunk * (job.z + 1) / job.s.count;
    if (A.splits > 1 && c_lo + wave < c_hi) load(b, c_lo + wave);
    if (!known) load_q(b);
    {
        const bool ok = qcc < A.columns && qcc / A.group < q.count;
        float mx = 0.0f;
        bool fin = true;
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) { fin = fin && isfinite(qv[i][j]); mx = fmaxf(mx, fabsf(qv[i][j])); }
        mx = fin ? mx : INFINITY;
        mx = fmaxf(mx, dppf<DPP_XOR1>(mx)); mx = fmaxf(mx, dppf<DPP_XOR2>(mx)); mx = fmaxf(mx, dppf<DPP_HALF_MIRROR>(mx));
        const bool bad = !(mx < INFINITY);
        const float sc = pow2_scale(bad ? 0.0f : mx, 14);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
#pragma unroll
            for (int j = 0; j < 8; ++j) qv[i][j] = bad || !ok ? 0.0f : qv[i][j];
            uint4 hi, lo;
            split8(qv[i], sc, hi, lo);
            const int at = seg * (D / 64) + i, s = at % KS, l = qc + 32 * (at / KS);
            s_q[(s * NP) * 64 + l] = hi;
            if (SPLIT) s_q[(s * NP + 1) * 64 + l] = lo;
        }
        if (seg == 0) s_sf[qc] = score_factor(A, sc, bad);
    }
    __syncthreads();
    const float sf = s_sf[col];
    if (A.pack_sf && job.z == 0) {   // the account's q
        const uint64_t at = ((uint64_t)b * A.a.kv_heads + g) * A.tiles + tile;
        if (A.pack)
            for (int i = tid; i < KS * NP * 64; i += 256) A.pack[at * (KS * NP * 64) + i] = s_q[i];
        if (tid < 32) A.pack_sf[at * 32 + tid] = s_sf[tid];
    }
    State<D> S;
    f4x kept[KEEP ? 4 : 1];   // a chunk's scores, written before the loads that the next chunk issues (a wait for loads waits for older stores)
    auto keep_scores = [&](uint32_t ci) {
        float *to = A.scores + ((((uint64_t)b * A.a.kv_heads + g) * ((A.a.positions + 31) / 32) + ci) * A.columns + c) * 32 + 4 * h;
        if (used)
#pragma unroll
            for (int j = 0; j < (KEEP ? 4 : 1); ++j) *reinterpret_cast<f4x *>(to + 8 * j) = kept[j];
    };
    uint32_t *vt = u.vt[wave];
#pragma unroll 1
    for (uint32_t ci = c_lo + wave; ci < c_hi; ci += 4) {
        const uint32_t pb = ci * 32;
        const KRow<D> kr = nx.k;
        if (lane < 32) {
            s_ks[wave][lane] = nx.ks;
            s_vs[wave][lane] = nx.vs;
        }
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const int bq = lane + 64 * i, dq = bq % (D / 4), pq = bq / (D / 4);
            const uint32_t *w = nx.v + 4 * i;
            const uint32_t a0 = perm(w[1], w[0], 0x05010400u), a1 = perm(w[3], w[2], 0x05010400u);
            const uint32_t a2 = perm(w[1], w[0], 0x07030602u), a3 = perm(w[3], w[2], 0x07030602u);
            vt[(4 * dq + 0) * 9 + pq] = perm(a1, a0, 0x05040100u);
            vt[(4 * dq + 1) * 9 + pq] = perm(a1, a0, 0x07060302u);
            vt[(4 * dq + 2) * 9 + pq] = perm(a3, a2, 0x05040100u);
            vt[(4 * dq + 3) * 9 + pq] = perm(a3, a2, 0x07060302u);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (KEEP && ci >= c_lo + 4) keep_scores(ci - 4);
        if (ci + 4 < c_hi) load(b, ci + 4);
        f16x dot = zero16();
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint4 kf = k_step<D>(kr, s);
            if (SPLIT) dot = mfma(kf, s_q[(s * NP + 1) * 64 + lane], dot);
            dot = mfma(kf, s_q[(s * NP) * 64 + lane], dot);
        }
        const bool edge = pb + 32 > q.len;   // the chunk holds nodes
        const uint32_t bits = edge ? visible(A, q, b, node, pb) : ~0u;
        uint4 phi[2], plo[2];
        weigh<D>(S, dot, sf, s_ks[wave], s_vs[wave], edge, bits, h, phi, plo, KEEP ? kept : nullptr);
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const uint32_t *row = vt + (32 * d + col) * 9;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint4 vf = i8x8_to_f16(row[4 * s + h], row[4 * s + 2 + h]);
                S.acc[d] = mfma(vf, plo[s], S.acc[d]);
                S.acc[d] = mfma(vf, phi[s], S.acc[d]);
            }
        }
    }
    if (KEEP && c_lo + wave < c_hi) keep_scores(c_lo + wave + (c_hi - 1 - c_lo - wave) / 4 * 4);   // the last chunk's
    S.close();
    // merge the 4 waves: 2 + 3 into 0 + 1, then 1 into 0
    float den = S.den + __shfl_xor(S.den, 32);
    __syncthreads();
#pragma unroll 1
    for (int nw = 2; nw; nw >>= 1) {
        if (c_hi - c_lo <= (uint32_t)nw) continue;   // (uniform) the others had no chunk
        if (wave >= nw && wave < 2 * nw) {
            const int slot = wave - nw;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) u.acc[slot][col][32 * d + 8 * (r >> 2) + 4 * h + (r & 3)] = S.acc[d][r];
            if (h == 0) { s_m[slot][col] = S.M; s_den[slot][col] = den; }
        }
        __syncthreads();
        if (wave < nw) {
            const float mo = s_m[wave][col], mn = fmaxf(S.M, mo);
            const float fa = S.M == mn ? 1.0f : exp2_fast(S.M - mn), fb = mo == mn ? 1.0f : exp2_fast(mo - mn);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    S.acc[d][r] = S.acc[d][r] * fa + u.acc[wave][col][32 * d + 8 * (r >> 2) + 4 * h + (r & 3)] * fb;
            den = den * fa + s_den[wave][col] * fb;
            S.M = mn;
        }
        __syncthreads();
    }
    if (wave == 0 && used) finish_column<T, D>(A, S, den, job, node, head, h);
}

// Many columns and much work.  The 4 waves of a workgroup take a tile of 32 columns of one kv head each and go through the
// same chunks of 32 positions, whose codes the workgroup stages in LDS as fp16 (K by rows; V transposed, a
// dim's 32 positions in the order of the second product's k): one conversion of a code for 128 columns.  Two
// buffers, so one barrier a chunk; the next chunk's codes are on their way.
// Instruction issue bounds it: 2 x 48 nodes of 32 heads over 65500 positions (f16, weights as hi + lo, so 24
// matrix instructions a chunk) take 167 us, 600 TFLOP/s of matrix work; the matrix pipe is busy a third of the
// cycles, the vector pipe under half, LDS two fifths, and a wave's softmax does not fit behind the other wave's
// products.  The same with chunks of 64 positions, with the next chunk's scores computed ahead, with three waves
// a SIMD (10 registers spilled): 157 .. 164 us, where this form had 162.
template <typename T, int D>
__global__ __launch_bounds__(256, 2) void qxa_wide(QxaArgs A) {
    constexpr bool SPLIT = two_halves_q<T>;
    constexpr int KS = D / 16, DT = D / 32;
    constexpr int KP = D + 8, VP = 40;   // fp16 from one row to the next: 16 rows' 16-byte pieces lie in 16 bank groups
    __shared__ __align__(16) union { struct { _Float16 k[2][32 * KP], v[2][D * VP]; } codes; _Float16 q[4][32 * KP]; float out[4][32 * 36]; } u;
    __shared__ __align__(16) float s_ks[2][32], s_vs[2][32];
    __shared__ float s_sf[4][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), col = lane & 31, h = lane >> 5;
    const uint32_t wgs = (A.tiles + 3) / 4, g = blockIdx.x / wgs, tile = blockIdx.x % wgs * 4 + wave;
    const Job job = job_of(A);
    const uint32_t b = job.b;
    const Seq q = sequence(A, b);
    if (job.s.count == 0 || blockIdx.x % wgs * 128 / A.group >= q.count) return;   // all tiles are behind count
    const Column mine = column(A, q, g, tile * 32 + col);
    const uint32_t node = mine.node, head = mine.head;
    const bool busy = tile < A.tiles && tile * 32 / A.group < q.count, used = mine.used;   // busy: of the wave
    const uint32_t total = q.len + q.count, nchunk = (total + 31) / 32;
    const uint32_t c_lo = (uint64_t)nchunk * job.z / job.s.count, c_hi = (uint64_t)nchunk * (job.z + 1) / job.s.count;
    // staging: K, a row's 16 bytes a thread; V, 4 positions x 4 dims.  Offsets inside a chunk fit 32 bits (the
    // row stride is below 2^26), the chunk's base is the same in all lanes.
    const bool stager = D == 128 || tid < 128;
    const uint32_t kpos = tid / (D / 16) % 32, kpiece = tid % (D / 16), dq = tid % (D / 4), pq = tid / (D / 4) % 8, row_bytes = (uint32_t)A.a.kv_row;
    const int8_t *kbase = A.a.k + b * A.a.kv_batch + g * D, *vbase = A.a.v + b * A.a.kv_batch + g * D;
    const float *sbase = (tid < 32 ? A.a.kscale : A.a.vscale) + b * A.a.scale_batch;
    struct Codes { nt4 k; uint32_t v[4]; float s; };   // a thread's part of a chunk
    Codes in{};
    auto load = [&](uint32_t ci, Codes &in) {
        const uint32_t pb = ci * 32, last = total - 1 - pb;   // (rows past the last read it again)
        const int8_t *kc = kbase + pb * A.a.kv_row, *vc = vbase + pb * A.a.kv_row;
        if (stager) {
            if (pb + 32 <= total) {
                in.k = *reinterpret_cast<const nt4 *>(kc + (kpos * row_bytes + 16 * kpiece));
#pragma unroll
                for (int r = 0; r < 4; ++r) in.v[r] = *reinterpret_cast<const uint32_t *>(vc + r * A.a.kv_row + (4 * pq * row_bytes + 4 * dq));
            } else {
                in.k = *reinterpret_cast<const nt4 *>(kc + (min(kpos, last) * row_bytes + 16 * kpiece));
#pragma unroll
                for (int r = 0; r < 4; ++r) in.v[r] = *reinterpret_cast<const uint32_t *>(vc + (min(4 * pq + r, last) * row_bytes + 4 * dq));
            }
        }
        if (tid < 64) in.s = sbase[pb + min((uint32_t)tid % 32, last)];
    };
    // positions 4 w .. 4 w + 3 (w = pq) are half w / 2 % 2 of the 16 bytes that lane half w % 2 reads in step w / 4;
    // the place of the 16 bytes turns with dim / 16, so that the lanes' writes spread over the banks
    const int slot = ((pq >> 2) * 2 + (pq & 1)) ^ ((dq >> 2) & 3), vat = 4 * dq * VP + 8 * slot + 4 * ((pq >> 1) & 1);
    auto stage_k = [&](uint32_t ci, const Codes &in) {
        if (stager) {
            uint4 *to = reinterpret_cast<uint4 *>(&u.codes.k[ci & 1][kpos * KP + 16 * kpiece]);
            to[0] = i8x8_to_f16(in.k.x, in.k.y);
            to[1] = i8x8_to_f16(in.k.z, in.k.w);
        }
        if (tid < 64) (tid < 32 ? s_ks : s_vs)[ci & 1][tid % 32] = in.s;
    };
    auto stage_v = [&](uint32_t ci, const Codes &in) {
        if (stager) {
            const uint32_t a0 = perm(in.v[1], in.v[0], 0x05010400u), a1 = perm(in.v[3], in.v[2], 0x05010400u);
            const uint32_t a2 = perm(in.v[1], in.v[0], 0x07030602u), a3 = perm(in.v[3], in.v[2], 0x07030602u);
            const uint4 v01 = i8x8_to_f16(perm(a1, a0, 0x05040100u), perm(a1, a0, 0x07060302u));
            const uint4 v23 = i8x8_to_f16(perm(a3, a2, 0x05040100u), perm(a3, a2, 0x07060302u));
            uint2 *vd = reinterpret_cast<uint2 *>(&u.codes.v[ci & 1][vat]);
            vd[0] = make_uint2(v01.x, v01.y);
            vd[VP / 4] = make_uint2(v01.z, v01.w);
            vd[2 * (VP / 4)] = make_uint2(v23.x, v23.y);
            vd[3 * (VP / 4)] = make_uint2(v23.z, v23.w);
        }
    };
    if (c_lo < c_hi) load(c_lo, in);
    uint4 qh[KS], ql[SPLIT ? KS : 1];
    float sf = 0.0f;
    if (busy) {   // q fragments: 8 lanes read a column's row, the wave's part of LDS hands each lane its column's half
        float v[4][D / 64][8];
        const int seg = lane & 7;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Column to = column(A, q, g, tile * 32 + (lane >> 3) + 8 * i);
            const T *row = (const T *)A.a.q + b * A.a.q_batch + (to.used ? to.node : 0) * A.a.q_node + (to.used ? to.head : g * A.group) * D + 8 * seg;
#pragma unroll
            for (int j = 0; j < D / 64; ++j) load8(row + 64 * j, v[i][j]);
        }
        float sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t m = 0;   // the largest magnitude's bits; infinity and NaN are beyond all others
#pragma unroll
            for (int j = 0; j < D / 64; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[i][j][e]) & 0x7fffffffu);
            m = max(m, __float_as_uint(dppf<DPP_XOR1>(__uint_as_float(m))));
            m = max(m, __float_as_uint(dppf<DPP_XOR2>(__uint_as_float(m))));
            m = max(m, __float_as_uint(dppf<DPP_HALF_MIRROR>(__uint_as_float(m))));
            const bool bad = m >= 0x7f800000u;
            sc[i] = pow2_scale(__uint_as_float(m), 14);
            if (seg == 0) s_sf[wave][(lane >> 3) + 8 * i] = score_factor(A, sc[i], bad);
        }
#pragma unroll
        for (int half = 0; half < (SPLIT ? 2 : 1); ++half) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
                    h8v x;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (half == 0) v[i][j][e] *= sc[i];
                        x[e] = (_Float16)v[i][j][e];
                        if (half == 0) v[i][j][e] -= (float)x[e];
                    }
                    *reinterpret_cast<h8v *>(&u.q[wave][((lane >> 3) + 8 * i) * KP + 8 * seg + 64 * j]) = x;
                }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const uint4 x = *reinterpret_cast<const uint4 *>(&u.q[wave][col * KP + (D / 2) * h + 8 * s]);
                if (half == 0) qh[s] = x;
                else ql[SPLIT ? s : 0] = x;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        sf = s_sf[wave][col];
        if (A.pack && job.z == 0) {   // the account's q
            const uint64_t at = ((uint64_t)b * A.a.kv_heads + g) * A.tiles + tile;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                uint4 *to = A.pack + (at * KS + s) * (SPLIT ? 128 : 64) + lane;
                to[0] = qh[s];
                if constexpr (SPLIT) to[64] = ql[s];
            }
            if (h == 0) A.pack_sf[at * 32 + col] = sf;
        }
    }
    State<D> S;
    __syncthreads();
#pragma unroll 1
    for (uint32_t ci = c_lo; ci < c_hi; ++ci) {
        stage_k(ci, in);
        stage_v(ci, in);
        if (ci + 1 < c_hi) load(ci + 1, in);
        __syncthreads();
        if (!busy) continue;
        const uint32_t pb = ci * 32;
        f16x dot = zero16();
        const _Float16 *kr = &u.codes.k[ci & 1][col * KP + (D / 2) * h], *vr = &u.codes.v[ci & 1][col * VP];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const uint4 kf = *reinterpret_cast<const uint4 *>(kr + 8 * s);
            if constexpr (SPLIT) dot = mfma(kf, ql[s], dot);
            dot = mfma(kf, qh[s], dot);
        }
        const bool edge = pb + 32 > q.len;   // the chunk holds nodes
        const uint32_t bits = edge ? visible(A, q, b, node, pb) : ~0u;
        uint4 phi[2], plo[2];
        weigh<D>(S, dot, sf, s_ks[ci & 1], s_vs[ci & 1], edge, bits, h, phi, plo);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint4 vf[DT];
#pragma unroll
            for (int d = 0; d < DT; ++d)
                vf[d] = *reinterpret_cast<const uint4 *>(vr + 32 * d * VP + 8 * ((2 * s + h) ^ ((2 * d + (col >> 4)) & 3)));
#pragma unroll
            for (int d = 0; d < DT; ++d) S.acc[d] = mfma(vf[d], plo[s], S.acc[d]);
#pragma unroll
            for (int d = 0; d < DT; ++d) S.acc[d] = mfma(vf[d], phi[s], S.acc[d]);
        }
    }
    S.close();
    const float den = S.den + __shfl_xor(S.den, 32);
    __syncthreads();
    if (!busy) return;
    // results: a tile of 32 dims after the other through the wave's part of LDS, so that 8 lanes write a column's line
    const bool whole = A.splits == 1;
    const float inv = !whole ? 1.0f : den == 0.0f ? 0.0f : 1.0f / den;
    const uint64_t states = (uint64_t)(job.s.first + job.z) * A.a.nodes * A.a.heads;
    float *o = u.out[wave];
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            *reinterpret_cast<f4x *>(o + col * 36 + 8 * k + 4 * h) = f4x{S.acc[d][4 * k] * inv, S.acc[d][4 * k + 1] * inv, S.acc[d][4 * k + 2] * inv,
                                                                       S.acc[d][4 * k + 3] * inv};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Column to = column(A, q, g, tile * 32 + (lane >> 3) + 8 * i);
            const float4 x = *reinterpret_cast<const float4 *>(o + ((lane >> 3) + 8 * i) * 36 + 4 * (lane & 7));
            const uint32_t dim = 32 * d + 4 * (lane & 7);
            if (!to.used) continue;
            if (whole) store4((T *)A.a.out + b * A.a.out_batch + to.node * A.a.out_node + to.head * D + dim, x);
            else store4(A.part + (states + to.node * A.a.heads + to.head) * D + dim, x);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (used && h == 0) finish_sums(A, S.M, den, whole, ((uint64_t)b * A.a.nodes + node) * A.a.heads + head, states + node * A.a.heads + head);
}

// The splits of a row joined: a workgroup a row, its 256 / (D / 4) strips of threads every so many splits, the
// strips in order.  (A wave a row, a split's state after the other: 12 us for 32 splits of 128 rows.)  A
// chain of loads bounds it: 4 us for 11 splits of 512 rows, 10.6 for 2 x 1536 rows of 20 splits.
template <typename T, int D>
__global__ __launch_bounds__(256) void qxa_join(QxaArgs A) {
    constexpr int W = D / 4, STRIPS = 256 / W;
    __shared__ float s_m[STRIPS], s_den[STRIPS];
    __shared__ __align__(16) float s_v[STRIPS][D];
    const uint64_t rows = (uint64_t)A.a.nodes * A.a.heads, row = blockIdx.x;
    const int at = threadIdx.x % W, strip = threadIdx.x / W;
    const uint32_t head = row % A.a.heads, node = row / A.a.heads % A.a.nodes, b = row / A.a.heads / A.a.nodes;
    if (node >= sequence(A, b).count) return;
    const Splits sp = splits_of(A, b);
    const uint64_t first = sp.first * rows + node * A.a.heads + head;   // the row's first state; the next lie `rows` apart
    float m = -INFINITY, den = 0.0f;
    f4x v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (uint32_t z = strip; z < sp.count; z += STRIPS) {
        const float2 s = A.md[first + z * rows];
        const f4x x = *reinterpret_cast<const f4x *>(A.part + (first + z * rows) * D + 4 * at);
        const float mn = fmaxf(m, s.x), f = m == mn ? 1.0f : exp2_fast(m - mn), fz = s.x == mn ? 1.0f : exp2_fast(s.x - mn);
        den = fmaf(den, f, s.y * fz);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = fmaf(v[i], f, x[i] * fz);
        m = mn;
    }
    if (at == 0) { s_m[strip] = m; s_den[strip] = den; }
    *reinterpret_cast<f4x *>(&s_v[strip][4 * at]) = v;
    __syncthreads();
    if (threadIdx.x >= W) return;
#pragma unroll
    for (int k = 1; k < STRIPS; ++k) {
        const float mn = fmaxf(m, s_m[k]), f = m == mn ? 1.0f : exp2_fast(m - mn), fz = s_m[k] == mn ? 1.0f : exp2_fast(s_m[k] - mn);
        const f4x x = *reinterpret_cast<const f4x *>(&s_v[k][4 * at]);
        den = fmaf(den, f, s_den[k] * fz);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = fmaf(v[i], f, x[i] * fz);
        m = mn;
    }
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
    store4((T *)A.a.out + b * A.a.out_batch + node * A.a.out_node + head * D + 4 * at, make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv));
    if (at == 0) finish_row(A, m, den, row);
}

namespace {
// The exponent of a weight, of dot * kscale: as it was for the row's own sums
DEV float weight_exponent(float s, float sf, float M, bool far) { return far ? s * sf - M : fmaf(s, sf, -M); }
}  // namespace

// account[p] = decay * account[p] + sum over nodes and heads of 2^(s - M) / denominator, of kept scores.  A wave takes 32
// positions, 8 lanes of 4 positions a row and every eighth row; rows and strips are added up in a fixed order.
__global__ __launch_bounds__(256) void qxa_account_kept(QxaArgs A) {
    const uint32_t lane = threadIdx.x & 63, quad = lane & 7, b = blockIdx.y;
    const Seq q = sequence(A, b);
    const uint32_t total = q.len + q.count, nchunk = (total + 31) / 32, inuse = q.count * A.group, rows = A.a.kv_heads * inuse;
    for (uint32_t ci = blockIdx.x * 4 + wave_id(); ci < nchunk; ci += gridDim.x * 4) {
        f4x sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (uint32_t r = lane >> 3; r < rows; r += 8) {
            const uint32_t g = r / inuse, c = r % inuse, node = c / A.group, head = g * A.group + c % A.group;
            const f4x s = *reinterpret_cast<const f4x *>(
                A.scores + ((((uint64_t)b * A.a.kv_heads + g) * ((A.a.positions + 31) / 32) + ci) * A.columns + c) * 32 + 4 * quad);
            const float2 norm = A.norm[((uint64_t)b * A.a.nodes + node) * A.a.heads + head];
            const float sf = A.pack_sf[((uint64_t)b * A.a.kv_heads + g) * 32 + c];   // (one tile of columns)
            const bool far = fabsf(norm.x) >= FAR;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += s[i] == -INFINITY ? 0.0f : exp2_fast(weight_exponent(s[i], sf, norm.x, far)) * norm.y;   // (not seen: 0, of a NaN row as well)
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // over the strips
            float v = sum[i];
            v += dppf<DPP_ROR8>(v);
            const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
            const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            sum[i] = __uint_as_float(y[0]) + __uint_as_float(y[1]);
        }
        const uint32_t p = ci * 32 + 4 * quad;
        if (lane >= 8) continue;
        float *to = A.a.account + b * A.a.account_batch + p;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p + i < total) to[i] = to[i] * A.a.decay + sum[i];
    }
}

// The same, the scores computed again from the q that the attention has left as matrix operands.  A wave keeps, per lane, its column's sums of the 16
// positions that its registers hold; columns and waves are added up in a fixed order, and no two
// workgroups add to one position.  SHARE waves take the same 32 positions and every SHARE-th (kv head, tile): 8
// where there are few positions, whose chain of pairs would be the time; else 1 and four chunks a
// workgroup, which then read each q from the first-level cache (calls of 16 nodes, BF16: over 16000 positions 42.1 us with
// 8 and 46.7 with 1, over 30000 57.3 and 52.8).  16 nodes of 32 heads over 1500 positions: 9.5 us, a chain
// of latencies (lengths, scales, K and q, two pairs a wave, the sums); of long ones the matrix instructions bound it.
template <typename T, int D, int SHARE>
__global__ __launch_bounds__(SHARE == 1 ? 256 : 64 * SHARE, 1) void qxa_account(QxaArgs A) {
    constexpr bool SPLIT = two_halves_q<T>;
    constexpr int KS = D / 16, NP = SPLIT ? 2 : 1, CHUNKS = SHARE == 1 ? 4 : 1;
    __shared__ float s_sum[SHARE == 1 ? 1 : SHARE][32];
    const int lane = threadIdx.x & 63, wave = wave_id(), col = lane & 31, h = lane >> 5;
    const uint32_t b = blockIdx.y;
    const Seq q = sequence(A, b);
    const uint32_t total = q.len + q.count, nchunk = (total + 31) / 32;
    const uint32_t tiles = min(A.tiles, (q.count * A.group + 31) / 32), pairs = A.a.kv_heads * tiles;   // those with nodes in use
    for (uint32_t c0 = blockIdx.x * CHUNKS; c0 < nchunk; c0 += gridDim.x * CHUNKS) {
        const uint32_t ci = c0 + (SHARE == 1 ? wave : 0), pb = ci * 32;
        float sum[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[r] = 0.0f;
        if (ci < nchunk) {
            const uint32_t pk = min(pb + col, total - 1);
            const bool edge = pb + 32 > q.len;
            float ks[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) ks[r] = A.a.kscale[b * A.a.scale_batch + min(pb + 8 * (r >> 2) + 4 * h + (r & 3), total - 1)];
            uint4 kf[KS];
            uint32_t held = ~0u;   // the kv head whose codes kf holds
#pragma unroll 1
            for (uint32_t pair = SHARE == 1 ? 0 : wave; pair < pairs; pair += SHARE) {
                const uint32_t g = pair / tiles, tile = pair % tiles, c = tile * 32 + col;
                const uint32_t node = min(c / A.group, A.a.nodes - 1), head = g * A.group + c % A.group;
                const bool used = c < A.columns && node < q.count;
                const uint64_t at = ((uint64_t)b * A.a.kv_heads + g) * A.tiles + tile;
                const uint4 *qp = A.pack + at * (KS * NP * 64) + lane;
                uint4 qf[KS * NP];
#pragma unroll
                for (int s = 0; s < KS * NP; ++s) qf[s] = qp[64 * s];
                const float sf = A.pack_sf[at * 32 + col];
                const float2 norm = used ? A.norm[((uint64_t)b * A.a.nodes + node) * A.a.heads + head] : make_float2(0.0f, 0.0f);
                if (g != held) {
                    const KRow<D> kr = load_k<D>(A, b, g, pk, h);
#pragma unroll
                    for (int s = 0; s < KS; ++s) kf[s] = k_step<D>(kr, s);
                    held = g;
                }
                f16x dot = zero16();
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    if constexpr (SPLIT) dot = mfma(kf[s], qf[s * NP + 1], dot);
                    dot = mfma(kf[s], qf[s * NP], dot);
                }
                // (a column that is not used or sees nothing adds 1 x 0)
                const float f = norm.y == 0.0f ? 0.0f : sf;
                const bool far = fabsf(norm.x) >= FAR;
                float e[16];
                if (__ballot(far) == 0) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) e[r] = exp2_fast(weight_exponent(dot[r] * ks[r], f, norm.x, false));
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) e[r] = exp2_fast(weight_exponent(dot[r] * ks[r], f, norm.x, far));
                }
                if (edge) {
                    const uint32_t bits = visible(A, q, b, node, pb) >> (4 * h);
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum[r] = seen(bits, r) && norm.y != 0.0f ? fmaf(e[r], norm.y, sum[r]) : sum[r];
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum[r] = fmaf(e[r], norm.y, sum[r]);
                }
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {   // over the 32 columns
                float v = sum[r];
                v += dppf<DPP_XOR1>(v); v += dppf<DPP_XOR2>(v); v += dppf<DPP_ROR4>(v); v += dppf<DPP_ROR8>(v);
                const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
                sum[r] = __uint_as_float(x[0]) + __uint_as_float(x[1]);
            }
        }
        float mine = 0.0f;   // position pb + lane % 32's
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int p = 8 * (r >> 2) + (r & 3);   // + 4 h
            const float lo = rdlanef(sum[r], 0), hi = rdlanef(sum[r], 32);
            mine = col == p ? lo : col == p + 4 ? hi : mine;
        }
        if constexpr (SHARE > 1) {
            if (h == 0) s_sum[wave][col] = mine;
            __syncthreads();
            mine = 0.0f;
#pragma unroll
            for (int w = 0; w < SHARE; ++w) mine += s_sum[w][col];
            __syncthreads();
        }
        if (h == 0 && (SHARE == 1 || wave == 0) && pb + col < total) {
            float *to = A.a.account + b * A.a.account_batch + pb + col;
            *to = *to * A.a.decay + mine;
        }
    }
}

namespace {
template <typename T, int D> hipError_t launch(const QxaArgs &A, hipStream_t s) {
    const uint64_t rows = (uint64_t)A.a.batch * A.a.nodes * A.a.heads;
    const bool shared = A.a.batch <= 64 && A.splits > 1;   // (a sequence's number of splits is rounded down, but at least one)
    const dim3 grid(A.a.kv_heads * A.wgs, shared && A.a.batch > 1 ? 2 * A.splits + A.a.batch : A.splits, shared ? 1 : A.a.batch);
    auto *kernel = A.wide ? qxa_wide<T, D> : A.scores ? qxa_tree<T, D, true> : qxa_tree<T, D, false>;
    hipError_t e = qxg_launch(kernel, grid, dim3(256), 0, s, A);
    if (e == hipSuccess && A.splits > 1) e = qxg_launch(qxa_join<T, D>, dim3((unsigned)rows), dim3(256), 0, s, A);
    if (e != hipSuccess || !A.a.account) return e;
    const uint64_t chunks = ((uint64_t)A.a.max_len + A.a.nodes + 31) / 32;
    const auto in_fours = [&] { return dim3((unsigned)std::min<uint64_t>(65535, (chunks + 3) / 4), A.a.batch); };
    if (A.scores) return qxg_launch(qxa_account_kept, in_fours(), dim3(256), 0, s, A);
    if (chunks * A.a.batch < 768) return qxg_launch(qxa_account<T, D, 8>, dim3((unsigned)chunks, A.a.batch), dim3(512), 0, s, A);
    return qxg_launch(qxa_account<T, D, 1>, in_fours(), dim3(256), 0, s, A);
}
}  // namespace

hipError_t qxa_launch(const QxaArgs &A, hipStream_t s) {
    if (A.a.type == QXG_TYPE_F32) return A.a.dim == 64 ? launch<float, 64>(A, s) : launch<float, 128>(A, s);
    if (A.a.type == QXG_TYPE_F16) return A.a.dim == 64 ? launch<_Float16, 64>(A, s) : launch<_Float16, 128>(A, s);
    return A.a.dim == 64 ? launch<__bf16, 64>(A, s) : launch<__bf16, 128>(A, s);
}
