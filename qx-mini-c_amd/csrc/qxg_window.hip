// Causal attention over a cache of 8 or 4 bits, whole or within a window with sinks (qxg_cache_attention).
//
// Mathematics.  One pass with a base-2 softmax: a column keeps a reference M, a whole number that follows the running maximum to
// within 2^8, the sum of e = 2^(s - M) and the context, the sum of e v; both are scaled by a power of two when M moves.
// All products are on the matrix cores in bf16, with f32 sums.  Codes are exact there: INT8 ones as whole numbers, whose scales
// multiply the scores and the weights e; E2M1 ones with their power of two.  What is not, q and the weights, is taken as the sum of
// several bf16 numbers: 3 for f32 (24 bits), for 16-bit types q as it is (f16: 2) and the weights as 2 (17 bits: their error is
// 2^-18, where the result's rounding is 2^-12 or 2^-9).  bf16 has f32's range, so weights far below their row's largest keep their bits,
// of which many may outweigh it; in f16 they would need a window that moves.  (Pieces below 2^-126 may count as 0.)
// The exponent s - M of a score in base 2 is one fma.  Where |M| is from FAR on, it is the product rounded as the maximum was, less
// M: an fma's would hold what that rounding left, half a step of the score, from 2^28 on more than the 8 that M allows, and from 2^31 on
// more than e has room for.
// (An f32 q over INT8 codes as a column's whole numbers, in products of 8 bits, is faster for a prompt, 40 us a call for 45 of 512 tokens of 32 / 4
// heads of 128 within 1024 + 4 positions, but a large value of q costs the others their low bits, from 2^22 times as large all of them.)
#include "qxg_cache.h"
#include "qxg_values.h"

namespace {
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef float f2v __attribute__((ext_vector_type(2)));
template <typename T> constexpr int Q_PIECES = sizeof(T) == 4 ? 3 : __is_same(T, _Float16) ? 2 : 1;
template <typename T> constexpr int P_PIECES = sizeof(T) == 4 ? 3 : 2;

DEV f4x mfma16(uint4 a, uint4 b, f4x c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}
DEV uint32_t pack_bf16(float lo, float hi) {   // to nearest
    const f2v x = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, b2v));
}
// v = p[0] + p[1] + ..., each to nearest.  What is left is v - 1 x hi + 0 x its neighbour, exact in f32: one instruction a value (the
// factors are hidden, or the compiler takes constants that stand for both halves).
template <int N> DEV void pieces8(float (&v)[8], uint4 (&p)[N]) {
    uint32_t first = 0x0000bf80u, second = 0xbf800000u;   // (-1, 0), (0, -1)
    asm("" : "+s"(first), "+s"(second));
#pragma unroll
    for (int n = 0; n < N; ++n) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
            if (n + 1 < N) {
                v[2 * i] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2v, w[i]), __builtin_bit_cast(b2v, first), v[2 * i], false);
                v[2 * i + 1] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2v, w[i]), __builtin_bit_cast(b2v, second), v[2 * i + 1], false);
            }
        }
        p[n] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
// 8 codes of 4 bits times a power of two, exact
DEV uint4 e2m1x8(uint32_t w, float scale) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3)));
}
// the power of two of byte i of a word of scales (all of these and their products with codes are normal numbers)
DEV float e8m0(uint32_t w, int i) { return __uint_as_float(min(max((w >> (8 * i)) & 255u, 2u), 252u) << 23); }
// A wave's scales of 32 positions in 8 bits, K's in lanes 0 .. 31 and V's in 32 .. 63: where one is not finite, the position's K scale
// becomes NaN and its V scale 0.  So a row that sees the position is NaN, and for one that does not its weight times the scale is 0.
DEV float finite_scales(uint32_t bits) {
    const float x = __uint_as_float(bits);
    const bool bad = !isfinite(x);
    const uint64_t all = __ballot(bad);
    const uint32_t lane = threadIdx.x & 63, either = (uint32_t)all | (uint32_t)(all >> 32);
    return either >> (lane & 31) & 1 ? (lane < 32 ? NAN : 0.0f) : x;
}
// Of 4 bits, likewise: the positions one of whose scale bytes (K's in lanes 0 .. 31, V's in 32 .. 63) is 255, NaN.  Its power of two counts as
// another's, so that for a row that does not see the position its weight times the value is 0; the scores of one that does become NaN.
DEV uint32_t nan_scales(uint32_t bytes) {
    const uint32_t x = ~bytes;   // a byte of 0: only where one is does the difference borrow
    const uint64_t all = __ballot(((x - 0x01010101u) & ~x & 0x80808080u) != 0);
    return (uint32_t)all | (uint32_t)(all >> 32);
}
DEV float code(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }
DEV uint4 codes8(uint32_t x, uint32_t y) {   // 8 INT8 codes
    return make_uint4(pack_bf16(code(x, 0), code(x, 1)), pack_bf16(code(x, 2), code(x, 3)), pack_bf16(code(y, 0), code(y, 1)), pack_bf16(code(y, 2), code(y, 3)));
}

constexpr float FAR = 4194304.0f;

struct Seq { uint32_t len, count; };   // of sequence b, clamped to the arrays
DEV Seq sequence(const QxwArgs &A, uint32_t b) {
    Seq s;
    s.count = min(A.a.counts ? A.a.counts[b] : A.a.tokens, min(A.a.tokens, A.a.positions));
    s.len = min(A.a.lens[b], A.a.positions - s.count);
    return s;
}
// The first position that a token at p sees behind the sinks
DEV uint32_t window_start(const QxwArgs &A, uint32_t p) { return A.a.window && p >= A.a.window ? p - A.a.window + 1 : 0; }
// The chunks of 32 positions that the tokens at positions p0 .. p1 see: `sinks` first ones, then those from `from` on
struct Chunks {
    uint32_t sinks, from, n;
    DEV uint32_t at(uint32_t i) const { return i < sinks ? i : from + (i - sinks); }
};
DEV Chunks chunks_of(const QxwArgs &A, uint32_t p0, uint32_t p1) {
    Chunks c;
    c.from = window_start(A, p0) / 32;
    c.sinks = min((uint32_t)(((uint64_t)A.a.sinks + 31) / 32), c.from);
    c.n = c.sinks + (p1 / 32 - c.from + 1);
    return c;
}
// Whether all of the positions pb .. pb + 31 are seen by all tokens at p0 .. p1
DEV bool all_seen(const QxwArgs &A, uint32_t pb, uint32_t p0, uint32_t p1) {
    return pb + 31 <= p0 && (window_start(A, p1) <= pb || pb + 32 <= A.a.sinks);
}
// The split's part of a list of n chunks; the splits that have chunks are the first ones.
struct Part { uint32_t lo, hi; };
DEV uint32_t split_size(const QxwArgs &A, uint32_t n) { return max(A.split_chunks, (n + A.splits - 1) / A.splits); }
DEV Part part_of(const QxwArgs &A, uint32_t n, uint32_t split) {
    const uint32_t size = split_size(A, n);
    return {min(n, split * size), min(n, (split + 1) * size)};
}
// A workgroup's place: kv head, tile of columns, split, sequence.  Workgroups go to the 8 XCDs in turn, each with an L2 of its own: the kv heads
// of a tile follow each other on one XCD, as a line of 128 bytes may hold several heads' codes.  Later tiles, which may see more, come first.
// A sequence's splits begin on another XCD than the one's before it: of shorter sequences the last ones are empty (16 of 10000 to
// 32000 positions of 4 bits in 8 splits 112 us, before 131).
struct Place { uint32_t g, tile, split, b; };
DEV Place place_of(const QxwArgs &A) {
    const uint32_t mine = blockIdx.x / 8;
    uint32_t at = mine / A.a.kv_heads * 8 + blockIdx.x % 8;
    Place p;
    p.g = mine % A.a.kv_heads;
    p.tile = A.tiles - 1 - at % A.tiles;
    at /= A.tiles;
    p.b = at / A.splits;   // (the batch or more: none)
    p.split = (at + p.b) % A.splits;
    return p;
}
DEV uint64_t state_at(const QxwArgs &A, uint32_t b, uint32_t split, uint32_t token, uint32_t head) {
    return (((uint64_t)b * A.splits + split) * A.a.tokens + token) * A.a.heads + head;
}
// A row sees its own position at least, so its denominator is 0 only where all of its scores are -inf (an infinite q, or dot products
// beyond f32): 1 / 0 makes the context NaN, as the formula is there, and lse is NaN with it.
DEV void finish_lse(const QxwArgs &A, float M, float den, uint32_t b, uint32_t token, uint32_t head) {
    if (A.a.lse) A.a.lse[((uint64_t)b * A.a.tokens + token) * A.a.heads + head] = den == 0.0f ? NAN : (M + __log2f(den)) * 0.69314718055994531f;
}
}  // namespace

// Few columns.  A workgroup takes 16 or 32 columns (CT tiles of 16) of one kv head and a split; its waves take the chunks in turn, each
// with a state of its own, and are joined at the end.
//
// What bounds it.  Long caches and few tokens: bytes; one token each of 16 sequences of 30000 positions, 32 / 8 heads of 128 in bf16 over 8 bits,
// 983 MB in 206 us, 4.8 TB/s (4 bits, 32000 positions: 557 MB in 141 us).  Otherwise the issue of instructions, about one in 4.7 cycles:
// a chunk of 16 columns of 128 dims is some 300 vector instructions, half of them the conversion of codes, and 28 to 48 matrix ones, which add up
// as a SIMD's waves all do the same; 512 tokens of 32 / 4 heads in f32 within 1024 + 4 positions 45 us a call (queued one after the other; under a tracer, at
// another clock, 48.5).  Tried without gain: 8 waves a
// workgroup (15.0 us and 14.3 for a token over 36 chunks), which share the SIMDs; contexts of 64 columns a wave, which spill.
// 16 x 1 token within 4096 + 16 took 42 us a call in a first form, which staged chunks in LDS for four waves of 16 columns each, 39 without the
// staging, and 33 to 36 with the present splits; 16 x 1 over 10000 to 32000 positions of 4 bits 165 in that form, and 130 without it and with the
// order of the kv heads on the XCDs (163 without that order), 95 to 107 with the smaller splits of batches.
//
// Tiles.  v_mfma_f32_16x16x32_bf16: lane l holds 8 values of k of row (column) l % 16, those of group l / 16; result register r of
// lane l is row 4 (l / 16) + r, column l % 16.  Scores have positions as rows, two tiles a chunk, and columns (token, head): a lane's
// weights are those of the positions 16 t + 4 (l / 16) + r, which with k = 4 t + r is an operand of the second product as
// they are.  The order of dims is free in the first product, so a lane takes D / 4 consecutive ones of its position's row: in 4
// bits one block, one scale.  In the second, a lane's rows are D / 16 consecutive dims, so it loads the codes of its 8 positions
// as they lie and turns them in registers, and its results are D / 4 consecutive dims.
template <typename T, int D, int BITS, int CT>
__global__ __launch_bounds__(256, CT == 2 || (D == 128 && (sizeof(T) == 4 || (__is_same(T, _Float16) && BITS == 8))) ? 2 : 3) void qxw_few(QxwArgs A) {
    constexpr int NQ = Q_PIECES<T>, NP = P_PIECES<T>, KS = D / 32, DT = D / 16, COLUMNS = 16 * CT;
    constexpr int KW = D * BITS / 128;                 // words of K a lane has of a position
    constexpr int VB = D / 16 * BITS / 8;              // bytes of V
    __shared__ __align__(16) float s_scale[4][2][BITS == 8 ? 1 : D / 32][32];   // of K and V, a block's positions
    __shared__ __align__(16) float s_acc[4][16][D + 4];
    __shared__ float s_m[4][16], s_den[4][16];
    const qxg_cache_attention_args &a = A.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63, u = lane & 15, w = lane >> 4;
    const int wave = wave_id();
    const Place place = place_of(A);
    const uint32_t g = place.g, tile = place.tile, b = place.b;
    if (b >= a.batch) return;
    const Seq q = sequence(A, b);
    const uint32_t first = tile * COLUMNS / A.group;   // the tile's first and last token
    if (first >= q.count) return;
    const uint32_t last = min((tile * COLUMNS + COLUMNS - 1) / A.group, q.count - 1), p0 = q.len + first, p1 = q.len + last;
    const Chunks list = chunks_of(A, p0, p1);
    const Part part = part_of(A, list.n, place.split);
    if (part.lo >= part.hi) return;
    uint32_t p[CT], start[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        p[c] = q.len + min((tile * COLUMNS + 16 * c + u) / A.group, last);
        start[c] = window_start(A, p[c]);
    }

    const uint8_t *kbase = (const uint8_t *)a.k + b * a.kv_batch + g * (D * BITS / 8), *vbase = (const uint8_t *)a.v + b * a.kv_batch + g * (D * BITS / 8);
    const uint8_t *scales = (const uint8_t *)(lane < 32 ? a.kscale : a.vscale) + b * a.scale_batch * (BITS == 8 ? 4 : 1) + (BITS == 8 ? 0 : g * (D / 32));
    const uint32_t row_bytes = (uint32_t)a.kv_row, scale_bytes = BITS == 8 ? 4u : (uint32_t)a.scale_row, end = a.positions - 1;
    struct { uint32_t k[2][KW]; uint32_t v[8][(VB + 3) / 4]; uint32_t scale; } in, next;   // a chunk's, the next one's
    // where a lane's rows are in a chunk (offsets there fit 32 bits: the row strides are below 2^26)
    uint32_t k_at[2], v_at[8], scale_at;
    auto rows = [&](uint32_t past) {
#pragma unroll
        for (int t = 0; t < 2; ++t) k_at[t] = min(16 * t + u, past) * row_bytes + w * (4 * KW);
#pragma unroll
        for (int i = 0; i < 8; ++i) v_at[i] = min(16 * (i / 4) + 4 * w + i % 4, past) * row_bytes + u * VB;
        scale_at = min(lane & 31, past) * scale_bytes;   // lanes 0 .. 31 those of K, 32 .. 63 those of V
    };
    rows(31);
    auto load = [&](uint32_t pb) {
        if (pb + 31 > end) rows(end - pb);   // the last chunk: positions past the array's last read it again, they are masked
        const uint8_t *k = kbase + (uint64_t)pb * row_bytes, *v = vbase + (uint64_t)pb * row_bytes, *s = scales + (uint64_t)pb * scale_bytes;
        if constexpr (BITS == 8 || D == 128) next.scale = *reinterpret_cast<const uint32_t *>(s + scale_at);
        else next.scale = *reinterpret_cast<const uint16_t *>(s + scale_at);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if constexpr (KW >= 4) {
#pragma unroll
                for (int i = 0; i < KW / 4; ++i) *reinterpret_cast<uint4 *>(&next.k[t][4 * i]) = reinterpret_cast<const uint4 *>(k + k_at[t])[i];
            } else *reinterpret_cast<uint2 *>(&next.k[t][0]) = *reinterpret_cast<const uint2 *>(k + k_at[t]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (VB == 8) *reinterpret_cast<uint2 *>(&next.v[i][0]) = *reinterpret_cast<const uint2 *>(v + v_at[i]);
            else if constexpr (VB == 4) next.v[i][0] = *reinterpret_cast<const uint32_t *>(v + v_at[i]);
            else next.v[i][0] = *reinterpret_cast<const uint16_t *>(v + v_at[i]);
        }
    };
    uint32_t ci = part.lo + wave;
    const bool busy = ci < part.hi;   // of the wave
    if (busy) load(list.at(ci) * 32);
    uint4 qf[CT][KS][NQ];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const uint32_t column = tile * COLUMNS + 16 * c + u;
        const T *row = (const T *)a.q + b * a.q_batch + min(column / A.group, last) * a.q_token + (g * A.group + column % A.group) * D + w * (D / 4);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float v[8];
            load8(row + 8 * s, v);
            pieces8<NQ>(v, qf[c][s]);
        }
    }
    float m[CT], den[CT];
    bool far = false;   // one of the wave's references is
    f4x acc[CT][DT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        m[c] = -INFINITY;
        den[c] = 0.0f;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[c][d] = f4x{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll 1
    for (; ci < part.hi; ci += 4) {
        const uint32_t pb = list.at(ci) * 32;
        in = next;
        if (ci + 4 < part.hi) load(list.at(ci + 4) * 32);
        if constexpr (BITS == 8) s_scale[wave][lane >> 5][0][lane & 31] = finite_scales(in.scale);
        else {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) s_scale[wave][lane >> 5][i][lane & 31] = e8m0(in.scale, i);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        f4x s[CT][2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int c = 0; c < CT; ++c) s[c][t] = f4x{0.0f, 0.0f, 0.0f, 0.0f};
            float scale = 1.0f;
            if constexpr (BITS == 4) scale = s_scale[wave][0][w * D / 128][16 * t + u];
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint4 kf;
                if constexpr (BITS == 4) kf = e2m1x8(in.k[t][k], scale);
                else kf = codes8(in.k[t][2 * k], in.k[t][2 * k + 1]);
#pragma unroll
                for (int n = NQ - 1; n >= 0; --n)
#pragma unroll
                    for (int c = 0; c < CT; ++c) s[c][t] = mfma16(kf, qf[c][k][n], s[c][t]);
            }
        }
        float vs[8];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const f4x x = *reinterpret_cast<const f4x *>(&s_scale[wave][1][BITS == 8 ? 0 : u * D / 512][16 * t + 4 * w]);
#pragma unroll
            for (int r = 0; r < 4; ++r) vs[4 * t + r] = x[r];
            if constexpr (BITS == 8) {
                const f4x ks = *reinterpret_cast<const f4x *>(&s_scale[wave][0][0][16 * t + 4 * w]);
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[c][t][r] *= ks[r];
            }
        }
        if constexpr (BITS == 4) {
            const uint32_t bad = nan_scales(in.scale);
            if (bad != 0) {
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[c][i / 4][i % 4] = bad >> (16 * (i / 4) + 4 * w + i % 4) & 1 ? NAN : s[c][i / 4][i % 4];
            }
        }
        if (!all_seen(A, pb, p0, p1)) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t j = pb + 16 * (i / 4) + 4 * w + i % 4;
                    s[c][i / 4][i % 4] = j <= p[c] && (j >= start[c] || j < a.sinks) ? s[c][i / 4][i % 4] : -INFINITY;
                }
        }
        float most[CT];
        bool over = false;
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            most[c] = s[c][0][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) most[c] = fmaxf(most[c], s[c][i / 4][i % 4]);
            most[c] *= A.scale2;
            over = over || most[c] - m[c] > 8.0f;   // (of infinities of one sign: no)
        }
        if (__ballot(over) != 0 || far) {   // M moves, of the columns where it has to
            far = false;
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                float x = fmaxf(most[c], __shfl_xor(most[c], 16));
                x = fmaxf(x, __shfl_xor(x, 32));
                const bool grow = x - m[c] > 8.0f;
                const float mn = grow ? rintf(x) : m[c], f = !grow || m[c] == -INFINITY ? 1.0f : exp2_fast(m[c] - mn);
                m[c] = mn;
                far = far || __ballot(fabsf(mn) >= FAR && mn > -INFINITY) != 0;
                den[c] *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[c][d][r] *= f;
            }
            if (far) {   // the exponents at once
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float M = m[c] == -INFINITY ? 0.0f : m[c], t = s[c][i / 4][i % 4] * A.scale2, rounded = t - M;
                        const float exact = fmaf(s[c][i / 4][i % 4], A.scale2, -M);
                        s[c][i / 4][i % 4] = fabsf(M) >= FAR ? rounded : exact;
                    }
            }
        }
        const float scale2 = far ? 1.0f : A.scale2;
        uint4 pf[CT][NP];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            const float M = m[c] == -INFINITY || far ? 0.0f : m[c];
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = exp2_fast(fmaf(s[c][i / 4][i % 4], scale2, -M));
            den[c] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
            if constexpr (BITS == 8) {
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] *= vs[i];
            }
            pieces8<NP>(e, pf[c]);
        }
        auto product = [&](int d, uint4 vf) {
#pragma unroll
            for (int n = NP - 1; n >= 0; --n)
#pragma unroll
                for (int c = 0; c < CT; ++c) acc[c][d] = mfma16(vf, pf[c][n], acc[c][d]);
        };
        if constexpr (BITS == 8) {
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = code(in.v[i][d / 4], d % 4);
                product(d, make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])));
            }
        } else {
            auto dims = [&](auto pair) {   // two dims: a byte of each position
                uint32_t x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(in.v[i][0], vs[i], pair.value));
                product(2 * pair.value, make_uint4(perm(x[1], x[0], 0x05040100u), perm(x[3], x[2], 0x05040100u), perm(x[5], x[4], 0x05040100u), perm(x[7], x[6], 0x05040100u)));
                product(2 * pair.value + 1, make_uint4(perm(x[1], x[0], 0x07060302u), perm(x[3], x[2], 0x07060302u), perm(x[5], x[4], 0x07060302u), perm(x[7], x[6], 0x07060302u)));
            };
            dims(std::integral_constant<int, 0>{});
            dims(std::integral_constant<int, 1>{});
            if constexpr (D == 128) {
                dims(std::integral_constant<int, 2>{});
                dims(std::integral_constant<int, 3>{});
            }
        }
    }
    // the waves' states, 16 columns after the other, a thread N dims of a column
    constexpr int N = D / 16;
    const uint32_t col = tid / 16, d0 = tid % 16 * N;
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        den[c] += __shfl_xor(den[c], 16);
        den[c] += __shfl_xor(den[c], 32);
        if (c) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < DT; d += 4)
                *reinterpret_cast<f4x *>(&s_acc[wave][u][w * (D / 4) + r * DT + d]) = f4x{acc[c][d][r], acc[c][d + 1][r], acc[c][d + 2][r], acc[c][d + 3][r]};
        if (lane < 16) { s_m[wave][u] = m[c]; s_den[wave][u] = den[c]; }
        __syncthreads();
        const uint32_t mine = tile * COLUMNS + 16 * c + col;
        if (mine / A.group > last) continue;
        float sum[N] = {}, all = 0.0f, M = s_m[0][col];
#pragma unroll
        for (int k = 1; k < 4; ++k) M = fmaxf(M, s_m[k][col]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float f = s_m[k][col] == M ? 1.0f : exp2_fast(s_m[k][col] - M);
            all = fmaf(s_den[k][col], f, all);
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] = fmaf(s_acc[k][col][d0 + i], f, sum[i]);
        }
        const uint32_t to = mine / A.group, h = g * A.group + mine % A.group;
        auto put = [&](auto *at) {
#pragma unroll
            for (int i = 0; i < N; i += 4) store4(at + i, make_float4(sum[i], sum[i + 1], sum[i + 2], sum[i + 3]));
        };
        if (A.splits == 1) {
            const float inv = 1.0f / all;
#pragma unroll
            for (int i = 0; i < N; ++i) sum[i] *= inv;
            put((T *)a.out + b * a.out_batch + to * a.out_token + h * D + d0);
            if (d0 == 0) finish_lse(A, M, all, b, to, h);
        } else {
            const uint64_t at = state_at(A, b, place.split, to, h);
            put(A.part + at * D + d0);
            if (d0 == 0) A.md[at] = make_float2(M, all);
        }
    }
}

// Many columns.  The WAVES waves of a workgroup take 32 columns of one kv head each and go through the same chunks of 32 positions,
// whose codes the workgroup stages in LDS as bf16 (K by rows; V transposed, a dim's 32 positions in the order of the second
// product's k).
//
// Tiles.  v_mfma_f32_32x32x16_bf16, rows positions, columns (token, head).  Lane half h of A and B holds dims (D / 2) h + 8 s + j of
// k-step s.  Result register r of lane l is position 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32: the k layout of the second
// product's B operand, so weights never leave their lane.
//
// A step works on three chunks at once, so that matrix and vector instructions do not wait for each other: the second product of
// chunk i - 1, the weights of chunk i, the scores of chunk i + 1.
//
// What bounds it: 2 x 4096 tokens of 32 / 8 heads of 128 within 2048 + 4 positions take 258 to 350 us on the card, as it clocks
// under the matrix cores' power, for products that a large matrix product's rate would do in 124 with one piece of the weights
// for their two: 24 matrix instructions of a chunk (768 cycles of a SIMD) and some 250 vector ones.  The first form, without the three chunks at once,
// took 560.  Other orders of the loop's parts, 8 waves a workgroup or raised priorities changed nothing.
namespace {
DEV f16x mfma32(uint4 a, uint4 b, f16x c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}
DEV float max_of_halves(float v) {   // of lanes l and l ^ 32
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
}  // namespace

template <int D>
__global__ __launch_bounds__(256, 2) void qxw_many(QxwArgs A) {
    using T = __bf16;
    constexpr int NP = P_PIECES<T>, KS = D / 16, DT = D / 32, COLUMNS = 128;
    constexpr int KP = D + 8, VP = 40;   // bf16 from one row to the next: 16 rows' 16-byte pieces lie in 16 bank groups
    constexpr int KV = D / 8, VR = KV / 4;   // a thread stages KV values of a chunk's K row, and VR positions x 4 dims of its V
    __shared__ __align__(16) union { struct { uint16_t k[2][32 * KP], v[4][D * VP]; } codes; float out[4][32 * 36]; } u;
    __shared__ __align__(16) float s_scale[4][2][32];   // of K (times scale2) and V
    const qxg_cache_attention_args &a = A.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 31, h = lane >> 5;
    const int wave = wave_id();
    const uint32_t g = blockIdx.x % a.kv_heads, tile = A.tiles - 1 - blockIdx.x / a.kv_heads, b = blockIdx.z;   // (those that see most first)
    const Seq q = sequence(A, b);
    const uint32_t first = tile * COLUMNS / A.group;
    if (first >= q.count) return;
    const uint32_t last = min((tile * COLUMNS + COLUMNS - 1) / A.group, q.count - 1);
    const Chunks list = chunks_of(A, q.len + first, q.len + last);
    const Part part = part_of(A, list.n, blockIdx.y);
    if (part.lo >= part.hi) return;
    // the wave's columns, the lane's
    const uint32_t c0 = tile * COLUMNS + 32 * wave, p0 = q.len + min(c0 / A.group, last), p1 = q.len + min((c0 + 31) / A.group, last);
    const uint32_t c = c0 + col, token = min(c / A.group, last), head = g * A.group + c % A.group, p = q.len + token, start = window_start(A, p);

    // staging
    const uint32_t kpos = tid / (D / KV), kpiece = tid % (D / KV), dq = tid % (D / 4), vt = tid / (D / 4);
    // (of 4 positions, the threads of a wave take those of both halves of 16 bytes: their writes use all banks)
    const uint32_t vpos = VR == 4 ? 4 * ((vt & 4) | (vt & 1) << 1 | (vt >> 1 & 1)) : VR * vt;
    // (bases are the workgroup's, offsets inside a chunk fit 32 bits: the row strides are below 2^26)
    const uint8_t *kbase = (const uint8_t *)a.k + b * a.kv_batch + g * D, *vbase = (const uint8_t *)a.v + b * a.kv_batch + g * D;
    const uint32_t *scales = (const uint32_t *)(lane < 32 ? a.kscale : a.vscale) + b * a.scale_batch;   // (a wave has those of both)
    const uint32_t total = q.len + q.count, n = part.hi - part.lo, row_bytes = (uint32_t)a.kv_row;
    const uint32_t kin = kpiece * KV, vin = dq * 4;   // bytes in a row
    struct { uint32_t k[KV / 4], v[VR], scale; } in;
    // where a lane's rows and scales are in a chunk
    uint32_t k_at = kpos * row_bytes + kin, v_at[VR], scale_at = lane & 31;
#pragma unroll
    for (int r = 0; r < VR; ++r) v_at[r] = (vpos + r) * row_bytes + vin;
    auto load = [&](uint32_t i) {   // (of a chunk behind the last that one's again)
        const uint32_t pb = list.at(part.lo + min(i, n - 1)) * 32;
        if (pb + 32 > total) {   // the last chunk: positions behind the last token's read that one's, they are masked
            const uint32_t past = total - 1 - pb;
            k_at = min(kpos, past) * row_bytes + kin;
#pragma unroll
            for (int r = 0; r < VR; ++r) v_at[r] = min(vpos + r, past) * row_bytes + vin;
            scale_at = min(lane & 31, past);
        }
        const uint8_t *krows = kbase + (uint64_t)pb * row_bytes, *vrows = vbase + (uint64_t)pb * row_bytes;
        if constexpr (KV == 16) *reinterpret_cast<uint4 *>(in.k) = *reinterpret_cast<const uint4 *>(krows + k_at);
        else *reinterpret_cast<uint2 *>(in.k) = *reinterpret_cast<const uint2 *>(krows + k_at);
#pragma unroll
        for (int r = 0; r < VR; ++r) in.v[r] = *reinterpret_cast<const uint32_t *>(vrows + v_at[r]);
        if (wave == 0) in.scale = scales[pb + scale_at];
    };
    auto stage_k = [&](uint32_t i) {
        uint4 *to = reinterpret_cast<uint4 *>(&u.codes.k[i & 1][kpos * KP + KV * kpiece]);
#pragma unroll
        for (int j = 0; j < KV / 8; ++j) to[j] = codes8(in.k[2 * j], in.k[2 * j + 1]);
        if (wave == 0) s_scale[i & 3][lane >> 5][lane & 31] = finite_scales(in.scale) * (lane < 32 ? A.scale2 : 1.0f);
    };
    // positions 4 w .. 4 w + 3 are half w / 2 % 2 of the 16 bytes that lane half w % 2 reads in step w / 4;
    // the place of the 16 bytes turns with dim / 16, so that the lanes' writes spread over the banks
    const int pq = vpos >> 2, slot = ((pq >> 2) * 2 + (pq & 1)) ^ ((dq >> 2) & 3), vat = 4 * dq * VP + 8 * slot + 4 * ((pq >> 1) & 1) + (vpos & 3);
    auto stage_v = [&](uint32_t i) {
        uint32_t w[4][VR / 2];   // a dim's positions
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int r = 0; r < VR; r += 2) w[d][r / 2] = pack_bf16(code(in.v[r], d), code(in.v[r + 1], d));
        uint32_t *to = reinterpret_cast<uint32_t *>(&u.codes.v[i & 3][vat]);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            if constexpr (VR == 4) *reinterpret_cast<uint2 *>(to + d * (VP / 2)) = make_uint2(w[d][0], w[d][1]);
            else to[d * (VP / 2)] = w[d][0];
        }
    };
    load(0);
    uint4 qf[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) qf[k] = reinterpret_cast<const uint4 *>((const T *)a.q + b * a.q_batch + token * a.q_token + head * D + h * (D / 2))[k];
    // the reference, how far over it a score may be (-inf: nothing is seen yet), this lane's sum
    float M = 0.0f, limit = -INFINITY, den = 0.0f;
    bool far = false;   // one of the wave's references is
    f16x acc[DT], s;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = zero16();
    uint4 pf[2][NP];   // the weights of the last chunk
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < NP; ++j) pf[k][j] = make_uint4(0, 0, 0, 0);
    const uint16_t *kr = &u.codes.k[0][col * KP + (D / 2) * h], *vr = &u.codes.v[0][col * VP];
    uint4 kf[KS], vf[2][DT];
    auto read_k = [&](uint32_t i) {
        const uint16_t *row = kr + (i & 1) * (32 * KP);
#pragma unroll
        for (int k = 0; k < KS; ++k) kf[k] = *reinterpret_cast<const uint4 *>(row + 8 * k);
    };
    auto read_v = [&](uint32_t i) {
        const uint16_t *row = vr + (i & 3) * (D * VP);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int d = 0; d < DT; ++d) vf[k][d] = *reinterpret_cast<const uint4 *>(row + 32 * d * VP + 8 * ((2 * k + h) ^ ((2 * d + (col >> 4)) & 3)));
    };
    auto scores = [&] {
        s = zero16();
#pragma unroll
        for (int k = 0; k < KS; ++k) s = mfma32(kf[k], qf[k], s);
    };
    auto context = [&] {   // acc += that of the chunk of pf
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = NP - 1; j >= 0; --j)
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[d] = mfma32(vf[k][d], pf[k][j], acc[d]);
    };
    for (uint32_t i = tid; i < D * VP / 2; i += 256) reinterpret_cast<uint32_t *>(u.codes.v[3])[i] = 0;   // (chunk -1 for the first step)
    stage_k(0);
    stage_v(0);
    load(1);
    __syncthreads();
    read_k(0);
    scores();
    stage_k(1);
    stage_v(1);
    load(2);
    __syncthreads();
#pragma unroll 1
    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t pb = list.at(part.lo + i) * 32;
        stage_k(i + 2);
        stage_v(i + 2);
        load(i + 3);
        read_v(i + 3);   // chunk i - 1's
        // exponents: scores, times the positions' scales, in base 2, less M
        float e[16];
        auto exponent = [&](int r, const f4x &ks) { return fmaf(s[r], ks[r % 4], -M); };
        auto scale_of = [&](int side, int j) { return *reinterpret_cast<const f4x *>(&s_scale[i & 3][side][8 * j + 4 * h]); };
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f4x ks = scale_of(0, j);
#pragma unroll
            for (int r = 4 * j; r < 4 * j + 4; ++r) e[r] = exponent(r, ks);
        }
        if (!all_seen(A, pb, p0, p1)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t j = pb + 8 * (r / 4) + 4 * h + r % 4;
                e[r] = j <= p && (j >= start || j < a.sinks) ? e[r] : -INFINITY;
            }
        }
        float most = e[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) most = fmaxf(most, e[r]);
        if (__ballot(most > limit) != 0 || far) {   // M moves, of the columns where it has to, and what was summed with it
            // (from the scores again: equal ones are to weigh the same in all chunks, however large)
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f4x ks = scale_of(0, j);
#pragma unroll
                for (int r = 4 * j; r < 4 * j + 4; ++r) {
                    const float t = s[r] * ks[r % 4];
                    top = fmaxf(top, e[r] == -INFINITY ? e[r] : t);
                }
            }
            top = max_of_halves(top);
            const bool grow = top - M > limit;
            const float mn = grow ? rintf(top) : M, f = !grow || limit < 0.0f ? 1.0f : exp2_fast(M - mn);
            M = mn;
            limit = grow ? 8.0f : limit;
            const bool away = fabsf(M) >= FAR;
            far = __ballot(away) != 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f4x ks = scale_of(0, j);
#pragma unroll
                for (int r = 4 * j; r < 4 * j + 4; ++r) {
                    const float t = s[r] * ks[r % 4], rounded = t - M, exact = exponent(r, ks), x = away ? rounded : exact;
                    e[r] = e[r] == -INFINITY ? e[r] : x;
                }
            }
            den *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= f;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int j = 0; j < NP; ++j) {   // (the last chunk's weights are still on their way)
                    uint32_t w[4] = {pf[k][j].x, pf[k][j].y, pf[k][j].z, pf[k][j].w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) w[x] = pack_bf16(__uint_as_float(w[x] << 16) * f, __uint_as_float(w[x] & 0xffff0000u) * f);
                    pf[k][j] = make_uint4(w[0], w[1], w[2], w[3]);
                }
        }
        read_k(i + 1);
        context();
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = exp2_fast(e[r]);
        float sum[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[r] = (e[r] + e[4 + r]) + (e[8 + r] + e[12 + r]);
        den += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f4x vs = scale_of(1, j);
#pragma unroll
            for (int r = 0; r < 4; ++r) e[4 * j + r] *= vs[r];
        }
        scores();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = e[8 * k + j];
            pieces8<NP>(x, pf[k]);
        }
        __syncthreads();
    }
    read_v(n - 1);
    context();
    __syncthreads();
    // results: a tile of 32 dims after the other through the wave's part of LDS, so that 8 lanes write a column's line
    const bool whole = A.splits == 1;
    den += __shfl_xor(den, 32);
    const float inv = whole ? 1.0f / den : 1.0f;
    float *o = u.out[wave];
#pragma unroll
    for (int d = 0; d < DT; ++d) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            *reinterpret_cast<f4x *>(o + col * 36 + 8 * k + 4 * h) = f4x{acc[d][4 * k] * inv, acc[d][4 * k + 1] * inv, acc[d][4 * k + 2] * inv, acc[d][4 * k + 3] * inv};
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t mine = c0 + (lane >> 3) + 8 * i, to = mine / A.group, th = g * A.group + mine % A.group, dim = 32 * d + 4 * (lane & 7);
            const float4 x = *reinterpret_cast<const float4 *>(o + ((lane >> 3) + 8 * i) * 36 + 4 * (lane & 7));
            if (to > last) continue;
            if (whole) store4((T *)a.out + b * a.out_batch + to * a.out_token + th * D + dim, x);
            else store4(A.part + state_at(A, b, blockIdx.y, to, th) * D + dim, x);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (h == 0 && c / A.group <= last) {
        if (whole) finish_lse(A, M, den, b, token, head);
        else A.md[state_at(A, b, blockIdx.y, token, head)] = make_float2(limit < 0.0f ? -INFINITY : M, den);
    }
}

// The splits of a row joined: a wave a row, its lanes the splits' references first, then D / 64 dims each.  A chain of latencies (4 to 6 us),
// or the states' bytes.
template <typename T, int D>
__global__ __launch_bounds__(256) void qxw_join(QxwArgs A) {
    const qxg_cache_attention_args &a = A.a;
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t row = (uint64_t)blockIdx.x * 4 + wave_id();
    if (row >= (uint64_t)a.batch * a.tokens * a.heads) return;
    const uint32_t head = row % a.heads, token = row / a.heads % a.tokens, b = row / a.heads / a.tokens;
    // (the first loads do not wait for the lengths that say how many of them count: a split's place is there, whatever it holds)
    constexpr uint32_t BATCH = 16;
    float x[BATCH][D / 64], next[BATCH][D / 64] = {};
    auto load = [&](uint32_t z0) {
#pragma unroll
        for (uint32_t k = 0; k < BATCH; ++k) {
            if (k % 4 == 0 && z0 + k >= A.splits) break;
            const float *from = A.part + state_at(A, b, min(z0 + k, A.splits - 1), token, head) * D + lane * (D / 64);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) next[k][i] = from[i];
        }
    };
    float2 md = A.md[state_at(A, b, min(lane, A.splits - 1), token, head)];
    load(0);
    const Seq q = sequence(A, b);
    if (token >= q.count) return;
    // the row's tile has as many splits as chunks for them
    const uint32_t column = token * A.group + head % A.group, tile = column / A.columns;
    const uint32_t p0 = q.len + tile * A.columns / A.group, p1 = q.len + min((tile * A.columns + A.columns - 1) / A.group, q.count - 1);
    const uint32_t n = chunks_of(A, p0, p1).n, size = split_size(A, n), splits = (n + size - 1) / size;
    float M = -INFINITY, den = 0.0f, sum[D / 64] = {};
    for (uint32_t z0 = 0; z0 < splits; z0 += 64) {
        const uint32_t many = min(splits - z0, 64u);
        if (z0) md = A.md[state_at(A, b, z0 + min(lane, many - 1), token, head)];
        if (lane >= many) md = make_float2(-INFINITY, 0.0f);
        const float mn = fmaxf(M, wave_max_f(md.x)), f = M == mn ? 1.0f : exp2_fast(M - mn);
        const float fz = lane >= many ? 0.0f : md.x == mn ? 1.0f : exp2_fast(md.x - mn);
        den = den * f + wave_total_f(md.y * fz);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) sum[i] *= f;
        M = mn;
        for (uint32_t z = 0; z < many; z += BATCH) {
#pragma unroll
            for (uint32_t k = 0; k < BATCH; ++k)
#pragma unroll
                for (int i = 0; i < D / 64; ++i) x[k][i] = next[k][i];
            if (z0 + z + BATCH < splits) load(z0 + z + BATCH);
#pragma unroll
            for (uint32_t k = 0; k < BATCH; ++k) {
                if (k % 4 == 0 && z + k >= many) break;
                const float scale = rdlanef(fz, (int)min(z + k, 63u));
#pragma unroll
                for (int i = 0; i < D / 64; ++i) sum[i] = z + k < many ? fmaf(x[k][i], scale, sum[i]) : sum[i];
            }
        }
    }
    const float inv = 1.0f / den;
    T *out = (T *)a.out + b * a.out_batch + token * a.out_token + head * D + lane * (D / 64);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) out[i] = (T)(sum[i] * inv);
    if (lane == 0) finish_lse(A, M, den, b, token, head);
}

namespace {
template <typename T, int D> hipError_t launch(const QxwArgs &A, hipStream_t s) {
    const uint32_t heads = A.a.kv_heads * A.tiles;
    const dim3 grid = A.columns != 128 ? dim3((A.tiles * A.splits * A.a.batch + 7) / 8 * 8 * A.a.kv_heads) : dim3(heads, A.splits, A.a.batch);
    auto *kernel = A.a.bits == 8 ? qxw_few<T, D, 8, 1> : qxw_few<T, D, 4, 1>;
    if constexpr (sizeof(T) == 2 || D == 64)
        if (A.columns == 32) kernel = A.a.bits == 8 ? qxw_few<T, D, 8, 2> : qxw_few<T, D, 4, 2>;
    if constexpr (__is_same(T, __bf16))
        if (A.columns == 128) kernel = qxw_many<D>;
    const hipError_t e = qxg_launch(kernel, grid, dim3(256), 0, s, A);
    if (e != hipSuccess || A.splits == 1) return e;
    const uint64_t rows = (uint64_t)A.a.batch * A.a.tokens * A.a.heads;
    return qxg_launch(qxw_join<T, D>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, A);
}
}  // namespace

hipError_t qxw_launch(const QxwArgs &A, hipStream_t s) {
    if (A.a.type == QXG_TYPE_F32) return A.a.dim == 64 ? launch<float, 64>(A, s) : launch<float, 128>(A, s);
    if (A.a.type == QXG_TYPE_F16) return A.a.dim == 64 ? launch<_Float16, 64>(A, s) : launch<_Float16, 128>(A, s);
    return A.a.dim == 64 ? launch<__bf16, 64>(A, s) : launch<__bf16, 128>(A, s);
}
