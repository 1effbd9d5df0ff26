// Eviction from a KV cache by accumulated attention weight (qxg_kv_select, qxg_kv_compact).
#include "qxg_dev.h"
#include "qxg_ops.h"

#include <type_traits>

namespace {
// Weights as unsigned numbers in their order, 0x007fffff (-inf) or more; NaN as -inf, -0 as +0
DEV uint32_t weight_rank(float w) {
    const uint32_t u = __float_as_uint(fmaxf(w, -INFINITY) + 0.0f);   // (the larger of NaN and a number is the number)
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
// sums of a wave's two counts (the same in all its lanes) over the waves before it, and over all 16
DEV uint2 waves_before(uint2 a, uint2 *s_w, uint2 &all) {
    const int wave = wave_id();
    if ((threadIdx.x & 63) == 0) s_w[wave] = a;
    __syncthreads();
    uint2 before = make_uint2(0, 0);
    all = make_uint2(0, 0);
#pragma unroll
    for (int w = 0; w < 16; ++w) {
        const uint2 x = s_w[w];
        if (w < wave) { before.x += x.x; before.y += x.y; }
        all.x += x.x;
        all.y += x.y;
    }
    return before;
}
struct Group { uint32_t len, kept; };
DEV Group group_of(const qxg_kv_select_args &A, uint32_t g) {
    Group x;
    x.len = min(A.lens[g], A.positions);
    x.kept = min(x.len, A.budget);
    return x;
}
// A group that is kept whole.  (kept may be lens: a wave that reads its length only after this finds the same.)
DEV void keep_all(const qxg_kv_select_args &A, uint32_t g, const Group &G, uint32_t *keep) {
    if (threadIdx.x == 0) A.kept[g] = G.kept;
    for (uint32_t p = threadIdx.x; p < G.len; p += 1024) keep[p] = p;
}
// rank of position p: the largest number for those kept in any case, 0 behind the end
DEV uint32_t rank_at(const qxg_kv_select_args &A, float w, uint32_t p, uint32_t len) {
    return p >= len ? 0u : p < A.sinks || p >= len - A.recent ? ~0u : weight_rank(w);
}
}  // namespace

namespace {
// The smallest rank among the block's k[] (E a thread, 0: none) that `want` of them reach, found two bits at a time
// in the low `bits` ones (an even number) below the bits of `least`; `above`: how many are larger.  (Or, found
// sooner: a number that exactly `want` of them are above.)  The count
// of ranks that reach a number is one ballot a wave and register; lanes 16 t + w of every wave add up the waves'
// counts of the step's number t.  The chain of barriers bounds it, so two bits a step (one bit a step: 1.3 us more for
// 700 positions).
template <int E>
DEV uint32_t block_nth(const uint32_t (&k)[E], uint32_t want, uint32_t least, int bits, uint32_t (&s_n)[2][64], uint32_t &above) {
    const int lane = threadIdx.x & 63, wave = wave_id();
    above = 0;
#pragma unroll 1
    for (int b = bits - 2; b >= 0; b -= 2) {
        uint32_t n[3] = {0, 0, 0};
#pragma unroll
        for (int i = 0; i < E; ++i)
#pragma unroll
            for (int t = 0; t < 3; ++t) n[t] += (uint32_t)__popcll(__ballot(k[i] >= (least | (uint32_t)(t + 1) << b)));
        uint32_t (&to)[64] = s_n[(b >> 1) & 1];
        if (lane < 3) to[16 * lane + wave] = lane == 0 ? n[0] : lane == 1 ? n[1] : n[2];
        __syncthreads();   // (the other half is written next, so one barrier a step is enough)
        uint32_t c = to[lane];   // (the last 16 are not used)
        c += (uint32_t)dppi<DPP_XOR1>((int)c); c += (uint32_t)dppi<DPP_XOR2>((int)c);
        c += (uint32_t)dppi<DPP_ROR4>((int)c); c += (uint32_t)dppi<DPP_ROR8>((int)c);
        uint32_t digit = 0;
#pragma unroll
        for (int t = 0; t < 3; ++t) {   // fewer reach each next number
            const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)c, 16 * t);
            if (all == want) {   // these and no others
                above = want;
                return (least | (uint32_t)(t + 1) << b) - 1;
            }
            if (all >= want) digit = t + 1;
            else { above = all; break; }
        }
        least |= digit << b;
    }
    return least;
}
// how many of a wave's ranks are above `least`, and how many are equal
template <int E> DEV uint2 count_kept(const uint32_t (&k)[E], uint32_t least) {
    uint2 n = make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        n.x += (uint32_t)__popcll(__ballot(k[i] > least));
        n.y += (uint32_t)__popcll(__ballot(k[i] == least));
    }
    return n;
}
// Lists the kept ones of a wave's 64 E positions from p0 on: ranks above `least`, and the lowest `need` equal ones.
// at: how many of either lie before p0; moved on.
template <int E>
DEV void list_kept(const uint32_t (&k)[E], uint32_t p0, uint32_t least, uint32_t need, uint2 &at, uint32_t *keep) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const uint64_t gt = __ballot(k[i] > least), eq = __ballot(k[i] == least);
        const uint32_t place = at.x + __builtin_amdgcn_mbcnt_hi((uint32_t)(gt >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)gt, 0));
        if (eq == 0 || at.y >= need) {   // (uniform)
            if (k[i] > least) keep[place + min(at.y, need)] = p0 + 64 * i + lane;
        } else {
            const uint32_t y = at.y + __builtin_amdgcn_mbcnt_hi((uint32_t)(eq >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)eq, 0));
            if (k[i] > least || (k[i] == least && y < need)) keep[place + min(y, need)] = p0 + 64 * i + lane;
        }
        at.x += (uint32_t)__popcll(gt);
        at.y += (uint32_t)__popcll(eq);
    }
}
// weights of a wave's 64 E positions from p0 on, those before `end`
template <int E>
DEV void load_weights(const float *acc, uint32_t p0, uint32_t end, float (&w)[E]) {
    const uint32_t lane = threadIdx.x & 63;
    if (p0 + 64 * E <= end) {   // (uniform)
        const float *p = acc + p0 + lane;
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = p[64 * i];
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = p0 + 64 * i + lane < end ? acc[p0 + 64 * i + lane] : 0.0f;
    }
}
// and their ranks, 0 from `end` on
template <int E>
DEV void ranks_of(const qxg_kv_select_args &A, const float (&w)[E], uint32_t p0, uint32_t end, uint32_t len, uint32_t (&k)[E]) {
    const uint32_t lane = threadIdx.x & 63;
    if (p0 >= A.sinks && p0 + 64 * E <= min(end, len - A.recent)) {   // (uniform; nothing kept in any case, nothing behind the end)
#pragma unroll
        for (int i = 0; i < E; ++i) k[i] = weight_rank(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const uint32_t p = p0 + 64 * i + lane;
            k[i] = p >= end ? 0u : rank_at(A, w[i], p, len);
        }
    }
}
// all batches of a wave's positions lo .. hi - 1, the next one's weights on their way: f(ranks, first position)
template <int E, typename F>
DEV void each_batch(const qxg_kv_select_args &A, const float *acc, uint32_t lo, uint32_t hi, uint32_t len, F f) {
    uint32_t k[E];
    float next[E];
    load_weights<E>(acc, lo, hi, next);
#pragma unroll 1
    for (uint32_t p0 = lo; p0 < hi; p0 += 64 * E) {
        ranks_of<E>(A, next, p0, hi, len, k);
        load_weights<E>(acc, p0 + 64 * E, hi, next);
        f(k, p0);
    }
}
// A group of at most 1024 E positions, more than the budget: a thread holds E positions' ranks in registers.
template <int E>
DEV void select_held(const qxg_kv_select_args &A, const float *acc, const Group &G, uint32_t *keep, uint32_t (&s_n)[2][64], uint2 *s_w) {
    const uint32_t p0 = 64 * E * wave_id();
    uint32_t k[E], above;
    float w[E];
    load_weights<E>(acc, p0, G.len, w);
    ranks_of<E>(A, w, p0, G.len, G.len, k);
    const uint32_t least = block_nth<E>(k, A.budget, 0, 32, s_n, above);
    uint2 all, at = waves_before(count_kept<E>(k, least), s_w, all);
    list_kept<E>(k, p0, least, A.budget - above, at, keep);
}
}  // namespace

// Up to 1024 E positions, a workgroup a group, in registers.  The
// counts of its steps bound it: 16 at most, 0.3 us each.  (Byte-wise histograms in LDS, their bins searched by one thread: 26 us
// for 700 positions.)
template <int E>
__global__ __launch_bounds__(1024) void qxe_select(qxg_kv_select_args A) {
    __shared__ uint32_t s_n[2][64];
    __shared__ uint2 s_w[16];
    const uint32_t g = blockIdx.x;
    const Group G = group_of(A, g);
    uint32_t *keep = A.keep + g * A.keep_group;
    if (G.len <= A.budget) return keep_all(A, g, G, keep);
    select_held<E>(A, A.account + g * A.account_group, G, keep, s_n, s_w);
    if (threadIdx.x == 0) A.kept[g] = G.kept;   // (kept may be lens: behind the barriers, so that every wave has its length)
}

// Caches of more positions; groups of up to 4096 go as above (700 of 131072: 8.2 us, as below 12.4; 4000: 9.3 and 13.9; with
// 16 ranks a thread 5000: 26.0 and 17.2).  A sixteenth of them a wave.  A histogram of the ranks' top 12 bits (each
// bin 8 times, by lane, as equal bins of a wave's lanes would be added one after the other), then the ranks of
// the bin that holds the smallest kept one go to LDS, where its other bits are found as above; a bin of more
// than ROOM ranks is halved further by another histogram.  The account is read three times, from the caches
// after the first, and the waves meet only between the readings.  The loads that one CU has on their way bound it:
// 131000 positions 62 us, 14 .. 17 a reading (35 GB/s; alike with twice as many registers loaded ahead, and with
// fewer instructions a rank), 3 the bins, 4 the last bits.  Shorter accounts in one workgroup's registers: 4096
// positions 12.5 us, 700 6.5.
__global__ __launch_bounds__(1024) void qxe_select_long(qxg_kv_select_args A) {
    constexpr int E = 8, BITS = 12, BINS = 1 << BITS, COPIES = 8, ROOM = 16384;
    __shared__ uint32_t s_hist[BINS * COPIES], s_n[2][64], s_digit, s_above, s_count, s_gt[16], s_eq[16];
    __shared__ uint8_t s_wave[ROOM];   // of a rank in LDS: the wave that holds its position
    __shared__ uint2 s_w[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const uint32_t g = blockIdx.x;
    const Group G = group_of(A, g);
    uint32_t *keep = A.keep + g * A.keep_group;
    const float *acc = A.account + g * A.account_group;
    if (G.len <= A.budget) return keep_all(A, g, G, keep);
    if (G.len <= 4096) {
        select_held<4>(A, acc, G, keep, s_n, s_w);
        if (tid == 0) A.kept[g] = G.kept;
        return;
    }
    const uint32_t part = (G.len + 1023) / 1024 * 64, lo = min(wave * part, G.len), hi = min(lo + part, G.len);
    uint32_t least = 0, above = 0;   // bits found, and ranks above them
    int shift = 32;                  // bits still to find
    bool counted = false;            // s_gt and s_eq hold the waves' numbers of kept ranks
    while (shift > 0) {
        const int bits = min(shift, BITS);
        for (int i = tid; i < BINS * COPIES / 4; i += 1024) reinterpret_cast<uint4 *>(s_hist)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        each_batch<E>(A, acc, lo, hi, G.len, [&](const uint32_t (&k)[E], uint32_t) {
            // (positions behind the end have rank 0, whose first 12 bits no other has)
            if (shift == 32) {   // no branch a rank
#pragma unroll
                for (int i = 0; i < E; ++i) atomicAdd(&s_hist[(k[i] >> (32 - BITS)) * COPIES + (lane & (COPIES - 1))], 1u);
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (k[i] >> shift == least >> shift)
                        atomicAdd(&s_hist[((k[i] >> (shift - bits)) & ((1u << bits) - 1u)) * COPIES + (lane & (COPIES - 1))], 1u);
            }
        });
        __syncthreads();
        // the bins from the top, four a thread
        uint32_t n[4] = {0, 0, 0, 0}, run = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int c = 0; c < COPIES; ++c) n[i] += s_hist[(BINS - 1 - 4 * tid - i) * COPIES + ((c + tid) & (COPIES - 1))];
            run += n[i];
        }
        const uint32_t mine = run;
        uint2 all;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {   // running count over the wave's lanes
            const uint32_t y = (uint32_t)__shfl_up((int)run, o);
            if (lane >= o) run += y;
        }
        uint32_t before = above + run - mine + waves_before(make_uint2((uint32_t)__shfl((int)run, 63), 0), s_w, all).x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (before < A.budget && before + n[i] >= A.budget) {
                s_digit = BINS - 1 - 4 * tid - i;
                s_above = before;
                s_count = n[i];
            }
            before += n[i];
        }
        __syncthreads();
        shift -= bits;
        least |= s_digit << shift;
        above = s_above;
        const uint32_t count = s_count;
        __syncthreads();
        if (shift && count <= ROOM) {
            if (tid == 0) s_count = 0;
            __syncthreads();
            const uint32_t width = 1u << shift;   // of the bin, from `least` on
            uint32_t larger = 0;
            each_batch<E>(A, acc, lo, hi, G.len, [&](const uint32_t (&k)[E], uint32_t) {
                uint32_t in = 0;
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    larger += (uint32_t)__popcll(__ballot(k[i] > least + (width - 1)));
                    in += (uint32_t)__popcll(__ballot(k[i] - least < width));
                }
                if (!in) return;
                uint32_t first = 0;
                if (lane == 0) first = atomicAdd(&s_count, in);
                first = (uint32_t)__builtin_amdgcn_readfirstlane((int)first);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const bool f = k[i] - least < width;
                    const uint64_t b = __ballot(f);
                    if (!b) continue;
                    if (f) {
                        const uint32_t to = first + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
                        s_hist[to] = k[i];   // (< count, in any order)
                        s_wave[to] = (uint8_t)wave;
                    }
                    first += (uint32_t)__popcll(b);
                }
            });
            if (lane == 0) { s_gt[wave] = larger; s_eq[wave] = 0; }
            __syncthreads();
            const auto rest = [&](auto size) {   // the bin's other bits, and whose ranks they are
                constexpr int N = decltype(size)::value;
                uint32_t k[N], more;
#pragma unroll
                for (int i = 0; i < N; ++i) k[i] = (uint32_t)(1024 * i + tid) < count ? s_hist[1024 * i + tid] : 0u;
                least = block_nth<N>(k, A.budget - above, least, shift, s_n, more);
                above += more;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (k[i] >= least) atomicAdd(&(k[i] > least ? s_gt : s_eq)[s_wave[1024 * i + tid]], 1u);
                __syncthreads();
            };
            if (count <= 4096) rest(std::integral_constant<int, 4>{});
            else rest(std::integral_constant<int, 16>{});
            shift = 0;
            counted = true;
        }
    }
    if (!counted) {
        uint2 own = make_uint2(0, 0);
        each_batch<E>(A, acc, lo, hi, G.len, [&](const uint32_t (&k)[E], uint32_t) {
            const uint2 n = count_kept<E>(k, least);
            own.x += n.x;
            own.y += n.y;
        });
        if (lane == 0) { s_gt[wave] = own.x; s_eq[wave] = own.y; }
        __syncthreads();
    }
    uint2 at = make_uint2(0, 0);
    for (int w = 0; w < wave; ++w) { at.x += s_gt[w]; at.y += s_eq[w]; }
    each_batch<E>(A, acc, lo, hi, G.len, [&](const uint32_t (&k)[E], uint32_t p0) { list_kept<E>(k, p0, least, A.budget - above, at, keep); });
    if (tid == 0) A.kept[g] = G.kept;   // (as above)
}

// Rows moved in place.  Tiles of R rows (32 KB of K, or one row) are claimed in order: a workgroup reads its tile's
// sources, says so, waits until the earlier tiles of its group whose sources lie where it is about to
// write have been read, and writes.  A claimed tile reads without waiting, and waits only for tiles
// claimed before it, so every wait ends (a bound on the polls ends it also where two calls share a workspace,
// which is not allowed).  Each row is read and written once: 48 groups of 2048 rows of
// 512 bytes 43 .. 48 us (200 MB), 3 of 32768 rows picked from four times as many 60 .. 65 (scattered rows).  (Strips of columns, each walked in order by
// one workgroup, left most of the GPU idle: 989 us for 3 groups of 32768 rows.)  state: the ticket, then
// a word a tile.
extern "C" __global__ __launch_bounds__(256) void qxe_clear(uint32_t *state, uint32_t n) {
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) state[i] = 0;
}
extern "C" __global__ __launch_bounds__(256) void qxe_compact(QxeCompact C) {
    const qxg_kv_compact_args &A = C.a;
    constexpr int U = QXE_UNITS / 256;
    __shared__ uint32_t s_ticket, s_keep[QXE_UNITS];
    const int tid = threadIdx.x;
    if (tid == 0) s_ticket = __hip_atomic_fetch_add(C.state, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const uint32_t ticket = s_ticket;
    if (ticket >= A.groups * C.tiles) return;
    const uint32_t g = ticket / C.tiles, tile = ticket % C.tiles, i0 = tile * C.rows;
    const uint32_t n = min(A.kept[g * A.kept_group], min(A.slots, A.positions - A.first));
    if (i0 >= n) return;
    const uint32_t *keep = A.keep + g * A.keep_group, here = min(C.rows, n - i0), to = A.first + i0;
    uint32_t *read = C.state + 1 + g * C.tiles;   // [tile] 1: its sources are in registers
    bool moves = false;
    for (uint32_t i = tid; i < here; i += 256) {
        const uint32_t p = keep[i0 + i];
        s_keep[i] = p;
        moves = moves || (p != to + i && p < A.positions);
    }
    const bool any = __syncthreads_or(moves);
    // the scales and accounts of rows tid, tid + 256, ..., and 16-byte units of the rows
    const float *acc = A.account ? A.account + g * A.account_group : nullptr;
    float *ks = A.kscale + g * A.scale_group, *vs = A.vscale + g * A.scale_group;
    if (acc) {
        float *out = A.account_out + g * A.account_out_group + to;
        for (uint32_t i = tid; i < here; i += 256)
            if (s_keep[i] < A.positions) out[i] = acc[s_keep[i]];
    }
    nt4 k[U], v[U];
    float sk[U], sv[U];
    uint64_t dst[U];
    if (any) {
        const uint8_t *kb = (const uint8_t *)A.k + g * A.kv_group, *vb = (const uint8_t *)A.v + g * A.kv_group;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint32_t x = tid + 256 * j, row = (x * C.inverse) >> 20, unit = x - row * C.units;
            const uint32_t p = row < here ? s_keep[row] : ~0u;
            dst[j] = ~0ull;
            if (p < A.positions && p != to + row) {
                const uint64_t off = p * A.kv_row + 16 * unit;
                k[j] = *reinterpret_cast<const nt4 *>(kb + off);
                v[j] = *reinterpret_cast<const nt4 *>(vb + off);
                dst[j] = (to + row) * A.kv_row + 16 * unit;
            }
            if (256 * j < C.rows) {   // (uniform)
                const uint32_t q = x < here ? s_keep[x] : ~0u;
                if (q < A.positions) { sk[j] = ks[q]; sv[j] = vs[q]; }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the wave's loads have returned (a barrier alone does not wait for them)
    __syncthreads();
    if (tid == 0) __hip_atomic_store(&read[tile], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (!any) return;
    for (uint32_t c = tile; c-- > 0;) {   // earlier tiles, the nearest first, 256 at a time
        const bool mine = c >= (uint32_t)tid;
        const uint32_t t = c - tid;
        bool wait = false;
        if (mine) {
            wait = keep[t * C.rows + C.rows - 1] >= to;   // its last source lies at or behind the first written row
            for (uint32_t polls = 0; wait && polls < 1u << 20; ++polls) {
                if (__hip_atomic_load(&read[t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) break;
                __builtin_amdgcn_s_sleep(1);
            }
        }
        // farther tiles' sources lie lower: none of them is awaited once one of these is not
        if (!__syncthreads_and(mine && wait)) break;
        c -= 255;
    }
    uint8_t *kb = (uint8_t *)A.k + g * A.kv_group, *vb = (uint8_t *)A.v + g * A.kv_group;
#pragma unroll
    for (int j = 0; j < U; ++j) {
        if (dst[j] != ~0ull) {
            *reinterpret_cast<nt4 *>(kb + dst[j]) = k[j];
            *reinterpret_cast<nt4 *>(vb + dst[j]) = v[j];
        }
        const uint32_t x = tid + 256 * j;
        if (256 * j < C.rows && x < here && s_keep[x] < A.positions) {
            ks[to + x] = sk[j];
            vs[to + x] = sv[j];
        }
    }
}

hipError_t qxe_launch_select(const qxg_kv_select_args &a, hipStream_t s) {
    auto *kernel = a.positions <= 1024 ? qxe_select<1> : a.positions <= 4096 ? qxe_select<4> : qxe_select_long;
    return qxg_launch(kernel, dim3(a.groups), dim3(1024), 0, s, a);
}
hipError_t qxe_launch_compact(const QxeCompact &C, hipStream_t s) {
    const uint32_t words = 1 + C.a.groups * C.tiles;
    const hipError_t e = qxg_launch(qxe_clear, dim3(std::min<uint32_t>(64, (words + 255) / 256)), dim3(256), 0, s, C.state, words);
    return e != hipSuccess ? e : qxg_launch(qxe_compact, dim3(C.a.groups * C.tiles), dim3(256), 0, s, C);
}
