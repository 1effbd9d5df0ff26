// Kernel arguments and launchers of the operators on device memory (include/qxg.h), between
// their host side (qxg_ops.hip) and their kernels (qxg_attend.hip, qxg_evict.hip, qxg_adjust.hip).
#pragma once
#include "qxg.h"
#include "qxg_internal.h"

// A launch that returns its error: the last error of the runtime, which may be one that the caller has yet to ask for, is
// not asked here.
template <typename... P>
hipError_t qxg_launch(void (*kernel)(P...), dim3 grid, dim3 block, uint32_t lds, hipStream_t s, P... args) {
    void *at[] = {(void *)&args...};
    return hipLaunchKernel((const void *)kernel, grid, block, at, lds, s);
}

// Tree attention.  A column is a (node, q head of the kv head) pair, node * group + head; a tile is
// 32 columns.  With several splits of the positions, a split's unnormalised context goes to part
// and its (reference, denominator) in base 2 to md, at [split of the batch][node][head].
struct QxaArgs {
    qxg_tree_attention_args a;
    uint32_t group, columns, tiles, words;
    uint32_t splits;   // of the batch; of a sequence beyond 64 sequences, and when it is 1
    uint32_t wide;     // tiles four at a time, chunks staged for all of them
    uint32_t wgs, wg_columns;   // workgroups of a kv head and split, columns of one
    float scale2;      // scale * log2(e)
    float *part;
    float2 *md;
    float2 *norm;      // with an account: a row's (M, 1 / denominator), [batch][node][head]: its weights are 2^(s - M) of that
    float *scores;     // with an account and few columns: dot * kscale, -inf where masked, [batch][kv head][chunk of 32 positions][column][32]
    uint4 *pack;       // with an account otherwise: q as matrix operands, [batch][kv head][tile][k-step][half][lane]
    float *pack_sf;    // with an account: [batch][kv head][tile][column] what turns dot * kscale into base-2 scores
};
hipError_t qxa_launch(const QxaArgs &A, hipStream_t s);

// Eviction.  A tile of the compaction is `rows` rows, QXE_UNITS 16-byte units of K (and of V) at most.
constexpr uint32_t QXE_UNITS = 2048;
struct QxeCompact {
    qxg_kv_compact_args a;
    uint32_t units, inverse;   // of a row; ceil(2^20 / units): x / units = x * inverse >> 20 for x < QXE_UNITS
    uint32_t rows, tiles;      // of a tile; of a group
    uint32_t *state;           // 1 + groups * tiles words
};
hipError_t qxe_launch_select(const qxg_kv_select_args &a, hipStream_t s);
hipError_t qxe_launch_compact(const QxeCompact &C, hipStream_t s);

// Logits.  Each of the 4 waves of a slice of a row leaves up to top_n keys, its largest among them, the
// others 0, and (maximum, sum of exponentials) to the join.
struct QxsArgs {
    qxg_adjust_logits_args a;
    uint32_t slices, words;
    uint32_t small;    // slices of one 16-byte step a thread instead of QXS_SLICE tokens
    uint64_t *keys;    // [rows][slices * 4][top_n]
    float2 *ms;        // [rows][slices * 4]
};
constexpr uint32_t QXS_SLICE = 4096, QXS_BIASES = 1024, QXS_HISTORY = (1u << 20) - 1;
hipError_t qxs_launch(const QxsArgs &A, hipStream_t s);

// the context's device (qxg_api.hip)
__attribute__((visibility("hidden"))) int qxg_ctx_device(const qxg_ctx *c);
