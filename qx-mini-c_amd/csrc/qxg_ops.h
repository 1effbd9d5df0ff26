// Kernel arguments and launchers of the operators on device memory (include/qxg.h), between
// their host side (qxg_ops.hip) and their kernels (qxg_attend.hip, qxg_evict.hip, qxg_adjust.hip).
#pragma once
#include "qxg.h"
#include "qxg_internal.h"

// Tree attention.  A column is a (node, q head of the kv head) pair, node * group + head; a tile is
// 32 columns.  With several splits of the positions, a split's unnormalised context goes to part
// and its (maximum, denominator) in base 2 to md, at [split][batch][node][head].
struct QxaArgs {
    qxg_tree_attention_args a;
    uint32_t group, columns, tiles, splits, words;
    float scale2;      // scale * log2(e)
    float *part;
    float2 *md;
    float *lse;        // the caller's, or the workspace's for the account
};
void qxa_launch(const QxaArgs &A, hipStream_t s);

// Eviction
void qxe_launch_select(const qxg_kv_select_args &a, hipStream_t s);
void qxe_launch_compact(const qxg_kv_compact_args &a, hipStream_t s);

// Logits.  A slice of a row leaves its top_n keys and (maximum, sum of exponentials) to the merge.
struct QxsArgs {
    qxg_adjust_logits_args a;
    uint32_t slices, words;
    uint64_t *keys;    // [rows][slices][top_n]
    float2 *ms;        // [rows][slices]
};
constexpr uint32_t QXS_SLICE = 4096;
void qxs_launch(const QxsArgs &A, hipStream_t s);

// the context's device (qxg_api.hip)
__attribute__((visibility("hidden"))) int qxg_ctx_device(const qxg_ctx *c);
