// Host side of the operators on device memory (include/qxg.h): argument checks, workspaces, launches.
// The checks of sizes come first and use no GPU.
#include "qxg_ops.h"

#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cmath>

namespace {
struct Err {
    char *err;
    uint64_t n;
    __attribute__((format(printf, 2, 3))) bool operator()(const char *fmt, ...) const {
        if (err && n) {
            va_list ap;
            va_start(ap, fmt);
            vsnprintf(err, (size_t)n, fmt, ap);
            va_end(ap);
        }
        return false;
    }
};

// bytes of a value; 0 for another type
uint32_t type_size(uint32_t t) { return t == QXG_TYPE_F32 ? 4 : t == QXG_TYPE_F16 || t == QXG_TYPE_BF16 ? 2 : 0; }

struct Arg {
    const void *p;
    const char *name;
    bool need;         // may not be NULL
    uint32_t align;
};

// Runs `go` with the context's GPU current (and the caller's GPU again after it), once every pointer is
// known to be memory of that GPU.
template <size_t N, typename F>
bool on_device(const qxg_ctx *c, const Arg (&args)[N], hipStream_t s, int wait, const Err &fail, F go) {
    if (!c) return fail("invalid context");
    const int dev = qxg_ctx_device(c);
    // An error of this call is reported by it and cleared, unless the caller had one pending before.
    const bool pending = hipPeekAtLastError() != hipSuccess;
    const auto clear = [&] { if (!pending) (void)hipGetLastError(); };
    for (const Arg &a : args) {
        if (!a.p) continue;
        hipPointerAttribute_t at{};
        if (hipPointerGetAttributes(&at, a.p) != hipSuccess) {
            clear();
            return fail("%s is not device memory of this library's HIP runtime", a.name);
        }
        if (at.type != hipMemoryTypeDevice || at.device != dev) return fail("%s is not memory of the context's device %d", a.name, dev);
    }
    int before = dev;
    hipError_t e = hipGetDevice(&before);
    if (e == hipSuccess && before != dev) e = hipSetDevice(dev);
    if (e != hipSuccess) {
        clear();
        return fail("hipSetDevice failed");
    }
    e = go();
    if (wait) {   // also for what a launch that failed has left before it
        const hipError_t w = hipStreamSynchronize(s);
        if (e == hipSuccess) e = w;
    }
    if (before != dev) (void)hipSetDevice(before);
    if (e == hipSuccess) return true;
    clear();
    return fail("%s", hipGetErrorString(e));
}
template <size_t N> bool pointers_ok(const Arg (&args)[N], const Err &fail) {
    for (const Arg &a : args) {
        if (!a.p && a.need) return fail("%s is NULL", a.name);
        if ((uintptr_t)a.p % a.align) return fail("%s is not aligned to %u bytes", a.name, a.align);
    }
    return true;
}
// Whether rows of `row` elements at i a + j b, i < na, j < nb, overlap.  (Most layouts are nested: the rows of one
// index lie in a run of their own.)
bool rows_overlap(uint64_t a, uint64_t na, uint64_t b, uint64_t nb, uint64_t row) {
    using wide = unsigned __int128;
    if (na < nb) { std::swap(a, b); std::swap(na, nb); }
    if (na == 1) return false;
    if (a < row) return true;
    if (nb == 1) return false;
    if (b < row) return true;
    if (a >= (wide)(nb - 1) * b + row || b >= (wide)(na - 1) * a + row) return false;
    for (uint64_t j = 1; j < nb; ++j) {   // the two rows (i, 0) next to (0, j)
        const wide at = (wide)j * b, i = at / a;
        if ((i && i < na && at - i * a < row) || (i + 1 < na && (i + 1) * a - at < row)) return true;
    }
    return false;
}
uint64_t up16(uint64_t v) { return (v + 15) & ~15ull; }

// ---- tree attention
// Which kernel takes a tree, and the splits of its positions over the batch (F32, 32 heads of 128 dims, in us; BF16 of 64
// dims has the same borders to within 2 us, but for 8 x 16 nodes over 1000 positions: 22 in splits, 16 without).
//
// The wide kernel's workgroups take four tiles at a time: a code is converted once for 128 columns, but a chunk's
// latency is a workgroup's, where the other kernel's four waves have a chunk each.  It gains from about 12000 chunks
// of all tiles on: 16 nodes, 4 kv heads, 12000 positions (6016 chunks) 31.8 against 26.9, 30000 (15008) 38.4 against 40.4; 64
// nodes, 4000 positions (8128) 33.8 against 28.6, 12000 (24128) 48.1 against 52.8.
//
// Splits: a workgroup a CU where the work is small, else two (480 of the 512 places: with all taken some workgroups of a launch
// waited for a second round, 217 instead of 162 for 2 x 48 nodes over 65500 positions): 16 nodes over 4000 positions
// (2016 chunks) with 240 workgroups 17.8, with 480 21.0; 64 nodes over 4000 (8128) 33.7 and 28.8.  None where a wave has few
// rounds of chunks anyway, as states and their join take 4, with a batch 5 to 10 (its shares are found in both
// kernels): 8 x 16 nodes, 8 kv heads, 500 positions (4 rounds) 17.2 without, 25.9 with; 8 rounds 24.0 and 27.6, but of
// 4 nodes (64 workgroups) 21.9 and 17.7; one tree of 64 nodes over 200 (3 rounds) 12.7 and 15.0, over 500 (5 rounds) 17.1 and 16.1.
void tree_splits(QxaArgs &A) {
    const qxg_tree_attention_args &a = A.a;
    const uint64_t chunks = ((uint64_t)a.max_len + a.nodes + 31) / 32;   // of a sequence
    const uint64_t work = (uint64_t)a.batch * a.kv_heads * A.tiles * chunks;
    A.wide = A.tiles > 2 && work > 12000;
    A.wg_columns = A.wide ? 128 : 32;
    A.wgs = (A.columns + A.wg_columns - 1) / A.wg_columns;
    const uint64_t wgs = (uint64_t)a.kv_heads * A.wgs;   // of one split
    const uint64_t rounds = (chunks + 3) / 4;            // of a wave of the kernel of few columns, without splits
    A.splits = 1;
    if (!A.wide && rounds <= (a.batch == 1 ? 3u : wgs * a.batch < 96 ? 4u : 8u)) return;
    const uint64_t target = !A.wide && work <= 3500 ? 240 : 480;
    const uint64_t most = std::max<uint64_t>(1, ((uint64_t)a.max_len + a.nodes) / 128);   // of a sequence: a chunk a wave
    if (a.batch > 64) {
        A.splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(target / (wgs * a.batch), most));
        return;
    }
    A.splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(target / wgs, most * a.batch));
    if (A.splits <= a.batch) A.splits = 1;   // (no more than one for each)
}
bool tree_plan(const qxg_tree_attention_args *p, QxaArgs &A, uint64_t &bytes, const Err &fail) {
    if (!p) return fail("invalid argument");
    const qxg_tree_attention_args &a = A.a = *p;
    const uint32_t size = type_size(a.type);
    if (!size) return fail("unsupported value type %u", a.type);
    if (!a.batch || a.batch > 65535) return fail("batch must be between 1 and 65535");
    if (!a.nodes || a.nodes > 1024) return fail("nodes must be between 1 and 1024");
    if (a.dim != 64 && a.dim != 128) return fail("dim must be 64 or 128");
    if (!a.kv_heads || !a.heads || a.heads % a.kv_heads || a.heads > 1024) return fail("heads must be a multiple of kv_heads, at most 1024");
    if (!a.positions || a.positions > 0x7fffffffu || a.max_len > 0x7fffffffu) return fail("positions and max_len must be below 2^31");
    if ((a.batch > 1 && (a.q_batch * size % 16 || a.out_batch * size % 16)) || (a.nodes > 1 && (a.q_node * size % 16 || a.out_node * size % 16)))
        return fail("the strides of q and out must be multiples of 16 bytes");
    if ((a.batch > 1 && a.kv_batch % 16) || (a.positions > 1 && a.kv_row % 16)) return fail("the strides of k and v must be multiples of 16 bytes");
    if (a.positions > 1 && a.kv_row >> 26) return fail("the row stride of k and v must be below 2^26 bytes");
    if (rows_overlap(a.out_batch, a.batch, a.out_node, a.nodes, (uint64_t)a.heads * a.dim)) return fail("rows of out overlap");
    if (a.out && a.out == a.q) return fail("out must be another array than q");
    if (a.account && a.batch > 1 && a.account_batch < a.positions) return fail("the accounts overlap");
    if (!std::isfinite(a.scale) || !(a.scale > 0.0f)) return fail("scale must be positive and finite");
    if (!std::isfinite(a.decay)) return fail("decay must be finite");
    A.group = a.heads / a.kv_heads;
    A.columns = a.nodes * A.group;
    A.tiles = (A.columns + 31) / 32;
    tree_splits(A);
    A.words = (a.nodes + 31) / 32;
    A.scale2 = (float)((double)a.scale * 1.4426950408889634);
    if (!std::isfinite(A.scale2)) return fail("scale * log2(e) must be finite");
    const uint64_t rows = (uint64_t)a.batch * a.nodes * a.heads;
    const uint64_t states = A.splits == 1 ? 0 : (a.batch > 64 ? (uint64_t)A.splits * a.batch : a.batch == 1 ? A.splits : 2ull * A.splits + a.batch) * a.nodes * a.heads;
    const uint64_t part = up16(states * a.dim * 4), md = up16(states * 8);
    // The account needs the scores again.  Of few columns they are kept (at most half as many bytes, written
    // and read, as the K codes have): single tokens over 4 x 30000 positions, 8 kv heads of 4 columns, take 67 us
    // instead of 90, of 8 columns 77, of 16 99 instead of 90.  Of more they are computed again from q, which the
    // attention leaves as matrix operands.
    const bool kept = a.account && A.columns * 16 <= a.dim;
    const uint64_t scores = kept ? (uint64_t)a.batch * a.kv_heads * (((uint64_t)a.positions + 31) / 32) * A.columns * 128 : 0;
    const uint64_t norm = a.account ? up16(rows * 8) : 0, tiles = a.account ? (uint64_t)a.batch * a.kv_heads * A.tiles : 0;
    const uint64_t sf = tiles * 128, pack = kept ? 0 : tiles * (a.dim / 16) * (a.type == QXG_TYPE_F32 ? 2 : 1) * 1024;
    uint8_t *w = (uint8_t *)a.workspace;
    A.part = (float *)w;
    A.md = (float2 *)(w + part);
    A.norm = a.account ? (float2 *)(w + part + md) : nullptr;
    A.pack_sf = a.account ? (float *)(w + part + md + norm) : nullptr;
    A.scores = kept ? (float *)(w + part + md + norm + sf) : nullptr;
    A.pack = pack ? (uint4 *)(w + part + md + norm + sf) : nullptr;
    bytes = part + md + norm + sf + scores + pack;
    return true;
}

// ---- eviction
bool select_ok(const qxg_kv_select_args *p, const Err &fail) {
    if (!p) return fail("invalid argument");
    if (!p->groups || p->groups >= 1u << 22) return fail("groups must be between 1 and 2^22 - 1");   // (a launch has less than 2^32 threads)
    if (!p->positions || p->positions > 0x7fffffffu || p->max_len > 0x7fffffffu) return fail("positions and max_len must be below 2^31");
    if (!p->budget) return fail("budget must be positive");
    if ((uint64_t)p->sinks + p->recent > p->budget) return fail("sinks + recent exceed the budget");
    if (p->groups > 1 && p->keep_group < p->budget) return fail("the lists of keep overlap");
    const uintptr_t lens = (uintptr_t)p->lens, kept = (uintptr_t)p->kept, bytes = (uintptr_t)p->groups * 4;
    if (kept != lens && kept < lens + bytes && lens < kept + bytes) return fail("kept overlaps lens (it may be lens itself)");
    return true;
}
bool compact_plan(const qxg_kv_compact_args *p, QxeCompact &C, uint64_t &bytes, const Err &fail) {
    if (!p) return fail("invalid argument");
    if (!p->groups || p->groups > 65535) return fail("groups must be between 1 and 65535");
    if (!p->positions || p->positions > 0x7fffffffu) return fail("positions must be below 2^31");
    if (!p->slots) return fail("slots must be positive");
    if (p->first >= p->positions) return fail("first is outside the cache");
    if (!p->row_bytes || p->row_bytes % 16 || p->row_bytes > 4096) return fail("row_bytes must be a multiple of 16 up to 4096");
    if ((p->groups > 1 && p->kv_group % 16) || (p->positions > 1 && p->kv_row % 16)) return fail("the strides of k and v must be multiples of 16 bytes");
    if (rows_overlap(p->kv_row, p->positions, p->kv_group, p->groups, p->row_bytes)) return fail("the rows of k and v overlap");
    if (p->groups > 1 && p->scale_group < p->positions) return fail("the scales of groups overlap");
    if (p->groups > 1 && p->account_out && p->account_out_group < p->positions) return fail("the accounts of groups overlap");
    if (!p->account != !p->account_out) return fail("account and account_out go together");
    if (p->account && p->account == p->account_out) return fail("account_out must be another array than account");
    C.a = *p;
    C.units = p->row_bytes / 16;
    C.inverse = ((1u << 20) + C.units - 1) / C.units;
    C.rows = QXE_UNITS / C.units;
    C.tiles = (std::min(p->slots, p->positions - p->first) + C.rows - 1) / C.rows;
    if ((uint64_t)p->groups * C.tiles >= 1u << 24) return fail("too many rows for one call");   // (a launch has less than 2^32 threads)
    C.state = (uint32_t *)p->workspace;
    bytes = up16(4 + 4ull * p->groups * C.tiles);
    return true;
}

// ---- logits
bool adjust_plan(const qxg_adjust_logits_args *p, QxsArgs &A, uint64_t &bytes, const Err &fail) {
    if (!p) return fail("invalid argument");
    const qxg_adjust_logits_args &a = A.a = *p;
    if (!type_size(a.type)) return fail("unsupported value type %u", a.type);
    if (!a.rows || a.rows > 65535) return fail("rows must be between 1 and 65535");
    if (!a.vocab || a.vocab > 0x7fffffffu) return fail("vocab must be between 1 and 2^31 - 1");
    if (a.top_n > QXG_MAX_TOPN) return fail("top_n must be at most %u", QXG_MAX_TOPN);
    if (a.biases > QXS_BIASES) return fail("biases must be at most %u", QXS_BIASES);
    if (a.rows > 1 && (a.logits_row < a.vocab || a.out_row < a.vocab)) return fail("rows of logits or out overlap");
    if (a.logits == a.out && a.rows > 1 && a.logits_row != a.out_row) return fail("in place, the row strides must be equal");
    if (a.history && !a.history_slots) return fail("history without slots");
    if (a.history_slots > QXS_HISTORY) return fail("history_slots must be at most %u", QXS_HISTORY);
    if (!a.history && (a.history_lens || a.prompt_lens)) return fail("history_lens or prompt_lens without history");
    if (!a.bias_ids != !a.bias_values || !a.bias_ids != !a.biases) return fail("bias_ids, bias_values and biases go together");
    if (!a.mask != !a.masks || (!a.mask && a.mask_rows)) return fail("mask, masks and mask_rows go together");
    if (a.mask && !a.mask_rows && a.masks < a.rows) return fail("fewer masks than rows without mask_rows");
    if (!a.top_n != !a.top_ids || (!a.top_n && a.top_logits)) return fail("top_n, top_ids and top_logits go together");
    // Few rows: small slices, so that the launch is not a few workgroups' chain of latencies (151936 F32 logits, best 8: one
    // row 10.3 us, 11.8 with large ones; 6 rows 12.1 and 12.6; 12 rows 15.4 and 13.8).
    const uint32_t tokens = 4096 / type_size(a.type);   // of a small slice
    A.small = (uint64_t)a.rows * ((a.vocab + QXS_SLICE - 1) / QXS_SLICE) < 256;
    A.slices = (a.vocab + (A.small ? tokens : QXS_SLICE) - 1) / (A.small ? tokens : QXS_SLICE);
    A.words = (a.vocab + 31) / 32;
    const uint64_t keys = up16((uint64_t)a.rows * A.slices * 4 * a.top_n * 8), ms = up16((uint64_t)a.rows * A.slices * 4 * 8);
    A.keys = (uint64_t *)a.workspace;
    A.ms = (float2 *)((uint8_t *)a.workspace + keys);
    bytes = keys + ms;
    return true;
}
bool workspace_ok(const void *p, uint64_t have, uint64_t need, const Err &fail) {
    return !need || (p && have >= need) || fail("the workspace holds %llu bytes; this call needs %llu", (unsigned long long)(p ? have : 0), (unsigned long long)need);
}
}  // namespace

extern "C" {

int qxg_tree_attention(qxg_ctx *c, const qxg_tree_attention_args *p, void *stream, int wait, char *err, uint64_t err_len) {
    const Err fail{err, err_len};
    QxaArgs A{};
    uint64_t need = 0;
    if (!tree_plan(p, A, need, fail)) return 0;
    const Arg args[] = {{p->q, "q", true, 16}, {p->k, "k", true, 16}, {p->v, "v", true, 16}, {p->kscale, "kscale", true, 4},
                        {p->vscale, "vscale", true, 4}, {p->lens, "lens", true, 4}, {p->counts, "counts", false, 4}, {p->mask, "mask", false, 4},
                        {p->out, "out", true, 16}, {p->lse, "lse", false, 4}, {p->account, "account", false, 4},
                        {p->workspace, "workspace", false, 16}};
    if (!pointers_ok(args, fail) || !workspace_ok(p->workspace, p->workspace_bytes, need, fail)) return 0;
    return on_device(c, args, (hipStream_t)stream, wait, fail, [&] { return qxa_launch(A, (hipStream_t)stream); });
}
uint64_t qxg_tree_attention_workspace(const qxg_tree_attention_args *p) {
    QxaArgs A{};
    uint64_t need = 0;
    return tree_plan(p, A, need, Err{}) ? need : 0;
}

int qxg_kv_select(qxg_ctx *c, const qxg_kv_select_args *p, void *stream, int wait, char *err, uint64_t err_len) {
    const Err fail{err, err_len};
    if (!select_ok(p, fail)) return 0;
    const Arg args[] = {{p->account, "account", true, 4}, {p->lens, "lens", true, 4}, {p->keep, "keep", true, 4}, {p->kept, "kept", true, 4}};
    if (!pointers_ok(args, fail)) return 0;
    return on_device(c, args, (hipStream_t)stream, wait, fail, [&] { return qxe_launch_select(*p, (hipStream_t)stream); });
}

int qxg_kv_compact(qxg_ctx *c, const qxg_kv_compact_args *p, void *stream, int wait, char *err, uint64_t err_len) {
    const Err fail{err, err_len};
    QxeCompact C{};
    uint64_t need = 0;
    if (!compact_plan(p, C, need, fail)) return 0;
    const Arg args[] = {{p->k, "k", true, 16}, {p->v, "v", true, 16}, {p->kscale, "kscale", true, 4}, {p->vscale, "vscale", true, 4},
                        {p->keep, "keep", true, 4}, {p->kept, "kept", true, 4}, {p->account, "account", false, 4},
                        {p->account_out, "account_out", false, 4}, {p->workspace, "workspace", false, 16}};
    if (!pointers_ok(args, fail) || !workspace_ok(p->workspace, p->workspace_bytes, need, fail)) return 0;
    return on_device(c, args, (hipStream_t)stream, wait, fail, [&] { return qxe_launch_compact(C, (hipStream_t)stream); });
}
uint64_t qxg_kv_compact_workspace(const qxg_kv_compact_args *p) {
    QxeCompact C{};
    uint64_t need = 0;
    return compact_plan(p, C, need, Err{}) ? need : 0;
}

int qxg_adjust_logits(qxg_ctx *c, const qxg_adjust_logits_args *p, void *stream, int wait, char *err, uint64_t err_len) {
    const Err fail{err, err_len};
    QxsArgs A{};
    uint64_t need = 0;
    if (!adjust_plan(p, A, need, fail)) return 0;
    const uint32_t size = type_size(p->type);
    const Arg args[] = {{p->logits, "logits", true, size}, {p->out, "out", true, size}, {p->history, "history", false, 4},
                        {p->history_lens, "history_lens", false, 4}, {p->prompt_lens, "prompt_lens", false, 4},
                        {p->penalties, "penalties", false, 4}, {p->temperature, "temperature", false, 4}, {p->bias_ids, "bias_ids", false, 4},
                        {p->bias_values, "bias_values", false, 4}, {p->mask, "mask", false, 4}, {p->mask_rows, "mask_rows", false, 4},
                        {p->top_ids, "top_ids", false, 4}, {p->top_logits, "top_logits", false, 4}, {p->lse, "lse", false, 4},
                        {p->workspace, "workspace", false, 16}};
    if (!pointers_ok(args, fail) || !workspace_ok(p->workspace, p->workspace_bytes, need, fail)) return 0;
    return on_device(c, args, (hipStream_t)stream, wait, fail, [&] { return qxs_launch(A, (hipStream_t)stream); });
}
uint64_t qxg_adjust_logits_workspace(const qxg_adjust_logits_args *p) {
    QxsArgs A{};
    uint64_t need = 0;
    return adjust_plan(p, A, need, Err{}) ? need : 0;
}

}  // extern "C"
