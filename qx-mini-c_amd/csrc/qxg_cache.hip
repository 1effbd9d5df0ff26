// Host side of the operators over a cache of 8 or 4 bits (include/qxg.h): argument checks, workspaces, launches.
// The checks of sizes come first and use no GPU.
#include "qxg_cache.h"
#include "qxg_ops_host.h"

namespace {
// What both calls ask of their sizes; rows of the cache of `row` bytes, `blocks` scales of a position.
template <typename A> bool sizes_ok(const A &a, const Err &fail) {
    if (!type_size(a.type)) return fail("unsupported value type %u", a.type);
    if (a.bits != 8 && a.bits != 4) return fail("bits must be 8 or 4");
    if (!a.batch || a.batch > 65535) return fail("batch must be between 1 and 65535");
    if (!a.tokens || a.tokens > 1u << 20) return fail("tokens must be between 1 and 2^20");
    if (a.dim != 64 && a.dim != 128) return fail("dim must be 64 or 128");
    if (!a.kv_heads || !a.heads || a.heads % a.kv_heads || a.heads > 1024) return fail("heads must be a multiple of kv_heads, at most 1024");
    if (!a.positions || a.positions > 0x7fffffffu) return fail("positions must be below 2^31");
    if ((a.batch > 1 && a.kv_batch % 16) || (a.positions > 1 && a.kv_row % 16)) return fail("the strides of the cache must be multiples of 16 bytes");
    if (a.positions > 1 && a.kv_row >> 26) return fail("the row stride of the cache must be below 2^26 bytes");
    const uint32_t blocks = a.dim / 32;
    if (a.bits == 4 && ((a.batch > 1 && a.scale_batch % blocks) || (a.positions > 1 && a.scale_row % blocks)))
        return fail("the strides of the scales must be multiples of %u bytes", blocks);
    if (a.bits == 4 && a.positions > 1 && a.scale_row >> 26) return fail("the row stride of the scales must be below 2^26 bytes");
    return true;
}
// bytes from one row to the next of an array [batch][tokens][..]
template <typename A> bool rows_aligned(const A &a, uint64_t batch, uint64_t token) {
    const uint32_t size = type_size(a.type);
    return (a.batch == 1 || batch * size % 16 == 0) && (a.tokens == 1 || token * size % 16 == 0);
}
// The rows of an array [batch][n][..] of `size` bytes an element and `row` elements a row
template <typename A> Rows rows_of(const A &a, const void *p, const char *name, uint64_t batch, uint64_t next, uint64_t n, uint64_t row, uint64_t size) {
    return {p, name, batch * size, a.batch, next * size, n, row * size};
}
template <typename A> Rows codes_of(const A &a, const void *p, const char *name) {
    return rows_of(a, p, name, a.kv_batch, a.kv_row, a.positions, (uint64_t)a.kv_heads * a.dim * a.bits / 8, 1);
}
template <typename A> Rows scales_of(const A &a, const void *p, const char *name) {
    return a.bits == 8 ? rows_of(a, p, name, a.scale_batch, 0, 1, a.positions, 4)
                       : rows_of(a, p, name, a.scale_batch, a.scale_row, a.positions, (uint64_t)a.kv_heads * a.dim / 32, 1);
}
// Refuses what is written, the first `written` arrays, where it shares memory with another of them.
template <size_t N> bool apart(const Rows (&rows)[N], size_t written, const Err &fail) {
    for (size_t i = 0; i < written; ++i)
        for (size_t j = i + 1; j < N; ++j)
            if (rows[i].p && rows[j].p && rows_meet(rows[i], rows[j])) return fail("%s and %s share memory", rows[i].name, rows[j].name);
    return true;
}

// ---- append
bool append_plan(const qxg_kv_append_args *p, QxkArgs &A, const Err &fail) {
    if (!p) return fail("invalid argument");
    const qxg_kv_append_args &a = A.a = *p;
    if (!sizes_ok(a, fail)) return false;
    if (a.kv_heads * a.dim > QXK_ROW) return fail("kv_heads * dim must be at most %u", QXK_ROW);
    if (!rows_aligned(a, a.q_batch, a.q_token) || !rows_aligned(a, a.k_batch, a.k_token) || !rows_aligned(a, a.v_batch, a.v_token) ||
        !rows_aligned(a, a.out_batch, a.out_token))
        return fail("the strides of q, k, v and q_out must be multiples of 16 bytes");
    if (rows_overlap(a.out_batch, a.batch, a.out_token, a.tokens, (uint64_t)a.heads * a.dim)) return fail("rows of q_out overlap");
    if (a.q == a.q_out && ((a.batch > 1 && a.q_batch != a.out_batch) || (a.tokens > 1 && a.q_token != a.out_token)))
        return fail("in place, the strides of q and q_out must be equal");
    if (a.q_out && (a.q_out == a.k || a.q_out == a.v)) return fail("q_out must be another array than k and v");
    if (rows_overlap(a.kv_row, a.positions, a.kv_batch, a.batch, (uint64_t)a.kv_heads * a.dim * a.bits / 8)) return fail("the rows of the cache overlap");
    if (a.bits == 8 ? a.batch > 1 && a.scale_batch < a.positions
                    : rows_overlap(a.scale_row, a.positions, a.scale_batch, a.batch, (uint64_t)a.kv_heads * a.dim / 32))
        return fail("the scales overlap");
    if (a.k_cache && a.k_cache == a.v_cache) return fail("v_cache must be another array than k_cache");
    if (a.kscale && a.kscale == a.vscale) return fail("vscale must be another array than kscale");
    if (a.rotated % 16 || a.rotated > a.dim) return fail("rotated must be a multiple of 16 up to dim");
    if (!a.rope != !a.rotated || !a.rope != !a.rope_positions) return fail("rope, rotated and rope_positions go together");
    if (a.rope_at && !a.rope) return fail("rope_at without rope");
    if ((a.q_norm || a.k_norm) && !(std::isfinite(a.eps) && a.eps >= 0.0f)) return fail("eps must be finite and not negative");
    const uint32_t units = QXK_LANES / (a.dim / 8);
    // Few tokens are shared out, a workgroup for each of their passes (one token of 32 q and 4 K and V heads of 128 in f32: 3.7 us against 5.7 in
    // one workgroup); many fill the card by themselves, and a workgroup that goes through all of a token's heads finds its angles once
    // (512 such tokens 8.0 us either way; 16384 in bf16 88 us against 118).
    const uint64_t passes = (a.heads + units - 1) / units + 1, tokens = (uint64_t)a.batch * a.tokens;
    if (tokens * passes >= 1u << 24) return fail("too many rows for one call");   // (a launch has less than 2^32 threads)
    A.parts = tokens < 512 ? (uint32_t)passes : 1;
    return true;
}

// ---- attention
// Columns of a tile and splits of its chunks.
//
// A CU does about as much with one workgroup as with several: its waves are bound by their instructions.  So what counts is how often the
// fullest CU has to go through a split's rounds (a round: 4 chunks, a wave each), 3 rounds' time to start, and of several splits
// the join, 8 rounds' time with its launch, and the states that they write and it reads, 4 MB a round's time.  The candidates fill
// the CUs 1 to 5 times, but for one that fills them once a split's rounds and the join's loads meet at sqrt(16 rounds).  us, one
// token of 32 / 8 heads of 128 in bf16: 16 sequences of 30000 positions of 8 bits within 4096 + 16 in 2, 3, 4 splits 33.5, 39.6, 36.3; 36
// of 8000 in 1 .. 5 splits 191, 165, 130, 129, 134; 1 of 30000 in 30 or 59 splits 19.7, 23.4; 24 of 3000 in 1, 2, 3 splits 36.6, 43.8,
// 43.5; 3 prompts of 1024 within 2000 + 40 in 1, 2, 3 splits 216, 271, 282.
// Sequences of a batch are of unlike lengths, taken as 13/16 of the longest on average: with small splits (12, 6 or 3 rounds) the CUs are
// done at about the same time, each with its share of the work, and workgroups start while others work.  16 sequences of 10000 to 32000
// positions of 4 bits in 2, 24, 48 splits 128, 101, 100 us, all of 32000 in 2, 23, 42 145, 142, 149; 36 of 2700 to 8000 of 8 bits in 4, 12
// splits 100, 87.  (Within a window the lists of sequences longer than it are of one length, and nothing is less there: their calls, and batches of
// equal lengths, may get more splits than they need.)
// Short lists stay whole: a token of 32 / 4 heads in f32 over 1024 + 4 positions takes 15 us on the card and 10 with the join, whose
// launch costs a program 3 to 5.
//
// With 32 columns a workgroup shares the codes' loads and conversion, and a round takes 1.4 times as long.  (f32 has registers for it with
// 64 dims: 512 tokens of 32 / 8 heads over 8000 positions of 8 bits 147 us with 16 and 120 with 32, of 4 bits 125 and 105; with 128
// dims it spills: of 32 / 4 heads 239 and 346, 191 and 189.)  us with 16 and 32, 32 / 4 heads of 128 in bf16: 512
// tokens over 8000 positions of 8 bits 223, 159, of 4 bits 154, 124; 8 x 5 over 6000 of 8 bits 37, 28; 256 over 600 17.8, 16.0; 32
// over 600 9.8, 11.5; one token each of 16 sequences of 32000 of 4 bits (4 columns) 141, 153.
// With 128, whose waves share them in LDS, more work is needed to pay: of 8 bits and a BF16 q, 512 tokens over 8000 positions
// (work 256000) 136 where 32 columns take 141, 2 x 4096 within 2048 + 4 (1600000) 271 and 313.  Two of its workgroups go on a CU.
void attention_splits(QxwArgs &A, uint64_t columns) {
    const qxg_cache_attention_args &a = A.a;
    // the chunks of a tile, at most
    const uint64_t positions = std::min<uint64_t>((uint64_t)a.max_len + a.tokens, a.positions), most = 128 / A.group + 2;   // tokens of a tile
    uint64_t chunks = (positions + 31) / 32;
    if (a.window) chunks = std::min(chunks, (a.window + most + 62) / 32 + ((uint64_t)a.sinks + 31) / 32);
    const uint64_t heads = (uint64_t)a.batch * a.kv_heads, states = columns * heads * a.dim * 8 >> 18;
    uint64_t least = ~0ull;
    auto consider = [&](uint32_t wide, uint64_t places, uint64_t round, uint64_t time) {   // the best splits with tiles of `wide` columns
        const uint64_t tiles = (columns + wide - 1) / wide, wgs = heads * tiles, rounds = (chunks + round - 1) / round;
        auto with = [&](uint64_t splits) {
            const uint64_t each = (rounds + splits - 1) / splits;   // (in sixteenths of a round of 16 columns)
            uint64_t busy = (wgs * splits + places - 1) / places * (each + 3);
            if (a.batch > 1) busy = std::min(busy, wgs * rounds * 13 / 16 / places + each + 3);
            const uint64_t cost = busy * time + (splits > 1 ? 128 + splits + splits * states : 0);
            if (cost >= least) return;
            least = cost;
            A.columns = wide;
            A.tiles = (uint32_t)tiles;
            A.split_chunks = (uint32_t)(each * round);
            A.splits = (uint32_t)((chunks + A.split_chunks - 1) / A.split_chunks);
        };
        with(1);
        for (uint64_t fill = 1; fill <= 5; ++fill) {
            uint64_t splits = std::min(places * fill / wgs, rounds);
            if (fill == 1) splits = std::min(splits, (uint64_t)std::sqrt(16.0 * rounds));
            if (splits > 1) with(splits);
        }
        for (const uint64_t each : {12, 6, 3})
            if (a.batch > 1 && rounds > each) with((rounds + each - 1) / each);
    };
    const uint64_t work = heads * ((columns + 15) / 16) * chunks;   // chunks of all tiles of 16 columns
    if (a.type == QXG_TYPE_BF16 && a.bits == 8 && columns >= 128 && work > 400000) return consider(128, 512, 1, 16);
    consider(16, 256, 4, 16);
    if (columns > 16 && (a.type != QXG_TYPE_F32 || a.dim == 64)) consider(32, 256, 4, 22);
}
bool attention_plan(const qxg_cache_attention_args *p, QxwArgs &A, uint64_t &bytes, const Err &fail) {
    if (!p) return fail("invalid argument");
    const qxg_cache_attention_args &a = A.a = *p;
    if (!sizes_ok(a, fail)) return false;
    if (a.max_len > 0x7fffffffu) return fail("max_len must be below 2^31");
    if (!rows_aligned(a, a.q_batch, a.q_token) || !rows_aligned(a, a.out_batch, a.out_token))
        return fail("the strides of q and out must be multiples of 16 bytes");
    if (rows_overlap(a.out_batch, a.batch, a.out_token, a.tokens, (uint64_t)a.heads * a.dim)) return fail("rows of out overlap");
    if (a.out && a.out == a.q) return fail("out must be another array than q");
    if (!std::isfinite(a.scale) || !(a.scale > 0.0f)) return fail("scale must be positive and finite");
    A.scale2 = (float)((double)a.scale * 1.4426950408889634);
    if (!std::isfinite(A.scale2)) return fail("scale * log2(e) must be finite");
    A.group = a.heads / a.kv_heads;
    const uint64_t columns = (uint64_t)a.tokens * A.group;
    attention_splits(A, columns);
    // (workgroups are launched in eights of a kv head's)
    if ((uint64_t)a.kv_heads * (((uint64_t)A.tiles * A.splits * a.batch + 7) / 8 * 8) >= 1u << 24 ||
        (uint64_t)a.batch * a.tokens * a.heads >= 1u << 26) return fail("too many rows for one call");   // (a launch has less than 2^32 threads)
    const uint64_t states = A.splits == 1 ? 0 : (uint64_t)A.splits * a.batch * a.tokens * a.heads;
    const uint64_t part = up16(states * a.dim * 4), md = up16(states * 8);
    A.part = (float *)a.workspace;
    A.md = (float2 *)((uint8_t *)a.workspace + part);
    bytes = part + md;
    return true;
}
}  // namespace

extern "C" {

int qxg_kv_append(qxg_ctx *c, const qxg_kv_append_args *p, void *stream, int wait, char *err, uint64_t err_len) {
    const Err fail{err, err_len};
    QxkArgs A{};
    if (!append_plan(p, A, fail)) return 0;
    const uint32_t scale = p->bits == 8 ? 4 : 1;
    const Arg args[] = {{p->q, "q", true, 16}, {p->k, "k", true, 16}, {p->v, "v", true, 16}, {p->q_out, "q_out", true, 16},
                        {p->k_cache, "k_cache", true, 16}, {p->v_cache, "v_cache", true, 16}, {p->kscale, "kscale", true, scale},
                        {p->vscale, "vscale", true, scale}, {p->lens, "lens", true, 4}, {p->counts, "counts", false, 4},
                        {p->q_norm, "q_norm", false, 4}, {p->k_norm, "k_norm", false, 4}, {p->rope, "rope", false, 4},
                        {p->rope_at, "rope_at", false, 4}};
    if (!pointers_ok(args, fail)) return 0;
    const uint32_t size = type_size(p->type);
    const uint64_t q_row = (uint64_t)p->heads * p->dim, row = (uint64_t)p->kv_heads * p->dim;
    const Rows q_out = rows_of(*p, p->q_out, "q_out", p->out_batch, p->out_token, p->tokens, q_row, size);
    const Rows rows[] = {q_out, codes_of(*p, p->k_cache, "k_cache"), codes_of(*p, p->v_cache, "v_cache"), scales_of(*p, p->kscale, "kscale"),
                         scales_of(*p, p->vscale, "vscale"), rows_of(*p, p->k, "k", p->k_batch, p->k_token, p->tokens, row, size),
                         rows_of(*p, p->v, "v", p->v_batch, p->v_token, p->tokens, row, size)};
    const Rows turned[] = {q_out, rows_of(*p, p->q == p->q_out ? nullptr : p->q, "q", p->q_batch, p->q_token, p->tokens, q_row, size)};
    if (!apart(rows, 5, fail) || !apart(turned, 1, fail)) return 0;
    return on_device(c, args, (hipStream_t)stream, wait, fail, [&] { return qxk_launch_append(A, (hipStream_t)stream); });
}

int qxg_cache_attention(qxg_ctx *c, const qxg_cache_attention_args *p, void *stream, int wait, char *err, uint64_t err_len) {
    const Err fail{err, err_len};
    QxwArgs A{};
    uint64_t need = 0;
    if (!attention_plan(p, A, need, fail)) return 0;
    const uint32_t scale = p->bits == 8 ? 4 : p->dim / 32;
    const Arg args[] = {{p->q, "q", true, 16}, {p->k, "k", true, 16}, {p->v, "v", true, 16}, {p->kscale, "kscale", true, scale},
                        {p->vscale, "vscale", true, scale}, {p->lens, "lens", true, 4}, {p->counts, "counts", false, 4},
                        {p->out, "out", true, 16}, {p->lse, "lse", false, 4}, {p->workspace, "workspace", false, 16}};
    if (!pointers_ok(args, fail) || !workspace_ok(p->workspace, p->workspace_bytes, need, fail)) return 0;
    const uint32_t size = type_size(p->type);
    const uint64_t row = (uint64_t)p->heads * p->dim;
    const Rows out = rows_of(*p, p->out, "out", p->out_batch, p->out_token, p->tokens, row, size);
    const Rows rows[] = {out, {p->lse, "lse", 0, 1, 0, 1, (uint64_t)p->batch * p->tokens * p->heads * 4}, codes_of(*p, p->k, "k"), codes_of(*p, p->v, "v"),
                         scales_of(*p, p->kscale, "kscale"), scales_of(*p, p->vscale, "vscale")};
    const Rows answers[] = {out, rows_of(*p, p->q, "q", p->q_batch, p->q_token, p->tokens, row, size)};
    if (!apart(rows, 2, fail) || !apart(answers, 1, fail)) return 0;
    return on_device(c, args, (hipStream_t)stream, wait, fail, [&] { return qxw_launch(A, (hipStream_t)stream); });
}
// (The plan goes by the value type as well; a program that asks before it has q's gets what all of them need.)
uint64_t qxg_cache_attention_workspace(const qxg_cache_attention_args *p) {
    QxwArgs A{};
    uint64_t most = 0;
    if (!attention_plan(p, A, most, Err{})) return 0;
    for (uint32_t type : {QXG_TYPE_F32, QXG_TYPE_F16, QXG_TYPE_BF16}) {
        qxg_cache_attention_args a = *p;
        a.type = type;
        uint64_t need = 0;
        if (attention_plan(&a, A, need, Err{})) most = std::max(most, need);
    }
    return most;
}

}  // extern "C"
