/* qxg — C ABI to the MI355X (gfx950) decode path.
 *
 * The reference has no process or device boundary: its state loop calls static
 * C functions over mmap'd weight spans (reference src/qx_format.c:5970-6733).  This
 * ABI is the seam that replaces those calls.  Each entry point below names the
 * reference function(s) it stands in for.  Conventions follow the reference C API
 * (reference include/qx_format.h:104-172): return 1 on success and 0 on failure,
 * with a message written into (err, err_len).  Pointers are host pointers, sizes
 * are plain integers, and calls are synchronous unless stated otherwise.  Each
 * context owns one HIP stream and its device buffers.  A context is not
 * thread-safe (the reference is single-threaded, src/qx_format.c:5984-5995).
 *
 * Fixed model geometry (reference --final-head manifest check,
 * src/qx_format.c:6120-6124): hidden 2048, 32 q heads / 4 kv heads of 128,
 * moe_intermediate 768, top-8 experts; vocab, experts (8..128) and layer count
 * come from the uploaded tensors.
 */
#ifndef QXG_H
#define QXG_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct qxg_ctx qxg_ctx;

/* Creates a context on HIP device `device`: stream, codebooks, RoPE table.
 * Stands in for the per-call setup of the reference state loop
 * (src/qx_format.c:6044-6160). */
int qxg_open(int device, qxg_ctx **out, char *err, uint64_t err_len);
void qxg_close(qxg_ctx *ctx);

/* Uploads one tensor of the QXF1 file (bytes = the tensor's mmap span) and repacks
 * quantized blocks on the device.  Replaces the per-call weight reads
 * qx_read_raw_span / qx_acquire_span (src/qx_format.c:1757-1773, 858-893).
 * ggml_type: 0 F32, 12 Q4_K, 13 Q5_K, 14 Q6_K, 17 IQ2_XS, 18 IQ3_XXS, 21 IQ3_S,
 * 22 IQ2_S, 23 IQ4_XS. */
int qxg_upload_tensor(qxg_ctx *ctx, const char *name, uint32_t ggml_type, const uint64_t dims[4],
                      const void *host_bytes, uint64_t nbytes, char *err, uint64_t err_len);

/* Resolves the uploaded tensors into layers [0, layers), checks every shape and
 * type (the checks of src/qx_format.c:5216-5235, 3610-3629), and sizes work
 * buffers.  need_head / need_embedding select whether output.* / token_embd.* must
 * be present.  Per layer: attn_q/k/v/output IQ4_XS or Q5_K; gate/up experts IQ2_XS
 * or IQ2_S (both the same); down experts IQ3_XXS, IQ4_XS or IQ3_S.  A model using any
 * format beyond IQ4_XS / IQ2_XS / IQ3_XXS decodes one kernel per phase; its prefill
 * (qxg_prefill / qxg_prefill_layer) stays batched on the matrix cores. */
int qxg_bind_model(qxg_ctx *ctx, uint32_t layers, int need_embedding, int need_head, char *err, uint64_t err_len);

/* Persistent INT8 KV cache [layers][ctx_tokens][512] for K and V plus one f32 scale
 * per (layer, position).  Same layout as the reference state loop
 * (src/qx_format.c:6138-6160, 6343-6400).  kv_format must be 1 (int8). */
int qxg_kv_create(qxg_ctx *ctx, uint32_t layers, uint32_t ctx_tokens, uint32_t kv_format, char *err, uint64_t err_len);
/* Copies rows [pos0, pos0+count) of one layer into / out of the device cache.
 * k, v: count*512 int8; kscale, vscale: count floats.  Used for QXKVSNP1
 * import/export (src/qx_format.c:5860-5968) and for seeded long-context tests. */
int qxg_kv_write(qxg_ctx *ctx, uint32_t layer, uint32_t pos0, uint32_t count, const int8_t *k, const int8_t *v,
                 const float *kscale, const float *vscale, char *err, uint64_t err_len);
int qxg_kv_read(qxg_ctx *ctx, uint32_t layer, uint32_t pos0, uint32_t count, int8_t *k, int8_t *v,
                float *kscale, float *vscale, char *err, uint64_t err_len);

/* QXKVSNP1 snapshots of the INT8 KV cache (the reference's accumulated-KV files,
 * qx_write_accumulated_kv_snapshot / qx_read_accumulated_kv_snapshot,
 * src/qx_format.c:5860-5968, used by --kv-snapshot-out / --kv-snapshot-in,
 * src/qx_format.c:6165-6177, 6629-6633).  File: 48-byte header ("QXKVSNP1", version 2,
 * layers, positions, ctx_tokens, kv_heads 4, head_dim 128, format 1 = int8, row bytes
 * 512, next_token, seed), per layer and position the K row, V row, K scale and V scale,
 * then the SHA-256 of all preceding bytes.  ctx_tokens must equal the cache's context.
 * qxg_kv_export writes layers [0, layers) x positions [0, positions) of the device cache;
 * qxg_kv_import checks the header (layers, ctx_tokens, kv geometry, int8, seed) and the
 * digest before writing positions [0, *positions_out) of every layer to the device. */
int qxg_kv_export(qxg_ctx *ctx, const char *path, uint32_t layers, uint32_t positions, uint32_t ctx_tokens,
                  uint32_t next_token, uint32_t seed, char *err, uint64_t err_len);
int qxg_kv_import(qxg_ctx *ctx, const char *path, uint32_t layers, uint32_t ctx_tokens, uint32_t seed,
                  uint32_t *positions_out, uint32_t *next_token_out, char *err, uint64_t err_len);
/* The same file format over host caches laid out as the reference's
 * ([layers][ctx_tokens][512] int8 rows, [layers*ctx_tokens] f32 scales); no device use. */
int qxg_kvsnap_write(const char *path, uint32_t layers, uint32_t positions, uint32_t ctx_tokens, uint32_t next_token,
                     uint32_t seed, const int8_t *k, const int8_t *v, const float *kscale, const float *vscale,
                     char *err, uint64_t err_len);
int qxg_kvsnap_read(const char *path, uint32_t layers, uint32_t ctx_tokens, uint32_t seed, int8_t *k, int8_t *v,
                    float *kscale, float *vscale, uint32_t *positions_out, uint32_t *next_token_out, char *err,
                    uint64_t err_len);

/* One full token at `position`: Q4_K embedding, every bound layer (attention with
 * INT8 KV append, then MoE), and if run_head the output RMSNorm, Q6_K head and
 * top_n (<= 32) ids by (logit desc, index asc).  The loop body of
 * qx_dump_prompt_state_loop_probe_summary (src/qx_format.c:6250-6627).
 * Any output pointer may be NULL.  layer_out: layers*2048 floats (the per-layer
 * "output" residual dumps, src/qx_format.c:6439).  Returns 0 on a non-finite
 * logit (src/qx_format.c:3715). */
int qxg_decode_token(qxg_ctx *ctx, uint32_t token, uint32_t position, int run_head,
                     float *residual_out, float *layer_out, float *logits, uint32_t top_n,
                     uint32_t *top_ids, double *top_logits, char *err, uint64_t err_len);

/* Greedy loop on the device: feeds prompt[0..n_prompt) at positions pos0.., then
 * generates n_gen tokens by argmax with the next token fed back on the device
 * (no host round trip per step).  tokens_out receives the n_gen generated ids.
 * Matches the step/phase sequence of src/qx_format.c:6250-6627 with temperature 0
 * (qx_sample_from_top, src/qx_format.c:3045-3057).  If elapsed_ms is non-NULL it
 * receives the device time of the whole loop (HIP events on the context stream). */
int qxg_generate(qxg_ctx *ctx, const uint32_t *prompt, uint32_t n_prompt, uint32_t n_gen, uint32_t pos0,
                 uint32_t *tokens_out, float *elapsed_ms, char *err, uint64_t err_len);

/* 1 when qxg_generate / qxg_decode_token run the persistent decode on this context (the
 * layer path set to 1, the f32 activation mode, every bound format one it decodes), else 0.
 * No reference counterpart. */
int qxg_persistent_path(const qxg_ctx *ctx);

/* qxg_generate with every step's records, for the reference's prompt state loop
 * (qx_dump_prompt_state_loop_probe_summary, src/qx_format.c:6250-6627, which prints them per
 * step and layer): one persistent launch over the S = n_prompt + n_gen - 1 steps, then the
 * top_n (<= 32) tokens of each head step ranked on the device and everything copied back in
 * bulk.  Persistent path only (qxg_persistent_path); the records live in device buffers
 * allocated for the call.  Outputs, any of which may be NULL, with L = the bound layers:
 *   tokens_out[S + 1]      the prompt, then each generated id at [step + 1];
 *   layer_out[S][L][2048]  each layer's output residual;
 *   attn_out, moe_out      [S][L][2048] each layer's attention output and MoE sum (before
 *                          their residual adds, as qxg_decode_halves);
 *   ids_out, weights_out   [S][L][8] the routing (as qxg_decode_routing);
 *   head_sums_out[S][L][32] each q head's sum of normalised attention weights;
 *   norm_out[S][2048], logits_out[S][vocab]   each head step's output-RMSNorm vector and
 *                          logits (steps before the last prompt token run no head: zeros);
 *   top_ids, top_logits    [S][top_n] each head step's best tokens, highest first (zeros
 *                          before the last prompt token);
 *   step_ms[S + 1]         the device clock at each step's start and at the end, in ms from
 *                          the first step's start;
 *   elapsed_ms             the device time of the launch (HIP events).
 * Returns 0 on a non-finite final logit (src/qx_format.c:3715) or a bad argument. */
int qxg_generate_recorded(qxg_ctx *ctx, const uint32_t *prompt, uint32_t n_prompt, uint32_t n_gen, uint32_t pos0,
                          uint32_t top_n, uint32_t *tokens_out, float *layer_out, float *attn_out, float *moe_out,
                          uint32_t *ids_out, double *weights_out, double *head_sums_out, float *norm_out, float *logits_out,
                          uint32_t *top_ids, double *top_logits, double *step_ms, float *elapsed_ms, char *err,
                          uint64_t err_len);

/* ---- same-input replay seams (host pointers in and out, synchronous) ---- */

/* Q4_K embedding row of `token` as 2048 floats, no norm on the full-MoE path:
 * replaces qx_fill_residual_vector_from_embedding (src/qx_format.c:3759-3793). */
int qxg_embed_token(qxg_ctx *ctx, uint32_t token, float *x_out, char *err, uint64_t err_len);

/* Decodes `nblocks` consecutive 256-value blocks of one type to f32, on the
 * device, from the repacked layout, with the reference's op order (bit-exact with
 * qx_decode_supported_block, src/qx_format.c:2206-2217). */
int qxg_dequant_blocks(qxg_ctx *ctx, uint32_t ggml_type, const void *raw, uint64_t nblocks, float *out,
                       char *err, uint64_t err_len);

/* INT8 KV quantization of one row of n <= 4096 f32 values on the device, with the same
 * device functions every kernel that appends a KV row uses: scale = max|x| / 127 over the
 * finite values (1 if zero), codes = lrintf(x / scale) clamped to +-127, non-finite -> 0.
 * Replaces qx_quantize_int8_vector (src/qx_format.c:4449-4463) as a same-input seam. */
int qxg_int8_quantize(qxg_ctx *ctx, const float *x, uint32_t n, int8_t *codes, float *scale, char *err, uint64_t err_len);

/* No counterpart in the reference: for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).
 * qxg_dequant_blocks with the raw blocks and the f32 output in device memory the caller
 * owns (raw_dev: nblocks blocks of the type's size; out_dev: nblocks * 256 floats) and
 * the repacked block planes in a static device workspace (one per GPU, held until the
 * process ends) instead of per-call allocations.  At most QXG_STATIC_MAX_BLOCKS blocks
 * per call; more fail with an error.  Allocates nothing; returns when the output is
 * written.  Every call on one GPU shares its workspace: calls that overlap on one GPU
 * (from several threads or contexts) are serialised by a per-GPU lock held from the
 * repack until the call has finished. */
#define QXG_STATIC_MAX_BLOCKS 4096u
int qxg_dequant_blocks_static(qxg_ctx *ctx, uint32_t ggml_type, const void *raw_dev, uint64_t nblocks, float *out_dev,
                              char *err, uint64_t err_len);

/* Attention block of `layer` for one token at `position` on residual x_in:
 * attn RMSNorm, K/V projections, k norm + RoPE, INT8 append at [layer][position],
 * Q projection/norm/RoPE, GQA softmax over 0..position, O projection.
 * attn_out = O*ctx (without the residual).  Replaces the attention half of the
 * layer loop (src/qx_format.c:6282-6423 and qx_rope_gqa_attention_partial,
 * 5051-5196).  kqv_out: 4096 floats, vcur_out: 512 floats (dump phases
 * "kqv-out" and "v-cur"). */
int qxg_attention_layer(qxg_ctx *ctx, uint32_t layer, uint32_t position, const float *x_in, float *attn_out,
                        float *kqv_out, float *vcur_out, char *err, uint64_t err_len);
/* qxg_attention_layer plus, when head_weight_sums is non-NULL, each q head's sum of its
 * normalised softmax weights (32 doubles): the reference reports their mean, minimum and
 * maximum as softmax_sum, softmax_sum_min, softmax_sum_max (src/qx_format.c:5154-5189,
 * printed at 6516-6523). */
int qxg_attention_layer_ex(qxg_ctx *ctx, uint32_t layer, uint32_t position, const float *x_in, float *attn_out,
                           float *kqv_out, float *vcur_out, double *head_weight_sums, char *err, uint64_t err_len);

/* The attention stage probe's computation (qx_dump_attention_stage_probe_summary,
 * src/qx_format.c:5478-5586): a single token attending to itself.  attn RMSNorm (norm_out,
 * 2048), V projection (vcur_out, 512), each q head's context = its kv head's V row, after
 * an fp16 round trip if f16_kv (kqv_out, 4096), O projection (attn_out, 2048), ffn_inp_out =
 * x_in + attn_out.  Fails with the reference's message on a non-finite output.  Output
 * pointers may be NULL. */
int qxg_attention_stage(qxg_ctx *ctx, uint32_t layer, int f16_kv, const float *x_in, float *norm_out,
                        float *vcur_out, float *kqv_out, float *attn_out, float *ffn_inp_out, char *err,
                        uint64_t err_len);

/* The MoE stage probe's computation (qx_dump_moe_stage_probe_summary, src/qx_format.c:
 * 5588-5725) on ffn input x_in: f32 router logits, f32 softmax probabilities, 8 picks by
 * probability, f32 renormalised weights, then per pick the gate, up, SwiGLU, down and
 * weighted down rows.  out receives QXG_MOE_STAGE_FLOATS(experts) floats, in order:
 * ffn_norm[2048], logits[E], probs[E], topk[8] (ids as floats), weights[8],
 * weights_sum[1], weights_norm[8], gate[8][768], up[8][768], swiglu[8][768],
 * down[8][2048], weighted[8][2048]; ids (may be NULL) the picks. */
#define QXG_MOE_STAGE_FLOATS(E) (2048u + 2u * (E) + 25u + 3u * 8u * 768u + 2u * 8u * 2048u)
int qxg_moe_stage(qxg_ctx *ctx, uint32_t layer, const float *x_in, float *out, uint32_t ids[8], char *err,
                  uint64_t err_len);

/* MoE block of `layer` on ffn_inp: replaces qx_apply_real_moe_layer
 * (src/qx_format.c:5198-5317).  layer_out = ffn_inp + moe; moe_out (may be NULL)
 * = the "ffn-moe-out" dump; ids/weights = selected experts in rank order. */
int qxg_moe_layer(qxg_ctx *ctx, uint32_t layer, const float *ffn_inp, float *layer_out, float *moe_out,
                  uint32_t ids[8], double weights[8], char *err, uint64_t err_len);

/* Output head on a residual: replaces qx_compute_real_final_head
 * (src/qx_format.c:3554-3738) as used by qx_dump_final_head_probe_summary
 * (src/qx_format.c:5369-5411).  norm_out: 2048 floats, logits: vocab floats. */
int qxg_final_head(qxg_ctx *ctx, const float *residual, float *norm_out, float *logits, uint32_t top_n,
                   uint32_t *top_ids, double *top_logits, char *err, uint64_t err_len);

/* Batched prefill: tokens[0..n) at positions position0.. through every bound layer
 * together (projection and expert GEMMs on the matrix cores), INT8 KV appended at
 * [layer][position0+i]; then, if run_head, the output RMSNorm, Q6_K head and top_n on
 * the last token.  Stands in for the reference's prompt steps, which run one token at a
 * time through the decode step with the head only on the last prompt token
 * (src/qx_format.c:6250-6547, sampling_step at 6253).  Chunks of 512 tokens run in
 * order; every per-layer format of the real checkpoint (IQ4_XS / Q5_K attention,
 * IQ2_XS / IQ2_S gate/up, IQ3_XXS / IQ3_S / IQ4_XS down) runs batched.  The q8_k_compat
 * mode takes those token steps on the device instead: one persistent launch over the
 * prompt where the persistent path serves the model and residual_out is NULL, else the
 * one-kernel-per-phase decode kernels one token at a time; either way the result equals
 * qxg_decode_token over the prompt on the same layer path.  So does an f32 prompt where the
 * GPU's memory does not hold the batched path's layout of the attention matrices (21 to 24 MB
 * a layer), which the first batched call after a bind makes.  Equal calls give equal bits.
 * residual_out (may be NULL): n*2048 floats, each token's residual after the
 * last layer.  logits / top_* as in qxg_decode_token.  elapsed_ms: device time of the
 * whole call (HIP events on the context stream). */
int qxg_prefill(qxg_ctx *ctx, const uint32_t *tokens, uint32_t n, uint32_t position0, int run_head,
                float *residual_out, float *logits, uint32_t top_n, uint32_t *top_ids, double *top_logits,
                float *elapsed_ms, char *err, uint64_t err_len);

/* Same-input replay of one prefill layer: n <= 512 residual rows x_in (n*2048) at
 * positions position0.. (KV rows appended as in qxg_prefill).  ffn_inp_out = x_in +
 * attention (the MoE input, dump phase "ffn-inp"), moe_out = the weighted expert sum
 * ("ffn-moe-out"), x_out = ffn_inp + moe; any output may be NULL.  The reference's
 * counterpart is n successive layer steps (src/qx_format.c:6282-6423, 5198-5317). */
int qxg_prefill_layer(qxg_ctx *ctx, uint32_t layer, uint32_t n, uint32_t position0, const float *x_in,
                      float *ffn_inp_out, float *moe_out, float *x_out, char *err, uint64_t err_len);

/* How the layers of a token are launched (no reference counterpart: the reference
 * runs one thread on the CPU).  1 (the default): one cooperative persistent kernel per
 * qxg_generate / qxg_decode_token call runs every step (embedding, all layers, head,
 * argmax), one workgroup per CU, its phases handed over through epoch-tagged device
 * words; 0: one kernel per phase, six per layer, each step replayed from a recorded
 * graph.  Both give the same results to the stated tolerance.  Drops the recorded decode
 * graph.  A model bound with formats beyond IQ4_XS / IQ2_XS / IQ3_XXS runs path 0
 * whatever is set here; the q8_k_compat mode runs either path (the persistent kernel has
 * a Q8_K instantiation). */
int qxg_set_layer_path(qxg_ctx *ctx, int persistent);

/* Activation format of the projections, experts and head: 0 "f32" (default), 1
 * "q8_k_compat" -- the reference's activation_format argument of the state loop and
 * stage probes (src/qx_format.c:5970-5972, 4217-4218, 5286-5288, 3565).  In
 * q8_k_compat the matvec inputs are quantized to Q8_K blocks (256 values, one f32
 * scale) and each weight type is dotted in integers; a non-finite activation or
 * expert row makes the call fail with the reference's message.  Decode follows
 * qxg_set_layer_path (the persistent kernel's Q8_K instantiation by default);
 * qxg_prefill runs token by token through the one-kernel-per-phase decode kernels in
 * this mode.  Drops the recorded decode graph. */
int qxg_set_activation(qxg_ctx *ctx, uint32_t activation_format, char *err, uint64_t err_len);

/* Routing of every layer in the last step run by qxg_decode_token (or the last step of
 * qxg_generate): ids[l*8 + r] the expert of rank r in layer l, weights[l*8 + r] its
 * renormalised weight, as qx_apply_real_moe_layer selects them (src/qx_format.c:5265-5290).
 * The reference keeps no such record; this is the readback the router parity tests use. */
int qxg_decode_routing(qxg_ctx *ctx, uint32_t layers, uint32_t *ids, double *weights, char *err, uint64_t err_len);

/* The two halves of every layer in the last step run by qxg_decode_token, before their
 * residual adds: attn_out[l*2048 ..] the attention output (the O projection of the
 * context; the reference's "attn-out" dump phase, src/qx_format.c:6420-6423) and
 * moe_out[l*2048 ..] the weighted expert sum ("ffn-moe-out", :5296-5309).  Either may be
 * NULL.  Same-input replay of each half on its own: the residual stream can be many orders
 * of magnitude larger than a half, so a layer output alone would hide an error in it. */
int qxg_decode_halves(qxg_ctx *ctx, uint32_t layers, float *attn_out, float *moe_out, char *err, uint64_t err_len);

/* Persistent decode only (no reference counterpart): from n = position + 1 >=
 * min_positions on, stage A attends by (kv head, 64-position chunk) over every workgroup
 * and merges the chunks' partial softmax results; below it the 32 q-head workgroups walk
 * the cache themselves.  Default 577 (measured crossover of the two); 1 chunks every position,
 * 4097 never. */
int qxg_set_attention_chunks(qxg_ctx *ctx, uint32_t min_positions);

/* The output-RMSNorm vector (2048 floats) of the last head step run by qxg_decode_token:
 * the normalised final residual the head consumed (src/qx_format.c:3655, the state loop's
 * final_norm_raw). */
int qxg_decode_final_norm(qxg_ctx *ctx, float *norm_out, char *err, uint64_t err_len);

/* Each q head's sum of its normalised attention weights in every layer of the last step run
 * by qxg_decode_token: sums[l*32 + h].  The state loop's per-layer softmax_sum fields
 * (src/qx_format.c:5183-5190, printed at :6494-6529); the reference keeps no other record. */
int qxg_decode_head_sums(qxg_ctx *ctx, uint32_t layers, double *sums, char *err, uint64_t err_len);

/* The cache rows of one position in layers [0, layers): k, v layers*512 int8 and the
 * scales, one strided copy each (qxg_kv_read per layer, batched for the state loop's
 * per-step K/V checksums, src/qx_format.c:6494-6529). */
int qxg_kv_read_position(qxg_ctx *ctx, uint32_t position, uint32_t layers, int8_t *k, int8_t *v, float *ks, float *vs,
                         char *err, uint64_t err_len);

/* Same-input seam of the Q8_K quantizer the q8_k_compat kernels use: n values (a
 * multiple of 256, at most 4096) -> n/256 blocks of 292 bytes in ggml's block_q8_K
 * layout {f32 d, int8 qs[256], int16 bsums[16]}.  Replaces qx_quantize_q8_k as exposed
 * by the reference's q8-k-activation-probe (src/qx_format.c:3891-3927, 4304-4345);
 * fails, like it, on a non-finite value or a bad length. */
int qxg_q8k_quantize(qxg_ctx *ctx, const float *x, uint32_t n, void *blocks_out, char *err, uint64_t err_len);

/* ---- operators on device memory (no reference counterpart) ----
 *
 * For programs that keep their activations and caches on the GPU: a drafted tree of tokens
 * attends over an INT8 cache of the context's format, the cache is kept within a budget, and
 * logits are adjusted and picked from.  Every pointer in the argument structs is device memory
 * of the context's GPU, owned by the caller and allocated by the HIP runtime that this library
 * uses; other pointers are refused.  A call queues its kernels on `stream` (a hipStream_t of
 * that GPU as void *; NULL: HIP's default stream) and returns; with wait != 0 it returns when
 * they have finished.  Work of other streams on the same memory is the caller's to order.  A
 * call allocates nothing and copies nothing, so it can be captured into a graph.  Its workspace
 * is the caller's: calls that may run at the same time (other streams, graphs) need one each.
 * The qxg_*_workspace functions return the bytes that a call with these arguments needs (0 if
 * it would be refused).  Indexes, lengths and counts in device memory are 32-bit unsigned and
 * clamped to the arrays' sizes by the kernels.  Calls do not touch the context's own buffers
 * and stream, and may be made from several threads on one context.
 *
 * Value types are GGML types: 0 F32, 1 F16, 30 BF16. */
#define QXG_TYPE_F32 0u
#define QXG_TYPE_F16 1u
#define QXG_TYPE_BF16 30u

/* Attention of a tree of drafted tokens (nodes) over an INT8 cache.  Sequence b has
 * lens[b] cached positions; its count = counts[b] nodes' K and V rows stand behind them at
 * positions lens[b] .. lens[b] + count - 1.  Node i sees every cached position and the nodes
 * that its mask row names (bit j % 32 of word j / 32: node j; a node that is to see itself has
 * its own bit set).  For q head h, kv head g = h / (heads / kv_heads):
 *     s[p] = scale * kscale[p] * sum_d q[i][h][d] k[p][g][d]        over the visible positions
 *     out[i][h] = sum_p softmax(s)[p] vscale[p] v[p][g]             (f32 sums, rounded once)
 *     lse[i][h] = log sum_p exp(s[p])
 * A row that sees nothing has out 0 and lse -inf.  What stands in positions that a row does not see
 * (scales that are infinite or NaN among them) does not reach it.  Rows of nodes at and behind
 * count are left as they were.  With account, each position's weight is added to it:
 *     account[p] = decay * account[p] + sum over nodes and heads of softmax(s)[p]
 * for p < lens[b] + count, in a fixed order (equal calls give equal bits).  The nodes' positions are among them: their
 * entries are the caller's to clear before a token takes the place of another, and to move with a path's rows that it keeps
 * (qxg_kv_compact's account_out).
 * An F32 q is multiplied as two halves of 11 bits each (F16 and BF16: as it is), the weights too (errors as of
 * f32 products, where vscale is 2^-99 or more).  nodes = 1 without a mask is ordinary decoding.  Rows of out that overlap, and accounts that do, are refused. */
typedef struct qxg_tree_attention_args {
    const void *q;            /* [batch][nodes][heads][dim] of `type`, 16-byte aligned */
    const int8_t *k, *v;      /* [batch][positions][kv_heads][dim], 16-byte aligned */
    const float *kscale, *vscale;   /* [batch][positions] */
    const uint32_t *lens;     /* [batch] cached positions; count + lens[b] is clamped to positions */
    const uint32_t *counts;   /* [batch] nodes in use, or NULL: all */
    const uint32_t *mask;     /* [batch][nodes][(nodes + 31) / 32], or NULL: node i sees nodes 0 .. i */
    void *out;                /* as q, 16-byte aligned; not overlapping q */
    float *lse;               /* [batch][nodes][heads], or NULL */
    float *account;           /* [batch][positions], or NULL */
    void *workspace;          /* 16-byte aligned */
    uint64_t workspace_bytes;
    uint64_t q_batch, q_node;         /* strides in elements; 16 bytes divide the strides' sizes */
    uint64_t out_batch, out_node;
    uint64_t kv_batch, kv_row;        /* of k and v, in bytes, multiples of 16; kv_row below 2^26 */
    uint64_t scale_batch;             /* of kscale and vscale, in floats */
    uint64_t account_batch;
    uint32_t type;
    uint32_t batch, nodes, heads, kv_heads;   /* batch <= 65535, nodes <= 1024, heads a multiple of kv_heads */
    uint32_t dim;             /* 64 or 128 */
    uint32_t positions;       /* of the cache arrays */
    uint32_t max_len;         /* about the longest of lens (shapes the launch; results hold for any) */
    float scale, decay;
} qxg_tree_attention_args;
int qxg_tree_attention(qxg_ctx *ctx, const qxg_tree_attention_args *args, void *stream, int wait, char *err, uint64_t err_len);
uint64_t qxg_tree_attention_workspace(const qxg_tree_attention_args *args);

/* Which positions of each group (a layer, a sequence) to keep within `budget`: the first `sinks`,
 * the last `recent`, and of those between the ones with the largest account (the lower position
 * where equal; NaN as -inf).  keep[g][0 .. kept[g]) receives them in ascending order, kept[g] =
 * min(lens[g], budget); the rest of keep is left as it was.  The account may be one for all groups
 * (account_group 0), the lists of keep may not overlap. */
typedef struct qxg_kv_select_args {
    const float *account;     /* [groups][positions] */
    const uint32_t *lens;     /* [groups] */
    uint32_t *keep;           /* [groups][budget] */
    uint32_t *kept;           /* [groups]; may be lens itself, which then holds the new lengths */
    uint64_t account_group, keep_group;   /* strides in elements */
    uint32_t groups, positions, budget, sinks, recent;   /* groups < 2^22, sinks + recent <= budget */
    uint32_t max_len;         /* below 2^31; not used: each group's own length, in device memory, decides */
} qxg_kv_select_args;
int qxg_kv_select(qxg_ctx *ctx, const qxg_kv_select_args *args, void *stream, int wait, char *err, uint64_t err_len);

/* Moves the rows of each group's cache in place: row first + i becomes what row keep[g][i] was,
 * for i < min(kept[g], slots).  keep[g] ascends strictly and keep[g][i] >= first + i, as
 * qxg_kv_select writes it, or as a program lists the accepted nodes of a tree behind its cached
 * positions (first = lens[b]); of a list that does not, the moved rows are undefined (never
 * anything else).  Rows at and behind first + kept[g] are left as they were.  account_out[first +
 * i] = account[keep[i]] in another array, whose other entries are left as they were.  Entries outside the cache are skipped.
 * first is the same for all groups: sequences of unlike lengths take a call each.  (Calls that share a workspace at the
 * same time, which is not allowed, end all the same; their moved rows are undefined.) */
typedef struct qxg_kv_compact_args {
    int8_t *k, *v;            /* [groups][positions][row_bytes], 16-byte aligned */
    float *kscale, *vscale;   /* [groups][positions] */
    const uint32_t *keep;     /* [groups][slots] */
    const uint32_t *kept;     /* [groups] */
    const float *account;     /* [groups][positions], or NULL with account_out */
    float *account_out;
    void *workspace;          /* 16-byte aligned */
    uint64_t workspace_bytes;
    uint64_t kv_group, kv_row;        /* in bytes, multiples of 16 */
    uint64_t scale_group;             /* in floats */
    uint64_t keep_group, kept_group;  /* in elements; 0: one list for all groups */
    uint64_t account_group, account_out_group;
    uint32_t groups, positions, slots, first, row_bytes;   /* groups <= 65535; row_bytes a multiple of 16, at most 4096 */
} qxg_kv_compact_args;
int qxg_kv_compact(qxg_ctx *ctx, const qxg_kv_compact_args *args, void *stream, int wait, char *err, uint64_t err_len);
uint64_t qxg_kv_compact_workspace(const qxg_kv_compact_args *args);

/* Penalties, biases, temperature and grammar mask on rows of logits, and the best tokens.  Per
 * row, for token v with logit x (f32 arithmetic, one rounding an operation, in this order):
 *     v anywhere in the history:                x = x > 0 ? x / repetition : x * repetition
 *     v occurs c > 0 times behind the prompt:   x = x - frequency * c;  x = x - presence
 *     v in the bias list:                       x = x + (its biases, added in list order)
 *                                               x = x / temperature
 *     the token's mask bit is 0:                x = -inf
 * out = x rounded once to the type; lse = log sum exp(x) (NaN if an x is); top_ids / top_logits = the
 * top_n tokens by (x desc, id asc), as qxg_final_head ranks them; NaN and -inf are never picked: where no
 * others are left the id is QXG_NO_TOKEN and the logit -inf.  History and bias entries that are no token (>= vocab)
 * are skipped, so unused entries can be filled with QXG_NO_TOKEN. */
#define QXG_NO_TOKEN 0xffffffffu
typedef struct qxg_adjust_logits_args {
    const void *logits;       /* [rows][vocab] of `type`; any alignment of the type */
    void *out;                /* as logits; may be logits itself with the same stride */
    const uint32_t *history;  /* [rows][history_slots], or NULL */
    const uint32_t *history_lens;   /* [rows] entries in use, or NULL: all */
    const uint32_t *prompt_lens;    /* [rows] entries that are prompt, or NULL: none */
    const float *penalties;   /* [rows][3] repetition, frequency, presence; NULL: 1, 0, 0 */
    const float *temperature; /* [rows], or NULL: 1 */
    const uint32_t *bias_ids; /* [rows][biases], or NULL */
    const float *bias_values;
    const uint32_t *mask;     /* [masks][(vocab + 31) / 32] bits, bit v % 32 of word v / 32, or NULL */
    const uint32_t *mask_rows;      /* [rows] the row's mask; no mask where >= masks; NULL: row r takes mask r */
    uint32_t *top_ids;        /* [rows][top_n], or NULL with top_n 0 */
    float *top_logits;        /* [rows][top_n], or NULL */
    float *lse;               /* [rows], or NULL */
    void *workspace;          /* 16-byte aligned */
    uint64_t workspace_bytes;
    uint64_t logits_row, out_row, history_row;   /* strides in elements */
    uint32_t type, rows, vocab, history_slots, biases, masks, top_n;   /* rows <= 65535, history_slots < 2^20, biases <= 1024, top_n <= 32 */
} qxg_adjust_logits_args;
int qxg_adjust_logits(qxg_ctx *ctx, const qxg_adjust_logits_args *args, void *stream, int wait, char *err, uint64_t err_len);
uint64_t qxg_adjust_logits_workspace(const qxg_adjust_logits_args *args);

/* ---- a cache of 8 or 4 bits: its rows from projections, and attention over it ----
 *
 * bits 8: the context's own format: k, v [batch][positions][kv_heads][dim] int8, kscale, vscale [batch][positions] f32.
 * bits 4: E2M1 values with an E8M0 scale for each 32 dims, as the OCP Microscaling formats define them but for the scales' ends: k, v
 * [batch][positions][kv_heads][dim / 2], dim 2 i in the low half of byte i; kscale, vscale [batch][positions][kv_heads][dim / 32]
 * bytes e, for 2^(e - 127), and 255 for NaN.  (The formats' 2^-127 and 2^-126, bytes 0 and 1, are read as 2^-125, and 2^126 and 2^127, bytes 253 and
 * 254, as 2^125: products with them leave f32's normal numbers.  qxg_kv_append writes none of the five.) */

/* The rows of new tokens on their way from a projection into attention and the cache.  Token i < counts[b] of sequence b
 * stands at position lens[b] + i.  Per head of q and k, in this order:
 *     y[d] = x[d] weight[d] / sqrt(mean(x^2) + eps)                    where there are weights
 *     (y[a], y[b]) = (y[a] c - y[b] s, y[a] s + y[b] c)                for the pairs j < rotated / 2: a = j, b = j + rotated / 2, or
 *                                                                      with `paired` a = 2 j, b = 2 j + 1; c = rope[at][j],
 *                                                                      s = rope[at][rotated / 2 + j], at = rope_at[b][i] or the position
 * q_out is that of q, in f32 and rounded once to the type.  The keys are worked out in 64 bits and rounded once to f32; they
 * and the values v are held in the cache at their position, a value that is not finite as 0:
 *     bits 8: scale = the position's largest magnitude / 127 (1 if that is 0), code = rint(x / scale), as qxg_int8_quantize
 *     bits 4: the least power of two, of 2^-125 to 2^125, of which a block's largest magnitude is not over 7 times; each value the
 *             nearest E2M1 value times it, of two equally near ones that of the even code, at most 6 times it
 * Rows of tokens at and behind counts, and all other positions, are left as they were.  q, k and v may be parts of one array's rows.
 * q_out may be q itself; otherwise outputs share memory with nothing else.  (Refused are q_out in q, and all outputs in each other and in k and v; rows
 * that lie between another array's are told apart where both arrays' strides are the same.)  at is clamped to the table's last row. */
typedef struct qxg_kv_append_args {
    const void *q;            /* [batch][tokens][heads][dim] of `type`, 16-byte aligned */
    const void *k, *v;        /* [batch][tokens][kv_heads][dim] of `type`, 16-byte aligned */
    void *q_out;              /* as q */
    void *k_cache, *v_cache;  /* 16-byte aligned */
    void *kscale, *vscale;
    const uint32_t *lens;     /* [batch] cached positions; lens[b] + count is clamped to positions */
    const uint32_t *counts;   /* [batch] tokens in use, or NULL: all */
    const float *q_norm, *k_norm;   /* [dim] weights, or NULL: no norm */
    const float *rope;        /* [rope_positions][rotated] cosines, then sines; or NULL with rotated 0 */
    const uint32_t *rope_at;  /* [batch][tokens] rows of the table, or NULL: the positions */
    uint64_t q_batch, q_token, k_batch, k_token, v_batch, v_token, out_batch, out_token;   /* strides in elements; 16 bytes divide their sizes */
    uint64_t kv_batch, kv_row;        /* of k_cache and v_cache, in bytes, multiples of 16; kv_row below 2^26 */
    uint64_t scale_batch, scale_row;  /* of kscale and vscale, in elements; bits 8: positions are contiguous, scale_row is not used */
    uint32_t type, bits, batch, tokens, heads, kv_heads;   /* batch <= 65535, tokens <= 2^20, heads a multiple of kv_heads, at most 1024 */
    uint32_t dim;             /* 64 or 128; kv_heads * dim <= 4096 */
    uint32_t positions;       /* of the cache arrays */
    uint32_t rotated, rope_positions, paired;   /* rotated: a multiple of 16 up to dim */
    float eps;
} qxg_kv_append_args;
int qxg_kv_append(qxg_ctx *ctx, const qxg_kv_append_args *args, void *stream, int wait, char *err, uint64_t err_len);

/* Causal attention of new tokens over a cache of 8 or 4 bits, whole or within a window.  The rows of count = counts[b] new tokens stand
 * behind lens[b] cached positions, as qxg_kv_append leaves them; token i is at p = lens[b] + i and sees the positions j <= p
 * with p - j < window or j < sinks (window 0: all of them).  As qxg_tree_attention otherwise:
 *     s[j] = scale * sum_d q[i][h][d] k[j][g][d],  out[i][h] = sum_j softmax(s)[j] v[j][g],  lse[i][h] = log sum_j exp(s[j])
 * with k and v the values that the cache stands for.  What stands in positions that a row does not see does not reach it; rows of
 * tokens at and behind count are left as they were; out shares memory with nothing else, nor does lse (refused: in each other, in
 * the cache, out in q).  tokens = 1 is single-token decoding.
 * Products are those of f32 numbers for an F32 q; for F16 and BF16 q enters them as it is, and the softmax weights with 17 bits (off by 2^-18 of a
 * term, where the result is rounded by 2^-12 or 2^-9).  Sums are f32, rounded once: a dot product, over 8 bits before it is multiplied by its
 * position's scale, has to be within f32, as scale times a position's scale has; weights are up to 2^8 before they are divided by their sum, so
 * values from 2^118 on may overflow.  A row that sees a scale that is not finite is NaN, and so is its lse, as are a row whose q is not finite
 * and one whose largest score is beyond f32. */
typedef struct qxg_cache_attention_args {
    const void *q;            /* [batch][tokens][heads][dim] of `type`, 16-byte aligned */
    const void *k, *v;        /* 16-byte aligned */
    const void *kscale, *vscale;
    const uint32_t *lens;     /* [batch] cached positions before the new tokens; lens[b] + count is clamped to positions */
    const uint32_t *counts;   /* [batch] tokens in use, or NULL: all */
    void *out;                /* as q, 16-byte aligned */
    float *lse;               /* [batch][tokens][heads], or NULL */
    void *workspace;          /* 16-byte aligned */
    uint64_t workspace_bytes;
    uint64_t q_batch, q_token, out_batch, out_token;   /* strides in elements; 16 bytes divide their sizes */
    uint64_t kv_batch, kv_row;        /* of k and v, in bytes, multiples of 16; kv_row below 2^26 */
    uint64_t scale_batch, scale_row;  /* of kscale and vscale, in elements; bits 8: positions are contiguous, scale_row is not used */
    uint32_t type, bits, batch, tokens, heads, kv_heads;   /* batch <= 65535, tokens <= 2^20, heads a multiple of kv_heads, at most 1024 */
    uint32_t dim;             /* 64 or 128 */
    uint32_t positions;       /* of the cache arrays */
    uint32_t max_len;         /* about the longest of lens (shapes the launch; results hold for any) */
    uint32_t window, sinks;
    float scale;
} qxg_cache_attention_args;
int qxg_cache_attention(qxg_ctx *ctx, const qxg_cache_attention_args *args, void *stream, int wait, char *err, uint64_t err_len);
uint64_t qxg_cache_attention_workspace(const qxg_cache_attention_args *args);

/* ---- measurement (no reference counterpart: the reference times with clock(),
 *      src/qx_format.c:6245, 6642-6653) ---- */

/* Average device time (ms) of one launch of kernel `which` over `iters` launches,
 * bracketed by HIP events on the context stream.  which: 0 gate/up experts,
 * 1 down experts, 2 Q/K/V projection, 3 O projection, 4 Q6_K head, 5 attention,
 * 6 router.  Uses layer `layer`'s weights and the current routing/KV state. */
int qxg_time_kernel(qxg_ctx *ctx, int which, uint32_t layer, uint32_t iters, float *avg_ms, char *err, uint64_t err_len);
/* Device bytes held by uploaded tensors (repacked; equal to the QXF1 tensor bytes). */
uint64_t qxg_device_bytes(const qxg_ctx *ctx);
/* In-situ timing: while enabled, qxg_generate / qxg_decode_token record a HIP
 * event pair around every launch of kernel `which` (numbering of
 * qxg_time_kernel, plus 7 the persistent layer kernel and, for qxg_prefill, 8 Q/K/V,
 * 9 O, 10 gate/up and 11 down GEMMs, 12 router logits, 13 attention; -1 disables).
 * qxg_profile_result sums the pairs. */
int qxg_profile_kernel(qxg_ctx *ctx, int which);
int qxg_profile_result(qxg_ctx *ctx, uint32_t *launches, double *total_ms);

#ifdef __cplusplus
}
#endif
#endif
