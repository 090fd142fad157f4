/*
 * vtq.h -- C ABI of libvtq, the MI355X (gfx950) backend for vitni-tensor's
 * quantized linear layer.
 *
 * The reference seam is the uniform Rust signature every dtype arm of
 * `linear_dispatch` calls (src/model/forward_quantized.rs:663-785), e.g.
 *
 *   pub fn linear_q4_k_integer(x: &[f32], w_q4k: &[u8], y_out: &mut [f32],
 *                              batch: usize, in_feat: usize, out_feat: usize)
 *       -> Result<()>                                  (src/ops/quant.rs:936-943)
 *
 * Each entry point below replaces one such function (citation on each) with
 * the same argument meaning: x[batch][in_feat] f32 row-major, w the GGUF
 * blocks of W[out_feat][in_feat] row-major, y[batch][out_feat] f32, all
 * outputs written.  Results are bit-identical to the reference CPU path.
 * Slices become (pointer, length) pairs; lengths are checked here where the
 * reference would panic on a short slice.
 *
 * Status codes mirror vitni_tensor::error::Error (src/error.rs:7-63):
 *   VTQ_OK                 Ok(())
 *   VTQ_E_INTERNAL         Error::Internal(&'static str)  (shape/length;
 *                          vtq_last_error() returns the reference's text)
 *   VTQ_E_GPU              Error::GpuError                (HIP failure)
 *   VTQ_E_NOT_IMPLEMENTED  Error::NotImplemented          (F16/other dtypes; a
 *                          request beyond the no-alloc entry point's scratch)
 *   VTQ_E_INVALID_ARGUMENT null pointer or context; Rust's types rule these out
 *   VTQ_E_MALFORMED        Error::Malformed               (GGUF parse, libvtq_runtime)
 *   VTQ_E_TRUNCATED        Error::Truncated               (GGUF parse, libvtq_runtime)
 *   VTQ_E_OVERFLOW         Error::Overflow                (GGUF parse, libvtq_runtime)
 *   VTQ_E_SHAPE_MISMATCH   Error::ShapeMismatch           (a norm weight whose length
 *                          is not the model dimension, rms_norm.rs:80-85)
 *   VTQ_E_INVALID_SHAPE    Error::InvalidShape            (empty prompt, prompt + new
 *                          tokens past seq_len, inference.rs:301-311)
 * No entry point aborts or panics.
 *
 * The operators of a batched serving step (the last part of this header) have
 * no counterpart in the reference, which serves one sequence with f32
 * activations; they use the same context, codes and error texts.
 *
 * Threading: a context is used by one host thread at a time (the reference's
 * Accelerator takes &mut self, src/accel/mod.rs:82).  Contexts on different
 * threads are independent.
 */
#ifndef VTQ_H
#define VTQ_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VTQ_OK 0
#define VTQ_E_INTERNAL 1
#define VTQ_E_GPU 2
#define VTQ_E_NOT_IMPLEMENTED 3
#define VTQ_E_INVALID_ARGUMENT 4
#define VTQ_E_MALFORMED 5
#define VTQ_E_TRUNCATED 6
#define VTQ_E_OVERFLOW 7
#define VTQ_E_SHAPE_MISMATCH 8
#define VTQ_E_INVALID_SHAPE 9

/* GGUF tensor type tags (src/model/gguf.rs:127-139). */
#define VTQ_TYPE_F32 0
#define VTQ_TYPE_F16 1
#define VTQ_TYPE_Q4_0 2
#define VTQ_TYPE_Q5_0 6
#define VTQ_TYPE_Q8_0 8
#define VTQ_TYPE_Q4_K 12
#define VTQ_TYPE_Q6_K 14
#define VTQ_TYPE_BF16 30 /* activations and caches of the serving operators only */

/* Numerical regime of the Q4_K arm, chosen by a Cargo feature in the
 * reference (src/model/forward_quantized.rs:704-725):
 *   VTQ_REGIME_INTEGER      `std-parallel` build: linear_q4_k_integer[_parallel]
 *   VTQ_REGIME_FLOAT_FUSED  default build:        linear_q4_k_fused
 * All other dtypes compute the same bits in both regimes. */
#define VTQ_REGIME_INTEGER 0
#define VTQ_REGIME_FLOAT_FUSED 1

typedef struct vtq_ctx vtq_ctx;

/* Create a context bound to HIP device `device`.  Replaces constructing the
 * reference's accelerator value (CpuAccelerator, src/accel/mod.rs:102-120). */
int vtq_create(int device, vtq_ctx **out);
void vtq_destroy(vtq_ctx *ctx);
/* Text of the last error on this context ("" after success); for
 * VTQ_E_INTERNAL it is the reference's Error::Internal message. */
const char *vtq_last_error(const vtq_ctx *ctx);
/* Library version string, "vtq <major>.<minor>.<patch> (gfx950)".  It names
 * the ABI of this header and of vtq_runtime.h together; 0.2.0 added the
 * trailing digest_v1 argument of vtqrt_run (a caller built against 0.1.0
 * headers must not load this library); 0.3.0 added vtqrt_set_prompt_mode
 * (no existing signature changed); 0.3.1 added the serving operators. */
const char *vtq_version(void);

/* ---- host-pointer entry points (synchronous; y is complete on return) ----
 * x, w, y are host memory owned by the caller.  w is uploaded once and cached
 * on the device keyed by (pointer, length): the reference's weights are
 * zero-copy views into a GGUF blob that lives for the model's lifetime
 * (src/model/quant_weights.rs:47-52), so the bytes behind a cached key must
 * not change until vtq_release_weights() drops it. */

/* src/model/forward_quantized.rs:663-785 linear_dispatch, for any batch. */
int vtq_linear(vtq_ctx *ctx, int ggml_type, int regime, const float *x, size_t x_len,
               const uint8_t *w, size_t w_len, float *y, size_t y_len, size_t batch,
               size_t in_feat, size_t out_feat);

/* src/ops/quant.rs:936-980 linear_q4_k_integer (and its row-parallel twin
 * :1149-1196, which computes the same bits). */
int vtq_linear_q4_k_integer(vtq_ctx *ctx, const float *x, size_t x_len, const uint8_t *w,
                            size_t w_len, float *y, size_t y_len, size_t batch, size_t in_feat,
                            size_t out_feat);
/* src/ops/quant.rs:1060-1096 linear_q6_k_integer (twin :1099-1146). */
int vtq_linear_q6_k_integer(vtq_ctx *ctx, const float *x, size_t x_len, const uint8_t *w,
                            size_t w_len, float *y, size_t y_len, size_t batch, size_t in_feat,
                            size_t out_feat);
/* src/ops/quant.rs:1433-1453 linear_q4_k_fused (twin :1386-1430). */
int vtq_linear_q4_k_fused(vtq_ctx *ctx, const float *x, size_t x_len, const uint8_t *w,
                          size_t w_len, float *y, size_t y_len, size_t batch, size_t in_feat,
                          size_t out_feat);
/* src/ops/quant.rs:1529-1565 linear_q4_0_cpu (exact-length checks kept). */
int vtq_linear_q4_0(vtq_ctx *ctx, const float *x, size_t x_len, const uint8_t *w, size_t w_len,
                    float *y, size_t y_len, size_t batch, size_t in_feat, size_t out_feat);

/* Drop the device copy cached for host weight pointer w (any length), or
 * every cached weight when w is NULL. */
int vtq_release_weights(vtq_ctx *ctx, const uint8_t *w);

/* ---- device-pointer entry point (asynchronous) ----
 * Same computation as vtq_linear, but d_x, d_w, d_y are device memory on the
 * context's device and the work is enqueued on `stream` (a hipStream_t, NULL
 * for the null stream) without synchronising.  d_x and d_w must be 16-byte
 * aligned, and d_w readable up to the next multiple of 16 bytes past w_len
 * (every hipMalloc or torch device allocation is: the kernels fetch whole
 * 16-byte chunks and ignore the bytes past the blob).  This is what a
 * device-resident forward step calls; it replaces the same linear_dispatch arm
 * as vtq_linear.  Calls that overlap in time on one context race on the
 * context's workspace.
 * A batch GEMM (Q4_K in the integer regime and Q6_K) keeps its quantized
 * activations in 8 MiB that the context allocates at a stream's first such
 * call, for its first eight streams, and frees with itself.  On further streams,
 * on hipStreamPerThread and under graph capture, Q6_K and Q4_K batches below
 * 32 rows take the form without a workspace, which passes over the weights once
 * per batch row; larger Q4_K batches share one workspace there. */
int vtq_linear_device(vtq_ctx *ctx, int ggml_type, int regime, const float *d_x,
                      const uint8_t *d_w, size_t w_len, float *d_y, size_t batch, size_t in_feat,
                      size_t out_feat, void *stream);

/* ---- allocation-free device entry point ----
 * No counterpart in the reference: it is for callers that cannot allocate
 * device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  Same computation, arguments and
 * errors as vtq_linear_device, but it calls no hipMalloc / hipFree: the
 * workspace of the GEMM that Q4_K batches of 32 rows and more take in the
 * integer regime (the quantized activations) lives in a fixed 32 MiB array on
 * each GPU, allocated when the library loads.  Requests whose workspace would
 * exceed it (vtq::q4k_gemm_workspace_bytes: about batch x in_feat x 1.14
 * bytes, batch capped at 8192 per chunk) return VTQ_E_NOT_IMPLEMENTED with a
 * message and launch nothing.  Smaller Q4_K batches and Q6_K take the form
 * without a workspace, one pass over the weights per batch row.  Rows longer
 * than the kernels hold (k-quant beyond 32768 inputs, the canonical dot beyond
 * 65536) keep their segments' sums in the array too (segments x batch x
 * out_feat x 4 bytes, plus one gathered segment of x per batch row for the
 * canonical dot), with the batch split into passes that fit; a single batch
 * row that does not fit is refused the same way.  All calls on one GPU share
 * that array: calls that use it and overlap in time on one device (any
 * context, any stream) race on it and must be serialised by the caller.
 * Every byte a call reads from the array is written earlier in the same call,
 * so nothing needs clearing between calls. */
int vtq_linear_device_noalloc(vtq_ctx *ctx, int ggml_type, int regime, const float *d_x,
                              const uint8_t *d_w, size_t w_len, float *d_y, size_t batch,
                              size_t in_feat, size_t out_feat, void *stream);

/* ---- operators of a batched serving step (device pointers, asynchronous) ----
 * Between the linears of a step that serves several sequences: an int8 linear
 * with scales per token and channel, rotary positions, appending to a paged
 * KV cache, and attention over it for a batch whose sequences share a prefix.
 * All pointers but the structs' own are device memory on the context's device;
 * the work is enqueued on `stream` (a hipStream_t of that device, NULL for the
 * null stream) without synchronising, whichever device is current, which stays
 * current.  Nothing is allocated, so every call may be captured into a graph,
 * and calls on different streams share no memory but the caller's.
 * `type` arguments take VTQ_TYPE_F32, VTQ_TYPE_F16 or VTQ_TYPE_BF16.  Leading
 * dimensions and strides count elements; the last dimension is contiguous.
 * Results do not change from run to run: no sums of a changing order.  Outputs
 * overlap neither each other's rows nor, but where a call says so, inputs.
 * Refusals: VTQ_E_INVALID_ARGUMENT (null or unaligned pointer, value out of its
 * range), VTQ_E_INVALID_SHAPE (sizes or strides that do not fit together) and
 * VTQ_E_NOT_IMPLEMENTED (type combinations and sizes beyond the kernels), with
 * a text, before anything is launched. */

/* Rows to 8 bits: scale[m] = max_k |x[m][k]| / 127 (f32, rounded once) and
 * q[m][k] = x[m][k] / scale[m] to the nearest whole number (the exact quotient;
 * ties to even; at most 127 in magnitude), 0 where the scale is 0.  A row that
 * holds an infinity or a NaN gets that as its scale and zeros, so its products
 * are NaN.  x has rows ld_x apart, q rows ld_q bytes apart (a multiple of 16, at
 * least n; q itself 16-byte aligned); the bytes from n to ld_q are set to 0.
 * n <= 131071.  Weights take the same call, one row per output channel. */
int vtq_quantize_i8_device(vtq_ctx *ctx, int x_type, const void *d_x, size_t ld_x, int8_t *d_q, size_t ld_q,
                           float *d_scale, size_t rows, size_t n, void *stream);

/* y[m][o] = x_scale[m] * w_scale[o] * sum_k xq[m][k] * wq[o][k] + bias[o]; the sum
 * is exact (32 bits: in_feat <= 131071), the rest f32, rounded once to y_type.
 * bias may be NULL.  xq and wq rows are ld_x and ld_w bytes apart (multiples of
 * 16, at least in_feat; 16-byte aligned), readable up to the next multiple of 16
 * past in_feat; in xq those bytes past in_feat must be 0, as the call above
 * leaves them.  y rows are ld_y apart.  in_feat 0 gives the bias alone. */
int vtq_linear_i8_device(vtq_ctx *ctx, const int8_t *d_xq, size_t ld_x, const float *d_x_scale, const int8_t *d_wq,
                         size_t ld_w, const float *d_w_scale, const float *d_bias, int y_type, void *d_y, size_t ld_y,
                         size_t batch, size_t in_feat, size_t out_feat, void *stream);

/* Rotary positions.  The first rot_dim elements of a head (even, 2 to 256) form
 * rot_dim / 2 pairs, (2i, 2i + 1) interleaved or (i, i + rot_dim / 2) by halves;
 * at position p pair i turns by the angle p * f_i:
 *   (a, b) -> magnitude * (a cos - b sin, a sin + b cos),  f_i = theta^(-2i / rot_dim) / factors[i].
 * scaling stretches f_i for contexts longer than the trained original_context:
 *   LINEAR  f_i / factor;
 *   BANDS   with t = original_context * f_i / 2 pi turns in the original context and
 *           k = (t - low) / (high - low) clamped to 0..1:  k f_i + (1 - k) f_i / factor
 *           (low, high: 1 and 4 where 0 is given);
 *   YARN    a ramp over the pair index between the pairs that make `high` and `low`
 *           turns (32 and 1 where 0 is given), rounded outwards to whole indices, and
 *           magnitude 0.1 ln(factor) + 1.
 * magnitude (at most 1e30), where it is not 0, replaces the rule's own.  A plan is plain memory:
 * it may be copied, and holds f_i as fractions of a turn in 64 bits (off by 4 2^-64
 * at most where no factor is below 1), so that p * f_i modulo a turn is right to
 * 2^-31 of a turn for every 32-bit position. */
#define VTQ_ROPE_INTERLEAVED 0
#define VTQ_ROPE_HALF 1
#define VTQ_ROPE_SCALE_NONE 0
#define VTQ_ROPE_SCALE_LINEAR 1
#define VTQ_ROPE_SCALE_BANDS 2
#define VTQ_ROPE_SCALE_YARN 3
typedef struct {
    int layout, scaling, rot_dim;
    int original_context;
    double theta, factor, low, high, magnitude;
    const float *factors; /* host, rot_dim / 2 values, or NULL: all 1 */
} vtq_rope_params;
typedef struct {
    int layout, rot_dim;
    float magnitude;
    int reserved;
    uint64_t turns[128];
} vtq_rope;
/* Fills *out on the host; ctx only takes the error text and may be NULL. */
int vtq_rope_plan(vtq_ctx *ctx, const vtq_rope_params *params, vtq_rope *out);

/* y[t][h] = x[t][h] rotated to position pos[t] (int32, negative ones turn
 * backwards); elements past rot_dim are copied.  x and y are tokens x heads x
 * head_dim with their own token and head strides; y may be x itself (the same
 * pointer and strides), and must not overlap it otherwise. */
int vtq_rope_device(vtq_ctx *ctx, const vtq_rope *rope, int type, const void *d_x, size_t x_token_stride,
                    size_t x_head_stride, void *d_y, size_t y_token_stride, size_t y_head_stride,
                    const int32_t *d_pos, size_t tokens, size_t heads, size_t head_dim, void *stream);

/* A paged KV cache: slot s of page p of KV head h is head_dim contiguous elements
 * at p * page_stride + h * head_stride + s * slot_stride, in k and v alike.
 * page_size is a power of two, 8 to 4096; head_dim a multiple of 8 up to 256; the
 * strides are multiples of 8 with slots and heads apart (at least head_dim), and k
 * and v 16-byte aligned.  So pages x heads x slots, pages x slots x heads and heads
 * x pages x slots all fit.  Limits: slot_stride below 2^24 and a page's slots
 * within 2^29 elements, head_stride and page_stride below 2^38, n_pages up to
 * INT_MAX, the whole within 2^46 elements. */
typedef struct {
    int type, page_size, kv_heads, head_dim;
    size_t n_pages;
    void *k, *v;
    size_t page_stride, head_stride, slot_stride;
} vtq_kv_cache;

/* A ragged batch.  Tokens q_start[b] to q_start[b + 1] of the call are the newest
 * of sequence b, which holds len[b] tokens of its own (these included) in the
 * slots of pages[b * max_pages + j], j = 0, 1, ..., behind a prefix of prefix_len
 * tokens that all sequences share in prefix_pages.  So token i of the n of a
 * sequence stands at position prefix_len + len[b] - n + i.
 * q_start (batch + 1, not decreasing, from 0), len and the page lists are device
 * memory, read when the work runs: a captured graph takes their new contents.
 * max_q is the host's idea of the longest sequence of tokens and max_len of the
 * longest own part (0: max_pages * page_size); they only choose how the work is
 * split.  Tokens of the call from q_start[batch] on are left alone, in every
 * output.  Page numbers outside the cache, and own tokens past max_pages pages,
 * are never read or written (see each call). */
typedef struct {
    int batch, max_pages, max_q, max_len, prefix_len;
    const int32_t *q_start, *len, *pages, *prefix_pages;
} vtq_kv_batch;

/* Writes the tokens' keys, rotated to their positions (rope NULL: as they are),
 * and values to their slots, rounded once to the cache's type, and, where d_q is
 * not NULL, the tokens' queries rotated to d_q_out (which may be d_q itself with
 * the same strides).  k and v are tokens x kv_heads x head_dim, q tokens x
 * heads x head_dim.  A token whose slot does not exist (a page number outside the
 * cache, a place below 0 or past max_pages pages) is not written.  Two tokens
 * must not share a slot: a page belongs to one sequence, or to the prefix. */
int vtq_kv_append_device(vtq_ctx *ctx, const vtq_kv_cache *cache, const vtq_kv_batch *batch, const vtq_rope *rope,
                         int type, size_t tokens, const void *d_k, size_t k_token_stride, size_t k_head_stride,
                         const void *d_v, size_t v_token_stride, size_t v_head_stride, size_t heads, const void *d_q,
                         size_t q_token_stride, size_t q_head_stride, void *d_q_out, size_t q_out_token_stride,
                         size_t q_out_head_stride, void *stream);

/* Attention of the batch's tokens over the prefix, which all of them see whole, and
 * the sequence's own tokens up to and including themselves:
 *   y[t][h] = sum_j softmax_j(scale * q[t][h] . k_j) v_j,  lse[t][h] = ln sum_j exp(scale * q . k_j),
 * query head h reading KV head h / (heads / kv_heads); heads is a multiple of
 * kv_heads.  The prefix is read once for all sequences.  A row that sees no key
 * gives zeros and an lse of -infinity; what stands in slots that a row does not
 * see never reaches it.  Keys in pages outside the cache count as zeros.  type is
 * the queries' and y's: the cache's own, or VTQ_TYPE_F32 with any cache.  lse
 * (f32, tokens x heads, or NULL) is in natural logarithms.  0 < scale <= 1e30.
 * Scores, maxima and sums are f32.  Where the queries are 16-bit, each weight is
 * rounded to their type before it meets its value: off by 2^-8 of itself (BF16), or
 * by 2^-11 of itself or 2^-32 of the row's largest, whichever is more (F16).  With
 * F32 queries weights stay f32, over a 16-bit cache too.
 * A row whose every score is -infinity counts as one that sees no key; a product
 * q . k past the range of f32 gives NaN, an lse past it an infinity.  y may be q
 * itself (the same pointer and strides), and must not overlap it otherwise.  A call
 * takes at most 2^23 tokens, 2^25 rows (tokens x heads) and 2^22 workgroups (to a
 * sequence, KV head and 32 rows of it).
 * d_ws is at least vtq_attention_workspace bytes, 256-byte aligned, for this call
 * alone until its work is done (calls that may overlap need one each); the size
 * depends on the host's numbers only, not on the lengths in device memory.  It is 0
 * where none is needed, and for numbers that the call refuses. */
size_t vtq_attention_workspace(const vtq_kv_cache *cache, const vtq_kv_batch *batch, int type, size_t tokens,
                               size_t heads);
int vtq_attention_device(vtq_ctx *ctx, const vtq_kv_cache *cache, const vtq_kv_batch *batch, int type, size_t tokens,
                         size_t heads, const void *d_q, size_t q_token_stride, size_t q_head_stride, void *d_y,
                         size_t y_token_stride, size_t y_head_stride, float *d_lse, float scale, void *d_ws,
                         size_t ws_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
