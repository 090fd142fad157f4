// vtq_serve_api.hip -- C entry points of the serving operators (the last part of
// include/vtq.h): the checks of vtq_serve_checks.h, then the launchers of
// vtq_serve.h.
#include "vtq_serve.h"

namespace {

using namespace vtq;

// The context's device is current inside a call, the caller's again after it.
struct OnDevice {
    int before = -1;
    hipError_t status;
    explicit OnDevice(int device) {
        status = hipGetDevice(&before);
        if (status == hipSuccess && before != device) status = hipSetDevice(device);
        else if (status == hipSuccess) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

RopeJob append_job(const vtq_kv_cache& cache, const vtq_kv_batch& batch, const vtq_rope* rope, size_t tokens, HeadRows k,
                   HeadRows v, size_t heads, HeadRows q, void* q_out, size_t q_out_token_stride,
                   size_t q_out_head_stride) {
    RopeJob j{};
    if (rope) j.rope = *rope;
    j.rotate = rope != nullptr;
    j.tokens = (int64_t)tokens;
    j.head_dim = cache.head_dim;
    j.x_heads = q.p && heads ? (int)heads : 0;
    j.kv_heads = cache.kv_heads;
    j.x = q;
    j.k = k;
    j.v = v;
    j.y = q_out;
    j.y_token_stride = (int64_t)q_out_token_stride;
    j.y_head_stride = (int64_t)q_out_head_stride;
    j.cache = cache;
    j.batch = batch;
    return j;
}

Scales scales_of(const vtq_kv8_cache& c) {
    return {c.block, c.k_scale, c.v_scale, (int64_t)c.scale_page_stride, (int64_t)c.scale_head_stride};
}

// Whether a workspace of `need` bytes is there; the text of what it lacks.
Refusal check_workspace(const void* d_ws, size_t bytes, size_t need) {
    if (need && (!d_ws || bytes < need)) return {VTQ_E_INVALID_ARGUMENT, "vtq: workspace too small"};
    if (need && !aligned(d_ws, 256)) return {VTQ_E_INVALID_ARGUMENT, "vtq: the workspace must be 256-byte aligned"};
    return {};
}

int run(vtq_ctx* ctx, hipError_t e) { return e == hipSuccess ? VTQ_OK : ctx_hip_error(ctx, e, "kernel launch"); }

}  // namespace

extern "C" {

int vtq_quantize_i8_device(vtq_ctx* ctx, int x_type, const void* d_x, size_t ld_x, int8_t* d_q, size_t ld_q,
                           float* d_scale, size_t rows, size_t n, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_quantize_i8(x_type, d_x, ld_x, d_q, ld_q, d_scale, rows, n)) return ctx_error(ctx, r.code,
            r.text);
    if (rows == 0) return VTQ_OK;
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    return run(ctx, launch_quantize_i8(x_type, d_x, ld_x, d_q, ld_q, d_scale, rows, (int)n,
                                       static_cast<hipStream_t>(stream)));
}

int vtq_linear_i8_device(vtq_ctx* ctx, const int8_t* d_xq, size_t ld_x, const float* d_x_scale, const int8_t* d_wq,
                         size_t ld_w, const float* d_w_scale, const float* d_bias, int y_type, void* d_y, size_t ld_y,
                         size_t batch, size_t in_feat, size_t out_feat, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_linear_i8(d_xq, ld_x, d_x_scale, d_wq, ld_w, d_w_scale, d_bias, y_type, d_y, ld_y, batch,
                                    in_feat, out_feat)) return ctx_error(ctx, r.code, r.text);
    if (batch == 0 || out_feat == 0) return VTQ_OK;
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    const I8Linear a{d_xq, d_wq, d_x_scale, d_w_scale, d_bias, d_y, ld_x, ld_w, ld_y, (int)batch, (int)in_feat,
                     (int)out_feat};
    return run(ctx, launch_linear_i8(a, y_type, static_cast<hipStream_t>(stream)));
}

int vtq_rope_plan(vtq_ctx* ctx, const vtq_rope_params* params, vtq_rope* out) {
    const Refusal r = plan_rope(params, out);
    return ctx_error(ctx, r.code, r.text);
}

int vtq_rope_device(vtq_ctx* ctx, const vtq_rope* rope, int type, const void* d_x, size_t x_token_stride,
                    size_t x_head_stride, void* d_y, size_t y_token_stride, size_t y_head_stride, const int32_t* d_pos,
                    size_t tokens, size_t heads, size_t head_dim, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_rope_call(rope, type, d_x, x_token_stride, x_head_stride, d_y, y_token_stride,
                                    y_head_stride, d_pos, tokens, heads, head_dim)) return ctx_error(ctx, r.code,
                                            r.text);
    if (tokens == 0 || heads == 0) return VTQ_OK;
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    RopeJob j{};
    j.rope = *rope;
    j.rotate = 1;
    j.tokens = (int64_t)tokens;
    j.head_dim = (int)head_dim;
    j.x_heads = (int)heads;
    j.x = HeadRows{d_x, (int64_t)x_token_stride, (int64_t)x_head_stride};
    j.y = d_y;
    j.y_token_stride = (int64_t)y_token_stride;
    j.y_head_stride = (int64_t)y_head_stride;
    j.pos = d_pos;
    return run(ctx, launch_rope(j, type, type, static_cast<hipStream_t>(stream)));
}

int vtq_kv_append_device(vtq_ctx* ctx, const vtq_kv_cache* cache, const vtq_kv_batch* batch, const vtq_rope* rope,
                         int type, size_t tokens, const void* d_k, size_t k_token_stride, size_t k_head_stride,
                         const void* d_v, size_t v_token_stride, size_t v_head_stride, size_t heads, const void* d_q,
                         size_t q_token_stride, size_t q_head_stride, void* d_q_out, size_t q_out_token_stride,
                         size_t q_out_head_stride, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_append(cache, batch, rope, type, tokens, d_k, k_token_stride, k_head_stride, d_v,
                                 v_token_stride, v_head_stride, heads, d_q, q_token_stride, q_head_stride, d_q_out,
                                         q_out_token_stride, q_out_head_stride)) return ctx_error(ctx, r.code, r.text);
    if (tokens == 0 || batch->batch == 0) return VTQ_OK;
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    const RopeJob j = append_job(*cache, *batch, rope, tokens, {d_k, (int64_t)k_token_stride, (int64_t)k_head_stride},
                                 {d_v, (int64_t)v_token_stride, (int64_t)v_head_stride}, heads,
                                 {d_q, (int64_t)q_token_stride, (int64_t)q_head_stride}, d_q_out, q_out_token_stride,
                                 q_out_head_stride);
    return run(ctx, launch_rope(j, type, cache->type, static_cast<hipStream_t>(stream)));
}

// 0 for numbers that vtq_attention_device refuses.
size_t vtq_attention_workspace(const vtq_kv_cache* cache, const vtq_kv_batch* batch, int type, size_t tokens,
                               size_t heads) {
    if (!cache || !batch || check_cache(cache) || check_batch(batch, cache, false)) return 0;
    if (type_bytes(type) == 0 || tokens > kMostTokens || heads > 65535 || heads % cache->kv_heads) return 0;
    if (!attention_fits(cache, batch, tokens, heads)) return 0;
    if (tokens == 0 || heads == 0 || batch->batch == 0) return 0;
    return attention_workspace(*cache, *batch, type, (int64_t)tokens, (int)heads);
}

int vtq_attention_device(vtq_ctx* ctx, const vtq_kv_cache* cache, const vtq_kv_batch* batch, int type, size_t tokens,
                         size_t heads, const void* d_q, size_t q_token_stride, size_t q_head_stride, void* d_y,
                         size_t y_token_stride, size_t y_head_stride, float* d_lse, float scale, void* d_ws,
                         size_t ws_bytes, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_attention(cache, batch, type, tokens, heads, d_q, q_token_stride, q_head_stride, d_y,
                                    y_token_stride, y_head_stride, d_lse, scale)) return ctx_error(ctx, r.code, r.text);
    if (tokens == 0 || heads == 0 || batch->batch == 0) return VTQ_OK;
    const size_t need = attention_workspace(*cache, *batch, type, (int64_t)tokens, (int)heads);
    if (need && (!d_ws || ws_bytes < need)) return ctx_error(ctx, VTQ_E_INVALID_ARGUMENT,
            "vtq: attention workspace too small");
    if (need && !aligned(d_ws, 256)) return ctx_error(ctx, VTQ_E_INVALID_ARGUMENT,
                                                      "vtq: the workspace must be 256-byte aligned");
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    Attention a{};
    a.cache = *cache;
    a.batch = *batch;
    a.tokens = (int64_t)tokens;
    a.heads = (int)heads;
    a.q = HeadRows{d_q, (int64_t)q_token_stride, (int64_t)q_head_stride};
    a.y = d_y;
    a.y_token_stride = (int64_t)y_token_stride;
    a.y_head_stride = (int64_t)y_head_stride;
    a.lse = d_lse;
    a.scale = scale;
    a.ws = d_ws;
    return run(ctx, launch_attention(a, type, static_cast<hipStream_t>(stream)));
}

int vtq_kv8_append_device(vtq_ctx* ctx, const vtq_kv8_cache* cache, const vtq_kv_batch* batch, const vtq_rope* rope,
                          int type, size_t tokens, const void* d_k, size_t k_token_stride, size_t k_head_stride,
                          const void* d_v, size_t v_token_stride, size_t v_head_stride, size_t heads, const void* d_q,
                          size_t q_token_stride, size_t q_head_stride, void* d_q_out, size_t q_out_token_stride,
                          size_t q_out_head_stride, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_kv8_append(cache, batch, rope, type, tokens, d_k, k_token_stride, k_head_stride, d_v,
                                     v_token_stride, v_head_stride, heads, d_q, q_token_stride, q_head_stride, d_q_out,
                                     q_out_token_stride, q_out_head_stride)) return ctx_error(ctx, r.code, r.text);
    if (tokens == 0 || batch->batch == 0) return VTQ_OK;
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    const RopeJob j = append_job(cache->cache, *batch, rope, tokens,
                                 {d_k, (int64_t)k_token_stride, (int64_t)k_head_stride},
                                 {d_v, (int64_t)v_token_stride, (int64_t)v_head_stride}, heads,
                                 {d_q, (int64_t)q_token_stride, (int64_t)q_head_stride}, d_q_out, q_out_token_stride,
                                 q_out_head_stride);
    return run(ctx, launch_kv8_append(j, scales_of(*cache), type, static_cast<hipStream_t>(stream)));
}

// 0 for numbers that vtq_kv8_attention_device refuses.
size_t vtq_kv8_attention_workspace(const vtq_kv8_cache* cache, const vtq_kv_batch* batch, int type, size_t tokens,
                                   size_t heads) {
    if (!cache || !batch || check_cache8(cache) || check_batch(batch, &cache->cache, false)) return 0;
    if (type_bytes(type) == 0 || tokens > kMostTokens || heads > 65535 || heads % cache->cache.kv_heads) return 0;
    if (!attention_fits(&cache->cache, batch, tokens, heads, most_kv8_workgroups(&cache->cache))) return 0;
    if (tokens == 0 || heads == 0 || batch->batch == 0) return 0;
    return kv8_attention_workspace(cache->cache, *batch, type, (int64_t)tokens, (int)heads);
}

int vtq_kv8_attention_device(vtq_ctx* ctx, const vtq_kv8_cache* cache, const vtq_kv_batch* batch, int type,
                             size_t tokens, size_t heads, const void* d_q, size_t q_token_stride, size_t q_head_stride,
                             void* d_y, size_t y_token_stride, size_t y_head_stride, float* d_lse, float scale,
                             void* d_ws, size_t ws_bytes, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_kv8_attention(cache, batch, type, tokens, heads, d_q, q_token_stride, q_head_stride, d_y,
                                        y_token_stride, y_head_stride, d_lse, scale)) return ctx_error(ctx, r.code, r.text);
    if (tokens == 0 || heads == 0 || batch->batch == 0) return VTQ_OK;
    const size_t need = kv8_attention_workspace(cache->cache, *batch, type, (int64_t)tokens, (int)heads);
    if (Refusal r = check_workspace(d_ws, ws_bytes, need)) return ctx_error(ctx, r.code, r.text);
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    Attention a{};
    a.cache = cache->cache;
    a.batch = *batch;
    a.tokens = (int64_t)tokens;
    a.heads = (int)heads;
    a.q = HeadRows{d_q, (int64_t)q_token_stride, (int64_t)q_head_stride};
    a.y = d_y;
    a.y_token_stride = (int64_t)y_token_stride;
    a.y_head_stride = (int64_t)y_head_stride;
    a.lse = d_lse;
    a.scale = scale;
    a.ws = d_ws;
    return run(ctx, launch_kv8_attention(a, scales_of(*cache), type, static_cast<hipStream_t>(stream)));
}

// 0 for numbers that vtq_beam_select_device refuses.
size_t vtq_beam_select_workspace(size_t groups, size_t beams, size_t vocab, size_t n_out) {
    if (!beam_select_fits(groups, beams, vocab, n_out) || !beams || !vocab || !n_out || !groups) return 0;
    return beam_select_workspace((int64_t)groups, (int64_t)beams, (int64_t)vocab, (int64_t)n_out);
}

int vtq_beam_select_device(vtq_ctx* ctx, int type, const void* d_logits, size_t ld, size_t groups, size_t beams,
                           size_t vocab, const float* d_score, const uint8_t* d_done, int end_token, size_t n_out,
                           float* d_out_score, int32_t* d_out_token, int32_t* d_out_parent, uint8_t* d_out_done,
                           void* d_ws, size_t ws_bytes, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_beam_select(type, d_logits, ld, groups, beams, vocab, d_score, d_done, end_token, n_out,
                                      d_out_score, d_out_token, d_out_parent, d_out_done)) return ctx_error(ctx, r.code,
                                              r.text);
    if (groups == 0) return VTQ_OK;
    const size_t need = beam_select_workspace((int64_t)groups, (int64_t)beams, (int64_t)vocab, (int64_t)n_out);
    if (Refusal r = check_workspace(d_ws, ws_bytes, need)) return ctx_error(ctx, r.code, r.text);
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    const BeamSelect a{d_logits, (int64_t)ld, (int)groups, (int)beams, (int)vocab, (int)n_out, end_token, d_score,
                       d_done, d_out_score, d_out_token, d_out_parent, d_out_done, d_ws};
    return run(ctx, launch_beam_select(a, type, static_cast<hipStream_t>(stream)));
}

size_t vtq_pages_reorder_workspace(size_t n_pages, size_t batch, size_t batch_out) {
    if (n_pages > kMostPages || batch > kMostReordered || batch_out > kMostReordered) return 0;
    return pages_reorder_workspace((int64_t)n_pages, (int64_t)batch_out);
}

int vtq_pages_reorder_device(vtq_ctx* ctx, size_t n_pages, int page_size, size_t max_pages, const int32_t* d_refs,
                             size_t batch, const int32_t* d_pages, const int32_t* d_len, size_t batch_out,
                             const int32_t* d_parent, const int32_t* d_grow, int32_t* d_new_refs, int32_t* d_new_pages,
                             int32_t* d_new_len, int32_t* d_copies, int32_t* d_info, void* d_ws, size_t ws_bytes,
                             void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_pages_reorder(n_pages, page_size, max_pages, d_refs, batch, d_pages, d_len, batch_out,
                                        d_parent, d_grow, d_new_refs, d_new_pages, d_new_len, d_copies,
                                        d_info)) return ctx_error(ctx, r.code, r.text);
    const size_t need = pages_reorder_workspace((int64_t)n_pages, (int64_t)batch_out);
    if (Refusal r = check_workspace(d_ws, ws_bytes, need)) return ctx_error(ctx, r.code, r.text);
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    const PagesReorder a{(int64_t)n_pages, page_size, (int)max_pages, (int)batch, (int)batch_out, d_refs, d_pages, d_len,
                         d_parent, d_grow, d_new_refs, d_new_pages, d_new_len, d_copies, d_info, d_ws};
    return run(ctx, launch_pages_reorder(a, static_cast<hipStream_t>(stream)));
}

size_t vtq_pages_compact_workspace(size_t n_pages) {
    return n_pages > kMostPages ? 0 : pages_compact_workspace((int64_t)n_pages);
}

int vtq_pages_compact_device(vtq_ctx* ctx, size_t n_pages, int page_size, const int32_t* d_refs, size_t n_entries,
                             const int32_t* d_pages, size_t n_prefix, const int32_t* d_prefix_pages,
                             int32_t* d_new_refs, int32_t* d_new_pages, int32_t* d_new_prefix_pages, int32_t* d_copies,
                             int32_t* d_info, void* d_ws, size_t ws_bytes, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_pages_compact(n_pages, page_size, d_refs, n_entries, d_pages, n_prefix, d_prefix_pages,
                                        d_new_refs, d_new_pages, d_new_prefix_pages, d_copies, d_info)) return
            ctx_error(ctx, r.code, r.text);
    const size_t need = pages_compact_workspace((int64_t)n_pages);
    if (Refusal r = check_workspace(d_ws, ws_bytes, need)) return ctx_error(ctx, r.code, r.text);
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    const PagesCompact a{(int64_t)n_pages, page_size, (int64_t)n_entries, (int64_t)n_prefix, d_refs, d_pages,
                         d_prefix_pages, d_new_refs, d_new_pages, d_new_prefix_pages, d_copies, d_info, d_ws};
    return run(ctx, launch_pages_compact(a, static_cast<hipStream_t>(stream)));
}

int vtq_pages_copy_device(vtq_ctx* ctx, const vtq_kv_cache* cache, size_t layers, size_t layer_stride,
                          const int32_t* d_copies, size_t max_copies, const int32_t* d_count, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_pages_copy(cache, layers, layer_stride, d_copies, max_copies, d_count)) return ctx_error(ctx,
            r.code, r.text);
    if (layers == 0 || max_copies == 0 || cache->n_pages == 0) return VTQ_OK;
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    const PagesCopy a{*cache, Scales{}, (int)layers, (int64_t)layer_stride, 0, d_copies, d_count, (int64_t)max_copies};
    return run(ctx, launch_pages_copy(a, static_cast<hipStream_t>(stream)));
}

int vtq_kv8_pages_copy_device(vtq_ctx* ctx, const vtq_kv8_cache* cache, size_t layers, size_t layer_stride,
                              size_t scale_layer_stride, const int32_t* d_copies, size_t max_copies,
                              const int32_t* d_count, void* stream) {
    if (!ctx) return VTQ_E_INVALID_ARGUMENT;
    ctx_error(ctx, VTQ_OK, "");
    if (Refusal r = check_kv8_pages_copy(cache, layers, layer_stride, scale_layer_stride, d_copies, max_copies,
                                         d_count)) return ctx_error(ctx, r.code, r.text);
    if (layers == 0 || max_copies == 0 || cache->cache.n_pages == 0) return VTQ_OK;
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    const PagesCopy a{cache->cache, scales_of(*cache), (int)layers, (int64_t)layer_stride, (int64_t)scale_layer_stride,
                      d_copies, d_count, (int64_t)max_copies};
    return run(ctx, launch_pages_copy(a, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
