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
    const bool with_q = d_q && heads;
    OnDevice on(ctx_device(ctx));
    if (on.status != hipSuccess) return ctx_hip_error(ctx, on.status, "hipSetDevice");
    RopeJob j{};
    if (rope) j.rope = *rope;
    j.rotate = rope != nullptr;
    j.tokens = (int64_t)tokens;
    j.head_dim = cache->head_dim;
    j.x_heads = with_q ? (int)heads : 0;
    j.kv_heads = cache->kv_heads;
    j.x = HeadRows{d_q, (int64_t)q_token_stride, (int64_t)q_head_stride};
    j.k = HeadRows{d_k, (int64_t)k_token_stride, (int64_t)k_head_stride};
    j.v = HeadRows{d_v, (int64_t)v_token_stride, (int64_t)v_head_stride};
    j.y = d_q_out;
    j.y_token_stride = (int64_t)q_out_token_stride;
    j.y_head_stride = (int64_t)q_out_head_stride;
    j.cache = *cache;
    j.batch = *batch;
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

}  // extern "C"
