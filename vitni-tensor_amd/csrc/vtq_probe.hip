// vtq_probe.hip -- helpers of the benchmark and the tests (libvtq_probe.so).
//
// Not part of the quantized-linear boundary (include/vtq.h).  The kernels
// exist only to measure what the hardware gives a plain access pattern on
// the same buffers the benchmark's GEMVs read, so that each GEMV's rate can
// be quoted against a measured read ceiling as well as the published peak.
// The queries name the form that the dispatch rules (vtq_rules.h) give a call,
// so that a test can say which kernel it covers; they touch no GPU.
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "vtq_attention_plan.h"
#include "vtq_i8_rules.h"
#include "vtq_rules.h"
#include "vtq_serve.h"

namespace {

// Read-only stream: every thread reads 16-byte words i = g, g + G, g + 2G, ...
// (g = global thread index, G = grid threads), one load in flight per thread,
// and folds them into one word.  The store happens only if that word equals
// a constant the data never produces in practice; it keeps the loads alive
// without adding write traffic.
__global__ __launch_bounds__(256) void stream_read_kernel(const uint4* __restrict__ p, size_t n16,
                                                          uint32_t* __restrict__ sink) {
    uint32_t acc = 0;
    const size_t stride = (size_t)gridDim.x * 256;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += stride) {
        const uint4 v = p[i];
        acc ^= v.x ^ v.y ^ v.z ^ v.w;
    }
    if (acc == 0x9E3779B9u) sink[blockIdx.x] = acc;
}

int told(const vtq::Refusal& r, const char** text) {
    if (text) *text = r.text;
    return r.code;
}

}  // namespace

extern "C" {

// Launches the read of `bytes` (a multiple of 16) starting at device pointer
// `p` on `stream` with `workgroups` workgroups of 256 threads; `sink` is a
// device buffer of at least `workgroups` words.  Returns a hipError_t value.
int vtqp_stream_read(const void* p, size_t bytes, int workgroups, void* sink, void* stream) {
    if (!p || !sink || workgroups <= 0 || bytes % 16 != 0) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(stream_read_kernel, dim3((unsigned)workgroups), dim3(256), 0, (hipStream_t)stream,
                       static_cast<const uint4*>(p), bytes / 16, static_cast<uint32_t*>(sink));
    return (int)hipGetLastError();
}

// The form a pinned-dot call takes: 0 one GEMV slice per batch row, else 10 *
// token tiles of a wave + waves to a tile.
int vtqp_canon_form(int fmt, int batch, int in_feat, int out_feat) {
    if (fmt < 0 || fmt > vtq::kCanonQ4KFloat || batch <= 0 || in_feat <= 0 || out_feat <= 0) return -1;
    const vtq::CanonFormat f = (vtq::CanonFormat)fmt;
    if (!vtq::canon_gemm_faster(f, batch, in_feat, out_feat)) return 0;
    long ns;
    const vtq::GmForm& g = vtq::kGmForms[vtq::gm_pick(f, batch, in_feat, out_feat, &ns)];
    return 10 * g.nt + g.cs;
}

// The form a k-quant call (Q4_K = 12 / Q6_K = 14, integer regime) takes: 0 one
// GEMV slice per batch row, 1 the LDS-operand kernel, 2 the per-wave kernel,
// 300 + piece the split-K kernel, 600 + piece the same with two token tiles to
// a wave.
int vtqp_kquant_form(int type, int batch, int in_feat, int out_feat) {
    if ((type != 12 && type != 14) || batch <= 0 || in_feat <= 0 || in_feat % 256 || out_feat <= 0) return -1;
    const int R = in_feat / 256, NR = (out_feat + 31) / 32;
    const int M = batch < vtq::kChunkM ? batch : vtq::kChunkM, Mt = (M + 31) / 32;
    if (type == 14) {
        if (!vtq::q6k_gemm_faster(batch, in_feat, out_feat)) return 0;
        if (const int C = vtq::q6k_two_tiles(R, NR, Mt)) return 600 + C;
        return 300 + vtq::sk_piece(R, NR * Mt);
    }
    if (!vtq::q4k_gemm_faster(batch, in_feat, out_feat)) return 0;
    const int form = vtq::gemm_form(R, out_feat, M, Mt);
    return form == 3 ? 300 + vtq::sk_piece(R, NR * Mt) : form == 2 ? 2 : 1;
}

// The form that an int8 product takes (I8Form in vtq_i8_rules.h).
int vtqp_i8_form(int batch, int in_feat, int out_feat) {
    if (batch <= 0 || in_feat < 0 || out_feat <= 0) return -1;
    return vtq::i8_form(batch, in_feat, out_feat);
}

// What the serving operators refuse: the status that a call with these arguments
// gets before anything is launched, and its text.
int vtqp_check_quantize_i8(const char** text, int x_type, const void* d_x, size_t ld_x, int8_t* d_q, size_t ld_q,
                           float* d_scale, size_t rows, size_t n) {
    return told(vtq::check_quantize_i8(x_type, d_x, ld_x, d_q, ld_q, d_scale, rows, n), text);
}
int vtqp_check_linear_i8(const char** text, const int8_t* d_xq, size_t ld_x, const float* d_x_scale,
                         const int8_t* d_wq, size_t ld_w, const float* d_w_scale, const float* d_bias, int y_type,
                                 void* d_y, size_t ld_y, size_t batch, size_t in_feat, size_t out_feat) {
    return told(vtq::check_linear_i8(d_xq, ld_x, d_x_scale, d_wq, ld_w, d_w_scale, d_bias, y_type, d_y, ld_y, batch,
                                     in_feat, out_feat), text);
}
int vtqp_check_rope_call(const char** text, const vtq_rope* rope, int type, const void* d_x, size_t x_token_stride,
                         size_t x_head_stride, void* d_y, size_t y_token_stride, size_t y_head_stride,
                                 const int32_t* d_pos, size_t tokens, size_t heads, size_t head_dim) {
    return told(vtq::check_rope_call(rope, type, d_x, x_token_stride, x_head_stride, d_y, y_token_stride,
                                     y_head_stride, d_pos, tokens, heads, head_dim), text);
}
int vtqp_check_append(const char** text, const vtq_kv_cache* cache, const vtq_kv_batch* batch, const vtq_rope* rope,
                      int type, size_t tokens, const void* d_k, size_t k_token_stride, size_t k_head_stride,
                              const void* d_v, size_t v_token_stride, size_t v_head_stride, size_t heads,
                                      const void* d_q, size_t q_token_stride, size_t q_head_stride, void* d_q_out,
                                              size_t q_out_token_stride, size_t q_out_head_stride) {
    return told(vtq::check_append(cache, batch, rope, type, tokens, d_k, k_token_stride, k_head_stride, d_v,
                                  v_token_stride, v_head_stride, heads, d_q, q_token_stride, q_head_stride, d_q_out,
                                          q_out_token_stride, q_out_head_stride), text);
}
int vtqp_check_attention(const char** text, const vtq_kv_cache* cache, const vtq_kv_batch* batch, int type,
                         size_t tokens, size_t heads, const void* d_q, size_t q_token_stride, size_t q_head_stride,
                                 void* d_y, size_t y_token_stride, size_t y_head_stride, float* d_lse, float scale) {
    return told(vtq::check_attention(cache, batch, type, tokens, heads, d_q, q_token_stride, q_head_stride, d_y,
                                     y_token_stride, y_head_stride, d_lse, scale), text);
}

// How an attention call that is not refused is split: AttentionPlan, 12 numbers in its
// order (vtq_attention_plan.h), and keys to each own range of a sequence of `keys`.
int vtqp_attention_plan(const vtq_kv_cache* cache, const vtq_kv_batch* batch, int type, size_t tokens, size_t heads,
                        int* out) {
    static_assert(sizeof(vtq::AttentionPlan) == 12 * sizeof(int), "plan");
    if (vtq::Refusal r = vtq::check_cache(cache)) return r.code;
    if (vtq::Refusal r = vtq::check_batch(batch, cache, false)) return r.code;
    if (!vtq::type_bytes(type) || !tokens || tokens > vtq::kMostTokens || !heads || heads > 65535 ||
        heads % cache->kv_heads || !batch->batch || !vtq::attention_fits(cache, batch, tokens, heads))
        return VTQ_E_INVALID_ARGUMENT;
    const vtq::AttentionPlan p = vtq::plan_attention(*cache, *batch, type, (int64_t)tokens, (int)heads);
    __builtin_memcpy(out, &p, sizeof p);
    return VTQ_OK;
}
int vtqp_own_chunk(int keys, int splits, int grain) { return vtq::own_chunk(keys, splits, grain); }

// Where a place of a sequence begins in the cache (vtq_serve.h).
int64_t vtqp_slot_of(const vtq_kv_cache* cache, const int32_t* pages, int max_pages, int64_t place) {
    return vtq::slot_of(*cache, pages, max_pages, place);
}

}  // extern "C"
