// vtq_serve_checks.h -- what the serving operators refuse, before anything is
// launched: host code without a kernel, so that tests can ask it (libvtq_probe.so)
// without a GPU.
#pragma once

#include <climits>
#include <cmath>
#include <cstddef>
#include <cstdint>

#include "../../include/vtq.h"

namespace vtq {

struct Refusal {
    int code = VTQ_OK;
    const char* text = "";
    explicit operator bool() const { return code != VTQ_OK; }
};

inline size_t type_bytes(int type) {
    return type == VTQ_TYPE_F32 ? 4 : type == VTQ_TYPE_F16 || type == VTQ_TYPE_BF16 ? 2 : 0;
}

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
constexpr size_t kMostStride = (size_t)1 << 40;  // no product of sizes below wraps 64 bits
constexpr size_t kMostTokens = (size_t)1 << 23;  // a workgroup a token stays below 2^32 threads

#define VTQ_REFUSE(cond, code, text) \
    if (cond) return Refusal{code, text}

inline Refusal check_rope(const vtq_rope* r) {
    VTQ_REFUSE(r->layout != VTQ_ROPE_INTERLEAVED && r->layout != VTQ_ROPE_HALF, VTQ_E_INVALID_ARGUMENT,
               "vtq: unknown rope layout");
    VTQ_REFUSE(r->rot_dim < 2 || r->rot_dim > 256 || r->rot_dim % 2, VTQ_E_INVALID_SHAPE,
               "vtq: rot_dim must be even, 2 to 256");
    return {};
}

inline Refusal check_cache_layout(const vtq_kv_cache* c) {
    VTQ_REFUSE(c->page_size < 8 || c->page_size > 4096 || (c->page_size & (c->page_size - 1)), VTQ_E_INVALID_SHAPE,
               "vtq: page_size must be a power of two, 8 to 4096");
    VTQ_REFUSE(c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8, VTQ_E_INVALID_SHAPE,
               "vtq: head_dim must be a multiple of 8, 8 to 256");
    VTQ_REFUSE(c->kv_heads < 1 || c->kv_heads > 65535, VTQ_E_INVALID_SHAPE, "vtq: kv_heads must be 1 to 65535");
    VTQ_REFUSE(c->n_pages > (size_t)INT_MAX, VTQ_E_NOT_IMPLEMENTED, "vtq: page count exceeds INT_MAX");
    VTQ_REFUSE(c->page_stride % 8 || c->head_stride % 8 || c->slot_stride % 8, VTQ_E_INVALID_SHAPE,
               "vtq: cache strides must be multiples of 8 elements");
    VTQ_REFUSE(c->slot_stride < (size_t)c->head_dim || (c->kv_heads > 1 && c->head_stride < (size_t)c->head_dim),
               VTQ_E_INVALID_SHAPE, "vtq: cache strides below head_dim");
    VTQ_REFUSE(c->slot_stride >= (size_t)1 << 24 || c->head_stride >= kMostStride / 4 ||
                   c->page_stride >= kMostStride / 4,
               VTQ_E_NOT_IMPLEMENTED, "vtq: cache stride too large");
    VTQ_REFUSE((size_t)c->page_size * c->slot_stride >= (size_t)1 << 29, VTQ_E_NOT_IMPLEMENTED,
               "vtq: the slots of a page span more than 2^29 elements");
    VTQ_REFUSE(c->n_pages * (c->page_stride / 8) > (size_t)1 << 43, VTQ_E_NOT_IMPLEMENTED, "vtq: cache too large");
    VTQ_REFUSE(c->n_pages && (!c->k || !c->v), VTQ_E_INVALID_ARGUMENT, "vtq: null cache");
    VTQ_REFUSE(!aligned(c->k, 16) || !aligned(c->v, 16), VTQ_E_INVALID_ARGUMENT,
               "vtq: the cache must be 16-byte aligned");
    return {};
}

inline Refusal check_cache(const vtq_kv_cache* c) {
    VTQ_REFUSE(type_bytes(c->type) == 0, VTQ_E_NOT_IMPLEMENTED, "vtq: cache type not F32 / F16 / BF16");
    return check_cache_layout(c);
}

inline Refusal check_cache8(const vtq_kv8_cache* c) {
    VTQ_REFUSE(c->cache.type != VTQ_TYPE_E4M3, VTQ_E_NOT_IMPLEMENTED, "vtq: the type of an 8-bit cache is E4M3");
    if (Refusal r = check_cache_layout(&c->cache)) return r;
    const vtq_kv_cache& b = c->cache;
    VTQ_REFUSE(b.page_size < 16, VTQ_E_INVALID_SHAPE, "vtq: pages of an 8-bit cache hold at least 16 tokens");
    VTQ_REFUSE(b.head_dim % 16 || b.page_stride % 16 || b.head_stride % 16 || b.slot_stride % 16, VTQ_E_INVALID_SHAPE,
               "vtq: head_dim and strides of an 8-bit cache must be multiples of 16");
    VTQ_REFUSE(c->block < 16 || c->block > b.page_size || (c->block & (c->block - 1)), VTQ_E_INVALID_SHAPE,
               "vtq: tokens to a scale must be a power of two, 16 to page_size");
    const size_t blocks = (size_t)(b.page_size / c->block);
    VTQ_REFUSE((b.kv_heads > 1 && c->scale_head_stride < blocks) || (b.n_pages > 1 && c->scale_page_stride < blocks),
               VTQ_E_INVALID_SHAPE, "vtq: scale strides below the blocks of a page");
    VTQ_REFUSE(c->scale_page_stride >= kMostStride / 4 || c->scale_head_stride >= kMostStride / 4 ||
                   b.n_pages * c->scale_page_stride > (size_t)1 << 46,
               VTQ_E_NOT_IMPLEMENTED, "vtq: scale stride too large");
    VTQ_REFUSE(b.n_pages && (!c->k_scale || !c->v_scale), VTQ_E_INVALID_ARGUMENT, "vtq: null scales");
    return {};
}

inline Refusal check_batch(const vtq_kv_batch* b, const vtq_kv_cache* c, bool reads_prefix) {
    VTQ_REFUSE(b->batch < 0 || b->max_pages < 0 || b->max_q < 0 || b->max_len < 0 || b->prefix_len < 0,
               VTQ_E_INVALID_ARGUMENT, "vtq: negative size in the batch");
    VTQ_REFUSE(b->batch > 1 << 20, VTQ_E_NOT_IMPLEMENTED, "vtq: more than 2^20 sequences");
    VTQ_REFUSE((int64_t)b->max_pages * c->page_size > INT_MAX / 2 || b->prefix_len > INT_MAX / 2, VTQ_E_NOT_IMPLEMENTED,
               "vtq: sequence length beyond 2^30");
    VTQ_REFUSE(b->batch && (!b->q_start || !b->len || (b->max_pages && !b->pages)), VTQ_E_INVALID_ARGUMENT,
               "vtq: null list in the batch");
    VTQ_REFUSE(reads_prefix && b->prefix_len && !b->prefix_pages, VTQ_E_INVALID_ARGUMENT, "vtq: null prefix_pages");
    VTQ_REFUSE(!aligned(b->q_start, 4) || !aligned(b->len, 4) || !aligned(b->pages, 4) ||
                   (reads_prefix && !aligned(b->prefix_pages, 4)),
               VTQ_E_INVALID_ARGUMENT, "vtq: list in the batch not aligned to its type");
    return {};
}

inline Refusal check_rows(const void* p, size_t token_stride, size_t head_stride, size_t head_dim, size_t heads,
                          int type, size_t tokens) {
    VTQ_REFUSE(!p, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    VTQ_REFUSE(!aligned(p, type_bytes(type)), VTQ_E_INVALID_ARGUMENT, "vtq: pointer not aligned to its type");
    VTQ_REFUSE((heads > 1 && head_stride < head_dim) || (tokens > 1 && token_stride < head_dim), VTQ_E_INVALID_SHAPE,
               "vtq: token or head stride below head_dim");
    VTQ_REFUSE(token_stride >= kMostStride / 4 || head_stride >= kMostStride / 4, VTQ_E_NOT_IMPLEMENTED,
               "vtq: stride too large");
    return {};
}

// Whether the launches stay below 2^32 threads: 256 of them to 4 rows of queries, and
// to a sequence, KV head and 32 rows.
inline bool attention_fits(const vtq_kv_cache* c, const vtq_kv_batch* b, size_t tokens, size_t heads,
                           size_t most = (size_t)1 << 22) {
    const size_t max_q = (size_t)b->max_q < tokens ? (size_t)b->max_q : tokens;
    return tokens * heads <= (size_t)1 << 25 &&
           (size_t)b->batch * (size_t)c->kv_heads * (max_q * (heads / (size_t)c->kv_heads) / 32 + 1) <= most;
}
// Over an 8-bit cache two workgroups take a head of more than 128 elements, in two ranges at least.
inline size_t most_kv8_workgroups(const vtq_kv_cache* c) { return (size_t)1 << (c->head_dim > 128 ? 20 : 22); }

// A plan from its parameters.
inline Refusal plan_rope(const vtq_rope_params* p, vtq_rope* out) {
    VTQ_REFUSE(!p || !out, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    vtq_rope r{};
    r.layout = p->layout;
    r.rot_dim = p->rot_dim;
    if (Refusal bad = check_rope(&r)) return bad;
    VTQ_REFUSE(p->scaling < VTQ_ROPE_SCALE_NONE || p->scaling > VTQ_ROPE_SCALE_YARN, VTQ_E_INVALID_ARGUMENT,
               "vtq: unknown rope scaling");
    VTQ_REFUSE(!std::isfinite(p->theta) || p->theta <= 1.0, VTQ_E_INVALID_ARGUMENT, "vtq: theta must be above 1");
    VTQ_REFUSE(!(p->magnitude >= 0.0 && p->magnitude <= 1e30), VTQ_E_INVALID_ARGUMENT,
               "vtq: magnitude must be 0 to 1e30");
    const bool ramp = p->scaling == VTQ_ROPE_SCALE_BANDS || p->scaling == VTQ_ROPE_SCALE_YARN;
    VTQ_REFUSE(p->scaling != VTQ_ROPE_SCALE_NONE && (!std::isfinite(p->factor) || p->factor < 1.0),
               VTQ_E_INVALID_ARGUMENT, "vtq: factor must be at least 1");
    VTQ_REFUSE(ramp && p->original_context <= 0, VTQ_E_INVALID_ARGUMENT, "vtq: original_context must be positive");
    const double two_pi = 6.283185307179586476925286766559;
    const bool bands = p->scaling == VTQ_ROPE_SCALE_BANDS;
    const double low = p->low != 0.0 ? p->low : 1.0, high = p->high != 0.0 ? p->high : bands ? 4.0 : 32.0;
    VTQ_REFUSE(ramp && !(low > 0.0 && high > low && std::isfinite(high)), VTQ_E_INVALID_ARGUMENT,
               "vtq: rope ramp must have 0 < low < high");
    const int dim = p->rot_dim;
    // the pair index (a real number) whose frequency makes `turns` turns in the original context
    auto index_at = [&](double turns) {
        return dim * std::log(p->original_context / (turns * two_pi)) / (2.0 * std::log(p->theta));
    };
    double first = 0.0, last = 0.0;
    if (p->scaling == VTQ_ROPE_SCALE_YARN) {
        first = std::fmax(std::floor(index_at(high)), 0.0);
        last = std::fmin(std::ceil(index_at(low)), dim - 1.0);
    }
    // Frequencies in the host's 64-bit mantissas: positions of up to 2^31 multiply what they
    // are off by, and doubles' 2^-53 would come out as 2^-22 of a radian.
    const long double full = 6.283185307179586476925286766559005768L;
    for (int i = 0; i < dim / 2; i++) {
        long double f = std::exp(-2.0L * i / dim * std::log((long double)p->theta));
        if (p->factors) {
            const double d = p->factors[i];
            VTQ_REFUSE(!std::isfinite(d) || d <= 0.0, VTQ_E_INVALID_ARGUMENT, "vtq: rope factors must be positive");
            f /= d;
        }
        long double keep = 1.0L;  // the share of the unscaled frequency
        if (p->scaling == VTQ_ROPE_SCALE_LINEAR) keep = 0.0L;
        else if (bands) keep = (p->original_context * f / full - low) / ((long double)high - low);
        else if (ramp) keep = 1.0L - (i - (long double)first) / std::fmax(last - first, 0.001);
        keep = std::fmin(1.0L, std::fmax(0.0L, keep));
        if (keep < 1.0L) f = keep * f + (1.0L - keep) * f / p->factor;
        // f <= 1 radian a position unless a factor below 1 says otherwise; whole turns do not count
        const long double turns = f / full;
        VTQ_REFUSE(!(turns < 1048576.0L), VTQ_E_INVALID_ARGUMENT, "vtq: rope frequency too large");
        r.turns[i] = (uint64_t)((turns - std::floor(turns)) * 18446744073709551616.0L);
    }
    r.magnitude = p->magnitude != 0.0                           ? (float)p->magnitude
                  : p->scaling == VTQ_ROPE_SCALE_YARN ? (float)(0.1 * std::log(p->factor) + 1.0)
                                                      : 1.0f;
    *out = r;
    return {};
}

inline Refusal check_quantize_i8(int x_type, const void* d_x, size_t ld_x, int8_t* d_q, size_t ld_q, float* d_scale,
                                 size_t rows, size_t n) {
    VTQ_REFUSE(type_bytes(x_type) == 0, VTQ_E_NOT_IMPLEMENTED, "vtq: activation type not F32 / F16 / BF16");
    VTQ_REFUSE(n > 131071 || rows > (size_t)INT_MAX, VTQ_E_NOT_IMPLEMENTED,
               "vtq: int8 rows hold at most 131071 inputs, and rows at most INT_MAX");
    VTQ_REFUSE(ld_q % 16 || ld_q < n || (rows > 1 && ld_x < n), VTQ_E_INVALID_SHAPE,
               "vtq: int8 rows start at multiples of 16 bytes and are at least as long as their inputs");
    VTQ_REFUSE(ld_x >= kMostStride || ld_q >= kMostStride, VTQ_E_NOT_IMPLEMENTED, "vtq: stride too large");
    if (rows == 0) return {};
    VTQ_REFUSE((n && !d_x) || (ld_q && !d_q) || !d_scale, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    VTQ_REFUSE(!aligned(d_x, type_bytes(x_type)) || !aligned(d_q, 16) || !aligned(d_scale, 4), VTQ_E_INVALID_ARGUMENT,
               "vtq: int8 data must be 16-byte aligned, x and scales to their type");
    return {};
}

inline Refusal check_linear_i8(const int8_t* d_xq, size_t ld_x, const float* d_x_scale, const int8_t* d_wq,
                               size_t ld_w, const float* d_w_scale, const float* d_bias, int y_type, void* d_y,
                                       size_t ld_y, size_t batch, size_t in_feat, size_t out_feat) {
    VTQ_REFUSE(type_bytes(y_type) == 0, VTQ_E_NOT_IMPLEMENTED, "vtq: output type not F32 / F16 / BF16");
    VTQ_REFUSE(in_feat > 131071 || batch > (size_t)INT_MAX / 2 || out_feat > (size_t)INT_MAX / 2, VTQ_E_NOT_IMPLEMENTED,
               "vtq: int8 rows hold at most 131071 inputs, and batch and out_feat at most INT_MAX / 2");
    VTQ_REFUSE(ld_x % 16 || ld_w % 16 || ld_x < in_feat || ld_w < in_feat || (batch > 1 && ld_y < out_feat),
               VTQ_E_INVALID_SHAPE,
               "vtq: int8 rows start at multiples of 16 bytes and are at least as long as their inputs");
    VTQ_REFUSE(ld_x >= (size_t)1 << 22 || ld_w >= (size_t)1 << 22 || ld_y >= kMostStride, VTQ_E_NOT_IMPLEMENTED,
               "vtq: stride too large");
    if (batch == 0 || out_feat == 0) return {};
    VTQ_REFUSE((in_feat && (!d_xq || !d_wq || !d_x_scale || !d_w_scale)) || !d_y, VTQ_E_INVALID_ARGUMENT,
               "vtq: null pointer");
    VTQ_REFUSE(!aligned(d_xq, 16) || !aligned(d_wq, 16) || !aligned(d_x_scale, 4) || !aligned(d_w_scale, 4) ||
                   !aligned(d_bias, 4) || !aligned(d_y, type_bytes(y_type)),
               VTQ_E_INVALID_ARGUMENT, "vtq: int8 data must be 16-byte aligned, y, scales and bias to their type");
    return {};
}

inline Refusal check_rope_call(const vtq_rope* rope, int type, const void* d_x, size_t x_token_stride,
                               size_t x_head_stride, void* d_y, size_t y_token_stride, size_t y_head_stride,
                                       const int32_t* d_pos, size_t tokens, size_t heads, size_t head_dim) {
    VTQ_REFUSE(!rope, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    if (Refusal r = check_rope(rope)) return r;
    VTQ_REFUSE(type_bytes(type) == 0, VTQ_E_NOT_IMPLEMENTED, "vtq: activation type not F32 / F16 / BF16");
    VTQ_REFUSE(tokens > kMostTokens || heads > 65535 || head_dim > 8192, VTQ_E_NOT_IMPLEMENTED,
               "vtq: too many tokens, heads or elements of a head");
    VTQ_REFUSE((size_t)rope->rot_dim > head_dim, VTQ_E_INVALID_SHAPE, "vtq: rot_dim exceeds head_dim");
    if (tokens == 0 || heads == 0) return {};
    if (Refusal r = check_rows(d_x, x_token_stride, x_head_stride, head_dim, heads, type, tokens)) return r;
    if (Refusal r = check_rows(d_y, y_token_stride, y_head_stride, head_dim, heads, type, tokens)) return r;
    VTQ_REFUSE(d_x == d_y && (x_token_stride != y_token_stride || x_head_stride != y_head_stride),
               VTQ_E_INVALID_SHAPE, "vtq: a rotation in place keeps its strides");
    VTQ_REFUSE(!d_pos || !aligned(d_pos, 4), VTQ_E_INVALID_ARGUMENT, "vtq: null or unaligned positions");
    return {};
}

// What an append's arguments have to be with a cache of any type.
inline Refusal check_append_rows(const vtq_kv_cache* cache, const vtq_kv_batch* batch, const vtq_rope* rope, int type,
                            size_t tokens, const void* d_k, size_t k_token_stride, size_t k_head_stride,
                                    const void* d_v, size_t v_token_stride, size_t v_head_stride, size_t heads,
                                            const void* d_q, size_t q_token_stride, size_t q_head_stride,
                                                    void* d_q_out, size_t q_out_token_stride,
                                                            size_t q_out_head_stride) {
    if (Refusal r = check_batch(batch, cache, false)) return r;
    VTQ_REFUSE(type_bytes(type) == 0, VTQ_E_NOT_IMPLEMENTED, "vtq: activation type not F32 / F16 / BF16");
    VTQ_REFUSE(tokens > kMostTokens || heads > 65535, VTQ_E_NOT_IMPLEMENTED, "vtq: too many tokens or heads");
    if (rope) {
        if (Refusal r = check_rope(rope)) return r;
        VTQ_REFUSE(rope->rot_dim > cache->head_dim, VTQ_E_INVALID_SHAPE, "vtq: rot_dim exceeds head_dim");
    }
    if (tokens == 0 || batch->batch == 0) return {};
    const size_t hd = cache->head_dim, hk = cache->kv_heads;
    if (Refusal r = check_rows(d_k, k_token_stride, k_head_stride, hd, hk, type, tokens)) return r;
    if (Refusal r = check_rows(d_v, v_token_stride, v_head_stride, hd, hk, type, tokens)) return r;
    const bool with_q = d_q && heads;
    if (with_q) {
        if (Refusal r = check_rows(d_q, q_token_stride, q_head_stride, hd, heads, type, tokens)) return r;
        if (Refusal r = check_rows(d_q_out, q_out_token_stride, q_out_head_stride, hd, heads, type, tokens)) return r;
        VTQ_REFUSE(d_q == d_q_out && (q_token_stride != q_out_token_stride || q_head_stride != q_out_head_stride),
                   VTQ_E_INVALID_SHAPE, "vtq: a rotation in place keeps its strides");
    }
    return {};
}

inline Refusal check_append(const vtq_kv_cache* cache, const vtq_kv_batch* batch, const vtq_rope* rope, int type,
                            size_t tokens, const void* d_k, size_t k_token_stride, size_t k_head_stride,
                            const void* d_v, size_t v_token_stride, size_t v_head_stride, size_t heads,
                            const void* d_q, size_t q_token_stride, size_t q_head_stride, void* d_q_out,
                            size_t q_out_token_stride, size_t q_out_head_stride) {
    VTQ_REFUSE(!cache || !batch, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    if (Refusal r = check_cache(cache)) return r;
    if (Refusal r = check_batch(batch, cache, false)) return r;
    VTQ_REFUSE(type_bytes(type) != 0 && type != VTQ_TYPE_F32 && type != cache->type, VTQ_E_NOT_IMPLEMENTED,
               "vtq: activations are F32 or of the cache's type");
    return check_append_rows(cache, batch, rope, type, tokens, d_k, k_token_stride, k_head_stride, d_v, v_token_stride,
                             v_head_stride, heads, d_q, q_token_stride, q_head_stride, d_q_out, q_out_token_stride,
                             q_out_head_stride);
}

inline Refusal check_kv8_append(const vtq_kv8_cache* cache, const vtq_kv_batch* batch, const vtq_rope* rope, int type,
                                size_t tokens, const void* d_k, size_t k_token_stride, size_t k_head_stride,
                                const void* d_v, size_t v_token_stride, size_t v_head_stride, size_t heads,
                                const void* d_q, size_t q_token_stride, size_t q_head_stride, void* d_q_out,
                                size_t q_out_token_stride, size_t q_out_head_stride) {
    VTQ_REFUSE(!cache || !batch, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    if (Refusal r = check_cache8(cache)) return r;
    // workgroups, one to 16 heads of a token at least, stay below 2^24 of 256 threads
    VTQ_REFUSE(tokens > kMostTokens || tokens * (size_t)cache->cache.kv_heads > (size_t)1 << 26, VTQ_E_NOT_IMPLEMENTED,
               "vtq: too many tokens or heads");
    return check_append_rows(&cache->cache, batch, rope, type, tokens, d_k, k_token_stride, k_head_stride, d_v,
                             v_token_stride, v_head_stride, heads, d_q, q_token_stride, q_head_stride, d_q_out,
                             q_out_token_stride, q_out_head_stride);
}

// What attention's arguments have to be with a cache of any type.
inline Refusal check_attention_rows(const vtq_kv_cache* cache, const vtq_kv_batch* batch, int type, size_t tokens,
                                    size_t heads, const void* d_q, size_t q_token_stride, size_t q_head_stride, void* d_y,
                                    size_t y_token_stride, size_t y_head_stride, float* d_lse, float scale,
                                    size_t most = (size_t)1 << 22) {
    VTQ_REFUSE(tokens > kMostTokens || heads > 65535, VTQ_E_NOT_IMPLEMENTED, "vtq: too many tokens or heads");
    VTQ_REFUSE(heads % cache->kv_heads, VTQ_E_INVALID_SHAPE, "vtq: heads must be a multiple of kv_heads");
    VTQ_REFUSE(!attention_fits(cache, batch, tokens, heads, most), VTQ_E_NOT_IMPLEMENTED, "vtq: more than 2^25 rows of queries");
    VTQ_REFUSE(!(scale > 0.0f && scale <= 1e30f), VTQ_E_INVALID_ARGUMENT, "vtq: scale must be positive, up to 1e30");
    if (tokens == 0 || heads == 0 || batch->batch == 0) return {};
    const size_t hd = cache->head_dim, es = type_bytes(type);
    if (Refusal r = check_rows(d_q, q_token_stride, q_head_stride, hd, heads, type, tokens)) return r;
    if (Refusal r = check_rows(d_y, y_token_stride, y_head_stride, hd, heads, type, tokens)) return r;
    VTQ_REFUSE(!aligned(d_q, 16) || !aligned(d_y, 16) || q_token_stride * es % 16 || q_head_stride * es % 16 ||
                   y_token_stride * es % 16 || y_head_stride * es % 16,
               VTQ_E_INVALID_ARGUMENT, "vtq: attention rows must start at multiples of 16 bytes");
    VTQ_REFUSE(d_q == d_y && (q_token_stride != y_token_stride || q_head_stride != y_head_stride),
               VTQ_E_INVALID_SHAPE, "vtq: attention in place keeps its strides");
    VTQ_REFUSE(d_lse && !aligned(d_lse, 4), VTQ_E_INVALID_ARGUMENT, "vtq: lse not aligned to its type");
    return {};
}

inline Refusal check_attention(const vtq_kv_cache* cache, const vtq_kv_batch* batch, int type, size_t tokens,
                               size_t heads, const void* d_q, size_t q_token_stride, size_t q_head_stride, void* d_y,
                               size_t y_token_stride, size_t y_head_stride, float* d_lse, float scale) {
    VTQ_REFUSE(!cache || !batch, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    if (Refusal r = check_cache(cache)) return r;
    if (Refusal r = check_batch(batch, cache, true)) return r;
    VTQ_REFUSE(type_bytes(type) == 0 || (type != VTQ_TYPE_F32 && type != cache->type), VTQ_E_NOT_IMPLEMENTED,
               "vtq: activations are F32 or of the cache's type");
    return check_attention_rows(cache, batch, type, tokens, heads, d_q, q_token_stride, q_head_stride, d_y,
                                y_token_stride, y_head_stride, d_lse, scale);
}

inline Refusal check_kv8_attention(const vtq_kv8_cache* cache, const vtq_kv_batch* batch, int type, size_t tokens,
                                   size_t heads, const void* d_q, size_t q_token_stride, size_t q_head_stride,
                                   void* d_y, size_t y_token_stride, size_t y_head_stride, float* d_lse, float scale) {
    VTQ_REFUSE(!cache || !batch, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    if (Refusal r = check_cache8(cache)) return r;
    if (Refusal r = check_batch(batch, &cache->cache, true)) return r;
    VTQ_REFUSE(type_bytes(type) == 0, VTQ_E_NOT_IMPLEMENTED, "vtq: activation type not F32 / F16 / BF16");
    return check_attention_rows(&cache->cache, batch, type, tokens, heads, d_q, q_token_stride, q_head_stride, d_y,
                                y_token_stride, y_head_stride, d_lse, scale, most_kv8_workgroups(&cache->cache));
}

constexpr size_t kMostKept = 64;  // continuations and beams of a group

inline bool beam_select_fits(size_t groups, size_t beams, size_t vocab, size_t n_out) {
    return beams <= kMostKept && n_out <= kMostKept && vocab <= (size_t)1 << 20 && groups <= (size_t)1 << 20 &&
           groups * beams <= (size_t)1 << 20;
}

inline Refusal check_beam_select(int type, const void* d_logits, size_t ld, size_t groups, size_t beams, size_t vocab,
                                 const float* d_score, const uint8_t* d_done, int end_token, size_t n_out,
                                 float* d_out_score, int32_t* d_out_token, int32_t* d_out_parent,
                                 uint8_t* d_out_done) {
    VTQ_REFUSE(type_bytes(type) == 0, VTQ_E_NOT_IMPLEMENTED, "vtq: logits type not F32 / F16 / BF16");
    VTQ_REFUSE(!beam_select_fits(groups, beams, vocab, n_out), VTQ_E_NOT_IMPLEMENTED, "vtq: at most 64 beams and continuations, 2^20 tokens and 2^20 rows");
    VTQ_REFUSE(beams == 0 || vocab == 0 || n_out == 0, VTQ_E_INVALID_SHAPE, "vtq: no beams, tokens or continuations");
    VTQ_REFUSE(groups * beams > 1 && ld < vocab, VTQ_E_INVALID_SHAPE, "vtq: rows of logits overlap");
    VTQ_REFUSE(ld >= kMostStride / 4, VTQ_E_NOT_IMPLEMENTED, "vtq: stride too large");
    VTQ_REFUSE(end_token >= 0 && (size_t)end_token >= vocab, VTQ_E_INVALID_ARGUMENT, "vtq: end_token outside the vocabulary");
    if (groups == 0) return {};
    VTQ_REFUSE(!d_logits || !d_score || !d_out_score || !d_out_token || !d_out_parent, VTQ_E_INVALID_ARGUMENT,
               "vtq: null pointer");
    VTQ_REFUSE(!aligned(d_logits, type_bytes(type)) || !aligned(d_score, 4) || !aligned(d_out_score, 4) ||
                   !aligned(d_out_token, 4) || !aligned(d_out_parent, 4),
               VTQ_E_INVALID_ARGUMENT, "vtq: pointer not aligned to its type");
    VTQ_REFUSE(n_out != beams && ((d_done && d_done == d_out_done) || d_score == d_out_score), VTQ_E_INVALID_SHAPE,
               "vtq: scores and ends are replaced in place only where n_out is beams");
    return {};
}

// Each workgroup adds up the counts of 1024 pages.
constexpr size_t kMostPages = (size_t)1 << 24;

inline Refusal check_pages(size_t n_pages, int page_size, const int32_t* d_refs, const int32_t* d_new_refs,
                           const int32_t* d_copies, const int32_t* d_info) {
    VTQ_REFUSE(n_pages > kMostPages, VTQ_E_NOT_IMPLEMENTED, "vtq: more than 2^24 pages");
    VTQ_REFUSE(page_size < 8 || page_size > 4096 || (page_size & (page_size - 1)), VTQ_E_INVALID_SHAPE,
               "vtq: page_size must be a power of two, 8 to 4096");
    VTQ_REFUSE((n_pages && (!d_refs || !d_new_refs)) || !d_info, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    VTQ_REFUSE(!aligned(d_refs, 4) || !aligned(d_new_refs, 4) || !aligned(d_copies, 4) || !aligned(d_info, 4),
               VTQ_E_INVALID_ARGUMENT, "vtq: list not aligned to its type");
    VTQ_REFUSE(n_pages && d_refs == d_new_refs, VTQ_E_INVALID_ARGUMENT, "vtq: the new lists stand beside the old ones");
    return {};
}

// Each sequence looks through the list of parents.
constexpr size_t kMostReordered = (size_t)1 << 16;

inline Refusal check_pages_reorder(size_t n_pages, int page_size, size_t max_pages, const int32_t* d_refs, size_t batch,
                                   const int32_t* d_pages, const int32_t* d_len, size_t batch_out,
                                   const int32_t* d_parent, const int32_t* d_grow, int32_t* d_new_refs,
                                   int32_t* d_new_pages, int32_t* d_new_len, int32_t* d_copies, int32_t* d_info) {
    if (Refusal r = check_pages(n_pages, page_size, d_refs, d_new_refs, d_copies, d_info)) return r;
    VTQ_REFUSE(batch > kMostReordered || batch_out > kMostReordered, VTQ_E_NOT_IMPLEMENTED,
               "vtq: more than 2^16 sequences");
    VTQ_REFUSE(max_pages > (size_t)(INT_MAX / 2) / page_size, VTQ_E_NOT_IMPLEMENTED, "vtq: page table too large");
    VTQ_REFUSE(batch && ((max_pages && !d_pages) || !d_len), VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    VTQ_REFUSE(batch_out && ((max_pages && !d_new_pages) || !d_new_len || !d_parent || !d_copies),
               VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    VTQ_REFUSE(!aligned(d_pages, 4) || !aligned(d_len, 4) || !aligned(d_parent, 4) || !aligned(d_grow, 4) ||
                   !aligned(d_new_pages, 4) || !aligned(d_new_len, 4),
               VTQ_E_INVALID_ARGUMENT, "vtq: list not aligned to its type");
    VTQ_REFUSE(batch && batch_out && (d_len == d_new_len || (max_pages && d_pages == d_new_pages)),
               VTQ_E_INVALID_ARGUMENT, "vtq: the new lists stand beside the old ones");
    return {};
}

inline Refusal check_pages_compact(size_t n_pages, int page_size, const int32_t* d_refs, size_t n_entries,
                                   const int32_t* d_pages, size_t n_prefix, const int32_t* d_prefix_pages,
                                   int32_t* d_new_refs, int32_t* d_new_pages, int32_t* d_new_prefix_pages,
                                   int32_t* d_copies, int32_t* d_info) {
    if (Refusal r = check_pages(n_pages, page_size, d_refs, d_new_refs, d_copies, d_info)) return r;
    VTQ_REFUSE(n_entries > (size_t)INT_MAX || n_prefix > (size_t)INT_MAX, VTQ_E_NOT_IMPLEMENTED,
               "vtq: page table too large");
    VTQ_REFUSE((n_pages > 1 && !d_copies) || (n_entries && (!d_pages || !d_new_pages)) ||
                   (n_prefix && (!d_prefix_pages || !d_new_prefix_pages)),
               VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    VTQ_REFUSE(!aligned(d_pages, 4) || !aligned(d_prefix_pages, 4) || !aligned(d_new_pages, 4) ||
                   !aligned(d_new_prefix_pages, 4),
               VTQ_E_INVALID_ARGUMENT, "vtq: list not aligned to its type");
    return {};
}

inline Refusal check_copies(const vtq_kv_cache* c, size_t layers, size_t layer_stride, const int32_t* d_copies,
                            size_t max_copies, const int32_t* d_count) {
    VTQ_REFUSE(layers > 65535 || max_copies > (size_t)INT_MAX, VTQ_E_NOT_IMPLEMENTED, "vtq: too many layers or copies");
    VTQ_REFUSE((size_t)c->kv_heads * c->page_size * c->head_dim > (size_t)1 << 31, VTQ_E_NOT_IMPLEMENTED,
               "vtq: pages of more than 2^31 elements");
    VTQ_REFUSE(layer_stride >= kMostStride || layers * (layer_stride / 8) > (size_t)1 << 43, VTQ_E_NOT_IMPLEMENTED,
               "vtq: layer stride too large");
    VTQ_REFUSE(layers > 1 && layer_stride == 0, VTQ_E_INVALID_SHAPE, "vtq: layers overlap");
    VTQ_REFUSE(layer_stride % (c->type == VTQ_TYPE_E4M3 ? 16 : 8), VTQ_E_INVALID_SHAPE,
               "vtq: the layer stride must be a multiple of 8 elements, of 16 in 8 bits");
    VTQ_REFUSE(layers && max_copies && !d_copies, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    VTQ_REFUSE(!aligned(d_copies, 4) || !aligned(d_count, 4), VTQ_E_INVALID_ARGUMENT,
               "vtq: list not aligned to its type");
    return {};
}

inline Refusal check_pages_copy(const vtq_kv_cache* cache, size_t layers, size_t layer_stride, const int32_t* d_copies,
                                size_t max_copies, const int32_t* d_count) {
    VTQ_REFUSE(!cache, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    if (Refusal r = check_cache(cache)) return r;
    return check_copies(cache, layers, layer_stride, d_copies, max_copies, d_count);
}

inline Refusal check_kv8_pages_copy(const vtq_kv8_cache* cache, size_t layers, size_t layer_stride,
                                    size_t scale_layer_stride, const int32_t* d_copies, size_t max_copies,
                                    const int32_t* d_count) {
    VTQ_REFUSE(!cache, VTQ_E_INVALID_ARGUMENT, "vtq: null pointer");
    if (Refusal r = check_cache8(cache)) return r;
    if (Refusal r = check_copies(&cache->cache, layers, layer_stride, d_copies, max_copies, d_count)) return r;
    VTQ_REFUSE(scale_layer_stride >= kMostStride || layers * scale_layer_stride > (size_t)1 << 46, VTQ_E_NOT_IMPLEMENTED,
               "vtq: layer stride too large");
    VTQ_REFUSE(layers > 1 && scale_layer_stride == 0, VTQ_E_INVALID_SHAPE, "vtq: layers overlap");
    return {};
}

#undef VTQ_REFUSE

}  // namespace vtq
