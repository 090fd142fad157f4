// vtq_serve.h -- internal interface of the serving operators: the launchers
// behind vtq_serve_api.hip and the device types they share.  Pointers are device
// pointers, arguments validated by the caller, launches asynchronous.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/vtq.h"
#include "vtq_serve_checks.h"

namespace vtq {

// The context's part in a call (vtq_api.hip).
int ctx_error(vtq_ctx* c, int code, const char* text) noexcept;
int ctx_hip_error(vtq_ctx* c, hipError_t e, const char* where) noexcept;
int ctx_device(const vtq_ctx* c);

// Calls f with a value of the C++ type behind a type tag.
template <class F>
hipError_t with_type(int type, F f) {
    if (type == VTQ_TYPE_F32) return f(float{});
    if (type == VTQ_TYPE_F16) return f(_Float16{});
    return f(__bf16{});
}

// Where place `place` of a sequence with these pages begins in the cache (elements,
// KV head 0), or -1 where it has no slot.
__host__ __device__ inline int64_t slot_of(const vtq_kv_cache& c, const int32_t* pages, int max_pages, int64_t place) {
    if (place < 0 || place / c.page_size >= max_pages) return -1;
    const int64_t page = pages[place / c.page_size];
    if (page < 0 || page >= (int64_t)c.n_pages) return -1;
    return page * (int64_t)c.page_stride + (place & (c.page_size - 1)) * (int64_t)c.slot_stride;
}

// tokens x heads x head_dim, strides in elements
struct HeadRows {
    const void* p;
    int64_t token_stride, head_stride;
};

hipError_t launch_quantize_i8(int type, const void* x, size_t ld_x, int8_t* q, size_t ld_q, float* scale, size_t rows,
                              int n, hipStream_t stream);

struct I8Linear {
    const int8_t *x, *w;
    const float *xs, *ws, *bias;
    void* y;
    size_t ld_x, ld_w, ld_y;
    int batch, in_feat, out_feat;
};
hipError_t launch_linear_i8(const I8Linear& a, int y_type, hipStream_t stream);

// Rotation of x to y, and (cache set) keys and values into their slots.
struct RopeJob {
    vtq_rope rope;
    int rotate;  // 0: every pair as it is
    int64_t tokens;
    int head_dim, x_heads, kv_heads;
    HeadRows x, k, v;
    void* y;
    int64_t y_token_stride, y_head_stride;
    const int32_t* pos;  // null: from the batch
    vtq_kv_cache cache;
    vtq_kv_batch batch;
};
hipError_t launch_rope(const RopeJob& j, int type, int cache_type, hipStream_t stream);

struct Attention {
    vtq_kv_cache cache;
    vtq_kv_batch batch;
    int64_t tokens;
    int heads;
    HeadRows q;
    void* y;
    int64_t y_token_stride, y_head_stride;
    float* lse;
    float scale;
    void* ws;
};
// Scales of an 8-bit cache.
struct Scales {
    int block;
    uint8_t *k, *v;
    int64_t page_stride, head_stride;
};

// The same append into an 8-bit cache.
hipError_t launch_kv8_append(const RopeJob& j, const Scales& s, int type, hipStream_t stream);

size_t attention_workspace(const vtq_kv_cache& cache, const vtq_kv_batch& batch, int type, int64_t tokens, int heads);
hipError_t launch_attention(const Attention& a, int type, hipStream_t stream);
size_t kv8_attention_workspace(const vtq_kv_cache& cache, const vtq_kv_batch& batch, int type, int64_t tokens, int heads);
hipError_t launch_kv8_attention(const Attention& a, const Scales& s, int type, hipStream_t stream);

struct BeamSelect {
    const void* logits;
    int64_t ld;
    int groups, beams, vocab, n_out, end_token;
    const float* score;
    const uint8_t* done;
    float* out_score;
    int32_t *out_token, *out_parent;
    uint8_t* out_done;
    void* ws;
};
size_t beam_select_workspace(int64_t groups, int64_t beams, int64_t vocab, int64_t n_out);
hipError_t launch_beam_select(const BeamSelect& a, int type, hipStream_t stream);

struct PagesReorder {
    int64_t n_pages;
    int page_size, max_pages, batch, batch_out;
    const int32_t *refs, *pages, *len, *parent, *grow;
    int32_t *new_refs, *new_pages, *new_len, *copies, *info;
    void* ws;
};
size_t pages_reorder_workspace(int64_t n_pages, int64_t batch_out);
hipError_t launch_pages_reorder(const PagesReorder& a, hipStream_t stream);

struct PagesCompact {
    int64_t n_pages;
    int page_size;
    int64_t n_entries, n_prefix;
    const int32_t *refs, *pages, *prefix_pages;
    int32_t *new_refs, *new_pages, *new_prefix_pages, *copies, *info;
    void* ws;
};
size_t pages_compact_workspace(int64_t n_pages);
hipError_t launch_pages_compact(const PagesCompact& a, hipStream_t stream);

struct PagesCopy {
    vtq_kv_cache cache;
    Scales scales;  // k null: none
    int layers;
    int64_t layer_stride, scale_layer_stride;
    const int32_t *copies, *count;
    int64_t max_copies;
};
hipError_t launch_pages_copy(const PagesCopy& a, hipStream_t stream);

}  // namespace vtq
