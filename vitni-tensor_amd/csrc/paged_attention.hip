// paged_attention.hip -- attention of a ragged batch over a prefix that all its
// sequences share and the pages of their own (gfx950).
//
//   y = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),  m = max_j scale q.k_j
//
// in one pass over the keys, with the running maximum and sum of each row in f32.
#include <type_traits>

#include "vtq_device.h"
#include "vtq_serve.h"

namespace vtq {
namespace {

// One wave a row: lane j scores key j of a chunk of 64, then the lanes share out the
// elements of the values.
template <class Q, class C>
__global__ __launch_bounds__(64) void attention_rows_kernel(Attention a) {
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x;
    const int h = (int)blockIdx.y, hd = a.cache.head_dim;
    int seq = 0;
    for (int b = 0; b < a.batch.batch; b += 64)
        seq += __popcll(__ballot(b + lane < a.batch.batch && a.batch.q_start[b + lane + 1] <= t));
    if (seq >= a.batch.batch) return;
    const int64_t place = (int64_t)a.batch.len[seq] - (a.batch.q_start[seq + 1] - t);
    const int64_t limit = min((int64_t)a.batch.max_pages * a.cache.page_size, place + 1);
    const int64_t keys = a.batch.prefix_len + max((int64_t)0, limit);
    const int64_t head_at = (int64_t)(h / (a.heads / a.cache.kv_heads)) * a.cache.head_stride;
    const Q* q = static_cast<const Q*>(a.q.p) + t * a.q.token_stride + h * a.q.head_stride;
    float m = -INFINITY, l = 0.0f, o[4] = {0, 0, 0, 0};
    for (int64_t j0 = 0; j0 < keys; j0 += 64) {
        const int64_t j = j0 + lane;
        int64_t at = -1;
        float s = -INFINITY;
        if (j < keys) {
            const bool own = j >= a.batch.prefix_len;
            const int64_t i = own ? j - a.batch.prefix_len : j;
            const int64_t page = own ? a.batch.pages[(int64_t)seq * a.batch.max_pages + i / a.cache.page_size]
                                     : a.batch.prefix_pages[i / a.cache.page_size];
            s = 0.0f;
            if (page >= 0 && page < (int64_t)a.cache.n_pages) {
                at = page * (int64_t)a.cache.page_stride + (i % a.cache.page_size) * (int64_t)a.cache.slot_stride + head_at;
                for (int d = 0; d < hd; d++) s = fmaf((float)q[d], (float)static_cast<const C*>(a.cache.k)[at + d], s);
            }
            s *= a.scale;
        }
        float top = s;
        for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x, 64));
        const float m1 = fmaxf(m, top), base = m1 == -INFINITY ? 0.0f : m1;
        const float shrink = expf(m - base), p = expf(s - base);
        float sum = p;
        for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x, 64);
        l = l * shrink + sum;
        m = m1;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] *= shrink;
        const int n = (int)min((int64_t)64, keys - j0);
        for (int k = 0; k < n; k++) {
            const float pk = __shfl(p, k, 64);
            const int64_t vk = __shfl(at, k, 64);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int d = lane + 64 * e;
                if (d < hd && vk >= 0) o[e] = fmaf(pk, (float)static_cast<const C*>(a.cache.v)[vk + d], o[e]);
            }
        }
    }
    Q* y = static_cast<Q*>(a.y) + t * a.y_token_stride + h * a.y_head_stride;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (lane + 64 * e < hd) y[lane + 64 * e] = (Q)(keys > 0 ? o[e] / l : 0.0f);
    if (a.lse && lane == 0) a.lse[t * a.heads + h] = keys > 0 ? m + logf(l) : -INFINITY;
}

}  // namespace

size_t attention_workspace(const vtq_kv_cache&, const vtq_kv_batch&, int, int64_t, int) { return 0; }

hipError_t launch_attention(const Attention& a, int type, hipStream_t stream) {
    const dim3 grid((unsigned)a.tokens, (unsigned)a.heads);
    return with_type(type, [&](auto q) {
        using Q = decltype(q);
        return with_type(a.cache.type, [&](auto c) {
            using C = decltype(c);
            if constexpr (!std::is_same_v<Q, C> && !std::is_same_v<Q, float>) {
                return hipErrorInvalidValue;
            } else {
                hipLaunchKernelGGL((attention_rows_kernel<Q, C>), grid, dim3(64), 0, stream, a);
                return hipGetLastError();
            }
        });
    });
}

}  // namespace vtq
