// rope_kv.hip -- rotary positions, and appending rotated keys and plain values to
// a paged cache (gfx950).
//
// Pair i of a head at position p turns by p * f_i.  f_i is kept as a fraction of
// a turn in 64 bits, so p * f_i modulo one turn is a 64-bit integer product: it
// loses nothing, and the fraction's own error (a few 2^-64) is 2^-31 of a turn at
// position 2^31, where a product in f32 is off by 0.06 rad at position 10^6.  The
// remainder, within an eighth of a turn of a quarter turn, goes through sine and
// cosine series in f64 (terms to x^13 and x^14: truncation below 2e-14 and 2e-15 on
// pi/4), rounded once to f32.
//
// The work is a copy: every element is read and written once.  A workgroup
// takes some heads of one token and computes that token's cosines and sines
// once, in LDS.  4096 tokens of 40 heads of 128 bf16: 15.3 us, 5.5 TB/s; 4920
// f32 tokens of 48 heads of 80, appended as f16: 33.6 us, 4.1 TB/s; 8 tokens of
// 36 heads 2.8 us and 32 appended ones 3.6 us inside a graph, a launch's own
// time.
#include "vtq_rope.h"

namespace vtq {
namespace {

// Workgroup (token, group of heads): heads 0..x_heads-1 are x, then the keys, then
// the values.  N elements to a thread's access; N = 1 takes any alignment.
template <class T, class C, int N>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeJob j, int heads_per_group) {
    const int64_t t = (int64_t)blockIdx.x;
    int64_t pos, place = 0;
    int seq = 0;
    if (j.pos) {
        pos = j.pos[t];
    } else {
        seq = sequence_of(j.batch, t);
        if (seq >= j.batch.batch) return;
        // the newest token of the sequence is the one before its end
        place = (int64_t)j.batch.len[seq] - (j.batch.q_start[seq + 1] - t);
        pos = j.batch.prefix_len + place;
    }
    __shared__ float2 cs[128];
    const int rot = j.rotate ? j.rope.rot_dim : 0;
    for (int i = threadIdx.x; i < rot / 2; i += kRopeThreads) {
        float2 w = turn_cos_sin((uint64_t)pos * j.rope.turns[i]);
        cs[i] = make_float2(w.x * j.rope.magnitude, w.y * j.rope.magnitude);
    }
    __syncthreads();
    // the token's slot
    const int64_t slot_at =
        j.kv_heads ? slot_of(j.cache, j.batch.pages + (int64_t)seq * j.batch.max_pages, j.batch.max_pages, place) : -1;
    const bool half = j.rope.layout == VTQ_ROPE_HALF;
    const int all = j.x_heads + 2 * j.kv_heads;
    const int h0 = (int)blockIdx.y * heads_per_group, h1 = min(all, h0 + heads_per_group);
    const int units_rot = rotated_units(j.head_dim, rot, half, N), units_plain = j.head_dim / N;
    const int most = units_plain;
    for (int w = threadIdx.x; w < (h1 - h0) * most; w += kRopeThreads) {
        const int h = h0 + w / most, u = w % most;
        const bool is_v = h >= j.x_heads + j.kv_heads;
        if (u >= (is_v ? units_plain : units_rot)) continue;
        if (h < j.x_heads) {
            const T* src = static_cast<const T*>(j.x.p) + t * j.x.token_stride + h * j.x.head_stride;
            T* dst = static_cast<T*>(j.y) + t * j.y_token_stride + h * j.y_head_stride;
            rotate_unit<T, T, N>(src, dst, cs, u, rot, half);
        } else if (slot_at >= 0) {
            const int hk = is_v ? h - j.x_heads - j.kv_heads : h - j.x_heads;
            const HeadRows& in = is_v ? j.v : j.k;
            const T* src = static_cast<const T*>(in.p) + t * in.token_stride + hk * in.head_stride;
            C* dst = static_cast<C*>(is_v ? j.cache.v : j.cache.k) + slot_at + hk * (int64_t)j.cache.head_stride;
            rotate_unit<T, C, N>(src, dst, cs, u, is_v ? 0 : rot, half);
        }
    }
}

}  // namespace

hipError_t launch_rope(const RopeJob& j, int type, int cache_type, hipStream_t stream) {
    const size_t es = type_bytes(type);
    const int n = rope_access(j, es);
    const int all = j.x_heads + 2 * j.kv_heads;
    // a workgroup a token, more where that leaves the chip idle
    const int64_t units = (int64_t)all * (j.head_dim / n);
    const int64_t most = (units + kRopeThreads - 1) / kRopeThreads;
    const int64_t groups = std::max<int64_t>(1, std::min<int64_t>({most, 1024 / j.tokens, (int64_t)all}));
    const int per = (int)((all + groups - 1) / groups);
    const dim3 grid((unsigned)j.tokens, (unsigned)((all + per - 1) / per));
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return with_type(cache_type, [&](auto c) {
            using C = decltype(c);
            if constexpr (!std::is_same_v<T, C> && !std::is_same_v<T, float>) {
                return hipErrorInvalidValue;
            } else {
                if (n == 8) {
                    hipLaunchKernelGGL((rope_kernel<T, C, 8>), grid, dim3(kRopeThreads), 0, stream, j, per);
                } else if (n == 4) {
                    if constexpr (sizeof(T) == 4)
                        hipLaunchKernelGGL((rope_kernel<T, C, 4>), grid, dim3(kRopeThreads), 0, stream, j, per);
                } else {
                    hipLaunchKernelGGL((rope_kernel<T, C, 1>), grid, dim3(kRopeThreads), 0, stream, j, per);
                }
                return hipGetLastError();
            }
        });
    });
}

}  // namespace vtq
