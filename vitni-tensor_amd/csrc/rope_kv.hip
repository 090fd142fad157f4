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
#include <algorithm>
#include <type_traits>

#include "vtq_device.h"
#include "vtq_serve.h"

namespace vtq {
namespace {

__device__ __forceinline__ float2 turn_cos_sin(uint64_t t) {
    const uint64_t quarter = (t + (1ull << 61)) >> 62;  // nearest, 0..3 (4 wraps to 0)
    const double x = (double)(int64_t)(t - (quarter << 62)) * (6.283185307179586476925286766559 / 18446744073709551616.0);
    const double z = x * x;
    double s = 1.0 / 6227020800.0;
    s = fma(s, z, -1.0 / 39916800.0);
    s = fma(s, z, 1.0 / 362880.0);
    s = fma(s, z, -1.0 / 5040.0);
    s = fma(s, z, 1.0 / 120.0);
    s = fma(s, z, -1.0 / 6.0);
    s = fma(s * z, x, x);
    double c = -1.0 / 87178291200.0;
    c = fma(c, z, 1.0 / 479001600.0);
    c = fma(c, z, -1.0 / 3628800.0);
    c = fma(c, z, 1.0 / 40320.0);
    c = fma(c, z, -1.0 / 720.0);
    c = fma(c, z, 1.0 / 24.0);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const float cf = (float)((quarter & 1) ? s : c), sf = (float)((quarter & 1) ? c : s);
    // quarter 0: (c, s), 1: (-s, c), 2: (-c, -s), 3: (s, -c)
    return make_float2(quarter == 1 || quarter == 2 ? -cf : cf, quarter >= 2 ? -sf : sf);
}

template <class T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T v[N];
};

template <class T, class O, int N>
__device__ __forceinline__ void put(O* dst, const float (&f)[N]) {
    Pack<O, N> o;
#pragma unroll
    for (int i = 0; i < N; i++) o.v[i] = (O)f[i];
    *reinterpret_cast<Pack<O, N>*>(dst) = o;
}

// One unit of a head: N elements of each half of the pairs (HALF), N elements of
// whole pairs, or N elements that do not rotate.  cs: cosine and sine a pair.
template <class T, class O, int N>
__device__ __forceinline__ void rotate_unit(const T* src, O* dst, const float2* cs, int unit, int rot, bool half) {
    if (half && rot) {
        const int per = rot / 2 / N;
        if (unit < per) {
            const int i = unit * N;
            const Pack<T, N> a = *reinterpret_cast<const Pack<T, N>*>(src + i);
            const Pack<T, N> b = *reinterpret_cast<const Pack<T, N>*>(src + rot / 2 + i);
            float x[N], y[N];
#pragma unroll
            for (int k = 0; k < N; k++) {
                const float2 w = cs[i + k];
                x[k] = (float)a.v[k] * w.x - (float)b.v[k] * w.y;
                y[k] = (float)a.v[k] * w.y + (float)b.v[k] * w.x;
            }
            put<T, O, N>(dst + i, x);
            put<T, O, N>(dst + rot / 2 + i, y);
            return;
        }
        unit += per;  // the units past the rotated ones
    }
    if (N == 1 && !half) {  // both elements of a pair, one at a time
        if (unit < rot / 2) {
            const float2 w = cs[unit];
            const float a = (float)src[2 * unit], b = (float)src[2 * unit + 1];
            dst[2 * unit] = (O)(a * w.x - b * w.y);
            dst[2 * unit + 1] = (O)(a * w.y + b * w.x);
            return;
        }
        unit += rot / 2;
    }
    const int i = unit * N;
    const Pack<T, N> a = *reinterpret_cast<const Pack<T, N>*>(src + i);
    float x[N];
#pragma unroll
    for (int k = 0; k < N; k++) x[k] = (float)a.v[k];
    if constexpr (N > 1) {
        if (!half && i < rot) {
#pragma unroll
            for (int k = 0; k < N; k += 2) {
                const float2 w = cs[(i + k) / 2];
                const float p = x[k] * w.x - x[k + 1] * w.y, q = x[k] * w.y + x[k + 1] * w.x;
                x[k] = p, x[k + 1] = q;
            }
        }
    }
    put<T, O, N>(dst + i, x);
}

constexpr int kRopeThreads = 256;

// Workgroup (token, group of heads): heads 0..x_heads-1 are x, then the keys, then
// the values.  N elements to a thread's access; N = 1 takes any alignment.
template <class T, class C, int N>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeJob j, int heads_per_group) {
    const int64_t t = (int64_t)blockIdx.x;
    const int lane = threadIdx.x & 63;
    int64_t pos, place = 0;
    int seq = 0;
    if (j.pos) {
        pos = j.pos[t];
    } else {
        // the sequence whose end is the first one past t; every wave finds it for itself
        for (int b = 0; b < j.batch.batch; b += 64) {
            const bool before = b + lane < j.batch.batch && j.batch.q_start[b + lane + 1] <= t;
            seq += __popcll(__ballot(before));
        }
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
    const int rot_units = half || N == 1 ? rot / 2 / N : rot / N;
    const int units_rot = rot_units + (j.head_dim - rot) / N, units_plain = j.head_dim / N;
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

bool rows_aligned(const void* p, int64_t ts, int64_t hs, size_t bytes, size_t elem) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ts * elem % bytes == 0 && hs * elem % bytes == 0;
}

}  // namespace

hipError_t launch_rope(const RopeJob& j, int type, int cache_type, hipStream_t stream) {
    const size_t es = type_bytes(type);
    const int rot = j.rotate ? j.rope.rot_dim : 0;
    const bool half = j.rope.layout == VTQ_ROPE_HALF;
    // N elements to an access: the most that the alignment of every row and the
    // places where the rotation starts and ends allow
    auto fits = [&](int n) {
        const size_t bytes = std::min<size_t>(es * n, 16);
        if (j.head_dim % n || rot % n || (half && rot / 2 % n)) return false;
        if (j.x_heads && (!rows_aligned(j.x.p, j.x.token_stride, j.x.head_stride, bytes, es) ||
                          !rows_aligned(j.y, j.y_token_stride, j.y_head_stride, bytes, es)))
            return false;
        return !j.kv_heads || (rows_aligned(j.k.p, j.k.token_stride, j.k.head_stride, bytes, es) &&
                               rows_aligned(j.v.p, j.v.token_stride, j.v.head_stride, bytes, es));
    };
    // (f32 by 8, two 16-byte accesses, or by 4)
    const int n = fits(8) ? 8 : es == 4 && fits(4) ? 4 : 1;
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
