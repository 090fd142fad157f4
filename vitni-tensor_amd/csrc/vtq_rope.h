// vtq_rope.h -- rotation of a head's units to a token's position: what the kernels
// that rotate share (rope_kv.hip, kv8_append.hip).
#pragma once

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
// whole pairs, or N elements that do not rotate.  cs: cosine and sine a pair.  give(i, x)
// takes the elements from i on.
template <class T, int N, class Give>
__device__ __forceinline__ void rotated_unit(const T* src, const float2* cs, int unit, int rot, bool half, Give give) {
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
            give(i, x);
            give(rot / 2 + i, y);
            return;
        }
        unit += per;  // the units past the rotated ones
    }
    if constexpr (N == 1) {
        if (!half) {  // both elements of a pair, one at a time
            if (unit < rot / 2) {
                const float2 w = cs[unit];
                const float a = (float)src[2 * unit], b = (float)src[2 * unit + 1];
                float x[1] = {a * w.x - b * w.y}, y[1] = {a * w.y + b * w.x};
                give(2 * unit, x);
                give(2 * unit + 1, y);
                return;
            }
            unit += rot / 2;
        }
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
    give(i, x);
}

// The same, rounded to O.
template <class T, class O, int N>
__device__ __forceinline__ void rotate_unit(const T* src, O* dst, const float2* cs, int unit, int rot, bool half) {
    rotated_unit<T, N>(src, cs, unit, rot, half, [&](int i, const float (&x)[N]) { put<T, O, N>(dst + i, x); });
}

// The sequence of a batch whose tokens hold token t: the one whose end is the first past t
// (batch where there is none).  Every wave finds it for itself.
__device__ __forceinline__ int sequence_of(const vtq_kv_batch& b, int64_t t) {
    const int lane = threadIdx.x & 63;
    int seq = 0;
    for (int i = 0; i < b.batch; i += 64) {
        const bool before = i + lane < b.batch && b.q_start[i + lane + 1] <= t;
        seq += __popcll(__ballot(before));
    }
    return seq;
}

// Units of N elements that a row of `head` elements takes, its first `rot` rotated.
__host__ __device__ inline int rotated_units(int head, int rot, bool half, int n) {
    return (half || n == 1 ? rot / 2 / n : rot / n) + (head - rot) / n;
}

inline bool rows_aligned(const void* p, int64_t ts, int64_t hs, size_t bytes, size_t elem) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && ts * elem % bytes == 0 && hs * elem % bytes == 0;
}

// N elements to an access of a rotation: the most that the alignment of every row and the
// places where the rotation starts and ends allow (f32 by 8, two 16-byte accesses, or by 4).
inline int rope_access(const RopeJob& j, size_t es) {
    const int rot = j.rotate ? j.rope.rot_dim : 0;
    const bool half = j.rope.layout == VTQ_ROPE_HALF;
    auto fits = [&](int n) {
        const size_t bytes = std::min<size_t>(es * n, 16);
        if (j.head_dim % n || rot % n || (half && rot / 2 % n)) return false;
        if (j.x_heads && (!rows_aligned(j.x.p, j.x.token_stride, j.x.head_stride, bytes, es) ||
                          !rows_aligned(j.y, j.y_token_stride, j.y_head_stride, bytes, es)))
            return false;
        return !j.kv_heads || (rows_aligned(j.k.p, j.k.token_stride, j.k.head_stride, bytes, es) &&
                               rows_aligned(j.v.p, j.v.token_stride, j.v.head_stride, bytes, es));
    };
    return fits(8) ? 8 : es == 4 && fits(4) ? 4 : 1;
}

constexpr int kRopeThreads = 256;

}  // namespace
}  // namespace vtq
