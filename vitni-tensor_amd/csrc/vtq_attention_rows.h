// vtq_attention_rows.h -- what the attention kernels (cache_attention.hip, kv8_attention.hip)
// share: a call's job, a wave's rows, and how parts of a row end in it.
#pragma once

#include <type_traits>

#include "vtq_attention_plan.h"
#include "vtq_device.h"
#include "vtq_kernels.h"
#include "vtq_lds_load.h"
#include "vtq_serve.h"

namespace vtq {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr float kLog2E = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr int kWord3 = 0x00020000;  // raw buffer, stride 0

struct Job : AttentionPlan {
    Attention a;
    float c;          // scale * log2(e)
    float* part_o;    // [splits][tokens * heads][head_dim]
    float2* part_ml;  // [splits][tokens * heads]: maximum of q.k and sum
};

// What a wave has of a 32-row tile.
template <int D>
struct State {
    v16f o[D / 32];
    float m, l;  // maximum of q.k; sum of this lane's weights (the partner lane has the other keys')
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// x of both half-waves: {lanes 0-31's, lanes 32-63's} in every lane
__device__ __forceinline__ float2 halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// A lane number that the compiler knows nothing of: what is worked out from it stays
// behind this point, instead of in registers all through the loops before it.
__device__ __forceinline__ int late_lane() {
    int x = threadIdx.x & 63;
    asm volatile("" : "+v"(x));
    return x;
}

// Sums of values that lie near f32's end are held 2^-kDown as large as they count where LOWERS; the
// sign of a row's l, which is never negative, says so.
constexpr int kDown = 40;
constexpr float kToDown = 0x1p-40f, kFromDown = 0x1p40f;
template <bool LOWERS>
__device__ __forceinline__ bool lowered(float l) {
    return LOWERS && __float_as_int(l) < 0;
}

__device__ __forceinline__ void scale4(float4& x, float by) { x.x *= by, x.y *= by, x.z *= by, x.w *= by; }

// Finishes a row: y and lse, or a part.  o are elements d..d+3 of the row, which with l are
// 2^UP times as large as they count.
template <class Q, int UP, bool LOWERS = false>
__device__ __forceinline__ void put_row(const Job& j, int split, int64_t token, int head, int d, float4 o, float m,
                                        float l) {
    const Attention& a = j.a;
    const int64_t row = token * a.heads + head;
    if (j.prefix_splits + j.own_splits > 1) {
        const int64_t at = (int64_t)split * a.tokens * a.heads + row;
        *reinterpret_cast<float4*>(j.part_o + at * a.cache.head_dim + d) = o;
        if (d == 0) j.part_ml[at] = make_float2(m, l);
        return;
    }
    const bool down = lowered<LOWERS>(l);
    if constexpr (LOWERS) l = fabsf(l);
    const bool none = l == 0.0f && m == -INFINITY;
    const float inv = none ? 0.0f : 1.0f / l;
    scale4(o, inv);
    if constexpr (LOWERS) scale4(o, down ? kFromDown : 1.0f);
    Q* y = static_cast<Q*>(a.y) + token * a.y_token_stride + head * a.y_head_stride + d;
    typedef Q v4q __attribute__((ext_vector_type(4)));
    v4q r;
    r[0] = (Q)o.x, r[1] = (Q)o.y, r[2] = (Q)o.z, r[3] = (Q)o.w;
    *reinterpret_cast<v4q*>(y) = r;
    if (d == 0 && a.lse) a.lse[row] = none ? -INFINITY : fmaf(m, a.scale, (__log2f(l) - UP) * kLn2);
}

// Joins the parts of a row: one wave a row.  L lanes take the elements, 64 / L groups
// of them every so many parts; a part without weight (no keys) is not used, its sums
// may never have been written.  2048 rows of 128 take 5.4 us, 4096 6.9: a launch
// and two loads' latency more than traffic (6.0 and 7.5 where the parts' loads wait for
// their weights).
template <class Q, int L, int UP, bool LOWERS>
__global__ __launch_bounds__(256) void join_kernel(Job j) {
    constexpr int N = 64 / L, kAhead = 4;
    static_assert(kMostParts == 2 * 64, "parts lane and 64 + lane");
    const Attention& a = j.a;
    const int lane = threadIdx.x & 63, splits = j.prefix_splits + j.own_splits, hd = a.cache.head_dim;
    const int64_t rows = a.tokens * a.heads, row = (int64_t)blockIdx.x * 4 + wave_id();
    if (row >= rows) return;
    const int64_t token = row / a.heads;
    const bool live = token < a.batch.q_start[a.batch.batch];
    // the first parts load while their weights are worked out
    const int d = 4 * (lane % L), group = lane / L;
    const bool in = d < hd;
    const float* from = j.part_o + row * hd + (in ? d : 0);
    float4 x[kAhead];
    auto load = [&](int s0) {
#pragma unroll
        for (int i = 0; i < kAhead; i++)
            x[i] = *reinterpret_cast<const float4*>(from + min(s0 + i * N + group, splits - 1) * rows * hd);
    };
    load(0);
    // part lane and part 64 + lane
    float2 ml[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        ml[i] = 64 * i + lane < splits ? j.part_ml[(64 * i + lane) * rows + row] : make_float2(-INFINITY, 0.0f);
    // where one part is held lower, the others are brought to it
    const bool down = LOWERS && __ballot(lowered<LOWERS>(ml[0].y) || lowered<LOWERS>(ml[1].y)) != 0;
    float m = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) m = fmaxf(m, __shfl_xor(m, x, 64));
    const float base = m == -INFINITY ? 0.0f : m;
    float f[2], l = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        f[i] = __builtin_amdgcn_exp2f((ml[i].x - base) * j.c);
        l += (LOWERS ? fabsf(ml[i].y) : ml[i].y) * f[i];
    }
#pragma unroll
    for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x, 64);
    float4 o = make_float4(0, 0, 0, 0);
    auto add_parts = [&](auto lowers) {
        for (int s0 = 0; s0 < splits; s0 += N * kAhead) {
            if (s0) load(s0);
            float w[kAhead], has[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                const int s = s0 + i * N + group;
                w[i] = __shfl(s0 < 64 ? f[0] : f[1], s & 63, 64);
                const float sum = __shfl(s0 < 64 ? ml[0].y : ml[1].y, s & 63, 64);  // by every lane
                has[i] = s < splits ? sum : 0.0f;
                if constexpr (lowers.value) scale4(x[i], lowered<true>(has[i]) ? 1.0f : kToDown);
            }
#pragma unroll
            for (int i = 0; i < kAhead; i++) {
                const bool use = has[i] != 0.0f;
                o.x = use ? fmaf(x[i].x, w[i], o.x) : o.x, o.y = use ? fmaf(x[i].y, w[i], o.y) : o.y;
                o.z = use ? fmaf(x[i].z, w[i], o.z) : o.z, o.w = use ? fmaf(x[i].w, w[i], o.w) : o.w;
            }
        }
    };
    if (LOWERS && down) add_parts(std::bool_constant<LOWERS>{});
    else add_parts(std::false_type{});
#pragma unroll
    for (int x = L; x < 64; x *= 2) {
        o.x += __shfl_xor(o.x, x, 64), o.y += __shfl_xor(o.y, x, 64);
        o.z += __shfl_xor(o.z, x, 64), o.w += __shfl_xor(o.w, x, 64);
    }
    const bool none = m == -INFINITY && l == 0.0f;
    const float inv = none ? 0.0f : 1.0f / l;
    scale4(o, inv);
    if constexpr (LOWERS) scale4(o, down ? kFromDown : 1.0f);
    typedef Q v4q __attribute__((ext_vector_type(4)));
    if (live && in && group == 0) {
        v4q r;
        r[0] = (Q)o.x, r[1] = (Q)o.y, r[2] = (Q)o.z, r[3] = (Q)o.w;
        *reinterpret_cast<v4q*>(static_cast<Q*>(a.y) + token * a.y_token_stride + (row % a.heads) * a.y_head_stride + d) =
            r;
    }
    if (live && a.lse && lane == 0) a.lse[row] = none ? -INFINITY : fmaf(m, a.scale, (__log2f(l) - UP) * kLn2);
}

// The parts of every row, one after another, then their maxima and sums.
inline void place_parts(Job& j) {
    const size_t rows = (size_t)(j.prefix_splits + j.own_splits) * j.a.tokens * j.a.heads;
    j.part_o = static_cast<float*>(j.a.ws);
    j.part_ml = reinterpret_cast<float2*>(static_cast<char*>(j.a.ws) +
                                          (rows * j.a.cache.head_dim * sizeof(float) + 255) / 256 * 256);
}
inline size_t parts_bytes(const AttentionPlan& plan, int64_t tokens, int heads, int head_dim) {
    const size_t splits = plan.prefix_splits + plan.own_splits;
    return splits > 1 ? splits * tokens * heads * (head_dim * sizeof(float) + sizeof(float2)) + 256 : 0;
}

template <class Q, int D, int UP, bool LOWERS = false>
hipError_t launch_join(const Job& j, hipStream_t stream) {
    if (j.prefix_splits + j.own_splits == 1) return hipSuccess;
    hipLaunchKernelGGL((join_kernel<Q, D / 4, UP, LOWERS>), dim3((unsigned)((j.a.tokens * j.a.heads + 3) / 4)), dim3(256), 0,
                       stream, j);
    return hipGetLastError();
}

}  // namespace
}  // namespace vtq
