// kv8_append.hip -- appending rotated keys and plain values to a paged cache of 8-bit
// floats with a scale to each block of tokens and head (gfx950).
//
//   e = least exponent with max |x| <= 448 * 2^e over a block's new elements, and at
//   least that of the tokens before them;  stored: x / 2^e, rounded to e4m3.
//
// Scales are powers of two, so the quotient is exact but for the one rounding, and a
// block whose scale grows as it fills has its earlier elements shifted, not
// requantized: only what drops below e4m3's smallest normal value rounds again (a full
// scale would gain half a bit at most: e4m3 is a float, and 448 / 2^e lies within two).
//
// A workgroup takes a block of a sequence (the one that holds the call's first token in
// it) and some of its heads; a wave a head's keys or values: the maximum first, then the
// elements again, from the caches near by.  Queries are rotated by workgroups of their own in the same launch.
#include "vtq_rope.h"

namespace vtq {
namespace {

constexpr int kCosTokens = 16;  // tokens whose cosines are held at a time
constexpr int kMostRows = 32;   // heads' keys and values to a workgroup
constexpr int kLeast = -117, kMost = 119;  // exponents of scales: what they scale stays a normal bf16

struct Kv8Job : RopeJob {
    Scales s;
    int q_groups, q_per, rows_per;  // workgroups of queries and their heads; heads' keys and values to one
};

// Least e with top <= 448 * 2^e, 448 being 1.75 * 2^8.
__device__ __forceinline__ int exponent_for(float top) {
    const uint32_t bits = __float_as_uint(top);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return min(max(e, kLeast), kMost);
}

__device__ __forceinline__ float for_e4m3(float x, int e) {
    const float y = __builtin_amdgcn_fmed3f(__builtin_amdgcn_ldexpf(x, -e), -448.0f, 448.0f);
    return fabsf(x) < INFINITY ? y : __uint_as_float(0x7FC00000u);
}

// N elements, rounded to the nearest e4m3 value.
template <int N>
__device__ __forceinline__ void put8(uint8_t* dst, const float (&x)[N], int e) {
    if constexpr (N == 1) {
        *dst = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(for_e4m3(x[0], e), 0.0f, 0, false);
    } else {
        Pack<uint32_t, N / 4> w;
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            int v = __builtin_amdgcn_cvt_pk_fp8_f32(for_e4m3(x[4 * i], e), for_e4m3(x[4 * i + 1], e), 0, false);
            v = __builtin_amdgcn_cvt_pk_fp8_f32(for_e4m3(x[4 * i + 2], e), for_e4m3(x[4 * i + 3], e), v, true);
            w.v[i] = (uint32_t)v;
        }
        *reinterpret_cast<Pack<uint32_t, N / 4>*>(dst) = w;
    }
}

// 4 stored elements times 2^shift.
__device__ __forceinline__ uint32_t shifted4(uint32_t w, int shift) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    int v = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_ldexpf(a[0], shift), __builtin_amdgcn_ldexpf(a[1], shift),
                                            0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(__builtin_amdgcn_ldexpf(b[0], shift), __builtin_amdgcn_ldexpf(b[1], shift), v,
                                        true);
    return (uint32_t)v;
}

template <class T, int N>
__global__ __launch_bounds__(kRopeThreads) void kv8_append_kernel(Kv8Job j) {
    const int64_t t = (int64_t)blockIdx.x;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int seq = sequence_of(j.batch, t);
    if (seq >= j.batch.batch) return;
    const int64_t end = min((int64_t)j.batch.q_start[seq + 1], j.tokens);
    // the newest token of the sequence is the one before its end
    const int64_t place = (int64_t)j.batch.len[seq] - (j.batch.q_start[seq + 1] - t);
    const int rot = j.rotate ? j.rope.rot_dim : 0;
    const bool half = j.rope.layout == VTQ_ROPE_HALF;
    const int units_rot = rotated_units(j.head_dim, rot, half, N), units_plain = j.head_dim / N;
    __shared__ float2 cs[kCosTokens][128];
    __shared__ float top[kMostRows];
    // cosines and sines of `n` tokens from the one at `from` on
    auto turn = [&](int64_t from, int n) {
        for (int i = threadIdx.x; i < n * (rot / 2); i += kRopeThreads) {
            const int token = i / (rot / 2), pair = i % (rot / 2);
            const uint64_t pos = (uint64_t)(j.batch.prefix_len + from + token);
            const float2 w = turn_cos_sin(pos * j.rope.turns[pair]);
            cs[token][pair] = make_float2(w.x * j.rope.magnitude, w.y * j.rope.magnitude);
        }
    };
    if ((int)blockIdx.y < j.q_groups) {
        turn(place, 1);
        __syncthreads();
        const int h0 = (int)blockIdx.y * j.q_per, h1 = min(j.x_heads, h0 + j.q_per);
        for (int w = threadIdx.x; w < (h1 - h0) * units_plain; w += kRopeThreads) {
            const int h = h0 + w / units_plain, u = w % units_plain;
            if (u >= units_rot) continue;
            rotate_unit<T, T, N>(static_cast<const T*>(j.x.p) + t * j.x.token_stride + h * j.x.head_stride,
                                 static_cast<T*>(j.y) + t * j.y_token_stride + h * j.y_head_stride, cs[0], u, rot, half);
        }
        return;
    }
    // the call's first token in the block has the block
    const int block = j.s.block, before = (int)(place & (block - 1));
    if (place < 0 || (before != 0 && t != j.batch.q_start[seq])) return;
    const int64_t at = slot_of(j.cache, j.batch.pages + (int64_t)seq * j.batch.max_pages, j.batch.max_pages, place);
    if (at < 0) return;
    const int64_t page = j.batch.pages[(int64_t)seq * j.batch.max_pages + place / j.cache.page_size];
    const int count = (int)min(end - t, (int64_t)(block - before));
    const int64_t scale_at = page * j.s.page_stride + (place & (j.cache.page_size - 1)) / block;
    const int r0 = ((int)blockIdx.y - j.q_groups) * j.rows_per, r1 = min(2 * j.kv_heads, r0 + j.rows_per);
    const bool keys = r0 < j.kv_heads && rot;
    // f(i, x, token) with the elements of a row (keys of a head, then values of a head) of n tokens
    auto each = [&](int r, int c0, int n, auto f) {
        const bool is_v = r >= j.kv_heads;
        const int h = is_v ? r - j.kv_heads : r, units = is_v ? units_plain : units_rot;
        const HeadRows& in = is_v ? j.v : j.k;
        const T* src = static_cast<const T*>(in.p) + (t + c0) * in.token_stride + h * in.head_stride;
        for (int w = lane; w < n * units; w += 64) {
            const int token = w / units, u = w % units;
            rotated_unit<T, N>(src + token * in.token_stride, cs[token], u, is_v ? 0 : rot, half,
                               [&](int i, const float (&x)[N]) { f(i, x, c0 + token); });
        }
    };
    for (int c0 = 0; c0 < count; c0 += kCosTokens) {
        const int n = min(kCosTokens, count - c0);
        if (keys) {
            if (c0) __syncthreads();
            turn(place + c0, n);
            __syncthreads();
        }
        for (int r = r0 + wave; r < r1; r += 4) {
            float most = 0.0f;
            each(r, c0, n, [&](int, const float (&x)[N], int) {
#pragma unroll
                for (int k = 0; k < N; k++) most = fmaxf(most, fabsf(x[k]) < INFINITY ? fabsf(x[k]) : 0.0f);
            });
#pragma unroll
            for (int x = 1; x < 64; x *= 2) most = fmaxf(most, __shfl_xor(most, x, 64));
            if (lane == 0) top[r - r0] = c0 ? fmaxf(top[r - r0], most) : most;  // the same wave throughout
        }
    }
    __builtin_amdgcn_wave_barrier();
    for (int c0 = 0; c0 < count; c0 += kCosTokens) {
        const int n = min(kCosTokens, count - c0);
        if (keys && count > kCosTokens) {
            __syncthreads();
            turn(place + c0, n);
            __syncthreads();
        }
        for (int r = r0 + wave; r < r1; r += 4) {
            const bool is_v = r >= j.kv_heads;
            const int h = is_v ? r - j.kv_heads : r;
            uint8_t* dst = static_cast<uint8_t*>(is_v ? j.cache.v : j.cache.k) + at + h * (int64_t)j.cache.head_stride;
            uint8_t* scale = (is_v ? j.s.v : j.s.k) + scale_at + h * j.s.head_stride;
            const int slot = (int)j.cache.slot_stride;
            int e = exponent_for(top[r - r0]);
            if (before) {
                // (a second pass finds the scale that the first wrote, which is e already)
                const int old = min(max((int)*scale - 127, kLeast), kMost);
                if (e > old && c0 == 0)
                    for (int w = lane; w < before * (j.head_dim / 4); w += 64) {
                        uint32_t* x = reinterpret_cast<uint32_t*>(dst - (int64_t)(before - w / (j.head_dim / 4)) * slot) +
                                      w % (j.head_dim / 4);
                        *x = shifted4(*x, old - e);
                    }
                e = max(e, old);
            }
            if (lane == 0 && c0 == 0) *scale = (uint8_t)(e + 127);
            each(r, c0, n, [&](int i, const float (&x)[N], int token) { put8<N>(dst + (int64_t)token * slot + i, x, e); });
        }
    }
}

}  // namespace

hipError_t launch_kv8_append(const RopeJob& job, const Scales& s, int type, hipStream_t stream) {
    Kv8Job j{};
    static_cast<RopeJob&>(j) = job;
    j.s = s;
    const int n = rope_access(j, type_bytes(type));
    // workgroups to a token: the queries' heads and the rows of keys and values over as many
    // as keep the chip busy
    auto groups = [&](int rows, int64_t units, int least) {
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>({units, 1024 / j.tokens, (int64_t)rows}));
        return (int)std::max<int64_t>(most, least);
    };
    j.q_groups = j.x_heads ? groups(j.x_heads, ((int64_t)j.x_heads * (j.head_dim / n) + kRopeThreads - 1) / kRopeThreads, 1) : 0;
    if (j.q_groups) {
        j.q_per = (j.x_heads + j.q_groups - 1) / j.q_groups;
        j.q_groups = (j.x_heads + j.q_per - 1) / j.q_per;
    }
    const int rows = 2 * j.kv_heads;
    int kv_groups = groups(rows, (rows + 3) / 4, (rows + kMostRows - 1) / kMostRows);
    j.rows_per = (rows + kv_groups - 1) / kv_groups;
    kv_groups = (rows + j.rows_per - 1) / j.rows_per;
    const dim3 grid((unsigned)j.tokens, (unsigned)(j.q_groups + kv_groups));
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        if (n == 8) {
            hipLaunchKernelGGL((kv8_append_kernel<T, 8>), grid, dim3(kRopeThreads), 0, stream, j);
        } else if (n == 4) {
            if constexpr (sizeof(T) == 4)
                hipLaunchKernelGGL((kv8_append_kernel<T, 4>), grid, dim3(kRopeThreads), 0, stream, j);
        } else {
            hipLaunchKernelGGL((kv8_append_kernel<T, 1>), grid, dim3(kRopeThreads), 0, stream, j);
        }
        return hipGetLastError();
    });
}

}  // namespace vtq
