// i8_linear.hip -- activations to 8 bits a token, and the int8 product with scales
// per token and output channel (gfx950).
//
//   s_m = max_k |x_mk| / 127,  q_mk = x_mk / s_m rounded,  y_mn = s_m t_n sum_k q_mk w_nk + b_n
//
// Integer sums are exact in any order, so how K is split never shows.
#include "vtq_device.h"
#include "vtq_serve.h"

namespace vtq {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
constexpr int kWord3 = 0x00020000;  // raw buffer, stride 0

// ------------------------------------------------ quantization

// x / s to the nearest whole number, ties to even, of the exact quotient: the f32
// quotient may round onto a half, so the remainder decides.  x - q s is exact in one
// fma (a multiple of the smaller unit in the last place, below s in magnitude).
__device__ __forceinline__ int quotient(float x, float s) {
    float q = rintf(x / s);
    const float r = fmaf(-q, s, x), twice = 2.0f * fabsf(r);
    if (twice > s || (twice == s && ((int)q & 1))) q += (r < 0.0f) ? -1.0f : 1.0f;
    return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

constexpr int kQuantThreads = 256;

template <class T>
__global__ __launch_bounds__(kQuantThreads) void quantize_kernel(const T* x, size_t ld_x, int8_t* q, size_t ld_q,
                                                                 float* scale, int rows, int n) {
    __shared__ uint32_t top[kQuantThreads / 64];
    for (int m = (int)blockIdx.x; m < rows; m += (int)gridDim.x) {
        const T* xr = x + (size_t)m * ld_x;
        // the largest magnitude by its bits: a NaN is above an infinity above every number
        uint32_t a = 0;
        for (int k = threadIdx.x; k < n; k += kQuantThreads)
            a = max(a, __float_as_uint((float)xr[k]) & 0x7FFFFFFFu);
        for (int d = 1; d < 64; d *= 2) a = max(a, (uint32_t)__shfl_xor((int)a, d, 64));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = a;
        __syncthreads();
        for (int w = 0; w < kQuantThreads / 64; w++) a = max(a, top[w]);
        const bool finite = a < 0x7F800000u;
        const float s = finite ? __uint_as_float(a) / 127.0f : __uint_as_float(a);
        if (threadIdx.x == 0) scale[m] = s;
        for (size_t k = threadIdx.x; k < ld_q; k += kQuantThreads)
            q[(size_t)m * ld_q + k] = (int8_t)(k < (size_t)n && finite && s > 0.0f ? quotient((float)xr[k], s) : 0);
    }
}

// ------------------------------------------------ product

// A workgroup owns 16 output channels x 16 tokens, its waves every W-th 256 bytes of
// K; lane (r, g) of a wave takes the 64 bytes g of row r, channel and token alike (the
// order of K inside an MFMA is free as long as both operands share it).
template <class O, int W>
__global__ __launch_bounds__(W * 64) void i8_rows_kernel(I8Linear a) {
    __shared__ int part[W][16][17];
    const int lane = threadIdx.x & 63, wave = wave_id(), r = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16;
    const int k_end = (a.in_feat + 15) & ~15;
    const int n_rows = min(16, a.out_feat - n0), m_rows = min(16, a.batch - m0);
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<int8_t*>(a.w + (size_t)n0 * a.ld_w), (short)0, (int)((n_rows - 1) * a.ld_w + k_end), kWord3);
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<int8_t*>(a.x + (size_t)m0 * a.ld_x), (short)0, (int)((m_rows - 1) * a.ld_x + k_end), kWord3);
    v4i acc = {0, 0, 0, 0};
    for (int k = wave * 256; k < k_end; k += W * 256) {
        v4i wv[4], xv[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = k + g * 64 + i * 16;
            // rows past the last one and bytes past the row give zeros
            const int ow = at < k_end && r < n_rows ? (int)(r * a.ld_w) + at : -1;
            const int ox = at < k_end && r < m_rows ? (int)(r * a.ld_x) + at : -1;
            wv[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw, ow, 0, 0));
            xv[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, ox, 0, 0));
        }
#pragma unroll
        for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(xv[i], wv[i], acc, 0, 0, 0);
    }
    // acc: channel lane & 15, tokens 4 (lane >> 4) + 0..3
#pragma unroll
    for (int i = 0; i < 4; i++) part[wave][4 * g + i][r] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < 256; e += W * 64) {
        const int m = e >> 4, n = e & 15;
        if (m >= m_rows || n >= n_rows) continue;
        int sum = 0;
        for (int w = 0; w < W; w++) sum += part[w][m][n];
        float y = a.in_feat ? (float)sum * a.xs[m0 + m] * a.ws[n0 + n] : 0.0f;
        if (a.bias) y += a.bias[n0 + n];
        static_cast<O*>(a.y)[(size_t)(m0 + m) * a.ld_y + n0 + n] = (O)y;
    }
}

}  // namespace

hipError_t launch_quantize_i8(int type, const void* x, size_t ld_x, int8_t* q, size_t ld_q, float* scale, size_t rows,
                              int n, hipStream_t stream) {
    const unsigned grid = (unsigned)(rows < 65536 ? rows : 65536);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((quantize_kernel<T>), dim3(grid), dim3(kQuantThreads), 0, stream, static_cast<const T*>(x),
                           ld_x, q, ld_q, scale, (int)rows, n);
        return hipGetLastError();
    });
}

hipError_t launch_linear_i8(const I8Linear& a, int y_type, hipStream_t stream) {
    // a launch takes at most 65535 groups of tokens
    constexpr int kMost = 65535 * 16;
    for (int m0 = 0; m0 < a.batch; m0 += kMost) {
        I8Linear b = a;
        b.batch = a.batch - m0 < kMost ? a.batch - m0 : kMost;
        b.x = a.x + (size_t)m0 * a.ld_x;
        b.xs = a.xs + (a.in_feat ? m0 : 0);
        b.y = static_cast<char*>(a.y) + (size_t)m0 * a.ld_y * type_bytes(y_type);
        const dim3 grid((unsigned)((a.out_feat + 15) / 16), (unsigned)((b.batch + 15) / 16));
        const hipError_t e = with_type(y_type, [&](auto t) {
            hipLaunchKernelGGL((i8_rows_kernel<decltype(t), 4>), grid, dim3(256), 0, stream, b);
            return hipGetLastError();
        });
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace vtq
