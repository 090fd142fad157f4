// i8_linear.hip -- activations to 8 bits a token, and the int8 product with scales
// per token and output channel (gfx950).
//
//   s_m = max_k |x_mk| / 127,  q_mk = x_mk / s_m rounded,  y_mn = s_m t_n sum_k q_mk w_nk + b_n
//
// Integer sums are exact in any order, so how K is split never shows.
#include <algorithm>

#include "vtq_device.h"
#include "vtq_kernels.h"
#include "vtq_lds_load.h"
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

// One output: the sum to f32, its two scales and the bias, each rounded once, then the
// output's type.
template <class O>
__device__ __forceinline__ void store(const I8Linear& a, int m, int n, int sum) {
    float y = a.in_feat ? (float)sum * a.xs[m] * a.ws[n] : 0.0f;
    if (a.bias) y += a.bias[n];
    static_cast<O*>(a.y)[(size_t)m * a.ld_y + n] = (O)y;
}

// ------------------------------------------------ product, few tokens

// A workgroup owns 16 output channels x 16 MT tokens, its waves every W-th 256 bytes
// of K; lane (r, g) of a wave takes the 64 bytes g of row r, channel and token alike
// (the order of K inside an MFMA is free as long as both operands share it).
template <class O, int W, int MT>
__global__ __launch_bounds__(W * 64) void i8_rows_kernel(I8Linear a) {
    __shared__ int part[W][16 * MT][17];
    const int lane = threadIdx.x & 63, wave = wave_id(), r = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16 * MT;
    const int k_end = (a.in_feat + 15) & ~15;
    const int n_rows = min(16, a.out_feat - n0), m_rows = min(16 * MT, a.batch - m0);
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<int8_t*>(a.w + (size_t)n0 * a.ld_w), (short)0, (int)((n_rows - 1) * a.ld_w + k_end), kWord3);
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<int8_t*>(a.x + (size_t)m0 * a.ld_x), (short)0, (int)((m_rows - 1) * a.ld_x + k_end), kWord3);
    v4i acc[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) acc[t] = v4i{0, 0, 0, 0};
    for (int k = wave * 256; k < k_end; k += W * 256) {
        v4i wv[4], xv[MT][4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = k + g * 64 + i * 16;
            // rows past the last one and bytes past the row give zeros
            const int ow = at < k_end && r < n_rows ? (int)(r * a.ld_w) + at : -1;
            wv[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw, ow, 0, 0));
#pragma unroll
            for (int t = 0; t < MT; t++) {
                const int ox = at < k_end && 16 * t + r < m_rows ? (int)((16 * t + r) * a.ld_x) + at : -1;
                xv[t][i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, ox, 0, 0));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int t = 0; t < MT; t++)
                acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xv[t][i], wv[i], acc[t], 0, 0, 0);
    }
    // acc: channel lane & 15, tokens 4 (lane >> 4) + 0..3
#pragma unroll
    for (int t = 0; t < MT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) part[wave][16 * t + 4 * g + i][r] = acc[t][i];
    __syncthreads();
    for (int e = threadIdx.x; e < 256 * MT; e += W * 64) {
        const int m = e >> 4, n = e & 15;
        if (m >= m_rows || n >= n_rows) continue;
        int sum = 0;
#pragma unroll
        for (int w = 0; w < W; w++) sum += part[w][m][n];
        store<O>(a, m0 + m, n0 + n, sum);
    }
}

// ------------------------------------------------ product, many tokens

// A workgroup owns BM tokens x BN channels, a wave 32 TM x 32 TN of them on 32x32x32
// MFMAs.  Tiles of both operands go from memory straight to LDS, two stages of 128
// bytes of K; the 16-byte chunks of a row are permuted so that the 16 rows that a
// read takes at one column lie in different banks.
typedef int v16i __attribute__((ext_vector_type(16)));

template <int TM_, int TN_, int WM_, int WN_>
struct Tiles {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, W = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN;
    static constexpr int kStage = (BM + BN) * 128;
    static constexpr int kLoadsA = BM / 8 / W, kLoadsB = BN / 8 / W;  // 1 KiB (8 rows) each, a wave
};

__device__ __forceinline__ int chunk_of(int row, int c) { return c ^ ((row ^ ((row >> 3) & 1)) & 7); }

template <class O, class T>
__global__ __launch_bounds__(T::W * 64, T::W / 4 == 2 ? 2 : 1) void i8_tiles_kernel(I8Linear a, int m_tiles, int n_tiles) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = wave_id(), row = lane & 31, h = lane >> 5;
    // Workgroups go to the 8 XCDs in turn: each XCD takes one run of tiles, 8 token
    // tiles deep before the next channels, so that what it loads meets its own L2.
    const int tiles = m_tiles * n_tiles, per = (tiles + 7) / 8;
    const int t = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3);
    if (t >= tiles || (int)(blockIdx.x >> 3) >= per) return;
    const int band = t / (8 * n_tiles), deep = min(8, m_tiles - 8 * band), in_band = t - band * 8 * n_tiles;
    const int m0 = (8 * band + in_band % deep) * T::BM, n0 = in_band / deep * T::BN;
    const int k_end = (a.in_feat + 15) & ~15;
    const int m_rows = min(T::BM, a.batch - m0), n_rows = min(T::BN, a.out_feat - n0);
    const int8_t* xp = a.x + (size_t)m0 * a.ld_x;
    const int8_t* wp = a.w + (size_t)n0 * a.ld_w;
    const int x_bytes = (int)((m_rows - 1) * a.ld_x) + k_end, w_bytes = (int)((n_rows - 1) * a.ld_w) + k_end;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8*)lds;
    // this lane's part of a load: row lane / 8 of its 8, chunk lane % 8 in LDS
    uint32_t off_a[T::kLoadsA], off_b[T::kLoadsB];
    const auto at = [&](int r, size_t ld) { return (uint32_t)(r * ld) + 16u * chunk_of(r, lane & 7); };
#pragma unroll
    for (int i = 0; i < T::kLoadsA; i++) off_a[i] = at((wave * T::kLoadsA + i) * 8 + lane / 8, a.ld_x);
#pragma unroll
    for (int i = 0; i < T::kLoadsB; i++) off_b[i] = at((wave * T::kLoadsB + i) * 8 + lane / 8, a.ld_w);
    auto load = [&](int k, int stage) {
        const __amdgpu_buffer_rsrc_t rx =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(xp + k), (short)0, x_bytes - k, kWord3);
        const __amdgpu_buffer_rsrc_t rw =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(wp + k), (short)0, w_bytes - k, kWord3);
        const uint32_t to = lds0 + (uint32_t)stage * T::kStage;
        // chunks past the row's end, in the last step, read as zeros
        const auto cut = [&](uint32_t off, int r) {
            return k + 128 > k_end && k + 16 * chunk_of(r, lane & 7) >= k_end ? 0x7FFFFFF0u : off;
        };
#pragma unroll
        for (int i = 0; i < T::kLoadsA; i++) {
            const int first = (wave * T::kLoadsA + i) * 8;
            load_to_lds<16>(rx, cut(off_a[i], first + lane / 8), to + (uint32_t)first * 128u);
        }
#pragma unroll
        for (int i = 0; i < T::kLoadsB; i++) {
            const int first = (wave * T::kLoadsB + i) * 8;
            load_to_lds<16>(rw, cut(off_b[i], first + lane / 8), to + T::BM * 128u + (uint32_t)first * 128u);
        }
    };
    v16i acc[T::TM][T::TN];
#pragma unroll
    for (int i = 0; i < T::TM; i++)
#pragma unroll
        for (int j = 0; j < T::TN; j++) acc[i][j] = v16i{};
    const int wm = wave / T::WN * T::TM * 32, wn = wave % T::WN * T::TN * 32;
    load(0, 0);
    for (int k = 0, stage = 0; k < k_end; k += 128, stage ^= 1) {
        wait_vmcnt<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (k + 128 < k_end) load(k + 128, stage ^ 1);
        const uint8_t* la = lds + stage * T::kStage + (wm + row) * 128;
        const uint8_t* lb = lds + stage * T::kStage + (T::BM + wn + row) * 128;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            // rows 16 apart have the same permutation
            const int c = 16 * chunk_of(row, 2 * s + h);
            v4i av[T::TM], bv[T::TN];
#pragma unroll
            for (int i = 0; i < T::TM; i++) av[i] = *reinterpret_cast<const v4i*>(la + i * 32 * 128 + c);
#pragma unroll
            for (int j = 0; j < T::TN; j++) bv[j] = *reinterpret_cast<const v4i*>(lb + j * 32 * 128 + c);
#pragma unroll
            for (int i = 0; i < T::TM; i++)
#pragma unroll
                for (int j = 0; j < T::TN; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[i], bv[j], acc[i][j], 0, 0, 0);
        }
    }
    // acc: channel lane & 31, tokens 8 (r / 4) + 4 h + r % 4
#pragma unroll
    for (int j = 0; j < T::TN; j++) {
        const int n = wn + 32 * j + row;
        if (n >= n_rows) continue;
#pragma unroll
        for (int i = 0; i < T::TM; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const int m = wm + 32 * i + 8 * (r / 4) + 4 * h + r % 4;
                if (m < m_rows) store<O>(a, m0 + m, n0 + n, acc[i][j][r]);
            }
    }
}

using Tiles256 = Tiles<4, 2, 2, 4>;     // 256 x 256, 8 waves
using Tiles128 = Tiles<2, 2, 2, 2>;     // 128 x 128, 4 waves
using Tiles256x128 = Tiles<4, 2, 2, 2>;  // 4 waves

template <class O, class T>
hipError_t launch_tiles(const I8Linear& a, hipStream_t stream) {
    const int m_tiles = (a.batch + T::BM - 1) / T::BM, n_tiles = (a.out_feat + T::BN - 1) / T::BN;
    const void* f = reinterpret_cast<const void*>(&i8_tiles_kernel<O, T>);
    if (hipError_t e = allow_dynamic_lds(f, 2 * T::kStage)) return e;
    const int per = (m_tiles * n_tiles + 7) / 8;
    hipLaunchKernelGGL((i8_tiles_kernel<O, T>), dim3((unsigned)per * 8), dim3(T::W * 64), 2 * T::kStage, stream, a, m_tiles,
                       n_tiles);
    return hipGetLastError();
}

template <class O, int W, int MT>
hipError_t launch_rows(const I8Linear& a, hipStream_t stream) {
    hipLaunchKernelGGL((i8_rows_kernel<O, W, MT>), dim3((unsigned)((a.out_feat + 15) / 16), (unsigned)((a.batch + 16 * MT - 1) / (16 * MT))),
                       dim3(W * 64), 0, stream, a);
    return hipGetLastError();
}

template <class O>
hipError_t launch_form(const I8Linear& a, int form, hipStream_t stream) {
    switch (form) {
    case 0: return launch_rows<O, 4, 1>(a, stream);
    case 1: return launch_rows<O, 8, 1>(a, stream);
    case 2: return launch_rows<O, 4, 2>(a, stream);
    case 3: return launch_rows<O, 4, 4>(a, stream);
    case 4: return launch_tiles<O, Tiles128>(a, stream);
    case 5: return launch_tiles<O, Tiles256x128>(a, stream);
    default: return launch_tiles<O, Tiles256>(a, stream);
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
    const int form = a.batch <= 16 ? 1 : a.batch <= 32 ? 2 : a.batch <= 64 ? 3 : a.batch <= 1024 ? 4 : 6;
    // a launch takes a part of the tokens, so that its grid stays in range
    const int64_t most = ((int64_t)1 << 28) / (a.out_feat + 255) * 256;
    const int step = (int)std::max<int64_t>(256, std::min<int64_t>(most, 65535 * 16));
    for (int m0 = 0; m0 < a.batch; m0 += step) {
        I8Linear b = a;
        b.batch = std::min(step, a.batch - m0);
        b.x = a.x + (size_t)m0 * a.ld_x;
        b.xs = a.xs + (a.in_feat ? m0 : 0);
        b.y = static_cast<char*>(a.y) + (size_t)m0 * a.ld_y * type_bytes(y_type);
        const hipError_t e = with_type(y_type, [&](auto t) { return launch_form<decltype(t)>(b, form, stream); });
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace vtq
