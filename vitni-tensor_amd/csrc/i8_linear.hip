// i8_linear.hip -- activations to 8 bits a token, and the int8 product with scales
// per token and output channel (gfx950).
//
//   s_m = max_k |x_mk| / 127,  q_mk = x_mk / s_m rounded,  y_mn = s_m t_n sum_k q_mk w_nk + b_n
//
// Integer sums are exact in any order, so how K is split never shows.  Few tokens are
// bound by the weights' bytes, many by the matrix cores: vtq_i8_rules.h says which form
// takes a call.
#include <algorithm>

#include "vtq_device.h"
#include "vtq_i8_rules.h"
#include "vtq_kernels.h"
#include "vtq_lds_load.h"
#include "vtq_serve.h"

namespace vtq {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
constexpr int kWord3 = 0x00020000;  // raw buffer, stride 0

// ------------------------------------------------ quantization

// x / s to the nearest whole number, ties to even, of the exact quotient.  e is the
// nearest even one by the rounded reciprocal (off by two units in its last place at
// most: the quotient lies within 1 + 2^-15 of e); the remainder, exact in one fma (a
// multiple of the smaller unit in the last place, below 2 s in magnitude), says whether
// an odd neighbour is nearer, and a tie stays with e.
__device__ __forceinline__ int quotient(float x, float s, float half_inv) {
    const float e = rintf(x * half_inv), r = fmaf(-e, 2.0f * s, x), h = 0.5f * s;
    const int q = 2 * (int)e + (r > h ? 1 : 0) - (r < -h ? 1 : 0);
    return min(max(q, -127), 127);  // a scale of one subnormal step may be a third too small
}

// A thread takes 16 elements at a time, whole 16-byte pieces of the output; rows of up
// to 16384 stay in registers between the maximum and the rounding.  Rows of up to 1024
// elements take one wave of a workgroup's four, longer ones a workgroup.  One row of
// 4096 bf16 takes 3.4 us, a launch's own time (11.1 with an element at a time, twice
// read), 4001 rows 13.7 us, 3.6 TB/s; the rest is arithmetic (15.8 us with the remainder
// against the nearest number and a rule for ties, 4.2 for one row).
constexpr int kQuantMost = 1024;  // threads

template <class T>
__device__ __forceinline__ void load16(float (&f)[16], const T* p, int left, bool whole) {
    if (whole && left >= 16) {
        typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
        constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < 16 / N; i++) {
            const vec v = reinterpret_cast<const vec*>(p)[i];
#pragma unroll
            for (int e = 0; e < N; e++) f[i * N + e] = (float)v[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; e++) f[e] = e < left ? (float)p[e] : 0.0f;
    }
}

__device__ __forceinline__ uint32_t top_bits(const float (&f)[16]) {
    uint32_t a = 0;  // magnitudes by their bits: a NaN is above an infinity above every number
#pragma unroll
    for (int e = 0; e < 16; e++) a = max(a, __float_as_uint(f[e]) & 0x7FFFFFFFu);
    return a;
}

// tpr: threads of a row, 64 (the workgroup's waves have a row each) or the whole workgroup
template <class T>
__global__ __launch_bounds__(kQuantMost, 8) void quantize_kernel(const T* x, size_t ld_x, int8_t* q, size_t ld_q,
                                                              float* scale, int rows, int n, int tpr, bool whole) {
    __shared__ uint32_t top[kQuantMost / 64];
    const int per = (int)blockDim.x / tpr, t = (int)threadIdx.x % tpr;
    for (int64_t m0 = (int64_t)blockIdx.x * per; m0 < rows; m0 += (int64_t)gridDim.x * per) {
        const int64_t m = m0 + (int)threadIdx.x / tpr;
        const bool row = m < rows;
        const T* xr = x + (row ? m : 0) * ld_x;
        const int last = row ? n : 0;
        float f[16];
        load16(f, xr + 16 * t, last - 16 * t, whole);
        uint32_t a = top_bits(f);
        for (int k = 16 * (t + tpr); k < last; k += 16 * tpr) {
            float g[16];
            load16(g, xr + k, last - k, whole);
            a = max(a, top_bits(g));
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) a = max(a, (uint32_t)__shfl_xor((int)a, d, 64));
        if (tpr > 64) {
            if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = a;
            __syncthreads();
            for (int w = 0; w < tpr / 64; w++) a = max(a, top[w]);
            __syncthreads();
        }
        if (!row) continue;
        const float s = a < 0x7F800000u ? __uint_as_float(a) / 127.0f : __uint_as_float(a);
        const bool some = a < 0x7F800000u && s > 0.0f;
        // where the reciprocal would overflow, both are scaled: exact powers of two
        const float up = s < 0x1p-100f ? 0x1p100f : 1.0f, su = s * up, half_inv = some ? 0.5f / su : 0.0f;
        if (t == 0) scale[m] = s;
        for (size_t k = 16 * (size_t)t; k < ld_q; k += 16 * (size_t)tpr) {
            if (k != 16 * (size_t)t) load16(f, xr + k, n > (int64_t)k ? n - (int)k : 0, whole);
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                o[i] = 0;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    o[i] |= (uint32_t)((some ? quotient(f[4 * i + e] * up, su, half_inv) : 0) & 255) << (8 * e);
            }
            *reinterpret_cast<uint4*>(q + m * ld_q + k) = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// One output before its type: the sum to f32, its two scales and the bias, each rounded
// once.  (No inputs: scales that are not there count as 0.)
__device__ __forceinline__ float scaled(int sum, float xs, float ws, float bias) { return (float)sum * xs * ws + bias; }

// ------------------------------------------------ product, few tokens

// A workgroup owns 16 output channels x 16 tokens, its waves every fourth 256 bytes of
// K; lane (r, g) of a wave takes the 64 bytes g of row r, channel and token alike (the
// order of K inside an MFMA is free as long as both operands share it).  The next
// 256 bytes load while these multiply.  Bound by the weights: 1 x 11008 -> 4096 10.3 us,
// 4.4 TB/s (8 waves 11.6, 16 waves 12.4).
constexpr int kRowWaves = 4;
struct RowOperands {
    v4i w[4], x[4];
};

template <class O>
__global__ __launch_bounds__(kRowWaves * 64) void i8_rows_kernel(I8Linear a) {
    __shared__ int part[kRowWaves][16][17];
    const int lane = threadIdx.x & 63, wave = wave_id(), r = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16;
    const int k_end = (a.in_feat + 15) & ~15;
    const int n_rows = min(16, a.out_feat - n0), m_rows = min(16, a.batch - m0);
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<int8_t*>(a.w + (size_t)n0 * a.ld_w), (short)0, (int)((n_rows - 1) * a.ld_w + k_end), kWord3);
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<int8_t*>(a.x + (size_t)m0 * a.ld_x), (short)0, (int)((m_rows - 1) * a.ld_x + k_end), kWord3);
    v4i acc = {0, 0, 0, 0};
    auto load = [&](RowOperands& o, int k) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = k + g * 64 + i * 16;
            // rows past the last one and bytes past the row give zeros
            const int ow = at < k_end && r < n_rows ? (int)(r * a.ld_w) + at : -16;
            const int ox = at < k_end && r < m_rows ? (int)(r * a.ld_x) + at : -16;
            o.w[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rw, ow, 0, 0));
            o.x[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, ox, 0, 0));
        }
    };
    auto multiply = [&](const RowOperands& o) {
#pragma unroll
        for (int i = 0; i < 4; i++) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(o.x[i], o.w[i], acc, 0, 0, 0);
    };
    RowOperands u, v;
    int k = wave * 256;
    load(u, k);
    for (; k < k_end; k += 2 * kRowWaves * 256) {
        load(v, k + kRowWaves * 256);
        multiply(u);
        load(u, k + 2 * kRowWaves * 256);
        multiply(v);
    }
    // acc: channel lane & 15, tokens 4 (lane >> 4) + 0..3
#pragma unroll
    for (int i = 0; i < 4; i++) part[wave][4 * g + i][r] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < 256; e += kRowWaves * 64) {
        const int m = e >> 4, n = e & 15;
        if (m >= m_rows || n >= n_rows) continue;
        int sum = 0;
#pragma unroll
        for (int w = 0; w < kRowWaves; w++) sum += part[w][m][n];
        static_cast<O*>(a.y)[(size_t)(m0 + m) * a.ld_y + n0 + n] =
            (O)scaled(sum, a.in_feat ? a.xs[m0 + m] : 0.0f, a.in_feat ? a.ws[n0 + n] : 0.0f,
                      a.bias ? a.bias[n0 + n] : 0.0f);
    }
}

// ------------------------------------------------ product, many tokens

// A workgroup owns BM tokens x BN channels, a wave 32 TM x 32 TN of them on 32x32x32
// MFMAs.  Tiles of both operands go from memory straight to LDS, S stages of 128
// bytes of K; the 16-byte chunks of a row are permuted so that the 16 rows that a
// read takes at one column lie in different banks.  Operands are read one MFMA group
// ahead, across the stages' barrier too; loads past the last stage read zeros from
// nowhere, so that the count of those in flight stays the same.  Bound by the matrix
// cores and what feeds them: 4001 x 4096 -> 11008 165-200 us, about 2000 TOP/s; 512 x
// 4096 -> 14336 33 us, 1820 TOP/s.
typedef int v16i __attribute__((ext_vector_type(16)));

template <int TM_, int TN_, int WM_, int WN_, int S_, int PER_CU_>
struct Tiles {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, S = S_, PER_CU = PER_CU_;
    static constexpr int W = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN;
    static constexpr int kStage = (BM + BN) * 128;
    static constexpr int kLoadsA = BM / 8 / W, kLoadsB = BN / 8 / W;  // 1 KiB (8 rows) each, a wave
};

__device__ __forceinline__ int chunk_of(int row, int c) { return c ^ ((row ^ ((row >> 3) & 1)) & 7); }

template <class O, class T>
__global__ __launch_bounds__(T::W * 64, T::PER_CU * T::W / 4) void i8_tiles_kernel(I8Linear a, int m_tiles,
        int n_tiles) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ __attribute__((aligned(16))) float x_scale[T::BM], w_scale[T::BN], w_bias[T::BN];
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
            __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(xp + k), (short)0, k < k_end ? x_bytes - k : 0,
                                              kWord3);
        const __amdgpu_buffer_rsrc_t rw =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(wp + k), (short)0, k < k_end ? w_bytes - k : 0,
                                              kWord3);
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
    // operands of 32 inputs: step s of the stage at `from`
    struct Operands {
        v4i a[T::TM], b[T::TN];
    };
    auto read = [&](Operands& o, const uint8_t* from, int s) {
        const int c = 16 * chunk_of(row, 2 * s + h);  // rows 16 apart have the same permutation
#pragma unroll
        for (int i = 0; i < T::TM; i++) o.a[i] = *reinterpret_cast<const v4i*>(from + (wm + row + 32 * i) * 128 + c);
#pragma unroll
        for (int j = 0; j < T::TN; j++)
            o.b[j] = *reinterpret_cast<const v4i*>(from + (T::BM + wn + row + 32 * j) * 128 + c);
    };
    auto multiply = [&](const Operands& o) {
#pragma unroll
        for (int i = 0; i < T::TM; i++)
#pragma unroll
            for (int j = 0; j < T::TN; j++)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(o.b[j], o.a[i], acc[i][j], 0, 0, 0);
    };
    for (int m = threadIdx.x; m < T::BM; m += T::W * 64) x_scale[m] = m < m_rows && a.in_feat ? a.xs[m0 + m] : 0.0f;
    for (int n = threadIdx.x; n < T::BN; n += T::W * 64) {
        w_scale[n] = n < n_rows && a.in_feat ? a.ws[n0 + n] : 0.0f;
        w_bias[n] = n < n_rows && a.bias ? a.bias[n0 + n] : 0.0f;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // seen by all after the loop's barriers
    constexpr int kLoads = T::kLoadsA + T::kLoadsB;
#pragma unroll
    for (int i = 0; i < T::S; i++) load(128 * i, i);
    wait_vmcnt<(T::S - 1) * kLoads>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    Operands x[2];
    read(x[0], lds, 0);
    int stage = 0;
    for (int k = 0; k < k_end; k += 128) {
        const uint8_t* here = lds + stage * T::kStage;
#pragma unroll
        for (int s = 0; s < 3; s++) {
            read(x[(s + 1) & 1], here, s + 1);
            multiply(x[s & 1]);
        }
        // The stage's last operands are in registers: once every wave is here it is free
        // for the loads of S steps on, and the next one has landed.
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        wait_vmcnt<(T::S - 2) * kLoads>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int next = stage + 1 == T::S ? 0 : stage + 1;
        read(x[0], lds + next * T::kStage, 0);
        load(k + 128 * T::S, stage);
        multiply(x[1]);
        stage = next;
    }
    // The tile's outputs go through the wave's own part of LDS, 32 tokens at a time, so
    // that rows of 16-byte pieces leave (written as the MFMAs hold them, 256 x 256 of
    // bf16 took a workgroup 27 us).  acc: token lane & 31, channels 8 g + 4 h + e.
    wait_vmcnt<0>();  // the loads of zeros
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    typedef O o4 __attribute__((ext_vector_type(4)));
    constexpr int kRow = T::TN * 32 * (int)sizeof(O), kPitch = kRow + 16, kPieces = kRow / 16,
            kEach = 16 / (int)sizeof(O);
    static_assert(32 * kPitch * T::W <= T::S * T::kStage, "LDS of the epilogue");
    uint8_t* out = lds + wave * 32 * kPitch;
    O* y = static_cast<O*>(a.y) + (size_t)(m0 + wm) * a.ld_y + n0 + wn;
    const bool whole = reinterpret_cast<uintptr_t>(y) % 16 == 0 && a.ld_y * sizeof(O) % 16 == 0;
#pragma unroll
    for (int i = 0; i < T::TM; i++) {
        const float xs = x_scale[wm + 32 * i + row];
#pragma unroll
        for (int j = 0; j < T::TN; j++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const int n = 32 * j + 8 * g + 4 * h;
                const float4 ws = *reinterpret_cast<const float4*>(&w_scale[wn + n]);
                const float4 bias = *reinterpret_cast<const float4*>(&w_bias[wn + n]);
                o4 v;
                v[0] = (O)scaled(acc[i][j][4 * g], xs, ws.x, bias.x);
                v[1] = (O)scaled(acc[i][j][4 * g + 1], xs, ws.y, bias.y);
                v[2] = (O)scaled(acc[i][j][4 * g + 2], xs, ws.z, bias.z);
                v[3] = (O)scaled(acc[i][j][4 * g + 3], xs, ws.w, bias.w);
                *reinterpret_cast<o4*>(out + row * kPitch + n * (int)sizeof(O)) = v;
            }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // a wave's LDS accesses are in order
#pragma unroll
        for (int p = 0; p < 32 * kPieces / 64; p++) {
            const int m = (p * 64 + lane) / kPieces, c = (p * 64 + lane) % kPieces;
            if (wm + 32 * i + m >= m_rows) continue;
            const uint8_t* from = out + m * kPitch + c * 16;
            O* to = y + (size_t)(32 * i + m) * a.ld_y + c * kEach;
            if (whole && wn + (c + 1) * kEach <= n_rows) {
                *reinterpret_cast<v4i*>(to) = *reinterpret_cast<const v4i*>(from);
            } else {
                for (int e = 0; e < kEach; e++)
                    if (wn + c * kEach + e < n_rows) to[e] = reinterpret_cast<const O*>(from)[e];
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

using Tiles128 = Tiles<2, 2, 2, 2, 4, 1>;     // 128 x 128, deep: grids that leave a CU one workgroup
using Pair128 = Tiles<2, 1, 2, 4, 2, 2>;      // 128 x 128, two workgroups a CU
using Tiles128x256 = Tiles<2, 2, 2, 4, 3, 1>;
using Tiles256 = Tiles<4, 2, 2, 4, 2, 1>;

// ------------------------------------------------ product, some tens of tokens

// A workgroup owns 32 TM tokens x 32 channels, its 4 waves every fourth 128 bytes of K,
// each with tiles of its own in LDS, S deep: nothing waits for another wave until the
// sums are joined.  Bound by the weights: 19 x 11008 -> 4096 12.7 us, 3.6 TB/s.
template <class O, int TM, int S>
__global__ __launch_bounds__(256, 1) void i8_slices_kernel(I8Linear a) {
    constexpr int kStage = (TM + 1) * 4096, kLoads = (TM + 1) * 4, BM = 32 * TM;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = wave_id(), row = lane & 31, h = lane >> 5;
    const int n0 = (int)blockIdx.x * 32, m0 = (int)blockIdx.y * BM;
    const int k_end = (a.in_feat + 15) & ~15;
    const int m_rows = min(BM, a.batch - m0), n_rows = min(32, a.out_feat - n0);
    const int8_t* xp = a.x + (size_t)m0 * a.ld_x;
    const int8_t* wp = a.w + (size_t)n0 * a.ld_w;
    const int x_bytes = (int)((m_rows - 1) * a.ld_x) + k_end, w_bytes = (int)((n_rows - 1) * a.ld_w) + k_end;
    uint8_t* mine = lds + wave * S * kStage;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8*)mine;
    auto load = [&](int k, int stage) {
        const __amdgpu_buffer_rsrc_t rx =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(xp + k), (short)0, k < k_end ? x_bytes - k : 0,
                                              kWord3);
        const __amdgpu_buffer_rsrc_t rw =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(wp + k), (short)0, k < k_end ? w_bytes - k : 0,
                                              kWord3);
        const uint32_t to = lds0 + (uint32_t)stage * kStage;
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const bool is_w = i < 4;
            const int r = (is_w ? i : i - 4) * 8 + lane / 8, c = 16 * chunk_of(r, lane & 7);
            // chunks past the row's end, in the last step, read as zeros
            const uint32_t at = (uint32_t)(r * (is_w ? a.ld_w : a.ld_x)) + (uint32_t)c;
            const uint32_t off = k + 128 > k_end && k + c >= k_end ? 0x7FFFFFF0u : at;
            load_to_lds<16>(is_w ? rw : rx, off, to + 1024u * i);
        }
    };
    v16i acc[TM];
#pragma unroll
    for (int i = 0; i < TM; i++) acc[i] = v16i{};
    const int k0 = wave * 128;
#pragma unroll
    for (int i = 0; i < S; i++) load(k0 + 512 * i, i);
    int stage = 0;
    for (int k = k0; k < k_end; k += 512) {
        wait_vmcnt<(S - 1) * kLoads>();
        asm volatile("" ::: "memory");
        const uint8_t* from = mine + stage * kStage + row * 128;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const int c = 16 * chunk_of(row, 2 * s + h);
            const v4i w = *reinterpret_cast<const v4i*>(from + c);
#pragma unroll
            for (int i = 0; i < TM; i++)
                acc[i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(
                    w, *reinterpret_cast<const v4i*>(from + (i + 1) * 4096 + c), acc[i], 0, 0, 0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: free for the loads of S steps on
        load(k + 512 * S, stage);
        stage = stage + 1 == S ? 0 : stage + 1;
    }
    wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    // acc: token lane & 31, channels 8 g + 4 h + e.  Sums of a token: 32 channels and a pad.
    static_assert(BM * 36 * 4 <= S * kStage, "LDS of the sums");
    int* sums = reinterpret_cast<int*>(mine);
#pragma unroll
    for (int i = 0; i < TM; i++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *reinterpret_cast<v4i*>(sums + (32 * i + row) * 36 + 8 * g + 4 * h) =
                v4i{acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]};
    __syncthreads();
    for (int e = threadIdx.x; e < BM * 8; e += 256) {
        const int m = e / 8, n = e % 8 * 4;
        if (m >= m_rows || n >= n_rows) continue;
        v4i sum = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++)
            sum += *reinterpret_cast<const v4i*>(reinterpret_cast<const int*>(lds + w * S * kStage) + m * 36 + n);
        const float xs = a.in_feat ? a.xs[m0 + m] : 0.0f;
        O* y = static_cast<O*>(a.y) + (size_t)(m0 + m) * a.ld_y + n0 + n;
        typedef O o4 __attribute__((ext_vector_type(4)));
        o4 v;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool in = n + i < n_rows;
            v[i] = (O)scaled(sum[i], xs, in && a.in_feat ? a.ws[n0 + n + i] : 0.0f,
                             in && a.bias ? a.bias[n0 + n + i] : 0.0f);
        }
        if (n + 4 <= n_rows && reinterpret_cast<uintptr_t>(y) % sizeof(o4) == 0) {
            *reinterpret_cast<o4*>(y) = v;
        } else {
            for (int i = 0; i < 4 && n + i < n_rows; i++) y[i] = v[i];
        }
    }
}

template <class O, int TM, int S>
hipError_t launch_slices(const I8Linear& a, hipStream_t stream) {
    const void* f = reinterpret_cast<const void*>(&i8_slices_kernel<O, TM, S>);
    constexpr int bytes = 4 * S * (TM + 1) * 4096;
    if (hipError_t e = allow_dynamic_lds(f, bytes)) return e;
    hipLaunchKernelGGL((i8_slices_kernel<O, TM, S>),
                       dim3((unsigned)((a.out_feat + 31) / 32), (unsigned)((a.batch + 32 * TM - 1) / (32 * TM))),
                               dim3(256),
                       bytes, stream, a);
    return hipGetLastError();
}

template <class O, class T>
hipError_t launch_tiles(const I8Linear& a, hipStream_t stream) {
    const int m_tiles = (a.batch + T::BM - 1) / T::BM, n_tiles = (a.out_feat + T::BN - 1) / T::BN;
    const void* f = reinterpret_cast<const void*>(&i8_tiles_kernel<O, T>);
    if (hipError_t e = allow_dynamic_lds(f, T::S * T::kStage + 4096)) return e;
    const int per = (m_tiles * n_tiles + 7) / 8;
    hipLaunchKernelGGL((i8_tiles_kernel<O, T>), dim3((unsigned)per * 8), dim3(T::W * 64), T::S * T::kStage, stream,
                       a, m_tiles,
                       n_tiles);
    return hipGetLastError();
}

template <class O>
hipError_t launch_rows(const I8Linear& a, hipStream_t stream) {
    const dim3 grid((unsigned)((a.out_feat + 15) / 16), (unsigned)((a.batch + 15) / 16));
    hipLaunchKernelGGL((i8_rows_kernel<O>), grid, dim3(kRowWaves * 64), 0, stream, a);
    return hipGetLastError();
}

template <class O>
hipError_t launch_form(const I8Linear& a, I8Form form, hipStream_t stream) {
    switch (form) {
    case kI8Rows: return launch_rows<O>(a, stream);
    case kI8Slices32: return launch_slices<O, 1, 2>(a, stream);
    case kI8Slices64: return launch_slices<O, 2, 2>(a, stream);
    case kI8Slices128: return launch_slices<O, 4, 2>(a, stream);
    case kI8Tiles128: return launch_tiles<O, Tiles128>(a, stream);
    case kI8Pair128: return launch_tiles<O, Pair128>(a, stream);
    case kI8Tiles128x256: return launch_tiles<O, Tiles128x256>(a, stream);
    case kI8Tiles256: return launch_tiles<O, Tiles256>(a, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_quantize_i8(int type, const void* x, size_t ld_x, int8_t* q, size_t ld_q, float* scale, size_t rows,
                              int n, hipStream_t stream) {
    const size_t es = type_bytes(type);
    const bool whole = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (rows == 1 || ld_x * es % 16 == 0);
    const int tpr = n <= 1024 ? 64 : std::min(kQuantMost, (n + 1023) / 1024 * 64);
    const int threads = tpr == 64 ? 256 : tpr, per = threads / tpr;
    const unsigned grid = (unsigned)std::min<size_t>((rows + per - 1) / per, 1 << 20);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((quantize_kernel<T>), dim3(grid), dim3(threads), 0, stream, static_cast<const T*>(x),
                           ld_x, q,
                           ld_q, scale, (int)rows, n, tpr, whole);
        return hipGetLastError();
    });
}

hipError_t launch_linear_i8(const I8Linear& a, int y_type, hipStream_t stream) {
    // a launch takes a part of the channels and tokens, so that its grid stays in range
    // (at most a thread per output of the smallest tiles, 2^31, and 65535 in y)
    const int n_step = 1 << 20;
    for (int n0 = 0; n0 < a.out_feat; n0 += std::min(n_step, a.out_feat - n0)) {
        I8Linear b = a;
        b.out_feat = std::min(n_step, a.out_feat - n0);
        b.w = a.w + (size_t)n0 * a.ld_w;
        b.ws = a.in_feat ? a.ws + n0 : a.ws;
        b.bias = a.bias ? a.bias + n0 : nullptr;
        const int m_step = (int)std::min<int64_t>(((int64_t)1 << 31) / std::max(b.out_feat, 1024) / 256 * 256, 65535 * 16);
        for (int m0 = 0; m0 < a.batch; m0 += std::min(m_step, a.batch - m0)) {
            b.batch = std::min(m_step, a.batch - m0);
            b.x = a.x + (size_t)m0 * a.ld_x;
            b.xs = a.in_feat ? a.xs + m0 : a.xs;
            b.y = static_cast<char*>(a.y) + ((size_t)m0 * a.ld_y + n0) * type_bytes(y_type);
            const I8Form form = i8_form(b.batch, b.in_feat, b.out_feat);
            const hipError_t e = with_type(y_type, [&](auto t) { return launch_form<decltype(t)>(b, form, stream); });
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

}  // namespace vtq
