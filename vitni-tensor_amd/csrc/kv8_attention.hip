// kv8_attention.hip -- attention of a ragged batch over a paged cache of 8-bit floats
// with a scale to each block of tokens and head (gfx950).
//
//   y = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),  m = max_j scale q.k_j,
//   k_j = 2^a k8_j,  v_j = 2^b v8_j,  a and b those of key j's block
//
// Workgroups, key ranges, products and the join are as in cache_attention.hip: S^T = K Q^T
// and O^T += V^T P^T on 32x32 MFMAs, one pass with a running maximum and sum.  Tiles stay
// 8 bits wide from memory to the registers, half the bytes of a 16-bit cache; the conversion to
// bf16, two elements an instruction, multiplies by the block's power of two at no cost
// and loses nothing (4 significant bits of 8).  bf16 queries meet bf16 keys; f16 ones meet
// keys as f16, whose scores are scaled after; f32 ones are split into three bf16 parts,
// exactly.  Weights are rounded to one (bf16), two (f16) or three (f32) bf16 parts, so
// that every type runs at the 16-bit products' rate.
//
// K: a lane reads 16 elements of its key at once, for two products; the order of a head's
// elements inside them is free as long as the query has the same.  V's transpose is the
// 8-bit transposing read: 16 lanes give 8 keys x 16 elements and get an element of all 8
// each, which are the keys that this half-wave's weights are of.
//
// Heads of more than 128 elements: a workgroup has half of the values' elements, and works
// out all scores for them.  (The sums of all in one wave, 128 registers beside the query's 64,
// spilled in every loop: 26 sequences of 7 behind 8099 keys, f16, 565 us against 100.)
//
// Measured (8 KV heads of 128, groups of 4, bf16; 16-bit keys in brackets): 128 sequences behind
// 32768 keys with up to 1024 of their own 111 and 6 to join (145); the prefix alone 99 (98), 700
// TFLOP/s at 2.05 GHz, the same with one workgroup a CU and with two.  There a SIMD's vector
// instructions, 210 to a tile beside its 16 products and one started every 4.4 cycles, take 68 %
// of its cycles and its products 35 %: they hardly overlap.  Its two waves wait for memory or LDS
// in a quarter of theirs, and for the other's turn in another.  (Without the softmax 15 us
// less, without the conversions 7.)  The own keys alone 41 (88), 4.9 TB/s; 8 sequences of
// 32000 88 (160).
#include <type_traits>

#include "vtq_attention_rows.h"

namespace vtq {
namespace {

typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i lds_v2i;
typedef __attribute__((address_space(3))) const v4u lds_v4u;
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr float kLargestBf16 = 3.3895313892515355e38f;  // 2^128 - 2^120

struct Job8 : Job {
    Scales s;
    int block_shift;
    int prefix_inside;  // own workgroups take the prefix's keys first
};

template <int D>
struct Tile8 {
    static constexpr int kRow = D;                   // bytes of a key in LDS
    static constexpr int kChunks = D / 16;
    static constexpr int kLoadRows = 1024 / D;       // rows of one wave load
    static constexpr int kBytes = 32 * D;            // 32 keys
    static constexpr int kLoads = 16 / kLoadRows;    // loads of 16 keys of K or V
    // The 16-byte chunks of a row are permuted so that no read meets its neighbours in
    // the same bank: K is read 16 rows at one column, V 8 rows (0 to 3 and 8 to 11, or
    // these and 4) x 32 bytes.  Both repeat after 16 rows.
    __device__ static int k_chunk(int row, int c) {
        if (kChunks == 4) return c ^ ((row >> 2) & 3);
        return kChunks == 8 ? c ^ ((row ^ ((row >> 3) & 1)) & 7) : c ^ (row & 15);
    }
    __device__ static int v_chunk(int row, int c) {
        return kChunks == 4 ? c ^ ((row >> 2) & 2) : c ^ ((row & 2) | ((row >> 1) & 4));
    }
};

// Scales of 32 keys: 16 keys lie in one block.
struct TileScales {
    float k0, k1, v0, v1;
};

// Keys of a page list, 16 at a time, which lie in one page and one block.  A lane holds
// where 16 keys are and their scales, 64 lanes 1024 keys from `first` on.
struct Runs {
    const int32_t* list;
    int keys;   // keys that exist: later ones read as zeros
    int first;  // in 16 keys
    int low, high;      // bytes from the head's start, -1: outside the cache
    int scales;         // bytes: the keys' scale, the values' 16 bits above
    int down;           // the values' are this much lower: 0 or kDown, the same in every lane
};

// Values above 2^80 may add up past f32's end though their mean does not: weights of up to 2^8 times 2^30
// keys times 448 x 2^119 are 2^166.  From the first 1024 keys on that have such a scale, a wave takes
// all values 2^-kDown as large as they count, and its sums so far too.  Powers of two change no bits, so
// that rows that do not see such a block are what they are without it; only values below 2^-77, whose
// scale would be none of a bf16, are off, by 2^-77 at most.
constexpr int kLargeScale = 127 + 80;

template <int DK, int DV>
struct Loader8 {
    using TK = Tile8<DK>;
    using TV = Tile8<DV>;
    const char *k, *v;  // of this KV head; v: of this part of its elements
    const uint8_t *k_scale, *v_scale;
    int64_t page_bytes, scale_page;
    uint32_t slot_bytes;
    int k_bytes, v_bytes, n_pages, page_shift, page_mask, block_shift;  // of a key's, of a value's row
    uint32_t k_off[TK::kLoads], v_off[TV::kLoads];

    __device__ __forceinline__ void init(const Job8& j, int head, int part) {
        const vtq_kv_cache& c = j.a.cache;
        const int64_t at = (int64_t)head * (int64_t)c.head_stride;
        k = static_cast<const char*>(c.k) + at;
        v = static_cast<const char*>(c.v) + at + part * DV;
        k_scale = j.s.k + head * j.s.head_stride;
        v_scale = j.s.v + head * j.s.head_stride;
        page_bytes = (int64_t)c.page_stride;
        scale_page = j.s.page_stride;
        slot_bytes = (uint32_t)c.slot_stride;
        k_bytes = c.head_dim;
        v_bytes = min(c.head_dim - part * DV, DV);
        n_pages = (int)c.n_pages;
        page_shift = j.page_shift;
        page_mask = c.page_size - 1;
        block_shift = j.block_shift;
        const int lane = threadIdx.x & 63;
        // chunks past head_dim read past the end: zeros
        auto at_chunk = [&](int row, int c, int bytes) {
            return c * 16 < bytes ? (uint32_t)row * slot_bytes + (uint32_t)c * 16 : 0x7FFFFFF0u;
        };
#pragma unroll
        for (int i = 0; i < TK::kLoads; i++) {
            const int row = i * TK::kLoadRows + lane / TK::kChunks;
            k_off[i] = at_chunk(row, TK::k_chunk(row, lane % TK::kChunks), k_bytes);
        }
#pragma unroll
        for (int i = 0; i < TV::kLoads; i++) {
            const int row = i * TV::kLoadRows + lane / TV::kChunks;
            v_off[i] = at_chunk(row, TV::v_chunk(row, lane % TV::kChunks), v_bytes);
        }
    }
    // Holds the runs from `key`'s on; whether their values are lower now than those before.
    __device__ __forceinline__ bool hold(Runs& p, int key) const {
        const int lane = threadIdx.x & 63;
        p.first = key >> 4;
        const int at = min(p.first + lane, (p.keys - 1) >> 4) * 16;
        const int page = p.list[at >> page_shift], slot = at & page_mask;
        const bool there = (uint32_t)page < (uint32_t)n_pages;
        const int64_t byte = there ? (int64_t)page * page_bytes + (int64_t)((uint64_t)(uint32_t)slot * slot_bytes) : -1;
        p.low = (int)(uint32_t)byte;
        p.high = (int)(byte >> 32);
        const int64_t scale = there ? (int64_t)page * scale_page + (slot >> block_shift) : 0;
        const int of_keys = there ? min(max((int)k_scale[scale], 10), 246) : 127;
        const int of_values = there ? min(max((int)v_scale[scale], 10), 246) : 127;
        const bool lower = !p.down && __ballot(of_values > kLargeScale);
        p.down = lower ? kDown : p.down;
        p.scales = of_keys | max(of_values - p.down, 1) << 16;
        // waited for here: left to its use, the wait would stand in every tile, and be one for
        // all loads to LDS in flight as well
        asm volatile("" : "+v"(p.low), "+v"(p.high), "+v"(p.scales));
        return lower;
    }
    // the lane of `key`'s 16 keys (those past the end have any)
    __device__ __forceinline__ int lane_of(const Runs& p, int key) const { return ((key >> 4) - p.first) & 63; }
    __device__ __forceinline__ TileScales scales(const Runs& p, int key) const {
        const int a = __builtin_amdgcn_readlane(p.scales, lane_of(p, key));
        const int b = __builtin_amdgcn_readlane(p.scales, lane_of(p, key + 16));
        TileScales s;
        s.k0 = __int_as_float((a & 0xFF) << 23);
        s.k1 = __int_as_float((b & 0xFF) << 23);
        s.v0 = __int_as_float(a >> 16 << 23);
        s.v1 = __int_as_float(b >> 16 << 23);
        return s;
    }
    // 16 keys from `key` on: K to k_lds, V to v_lds.
    static constexpr int kLoads = TK::kLoads + TV::kLoads;
    __device__ __forceinline__ void load16(const Runs& p, int key, uint32_t k_lds, uint32_t v_lds) const {
        const int lane = lane_of(p, key);
        const uint32_t low = (uint32_t)__builtin_amdgcn_readlane(p.low, lane);
        const int high = __builtin_amdgcn_readlane(p.high, lane);
        const int64_t at = (int64_t)(((uint64_t)(uint32_t)high << 32) | low);
        const int rows = min(16, p.keys - key);
        const int before = (rows - 1) * (int)slot_bytes;
        const bool there = rows > 0 && high >= 0;  // nothing is read at an address of no bytes
        const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(k + at), (short)0,
                                                                            there ? before + k_bytes : 0, kWord3);
        const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(v + at), (short)0,
                                                                            there ? before + v_bytes : 0, kWord3);
#pragma unroll
        for (int i = 0; i < TK::kLoads; i++) load_to_lds<16>(rk, k_off[i], k_lds + 1024u * i);
#pragma unroll
        for (int i = 0; i < TV::kLoads; i++) load_to_lds<16>(rv, v_off[i], v_lds + 1024u * i);
    }
};

__device__ __forceinline__ float lower_scale(float x) {
    return __int_as_float(max(__float_as_int(x) - (kDown << 23), 1 << 23));
}

// ------------------------------------------------ one tile of 32 keys

template <class Q, int DK, int DV>
struct Compute8 {
    using TK = Tile8<DK>;
    using TV = Tile8<DV>;
    static constexpr bool kHalf = std::is_same_v<Q, _Float16>;
    static constexpr int P = std::is_same_v<Q, float> ? 3 : kHalf ? 2 : 1;  // parts of a weight
    static constexpr int PQ = kHalf ? 1 : P;                                 // parts of a query
    static constexpr bool kPairs = DK <= 128 && P < 3;  // two tiles at a time, where registers allow
    using K = std::conditional_t<kHalf, _Float16, __bf16>;
    typedef K v8k __attribute__((ext_vector_type(8)));
    // q of row lane & 31: element d of 32 c + 16 h + 8 s + 0..7 is v[part][2 c + s]
    struct Query {
        v8k v[PQ][DK / 16];
    };
    struct Weights {
        v8bf v[P][2];
    };
    using Rows = State<DV>;

    // 8 elements in parts: give(part, element, it)
    template <class Give>
    __device__ __forceinline__ static void split(const Q* p, bool in, Give give) {
        typedef Q v8q __attribute__((ext_vector_type(8)));
        v8q x = {};
        if (in) x = *reinterpret_cast<const v8q*>(p);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (PQ == 1) {
                give(0, e, x[e]);
            } else {
                float rest = x[e];
#pragma unroll
                for (int i = 0; i < PQ; i++) {
                    // a finite number that would round to an infinity leaves its rest to the other parts, as
                    // many bits as they hold; an infinity's own rest would be no number: the first has it all
                    const bool finite = i || fabsf(rest) < INFINITY;
                    const float near = i ? rest : __builtin_amdgcn_fmed3f(rest, -kLargestBf16, kLargestBf16);
                    const __bf16 part = (__bf16)(finite ? near : rest);
                    give(i, e, part);
                    rest = finite ? rest - (float)part : 0.0f;
                }
            }
        }
    }
    __device__ static void load_query(Query& q, const Q* p, bool valid, int head_dim) {
        const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int s = 0; s < DK / 16; s++) {
            const int d = 32 * (s / 2) + 16 * h + 8 * (s & 1);
            split(p + d, valid && d < head_dim, [&](int part, int e, auto x) { q.v[part][s][e] = x; });
        }
    }

    __device__ __forceinline__ static v8bf widen(uint32_t a, uint32_t b, float scale) {
        v8bf r;
        const v2bf x = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false);
        const v2bf y = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true);
        const v2bf z = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false);
        const v2bf w = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true);
        r[0] = x[0], r[1] = x[1], r[2] = y[0], r[3] = y[1], r[4] = z[0], r[5] = z[1], r[6] = w[0], r[7] = w[1];
        return r;
    }
    // 8 elements of a key, scaled, or (f16 has not the exponents) as they are
    __device__ __forceinline__ static v8k widen_key(uint32_t a, uint32_t b, float scale) {
        if constexpr (kHalf) {
            v8k r;
            const auto x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
            const auto y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
            const auto z = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
            const auto w = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
            r[0] = x[0], r[1] = x[1], r[2] = y[0], r[3] = y[1], r[4] = z[0], r[5] = z[1], r[6] = w[0], r[7] = w[1];
            return r;
        } else {
            return widen(a, b, scale);
        }
    }
    __device__ __forceinline__ static v16f mma(v8bf a, v8bf b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    __device__ __forceinline__ static v16f mma_key(v8k a, v8k b, v16f c) {
        if constexpr (kHalf) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
        else return mma(a, b, c);
    }
    // f16: scores of keys in the two blocks of 16 (registers 0 to 7, 8 to 15)
    __device__ __forceinline__ static void scale_scores(v16f& s, TileScales sc) {
        if constexpr (kHalf) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] *= r < 8 ? sc.k0 : sc.k1;
        }
    }

    // A tile's operands as they are in LDS, read ahead of their products.
    struct Keys {
        v4u x[DK / 32];
    };
    struct Values {
        v2i x[DV / 32][2];
    };
    // A row's chunks differ in bits that the permutation only flips, so one address makes them all
    // (tiles begin at multiples of a row): kept ones for each spilled.
    __device__ __forceinline__ static uint32_t keys_from(const uint8_t* k) {
        const int lane = threadIdx.x & 63, row = lane & 31, h = lane >> 5;
        return (uint32_t)(uintptr_t)(lds_u8*)k + (uint32_t)(row * TK::kRow + TK::k_chunk(row, h) * 16);
    }
    __device__ __forceinline__ static v4u key_at(uint32_t from, int c) {
        return *(lds_v4u*)(uintptr_t)(from ^ (uint32_t)(32 * c));
    }
    // elements 32 b + (lane & 31) of keys 16 i + 4 h + {0..3, 8..11}
    __device__ __forceinline__ static uint32_t values_from(const uint8_t* v) {
        const int lane = threadIdx.x & 63, h = lane >> 5, n = lane & 15, r = n >> 1;
        const int row = 4 * h + (r & 3) + 8 * (r >> 2), c = (lane >> 4) & 1;
        return (uint32_t)(uintptr_t)(lds_u8*)v + (uint32_t)(row * TV::kRow + TV::v_chunk(row, c) * 16 + (n & 1) * 8);
    }
    __device__ __forceinline__ static v2i values_at(uint32_t from, int b, int i) {
        return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(uintptr_t)((from ^ (uint32_t)(32 * b)) + 16 * TV::kRow * i));
    }
    __device__ __forceinline__ static void read_keys(Keys& r, const uint8_t* k) {
        const uint32_t from = keys_from(k);
#pragma unroll
        for (int c = 0; c < DK / 32; c++) r.x[c] = key_at(from, c);
    }
    __device__ __forceinline__ static void read_values(Values& r, const uint8_t* v) {
        const uint32_t from = values_from(v);
#pragma unroll
        for (int b = 0; b < DV / 32; b++)
#pragma unroll
            for (int i = 0; i < 2; i++) r.x[b][i] = values_at(from, b, i);
    }
    __device__ __forceinline__ static float key_scale(TileScales sc) { return threadIdx.x & 16 ? sc.k1 : sc.k0; }
    // scores of 32 keys: register 4i + e is key 8i + 4h + e, row lane & 31
    __device__ __forceinline__ static v16f scores(const uint8_t* k, const Query& q, TileScales sc) {
        const float scale = key_scale(sc);
        const uint32_t from = keys_from(k);
        v16f s = {};
#pragma unroll
        for (int c = 0; c < DK / 32; c++) {
            const v4u x = key_at(from, c);
            const v8k a = widen_key(x[0], x[1], scale), b = widen_key(x[2], x[3], scale);
#pragma unroll
            for (int i = PQ - 1; i >= 0; i--) {  // small parts first
                s = mma_key(a, q.v[i][2 * c], s);
                s = mma_key(b, q.v[i][2 * c + 1], s);
            }
        }
        scale_scores(s, sc);
        return s;
    }
    // two tiles' scores, two chains of products that do not wait for each other
    __device__ __forceinline__ static void scores(v16f (&s)[2], const Keys& k0, const Keys& k1, const Query& q, TileScales sc0,
                                                  TileScales sc1) {
        const float scale0 = key_scale(sc0), scale1 = key_scale(sc1);
        s[0] = s[1] = v16f{};
#pragma unroll
        for (int c = 0; c < DK / 32; c++) {
            const v8k a0 = widen_key(k0.x[c][0], k0.x[c][1], scale0), a1 = widen_key(k1.x[c][0], k1.x[c][1], scale1);
            const v8k b0 = widen_key(k0.x[c][2], k0.x[c][3], scale0), b1 = widen_key(k1.x[c][2], k1.x[c][3], scale1);
#pragma unroll
            for (int i = PQ - 1; i >= 0; i--) {
                s[0] = mma_key(a0, q.v[i][2 * c], s[0]);
                s[1] = mma_key(a1, q.v[i][2 * c], s[1]);
                s[0] = mma_key(b0, q.v[i][2 * c + 1], s[0]);
                s[1] = mma_key(b1, q.v[i][2 * c + 1], s[1]);
            }
        }
        scale_scores(s[0], sc0);
        scale_scores(s[1], sc1);
    }
    __device__ __forceinline__ static void add_values(State<DV>& st, const Values& v, const Weights& w, TileScales sc) {
#pragma unroll
        for (int b = 0; b < DV / 32; b++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const v8bf x = widen((uint32_t)v.x[b][i][0], (uint32_t)v.x[b][i][1], i ? sc.v1 : sc.v0);
#pragma unroll
                for (int p = P - 1; p >= 0; p--) st.o[b] = mma(x, w.v[p][i], st.o[b]);
            }
    }

    __device__ __forceinline__ static Weights weights(const v16f& p) {
        Weights w;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            // Off by 2^-8 (bf16), 2^-16 (f16) or 2^-24 (f32) of each at most; the sum is of the
            // unrounded ones, in f32.  In bf16 that leaves y 1.8e-3 off 64 bits, 1.6e-3 of which are
            // its own rounding (128 behind 32768 keys, in the norm); a second part would take half as
            // many products again.
            float rest = p[r];
#pragma unroll
            for (int i = 0; i < P; i++) {
                const __bf16 part = (__bf16)rest;
                w.v[i][r / 8][r & 7] = part;
                rest -= (float)part;
            }
        }
        return w;
    }

    // m follows the maximum only once it is 8 powers of two behind: weights up to 256
    // cost nothing, and rows rarely rescale.
    __device__ __forceinline__ static bool moved(float top, float m, float c) { return (top - m) * c > 8.0f; }
    // Scores of N tiles to weights, with the row's maximum and sum.
    template <int N>
    __device__ __forceinline__ static void softmax(State<DV>& st, Weights (&w)[N], v16f (&s)[N], float c) {
        float top = s[0][0];
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[i][r]);
        const float2 both = halves(top);
        top = fmaxf(both.x, both.y);
        const float before = st.m;
        if (__ballot(moved(top, before, c))) {
            const bool mine = moved(top, before, c);  // each row for itself
            const float shrink = mine ? __builtin_amdgcn_exp2f((before - top) * c) : 1.0f;
            st.m = mine ? top : before;
            st.l *= shrink;
#pragma unroll
            for (int b = 0; b < DV / 32; b++) st.o[b] *= shrink;
        }
        // the difference first, then the scale: see cache_attention.hip
        const float base = st.m == -INFINITY ? 0.0f : st.m;
        float sum[4] = {st.l, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < N; i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[i][r] = __builtin_amdgcn_exp2f((s[i][r] - base) * c);
                sum[r & 3] += s[i][r];
            }
            w[i] = weights(s[i]);
        }
        st.l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }

    // Whether a tile holds no NaN (7 bits set).
    __device__ __forceinline__ static bool all_numbers(const uint8_t* v) {
        const uint8_t* at = v + 16 * late_lane();
        uint32_t any = 0;
#pragma unroll 1
        for (int i = 0; i < TV::kBytes / 1024; i++) {
            const v4u x = *reinterpret_cast<const v4u*>(at + 1024 * i);
#pragma unroll
            for (int e = 0; e < 4; e++) any |= (x[e] & 0x7F7F7F7Fu) + 0x01010101u;
        }
        return __ballot((any & 0x80808080u) != 0) == 0;
    }

    // The numbers among codes, zeros for the others; 1 (0x38) for each of these, else 0.
    __device__ __forceinline__ static v8bf without_nans(v2i& x) {
        uint32_t none[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t is = ((((uint32_t)x[e] & 0x7F7F7F7Fu) + 0x01010101u) >> 7) & 0x01010101u;
            x[e] = (int)((uint32_t)x[e] & ~(is * 255u));
            none[e] = is * 0x38u;
        }
        return widen(none[0], none[1], 1.0f);
    }
    // x, or NaN where the bit is set (bits all the way: a mask of lanes for each would fill the scalars)
    __device__ __forceinline__ static float nan_where(float x, uint32_t bits, int bit) {
        return __uint_as_float(__float_as_uint(x) | ((uint32_t)((int)(bits << (31 - bit)) >> 31) & 0x7FC00000u));
    }
    // A tile that holds NaNs and that some row does not see whole: a weight of 0 does not silence a
    // NaN.  They become zeros here, and the elements of rows that see one are told: bit 16 (b % 2) + r of bits[b / 2].
    __device__ __forceinline__ static void take_nans(uint32_t (&bits)[DV / 64], Values& v, int key, int limit) {
        const int h = (threadIdx.x & 63) >> 5;
        v8bf seen[2];
#pragma unroll
        for (int r = 0; r < 16; r++)
            seen[r / 8][r & 7] = (__bf16)(key + 8 * (r / 4) + 4 * h + r % 4 < limit ? 1.0f : 0.0f);
#pragma unroll
        for (int b = 0; b < DV / 32; b++) {
            v16f bad = {};
#pragma unroll
            for (int i = 0; i < 2; i++) bad = mma(without_nans(v.x[b][i]), seen[i], bad);
#pragma unroll
            for (int r = 0; r < 16; r++) bits[b / 2] |= bad[r] > 0.0f ? 1u << (16 * (b & 1) + r) : 0u;
            asm volatile("" : "+v"(bits[b / 2]));       // bits, not 64 masks of lanes
            __builtin_amdgcn_sched_barrier(0);  // rare: few registers
        }
    }

    // Two tiles that every row sees whole: chains of products side by side, one maximum.
    __device__ __forceinline__ static void pair(State<DV>& st, const Query& q, const uint8_t* k, const uint8_t* v,
                                                TileScales s0, TileScales s1, float c) {
        Keys k0, k1;
        read_keys(k0, k);
        read_keys(k1, k + TK::kBytes);
        Values v0, v1;
        read_values(v0, v);
        v16f s[2];
        scores(s, k0, k1, q, s0, s1);
        read_values(v1, v + TV::kBytes);
        Weights w[2];
        softmax<2>(st, w, s, c);
        add_values(st, v0, w[0], s0);
        add_values(st, v1, w[1], s1);
    }

    // A tile from its keys to its values.  edge: some row may not see all of the 32 keys from
    // `key` on; limit: keys that this lane's row sees; low: that the wave's rows see at least;
    // there: keys that exist (later ones are zeros in LDS).
    __device__ __forceinline__ static void tile(State<DV>& st, const Query& q, const uint8_t* k, const uint8_t* v,
                                                TileScales sc, bool edge, int key, int limit, int low, int there, float c) {
        v16f s[1] = {scores(k, q, sc)};
        if (edge) {
            const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (key + 8 * (r / 4) + 4 * h + r % 4 >= limit) s[0][r] = -INFINITY;
        }
        Weights w[1];
        softmax<1>(st, w, s, c);
        Values x;
        read_values(x, v);
        const bool nans = edge && low < there && !all_numbers(v);
        uint32_t bad[DV / 64] = {};
        if (nans) take_nans(bad, x, key, limit);
        add_values(st, x, w[0], sc);
        if (nans) {
#pragma unroll
            for (int b = 0; b < DV / 32; b++)
#pragma unroll
                for (int r = 0; r < 16; r++)
                    st.o[b][r] = nan_where(st.o[b][r], bad[b / 2], 16 * (b & 1) + r);
        }
    }
    __device__ __forceinline__ static float sum(float l) {
        const float2 both = halves(l);
        return both.x + both.y;
    }
    // Four elements at a time: give(row, element / 4, them)
    template <class Give>
    __device__ __forceinline__ static void each(const State<DV>& st, Give give) {
        const int lane = late_lane();
#pragma unroll
        for (int b = 0; b < DV / 32; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const v16f& o = st.o[b];
                give(lane & 31, 8 * b + 2 * i + (lane >> 5), make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
            }
    }
};

// The same for 16 rows or fewer, a step's tokens of a group, by 16x16 products: half the products
// and half the weights (128 sequences behind 32768 keys 133 -> 127 us, 64 behind 8192 37 -> 34).
// A score of register r of tile t (of 16 keys) is key 8 t + 4 (g / 2) + 16 (g % 2) + r, g = lane / 16,
// so that a lane's keys lie in one block and its values in 8 rows.
template <class Q, int DK, int DV>
struct Few8 {
    using X = Compute8<Q, DK, DV>;
    using TK = Tile8<DK>;
    using TV = Tile8<DV>;
    using v8k = typename X::v8k;
    static constexpr int P = X::P, PQ = X::PQ;
    // q of row lane & 15: element d of 64 c + 16 g + 8 s + 0..7 is v[part][2 c + s]
    struct Query {
        v8k v[PQ][DK / 32];
    };
    struct Rows {
        v4f o[DV / 16];  // register r of o[b]: element 16 b + 4 g + r
        float m, l;
    };
    struct Weights {
        v8bf v[P];
    };

    __device__ __forceinline__ static int group() { return (threadIdx.x & 63) >> 4; }
    __device__ static void load_query(Query& q, const Q* p, bool valid, int head_dim) {
#pragma unroll
        for (int s = 0; s < DK / 32; s++) {
            const int d = 64 * (s / 2) + 16 * group() + 8 * (s & 1);
            X::split(p + d, valid && d < head_dim, [&](int part, int e, auto x) { q.v[part][s][e] = x; });
        }
    }
    __device__ __forceinline__ static int key_of(int t, int g, int r) { return 8 * t + 4 * (g >> 1) + 16 * (g & 1) + r; }
    __device__ __forceinline__ static v4f mma(v8bf a, v8bf b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    __device__ __forceinline__ static v4f mma_key(v8k a, v8k b, v4f c) {
        if constexpr (X::kHalf) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
        else return mma(a, b, c);
    }
    // where this lane reads values: rows of its keys
    __device__ __forceinline__ static uint32_t values_from(const uint8_t* v) {
        const int n = threadIdx.x & 15, row = key_of(n >> 3, group(), (n >> 1) & 3);
        return (uint32_t)(uintptr_t)(lds_u8*)v + (uint32_t)(row * TV::kRow + TV::v_chunk(row, 0) * 16 + (n & 1) * 8);
    }
    __device__ __forceinline__ static v2i values_at(uint32_t from, int b) {
        return __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(uintptr_t)(from ^ (uint32_t)(16 * b)));
    }
    __device__ __forceinline__ static void scores(v4f (&s)[2], const uint8_t* k, const Query& q, TileScales sc) {
        const int m = threadIdx.x & 15;
        const float scale = m & 4 ? sc.k1 : sc.k0;
        v4u x[2][DK / 64];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int row = key_of(t, m >> 2, m & 3);
            const uint32_t from = (uint32_t)(uintptr_t)(lds_u8*)k + (uint32_t)(row * TK::kRow + TK::k_chunk(row, group()) * 16);
#pragma unroll
            for (int c = 0; c < DK / 64; c++) x[t][c] = *(lds_v4u*)(uintptr_t)(from ^ (uint32_t)(64 * c));
        }
        s[0] = s[1] = v4f{};
#pragma unroll
        for (int c = 0; c < DK / 64; c++)
#pragma unroll
            for (int half = 0; half < 2; half++)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const v8k a = X::widen_key(x[t][c][2 * half], x[t][c][2 * half + 1], scale);
#pragma unroll
                    for (int i = PQ - 1; i >= 0; i--) s[t] = mma_key(a, q.v[i][2 * c + half], s[t]);
                }
        if constexpr (X::kHalf) {
            const float mine = group() & 1 ? sc.k1 : sc.k0;
#pragma unroll
            for (int t = 0; t < 2; t++) s[t] *= mine;
        }
    }
    // x of the lane's row in the four groups
    template <class F>
    __device__ __forceinline__ static float of_groups(float x, F join) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        const float2 y = halves(join(__uint_as_float(r[0]), __uint_as_float(r[1])));
        return join(y.x, y.y);
    }
    __device__ __forceinline__ static float sum(float l) {
        return of_groups(l, [](float a, float b) { return a + b; });
    }
    __device__ __forceinline__ static void softmax(Rows& st, Weights& w, v4f (&s)[2], float c) {
        float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int r = 1; r < 4; r++) top = fmaxf(top, fmaxf(s[0][r], s[1][r]));
        top = of_groups(top, [](float a, float b) { return fmaxf(a, b); });
        const float before = st.m;
        if (__ballot(X::moved(top, before, c))) {
            const bool mine = X::moved(top, before, c);
            const float shrink = mine ? __builtin_amdgcn_exp2f((before - top) * c) : 1.0f;
            st.m = mine ? top : before;
            st.l *= shrink;
#pragma unroll
            for (int b = 0; b < DV / 16; b++) st.o[b] *= shrink;
        }
        const float base = st.m == -INFINITY ? 0.0f : st.m;
        float sum[2] = {st.l, 0.0f};
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float rest = __builtin_amdgcn_exp2f((s[t][r] - base) * c);
                sum[t] += rest;
#pragma unroll
                for (int i = 0; i < P; i++) {
                    const __bf16 part = (__bf16)rest;
                    w.v[i][4 * t + r] = part;
                    rest -= (float)part;
                }
            }
        st.l = sum[0] + sum[1];
    }
    __device__ __forceinline__ static float value_scale(TileScales sc) { return group() & 1 ? sc.v1 : sc.v0; }
    // bit 4 b + r, as above
    __device__ __forceinline__ static uint32_t take_nans(v2i (&x)[DV / 16], int key, int limit) {
        v8bf seen;
#pragma unroll
        for (int e = 0; e < 8; e++) seen[e] = (__bf16)(key + key_of(e / 4, group(), e % 4) < limit ? 1.0f : 0.0f);
        uint32_t bits = 0;
#pragma unroll
        for (int b = 0; b < DV / 16; b++) {
            const v4f bad = mma(X::without_nans(x[b]), seen, v4f{});
#pragma unroll
            for (int r = 0; r < 4; r++) bits |= bad[r] > 0.0f ? 1u << (4 * b + r) : 0u;
            asm volatile("" : "+v"(bits));
            __builtin_amdgcn_sched_barrier(0);  // rare: few registers
        }
        return bits;
    }
    __device__ __forceinline__ static void tile(Rows& st, const Query& q, const uint8_t* k, const uint8_t* v, TileScales sc,
                                                bool edge, int key, int limit, int low, int there, float c) {
        v4f s[2];
        scores(s, k, q, sc);
        if (edge) {
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (key + key_of(t, group(), r) >= limit) s[t][r] = -INFINITY;
        }
        Weights w;
        softmax(st, w, s, c);
        const uint32_t from = values_from(v);
        const float scale = value_scale(sc);
        v2i x[DV / 16];
#pragma unroll
        for (int b = 0; b < DV / 16; b++) x[b] = values_at(from, b);
        const bool nans = edge && low < there && !X::all_numbers(v);
        uint32_t bad = 0;
        if (nans) bad = take_nans(x, key, limit);
#pragma unroll
        for (int b = 0; b < DV / 16; b++) {
            const v8bf a = X::widen((uint32_t)x[b][0], (uint32_t)x[b][1], scale);
#pragma unroll
            for (int p = P - 1; p >= 0; p--) st.o[b] = mma(a, w.v[p], st.o[b]);
        }
        if (nans) {
#pragma unroll
            for (int b = 0; b < DV / 16; b++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    st.o[b][r] = X::nan_where(st.o[b][r], bad, 4 * b + r);
        }
    }
    // Four elements at a time: give(row, element / 4, them)
    template <class Give>
    __device__ __forceinline__ static void each(const Rows& st, Give give) {
        const int lane = late_lane();
#pragma unroll
        for (int b = 0; b < DV / 16; b++)
            give(lane & 15, 4 * b + (lane >> 4), make_float4(st.o[b][0], st.o[b][1], st.o[b][2], st.o[b][3]));
    }
};

// ------------------------------------------------ workgroups

constexpr int kWaves8 = 4;

template <class Q, int DK, int DV>
struct Config8 {
    static constexpr int kTile = Tile8<DK>::kBytes + Tile8<DV>::kBytes;  // 32 keys of K and V
    // two stages of a tile a wave, or four of two tiles shared; the merge of the waves' rows takes
    // 32 x DV x 4 bytes of each
    static constexpr int kLds = kWaves8 * 2 * kTile;
    static_assert(2 * kTile >= 128 * DV, "the merge");
    static constexpr int kPerCu = kLds <= 80 * 1024 && !(std::is_same_v<Q, float> && DK > 64) ? 2 : 1;
};

// R: rows of a tile that the waves share, 16 or 32.
template <class Q, int DK, int DV, int R>
__global__ __launch_bounds__((kWaves8 * 64), (Config8<Q, DK, DV>::kPerCu)) void kv8_attention_kernel(Job8 j) {
    using Cfg = Config8<Q, DK, DV>;
    using TK = Tile8<DK>;
    using TV = Tile8<DV>;
    using X = Compute8<Q, DK, DV>;
    using Y = std::conditional_t<R == 16, Few8<Q, DK, DV>, X>;  // of rows that the waves share
    constexpr int W = kWaves8, kParts = DK / DV;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float2 wave_ml[W][32];
    const Attention& a = j.a;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int hd = a.cache.head_dim, G = j.group, kv_heads = a.cache.kv_heads;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8*)lds;

    // Which part of the work.  Workgroups go to the 8 XCDs in turn; the row tiles of the same keys
    // follow each other on one, or on as many as share them.
    const int xcd = (int)(blockIdx.x & 7);
    const int64_t s = blockIdx.x >> 3;
    const bool prefix = s < j.prefix_per_xcd;
    const int64_t mine = prefix ? s : s - j.prefix_per_xcd;
    const int row_tiles = prefix ? j.prefix_rows : j.own_rows;
    const int splits = prefix ? j.prefix_splits : j.own_splits;
    const bool shared = prefix ? j.shared_prefix : j.shared_own;
    const int all_tiles = row_tiles * kParts;
    const int64_t units = (int64_t)kv_heads * splits * (prefix ? 1 : a.batch.batch), turns = units / 8;
    int unit, tile;  // KV head, then key range, then sequence; row tiles of the parts
    if (mine < turns * all_tiles) {
        unit = (int)(mine / all_tiles) * 8 + xcd;
        tile = (int)(mine % all_tiles);
    } else {
        const int last = (int)(units % 8), share = xcds_of(last);
        if (xcd >= last * share) return;
        unit = (int)turns * 8 + xcd % last;
        tile = (int)(mine - turns * all_tiles) * share + xcd / last;
        if (tile >= all_tiles) return;
    }
    const int part = tile / row_tiles;
    // a prompt's last rows, which see the most keys, first
    const int row_tile = prefix ? tile % row_tiles : row_tiles - 1 - tile % row_tiles;
    const int kv_head = unit % kv_heads;
    unit /= kv_heads;
    const int split = unit % splits, seq = unit / splits;

    // tokens, keys and the key range
    const int64_t all = min((int64_t)max(uniform(a.batch.q_start[a.batch.batch]), 0), a.tokens);
    int64_t t0 = 0, t1 = all;
    Runs runs;
    const int32_t* own_list = nullptr;
    int k0, k1, unseen = 0;  // row of token t sees keys below  t - t0 + 1 + unseen  (own keys)
    if (prefix) {
        runs.list = a.batch.prefix_pages;
        runs.keys = a.batch.prefix_len;
        k0 = split * j.prefix_chunk;
        k1 = min(runs.keys, k0 + j.prefix_chunk);
    } else {
        t0 = min(max((int64_t)uniform(a.batch.q_start[seq]), (int64_t)0), all);
        t1 = min(max((int64_t)uniform(a.batch.q_start[seq + 1]), t0), all);
        runs.list = own_list = a.batch.pages + (int64_t)seq * a.batch.max_pages;
        const int len = uniform(min(max(a.batch.len[seq], -(1 << 29)), 1 << 30));
        runs.keys = min(max(len, 0), a.batch.max_pages << j.page_shift);
        unseen = len - (int)(t1 - t0);
        const int chunk = own_chunk(runs.keys, splits, j.own_grain);
        k0 = (int)min((int64_t)split * chunk, (int64_t)runs.keys);
        k1 = min(runs.keys, k0 + chunk);
    }
    const int n_rows = (int)min((t1 - t0) * G, (int64_t)INT32_MAX);
    const int tile_rows = shared ? W * 32 : R;
    Loader8<DK, DV> from;
    from.init(j, kv_head, part);

    // own workgroups take every row_tiles-th tile of a sequence's rows
    for (int r0 = row_tile * tile_rows; r0 < n_rows; r0 += row_tiles * tile_rows) {
        const int rows = min(tile_rows, n_rows - r0);
        const int r = r0 + (shared ? wave * 32 + (lane & 31) : lane & (R - 1));
        const bool valid = r < n_rows;
        const int64_t token = t0 + r / G;
        const int head = kv_head * G + r % G;
        // keys that a row sees; rows that do not exist see all
        const int limit = !valid || prefix ? k1 : min(max(unseen + 1 + r / G, 0), k1);
        int low = limit, high = valid ? limit : 0;
#pragma unroll
        for (int x = 1; x < 32; x *= 2) low = min(low, __shfl_xor(low, x, 64)), high = max(high, __shfl_xor(high, x, 64));
        low = uniform(low);
        high = uniform(high);
        // the last row of the tile sees the most
        const int last_row = r0 + rows - 1;
        const int end = prefix ? k1 : min(max(unseen + 1 + last_row / G, 0), k1);
        const int first_limit = prefix ? k1 : min(max(unseen + 1 + r0 / G, 0), k1);  // the first row's, the least
        const int tiles = end > k0 ? (end - k0 + 31) / 32 : 0;  // of 32 keys
        const int whole = (first_limit - k0) / 32;              // tiles that every row sees whole
        const Q* q_row = static_cast<const Q*>(a.q.p) + token * a.q.token_stride + head * a.q.head_stride;
        const int out_split = prefix ? split : j.prefix_splits + split;
        auto clear = [&](auto& st) {
            st.m = -INFINITY;
            st.l = 0.0f;
            runs.down = 0;
            for (auto& o : st.o) o = std::remove_reference_t<decltype(o)>{};
        };
        auto hold = [&](auto& st, int key) {
            const bool lower = from.hold(runs, key);
            if (lower)
                for (auto& o : st.o) o *= kToDown;
            return lower;
        };
        // the query's loads are waited for before the loops, as those of hold()
        auto wait_for = [&](auto& q) {
            for (auto& part : q.v)
                for (auto& x : part) asm volatile("" : "+v"(x));
        };
        if (shared) {
            typename X::Query q;
            typename X::Rows st;
            X::load_query(q, q_row, valid, hd);
            clear(st);
            // the prefix's keys, where they are this workgroup's too (never beside 16 rows), then its own
            const bool inside = R == 32 && j.prefix_inside;
            for (int of_prefix = inside && !prefix && split == 0; of_prefix >= 0; of_prefix--) {
                const int begin = of_prefix ? 0 : k0, stop = of_prefix ? a.batch.prefix_len : end;
                const int tiles = stop > begin ? (stop - begin + 31) / 32 : 0;  // of 32 keys
                if (tiles == 0) continue;
                // tiles that every row sees whole; keys that this row, and the wave's rows at least and at most, see
                const int whole = ((of_prefix ? stop : first_limit) - begin) / 32, sees = of_prefix ? stop : limit;
                const int least = of_prefix ? stop : low, most = !of_prefix ? high : __ballot(valid) ? stop : 0;
                if (inside) runs.list = of_prefix ? a.batch.prefix_pages : own_list;
                runs.keys = stop;  // past the last row's sight nothing is read
                hold(st, begin);
                wait_for(q);
                // stages of two tiles (K, then V), S - 1 of them ahead; a wave loads 16 of the 64 keys
                constexpr int kStage = 2 * Cfg::kTile, S = Cfg::kLds / kStage;
                const int stages = (tiles + 1) / 2;
                int n = 0, at = 0;
                // Every step loads a stage, past the end too (zeros from nowhere), so that the count of
                // those in flight stays the same.
                auto load_stage = [&](int m, int to) {
                    const int key = begin + 64 * m;
                    const uint32_t stage = lds0 + (uint32_t)(to * kStage);
                    from.load16(runs, key + 16 * wave, stage + 16 * wave * TK::kRow,
                                stage + 2 * TK::kBytes + 16 * wave * TV::kRow);
                };
#pragma unroll
                for (int i = 0; i < S - 1; i++) load_stage(i, i);
                TileScales here0, here1;
                // the stage that n is, and a later one's loads
                auto next_stage = [&] {
                    wait_vmcnt<(S - 2) * from.kLoads>();
                    // all waves have read what the loads after this overwrite
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                    // (what is held begins at the tiles at hand, whose scales are read from it too; the first
                    // stages ahead are held from `begin` on)
                    const int ahead = n + S - 1;
                    if ((min(begin + 64 * ahead + 64, runs.keys) - 1) / 16 - runs.first >= 64) hold(st, begin + 64 * n);
                    load_stage(ahead, at == 0 ? S - 1 : at - 1);
                    here0 = from.scales(runs, begin + 64 * n), here1 = from.scales(runs, begin + 64 * n + 32);
                    const uint8_t* k = lds + at * kStage;
                    at = at + 1 == S ? 0 : at + 1;
                    return k;
                };
                if constexpr (X::kPairs) {
                    for (; 2 * n + 2 <= min(whole, tiles); n++) {
                        const uint8_t* k = next_stage();
                        X::pair(st, q, k, k + 2 * TK::kBytes, here0, here1, j.c);
                    }
                }
                for (; n < stages; n++) {
                    const uint8_t* k = next_stage();
#pragma unroll 1
                    for (int i = 0; i < 2; i++) {
                        const int key = begin + 64 * n + 32 * i;
                        const TileScales sc = i ? here1 : here0;
                        if (2 * n + i < tiles && key < most)
                            X::tile(st, q, k + i * TK::kBytes, k + 2 * TK::kBytes + i * TV::kBytes, sc, 2 * n + i >= whole, key,
                                    sees, least, runs.keys, j.c);
                    }
                }
                wait_vmcnt<0>();
                // the next keys' or row tile's loads overwrite what other waves may still read
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
            st.l = X::sum(st.l);
            if (runs.down) st.l = -st.l;
            const int first_row = r0 + wave * 32;
            X::each(st, [&](int late_row, int chunk, float4 o) {
                const int row = first_row + late_row, d = DV * part + 4 * chunk;
                if (row < n_rows && d < hd)
                    put_row<Q, 0, true>(j, out_split, t0 + row / G, kv_head * G + row % G, d, o, st.m, st.l);
            });
            continue;
        }
        // The waves share the rows: each takes every fourth tile.
        {
            typename Y::Query q;
            typename Y::Rows st;
            Y::load_query(q, q_row, valid, hd);
            clear(st);
            runs.keys = end;  // past the last row's sight nothing is read
            if (tiles > 0) hold(st, k0);
            wait_for(q);
            if (wave < tiles) {
                // a wave's two stages of a tile
                const uint8_t* mine8 = lds + wave * 2 * Cfg::kTile;
                const uint32_t to = lds0 + (uint32_t)wave * 2 * Cfg::kTile;
                auto load = [&](int n, int at) {
                    const int key = k0 + 32 * n;
                    const uint32_t stage = to + (uint32_t)(at * Cfg::kTile);
                    from.load16(runs, key, stage, stage + TK::kBytes);
                    from.load16(runs, key + 16, stage + 16 * TK::kRow, stage + TK::kBytes + 16 * TV::kRow);
                    return from.scales(runs, key);
                };
                TileScales here = load(wave, 0), next = load(wave + W, 1);
                int n = wave, at = 0;
                // Every step loads the tile two steps on, past the end too (zeros from nowhere), so
                // that the count of those in flight stays the same.
                for (; n < tiles; n += W, at ^= 1) {
                    const uint8_t* k = mine8 + at * Cfg::kTile;
                    wait_vmcnt<2 * from.kLoads>();
                    asm volatile("" ::: "memory");
                    Y::tile(st, q, k, k + TK::kBytes, here, n >= whole, k0 + 32 * n, limit, low, runs.keys, j.c);
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    here = next;
                    const int key = k0 + 32 * (n + 2 * W);  // (the first two tiles are held from k0 on)
                    if ((min(key + 32, runs.keys) - 1) / 16 - runs.first >= 64 && hold(st, key)) {
                        here.v0 = lower_scale(here.v0);
                        here.v1 = lower_scale(here.v1);
                    }
                    next = load(n + 2 * W, at);
                }
                wait_vmcnt<0>();
                asm volatile("" ::: "memory");
            }
            st.l = Y::sum(st.l);
            if (runs.down) st.l = -st.l;
            // each wave's part of the rows in its own part of LDS
            float* mine = reinterpret_cast<float*>(lds + wave * 2 * Cfg::kTile);
            asm volatile("" ::: "memory");
            Y::each(st, [&](int row, int chunk, float4 o) {
                *reinterpret_cast<float4*>(mine + row * DV + 4 * (chunk ^ (row & 15))) = o;
            });
            const int late = late_lane();
            if (late < R) wave_ml[wave][late] = make_float2(st.m, st.l);
        }
        __syncthreads();
        const int late = late_lane();
        for (int e = wave * 64 + late; e < rows * (DV / 4); e += W * 64) {
            const int rr = e / (DV / 4), c = e % (DV / 4), d = DV * part + 4 * c;
            if (d >= hd) continue;
            float m = -INFINITY;
            bool down = false;  // some wave's are held lower: the others' are brought to it
#pragma unroll
            for (int w = 0; w < W; w++) m = fmaxf(m, wave_ml[w][rr].x), down |= lowered<true>(wave_ml[w][rr].y);
            const float base = m == -INFINITY ? 0.0f : m;
            float l = 0.0f;
            float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float2 ml = wave_ml[w][rr];
                const float f = __builtin_amdgcn_exp2f((ml.x - base) * j.c);
                float4 x = *reinterpret_cast<const float4*>(
                    reinterpret_cast<const float*>(lds + w * 2 * Cfg::kTile) + rr * DV + 4 * (c ^ (rr & 15)));
                scale4(x, down && !lowered<true>(ml.y) ? kToDown : 1.0f);
                l = fmaf(fabsf(ml.y), f, l);
                o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
            }
            put_row<Q, 0, true>(j, out_split, t0 + (r0 + rr) / G, kv_head * G + (r0 + rr) % G, d, o, m, down ? -l : l);
        }
        __syncthreads();
    }
}

template <class Q, int DK, int DV>
hipError_t launch_of(const Job8& j, hipStream_t stream) {
    constexpr int kLds = Config8<Q, DK, DV>::kLds;
    const int64_t prefix_rows = j.prefix_splits ? j.a.tokens * j.group : 0;
    const int64_t own_rows = std::min<int64_t>(std::max(1, j.a.batch.max_q), j.a.tokens) * j.group;
    // 16 rows by the hint are two tiles, or more, where it is wrong
    const bool few = !j.shared_own && own_rows <= 16 && (j.shared_prefix || prefix_rows <= 16);
    auto launch = [&](void (*kernel)(Job8)) {
        if (hipError_t e = allow_dynamic_lds(reinterpret_cast<const void*>(kernel), kLds + 2048)) return e;
        hipLaunchKernelGGL(kernel, dim3(8u * (unsigned)(j.prefix_per_xcd + j.own_per_xcd)), dim3(kWaves8 * 64), kLds,
                           stream, j);
        return hipGetLastError();
    };
    if (hipError_t e = few ? launch(kv8_attention_kernel<Q, DK, DV, 16>) : launch(kv8_attention_kernel<Q, DK, DV, 32>)) return e;
    return launch_join<Q, DK, 0, true>(j, stream);
}

}  // namespace

size_t kv8_attention_workspace(const vtq_kv_cache& cache, const vtq_kv_batch& batch, int type, int64_t tokens,
                               int heads) {
    return parts_bytes(plan_kv8_attention(cache, batch, type, tokens, heads), tokens, heads, cache.head_dim);
}

hipError_t launch_kv8_attention(const Attention& a, const Scales& s, int type, hipStream_t stream) {
    Job8 j{};
    bool inside;
    static_cast<AttentionPlan&>(j) = plan_kv8_attention(a.cache, a.batch, type, a.tokens, a.heads, &inside);
    j.prefix_inside = inside;
    j.a = a;
    j.c = a.scale * kLog2E;
    j.s = s;
    j.block_shift = __builtin_ctz((unsigned)s.block);
    place_parts(j);
    return with_type(type, [&](auto q) {
        using Q = decltype(q);
        if (a.cache.head_dim <= 64) return launch_of<Q, 64, 64>(j, stream);
        if (a.cache.head_dim <= 128) return launch_of<Q, 128, 128>(j, stream);
        return launch_of<Q, 256, 128>(j, stream);
    });
}

}  // namespace vtq
