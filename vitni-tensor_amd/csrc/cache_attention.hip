// cache_attention.hip -- attention of a ragged batch over a prefix that all its
// sequences share and the pages of their own (gfx950).
//
//   y = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m),  m = max_j scale q.k_j
//
// One pass over the keys, with the running maximum and sum of each row in f32.
// The prefix is one matrix of keys for the rows of every sequence (tokens x the
// query heads of a KV head): workgroups take 32 rows a wave against tiles that the
// waves share.  A sequence's own keys meet few rows (the query heads of its one
// token): there the waves of a workgroup take different tiles against the same 32
// rows, and merge at the end.  Both kinds of workgroup are one launch, mixed, so
// that the prefix's matrix work runs beside the other's memory traffic.  Key ranges
// are split to fill the chip; a second launch joins the parts of a row by their
// maxima and sums.  The order of every sum goes by sizes alone.
//
// Per 32 keys and 32 rows, S^T = K Q^T and O^T += V^T P^T on 32x32 MFMAs.  Lane l
// then holds row l & 31 and keys 8i + 4(l >> 5) + e of a tile, a maximum or sum over
// keys stays within a lane and its partner, and the registers of P^T are the second
// product's operand as they are: the order of keys inside an MFMA is free, so V is
// read in the order that P has.  V's transpose comes from the LDS transposing read.
// f32 queries multiply in f32 (32x32x2 MFMAs; 16-bit keys and values widen exactly).
//
// bf16, 32 heads on 8 of 128: 64 sequences of up to 512 keys alone 22.8 us, 4.6 TB/s;
// behind a prefix of 8192 45 us; 128 of up to 1024 behind 32768 138 us, 510 TFLOP/s and
// 3.9 TB/s at once; that prefix alone 97-103 us, 670-690 TFLOP/s.  Own keys are bound by
// memory, prefix tiles by one wave's chain of products, exponentials and LDS reads
// (the matrix cores are busy 28 % of the time; keys from one hot page are 10 % faster).
// Prompts are far from this: one of 4096 tokens 201 us, 680 TFLOP/s; on 2 KV heads 555,
// where the row tiles of a KV head stay on one XCD and the others idle.  Heads of 256
// elements spill in the loops (26 sequences of 7 behind 8099, f16: 120 us, 165 TFLOP/s).
#include <type_traits>

#include "vtq_attention_rows.h"

namespace vtq {
namespace {

typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint16_t v8us __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// Weights, and what is summed with them, are 2^kUp times as large as they count.  In f16
// the 2^8 that a weight may be ahead of the maximum times 2^7 stay within 65504, and what
// is lost below the smallest step is 2^-32 of the largest weight instead of 2^-25 (500 keys
// of 2^-26 counted for nothing beside one of 1).  bf16 and f32 have exponents enough.
template <class Q>
constexpr int kUpOf = std::is_same_v<Q, _Float16> ? 7 : 0;
template <class Q>
constexpr float kUp = kUpOf<Q>;

template <class C, int D>
struct Tile {
    static constexpr int kRow = D * (int)sizeof(C);    // bytes of a key in LDS
    static constexpr int kChunks = kRow / 16;
    static constexpr int kLoadRows = 1024 / kRow;      // rows of one wave load
    static constexpr int kBytes = 32 * kRow;           // 32 keys
    static constexpr int kLoads = 32 / kLoadRows;
    // The 16-byte chunks of a row are permuted so that no read meets its neighbours
    // in the same bank: K is read 32 rows at one column, V (16 bits) 4 rows x 32
    // bytes, V (f32) two rows x 128 bytes.
    __device__ static int k_chunk(int row, int c) {
        return kChunks == 8 ? c ^ ((row ^ ((row >> 3) & 1)) & 7) : c ^ (row & 15);
    }
    __device__ static int v_chunk(int row, int c) {
        if (sizeof(C) == 4) return c ^ (((row >> 2) & 1) << 3);
        return kChunks == 8 ? c ^ ((row & 3) << 1) : c ^ ((row & 7) << 1);
    }
};

// Where keys come from: a page list with its length in keys.  The byte offsets of up to
// 64 pages are held a lane each (-1: outside the cache).
struct Pages {
    const int32_t* list;
    int keys;     // keys that exist: later ones read as zeros
    int shift;
    int first;    // page that lane 0 holds
    int low, high;
};

// Loads of a wave, 8 keys of K or V at a time: 8 keys lie in one page, so their address
// is worked out once, in scalar registers, and the lanes' offsets from it stay the same.
template <class C, int D>
struct Loader {
    using T = Tile<C, D>;
    static constexpr int kLoads8 = 8 / T::kLoadRows;  // loads of 8 keys
    const char *k, *v;                                 // of this KV head
    int64_t page_bytes;
    uint32_t slot_bytes, row_bytes;
    int n_pages, page_mask;
    uint32_t k_off[2][kLoads8], v_off[kLoads8];  // the permutations repeat after 16 (K) and 8 (V) rows

    __device__ __forceinline__ void init(const vtq_kv_cache& c, int head) {
        const int64_t at = (int64_t)head * (int64_t)c.head_stride * (int64_t)sizeof(C);
        k = static_cast<const char*>(c.k) + at;
        v = static_cast<const char*>(c.v) + at;
        page_bytes = (int64_t)c.page_stride * (int64_t)sizeof(C);
        slot_bytes = (uint32_t)(c.slot_stride * sizeof(C));
        row_bytes = (uint32_t)c.head_dim * (uint32_t)sizeof(C);
        n_pages = (int)c.n_pages;
        page_mask = c.page_size - 1;
        const int lane = threadIdx.x & 63, chunk = lane % T::kChunks;
#pragma unroll
        for (int i = 0; i < kLoads8; i++) {
            const int row = i * T::kLoadRows + lane / T::kChunks;
            // chunks past head_dim read past the end: zeros
            auto at_chunk = [&](int c) {
                return (uint32_t)c * 16 < row_bytes ? (uint32_t)row * slot_bytes + (uint32_t)c * 16 : 0x7FFFFFF0u;
            };
            k_off[0][i] = at_chunk(T::k_chunk(row, chunk));
            k_off[1][i] = at_chunk(T::k_chunk(8 + row, chunk));
            v_off[i] = at_chunk(T::v_chunk(row, chunk));
        }
    }
    // Holds the pages from `key`'s on.
    __device__ __forceinline__ void hold(Pages& p, int key) const {
        const int lane = threadIdx.x & 63, last = (p.keys - 1) >> p.shift;
        p.first = key >> p.shift;
        const int page = p.list[min(p.first + lane, last)];
        const int64_t at = (uint32_t)page < (uint32_t)n_pages ? (int64_t)page * page_bytes : -1;
        p.low = (int)(uint32_t)at;
        p.high = (int)(at >> 32);
        // waited for here: left to its use, the wait would stand in every tile, and be one for
        // all loads to LDS in flight as well
        asm volatile("" : "+v"(p.low), "+v"(p.high));
    }
    // Where 8 keys from `row` on are, and how many bytes of them exist.
    struct Run {
        int64_t at;
        int bytes;
    };
    __device__ __forceinline__ Run run(const Pages& p, int row) const {
        const int lane = ((row >> p.shift) - p.first) & 63;
        const uint32_t low = (uint32_t)__builtin_amdgcn_readlane(p.low, lane);
        const int high = __builtin_amdgcn_readlane(p.high, lane);
        Run r;
        r.at = (int64_t)(((uint64_t)(uint32_t)high << 32) | low) +
               (int64_t)(uint32_t)((uint32_t)(row & page_mask) * slot_bytes);  // a page's slots span less than 2^31
        const int rows = min(8, p.keys - row);
        r.bytes = (rows - 1) * (int)slot_bytes + (int)row_bytes;
        r.bytes = rows > 0 ? r.bytes : 0;
        r.bytes = high >= 0 ? r.bytes : 0;  // nothing is read at an address of no bytes
        return r;
    }
    // 8 keys of K or V into lds; odd: the second 8 of 16 rows.
    template <bool V>
    __device__ __forceinline__ void load8(const Run& r, bool odd, uint32_t lds) const {
        const __amdgpu_buffer_rsrc_t rs =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>((V ? v : k) + r.at), (short)0, r.bytes, kWord3);
#pragma unroll
        for (int i = 0; i < kLoads8; i++)
            load_to_lds<16>(rs, V ? v_off[i] : odd ? k_off[1][i] : k_off[0][i], lds + 1024u * i);
    }
};

// ------------------------------------------------ one tile of 32 keys

template <class Q, class C, int D>
struct Compute {
    using T = Tile<C, D>;
    static constexpr bool kWide = std::is_same_v<Q, float>;  // f32 products
    static constexpr bool kPairs = !kWide && D <= 128;        // two tiles at a time, where registers allow
    static constexpr int kStep = sizeof(C) == 4 ? 8 : 16;     // elements of a head that both half-waves read at once
    typedef Q v8q __attribute__((ext_vector_type(8)));
    typedef C v8c __attribute__((ext_vector_type(8)));
    typedef C v4c __attribute__((ext_vector_type(4)));
    // q of row lane & 31: per step, this half-wave's elements
    struct Query {
        std::conditional_t<kWide, float, v8q> v[kWide ? D / 2 : D / 16];
    };

    __device__ static void load_query(Query& q, const Q* p, bool valid, int head_dim) {
        const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int s = 0; s < D / kStep; s++) {
            const int d = s * kStep + h * (kStep / 2);
            const bool in = valid && d < head_dim;
            if constexpr (!kWide) {
                v8q z;
#pragma unroll
                for (int j = 0; j < 8; j++) z[j] = (Q)0.0f;
                q.v[s] = in ? *reinterpret_cast<const v8q*>(p + d) : z;
            } else {
#pragma unroll
                for (int j = 0; j < kStep / 2; j += 4) {
                    const float4 f = in ? *reinterpret_cast<const float4*>(p + d + j) : make_float4(0, 0, 0, 0);
                    q.v[s * (kStep / 2) + j] = f.x, q.v[s * (kStep / 2) + j + 1] = f.y;
                    q.v[s * (kStep / 2) + j + 2] = f.z, q.v[s * (kStep / 2) + j + 3] = f.w;
                }
            }
        }
    }

    __device__ static v16f mma(v8q a, v8q b, v16f c) {
        if constexpr (std::is_same_v<Q, __bf16>) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
        else if constexpr (std::is_same_v<Q, _Float16>) return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
        else return c;
    }

    // scores of 32 keys: register 4i + e is key 8i + 4h + e, row lane & 31
    __device__ static v16f scores(const uint8_t* k, const Query& q) {
        const int lane = threadIdx.x & 63, row = lane & 31, h = lane >> 5;
        v16f s = {};
#pragma unroll
        for (int i = 0; i < D / kStep; i++) {
            const uint8_t* at = k + row * T::kRow + T::k_chunk(row, 2 * i + h) * 16;
            if constexpr (!kWide) {
                s = mma(*reinterpret_cast<const v8q*>(at), q.v[i], s);
            } else if constexpr (sizeof(C) == 4) {
                const float4 f = *reinterpret_cast<const float4*>(at);
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(f.x, q.v[4 * i], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(f.y, q.v[4 * i + 1], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(f.z, q.v[4 * i + 2], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(f.w, q.v[4 * i + 3], s, 0, 0, 0);
            } else {
                const v8c f = *reinterpret_cast<const v8c*>(at);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    s = __builtin_amdgcn_mfma_f32_32x32x2f32((float)f[j], q.v[8 * i + j], s, 0, 0, 0);
            }
        }
        return s;
    }

    // elements 32 db + (lane & 31) of keys 8i + 4h + 0..3
    __device__ static v4c values4(const uint8_t* v, int db, int i) {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        if constexpr (sizeof(C) == 4) {
            v4c x;
            const int d = 32 * db + (lane & 31);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = 8 * i + 4 * h + e;
                x[e] = *reinterpret_cast<const float*>(v + row * T::kRow + T::v_chunk(row, d / 4) * 16 + (d & 3) * 4);
            }
            return x;
        } else {
            const int n = lane & 15, row = 8 * i + 4 * h + n / 4;
            const int c = 4 * db + 2 * ((lane >> 4) & 1) + ((n & 3) >> 1);
            const uint8_t* at = v + row * T::kRow + T::v_chunk(row, c) * 16 + (n & 1) * 8;
            return __builtin_bit_cast(v4c, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at)));
        }
    }

    // What the second product takes of a value: itself; itself where it is finite, else 0;
    // 1 where it is infinite with this sign or no number, else 0.
    enum Part { kAll, kFinite, kPlusInfinite, kMinusInfinite };
    template <Part P>
    __device__ static v4c part_of(v4c x) {
        if constexpr (P != kAll) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float f = (float)x[e];
                if constexpr (P == kFinite) x[e] = fabsf(f) < INFINITY ? x[e] : (C)0.0f;
                if constexpr (P == kPlusInfinite) x[e] = !(f < INFINITY) ? (C)1.0f : (C)0.0f;
                if constexpr (P == kMinusInfinite) x[e] = !(f > -INFINITY) ? (C)1.0f : (C)0.0f;
            }
        }
        return x;
    }

    struct Weights {
        std::conditional_t<kWide, v16f, v8q> v[kWide ? 1 : 2];
    };
    __device__ static Weights weights(v16f p) {
        Weights w;
        if constexpr (kWide) {
            w.v[0] = p;
        } else {
            // Rounded to the values' type, so that the second product runs at that type's rate
            // (f32's is a sixteenth): off by 2^-8 (bf16) or 2^-11 (f16) of each at most, in f16 or
            // by 2^-32 of the largest.  The sum is of the unrounded ones, in f32.
#pragma unroll
            for (int j = 0; j < 8; j++) w.v[0][j] = (Q)p[j], w.v[1][j] = (Q)p[8 + j];
        }
        return w;
    }

    // o + V^T P^T for elements 32 db .. of a head
    template <Part P>
    __device__ static v16f add_values(const uint8_t* v, const Weights& w, int db, v16f o) {
#pragma unroll
        for (int i = 0; i < 4; i += kWide ? 1 : 2) {
            const v4c a = part_of<P>(values4(v, db, i));
            if constexpr (kWide) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    o = __builtin_amdgcn_mfma_f32_32x32x2f32((float)a[e], w.v[0][4 * i + e], o, 0, 0, 0);
            } else {
                const v4c b = part_of<P>(values4(v, db, i + 1));
                v8q x;
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = a[e], x[4 + e] = b[e];
                o = mma(x, w.v[i / 2], o);
            }
        }
        return o;
    }

    // 16-bit operands of a tile, read ahead of their products
    struct Keys {
        v8q v[kWide ? 1 : D / 16];
    };
    struct Values {
        v8q v[kWide ? 1 : D / 32][2];
    };
    __device__ static void read_keys(Keys& x, const uint8_t* k) {
        const int lane = threadIdx.x & 63, row = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i = 0; i < D / 16; i++)
            x.v[i] = *reinterpret_cast<const v8q*>(k + row * T::kRow + T::k_chunk(row, 2 * i + h) * 16);
    }
    __device__ static void read_values(Values& x, const uint8_t* v) {
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const v4c lo = values4(v, b, 2 * i), hi = values4(v, b, 2 * i + 1);
#pragma unroll
                for (int e = 0; e < 4; e++) x.v[b][i][e] = lo[e], x.v[b][i][4 + e] = hi[e];
            }
    }
    // two tiles' scores, two chains of products that do not wait for each other
    __device__ static void scores(v16f (&s)[2], const Keys (&x)[2], const Query& q) {
        s[0] = s[1] = v16f{};
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            s[0] = mma(x[0].v[i], q.v[i], s[0]);
            s[1] = mma(x[1].v[i], q.v[i], s[1]);
        }
    }
    __device__ static void add_values(State<D>& st, const Values& x, const Weights& w) {
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int i = 0; i < 2; i++) st.o[b] = mma(x.v[b][i], w.v[i], st.o[b]);
    }

    // Scores of N tiles to weights, with the row's maximum and sum.
    template <int N>
    __device__ __forceinline__ static void softmax(State<D>& st, Weights (&w)[N], v16f (&s)[N], float c) {
        float top = s[0][0];
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) top = fmaxf(top, s[i][r]);
        const float2 both = halves(top);
        top = fmaxf(both.x, both.y);
        // m follows the maximum only once it is 8 powers of two behind: weights up to 256
        // cost nothing, and rows rarely rescale
        const bool moves = (top - st.m) * c > 8.0f;  // each row for itself
        if (__ballot(moves)) {
            const float shrink = moves ? __builtin_amdgcn_exp2f((st.m - top) * c) : 1.0f;
            st.m = moves ? top : st.m;
            st.l *= shrink;
#pragma unroll
            for (int b = 0; b < D / 32; b++) st.o[b] *= shrink;
        }
        // The difference first, then the scale, here and wherever sums meet: the product m c, rounded,
        // would be off by a power of two and more from scores of 2^24 on, and exp2 leave its range
        const float base = st.m == -INFINITY ? 0.0f : st.m;
        float sum[4] = {st.l, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < N; i++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[i][r] = __builtin_amdgcn_exp2f(fmaf(s[i][r] - base, c, kUp<Q>));
                sum[r & 3] += s[i][r];
            }
            w[i] = weights(s[i]);
        }
        st.l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }

    // Whether a tile holds no infinity and no NaN: the largest exponent of all.  (Without it
    // every tile on a causal edge took three products: a prompt of 52 tokens of 256 elements
    // 42 us, 28 with it.)
    __device__ __forceinline__ static bool all_finite(const uint8_t* v) {
        const uint8_t* at = v + 16 * late_lane();
        if constexpr (sizeof(C) == 4) {
            uint32_t top = 0;
#pragma unroll 1  // few registers: all sums are live
            for (int i = 0; i < T::kBytes / 1024; i++) {
                const v4u x = *reinterpret_cast<const v4u*>(at + 1024 * i);
#pragma unroll
                for (int e = 0; e < 4; e++) top = max(top, x[e] & 0x7FFFFFFFu);
            }
            return __ballot(top >= 0x7F800000u) == 0;
        } else {
            v8us top = {};
#pragma unroll 1  // few registers: all sums are live
            for (int i = 0; i < T::kBytes / 1024; i++)
                top = __builtin_elementwise_max(top, *reinterpret_cast<const v8us*>(at + 1024 * i) & (uint16_t)0x7FFF);
            uint16_t most = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) most = max(most, top[e]);
            return __ballot(most >= (std::is_same_v<C, __bf16> ? 0x7F80 : 0x7C00)) == 0;
        }
    }

    // The values of a tile that some row does not see whole.  low: the keys that the wave's
    // rows see at least; there: keys that exist (later ones are zeros in LDS).
    __device__ __forceinline__ static void add_edge(State<D>& st, const Weights& w, const uint8_t* v, int key, int limit,
                                                    int low, int there) {
        const int h = (threadIdx.x & 63) >> 5;
        if (low >= there) {
#pragma unroll
            for (int b = 0; b < D / 32; b++) st.o[b] = add_values<kAll>(v, w, b, st.o[b]);
            return;
        }
        // Some row sees less than what is there, and a weight of 0 does not silence a value
        // that is not finite: such values count as zeros here, and the rows that see one
        // get its infinity (or NaN, the sum of both) on top.
        v16f sees;
#pragma unroll
        for (int r = 0; r < 16; r++) sees[r] = key + 8 * (r / 4) + 4 * h + r % 4 < limit ? 1.0f : 0.0f;
        const Weights seen = weights(sees);
#pragma unroll
        for (int b = 0; b < D / 32; b++) {
            st.o[b] = add_values<kFinite>(v, w, b, st.o[b]);
            const v16f up = add_values<kPlusInfinite>(v, seen, b, v16f{});
#pragma unroll
            for (int r = 0; r < 16; r++) st.o[b][r] += up[r] > 0.0f ? INFINITY : 0.0f;
            const v16f down = add_values<kMinusInfinite>(v, seen, b, v16f{});
#pragma unroll
            for (int r = 0; r < 16; r++) st.o[b][r] -= down[r] > 0.0f ? INFINITY : 0.0f;
        }
    }

    // A tile from its keys to its values.  EDGE: some row may not see all of the 32 keys from
    // `key` on; limit: keys that this lane's row sees.
    template <bool EDGE, class Between>
    __device__ __forceinline__ static void tile(State<D>& st, const Query& q, const uint8_t* k, const uint8_t* v, int key,
                                                int limit, int low, int there, float c, Between between) {
        v16f s[1] = {scores(k, q)};
        between();  // K is read; V's loads may still be on their way
        if constexpr (EDGE) {
            if (low < there && all_finite(v)) low = there;
            const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (key + 8 * (r / 4) + 4 * h + r % 4 >= limit) s[0][r] = -INFINITY;
        }
        Weights w[1];
        softmax<1>(st, w, s, c);
        if constexpr (EDGE) {
            add_edge(st, w[0], v, key, limit, low, there);
        } else {
#pragma unroll
            for (int b = 0; b < D / 32; b++) st.o[b] = add_values<kAll>(v, w[0], b, st.o[b]);
        }
    }
};

// ------------------------------------------------ workgroups

template <class Q, class C, int D>
struct Config {
    static constexpr int kTile = Tile<C, D>::kBytes;         // 32 keys of K or V
    static constexpr int kWaves = kTile > 16384 ? 2 : 4;
    static constexpr int kLds = kWaves * 2 * kTile;           // a tile of K and V a wave, or two stages shared
    // workgroups of a CU: f32 queries of 128 elements and more take the registers of two
    static constexpr int kPerCu = kLds <= 80 * 1024 && !(std::is_same_v<Q, float> && D > 64) ? 2 : 1;
};

template <class Q, class C, int D>
__global__ __launch_bounds__((Config<Q, C, D>::kWaves * 64), (Config<Q, C, D>::kPerCu)) void attention_kernel(Job j) {
    using Cfg = Config<Q, C, D>;
    using T = Tile<C, D>;
    using X = Compute<Q, C, D>;
    constexpr int W = Cfg::kWaves;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float2 wave_ml[W][32];
    const Attention& a = j.a;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int hd = a.cache.head_dim, G = j.group, kv_heads = a.cache.kv_heads;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8*)lds;

    // Which part of the work.  Workgroups go to the 8 XCDs in turn: the row tiles of the
    // same keys follow each other on one XCD, where its L2 has the keys; prefix and own
    // workgroups are evenly mixed on each.
    const int xcd = (int)(blockIdx.x & 7);
    const int64_t s = blockIdx.x >> 3;
    const bool prefix = s < j.prefix_per_xcd;
    const int64_t mine = prefix ? s : s - j.prefix_per_xcd;
    const int row_tiles = prefix ? j.prefix_rows : j.own_rows;
    const int splits = prefix ? j.prefix_splits : j.own_splits;
    const bool shared = prefix ? j.shared_prefix : j.shared_own;
    const int row_tile = (int)(mine % row_tiles);
    int unit = (int)(mine / row_tiles) * 8 + xcd;  // KV head, then key range, then sequence
    const int kv_head = unit % kv_heads;
    unit /= kv_heads;
    const int split = unit % splits, seq = unit / splits;
    if (seq >= (prefix ? 1 : a.batch.batch)) return;

    // tokens, keys and the key range
    const int64_t all = min((int64_t)max(uniform(a.batch.q_start[a.batch.batch]), 0), a.tokens);
    int64_t t0 = 0, t1 = all;
    Pages pages;
    pages.shift = j.page_shift;
    int k0, k1, unseen = 0;  // row of token t sees keys below  t - t0 + 1 + unseen  (own keys)
    if (prefix) {
        pages.list = a.batch.prefix_pages;
        pages.keys = a.batch.prefix_len;
        k0 = split * j.prefix_chunk;
        k1 = min(pages.keys, k0 + j.prefix_chunk);
    } else {
        t0 = min(max((int64_t)uniform(a.batch.q_start[seq]), (int64_t)0), all);
        t1 = min(max((int64_t)uniform(a.batch.q_start[seq + 1]), t0), all);
        pages.list = a.batch.pages + (int64_t)seq * a.batch.max_pages;
        const int len = uniform(min(max(a.batch.len[seq], -(1 << 29)), 1 << 30));
        pages.keys = min(max(len, 0), a.batch.max_pages << j.page_shift);
        unseen = len - (int)(t1 - t0);
        const int chunk = own_chunk(pages.keys, splits, j.own_grain);
        k0 = (int)min((int64_t)split * chunk, (int64_t)pages.keys);
        k1 = min(pages.keys, k0 + chunk);
    }
    const int n_rows = (int)min((t1 - t0) * G, (int64_t)INT32_MAX);
    const int tile_rows = shared ? W * 32 : 32;
    Loader<C, D> from;
    from.init(a.cache, kv_head);

    // own workgroups take every row_tiles-th tile of a sequence's rows
    for (int r0 = row_tile * tile_rows; r0 < n_rows; r0 += row_tiles * tile_rows) {
        const int r = r0 + (shared ? wave * 32 : 0) + (lane & 31);
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
        const int last_row = min(n_rows, r0 + tile_rows) - 1;
        const int end = prefix ? k1 : min(max(unseen + 1 + last_row / G, 0), k1);
        const int first_limit = prefix ? k1 : min(max(unseen + 1 + r0 / G, 0), k1);  // the first row's, the least
        const int tiles = end > k0 ? (end - k0 + 31) / 32 : 0;  // of 32 keys
        typename X::Query q;
        X::load_query(q, static_cast<const Q*>(a.q.p) + token * a.q.token_stride + head * a.q.head_stride, valid, hd);
        State<D> st;
        st.m = -INFINITY;
        st.l = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; i++) st.o[i] = v16f{};
        if (tiles > 0) {
            const int whole = (first_limit - k0) / 32;  // tiles that every row sees whole
            pages.keys = end;  // past the last row's sight nothing is read
            from.hold(pages, k0);
            auto holds = [&](int key) {
                if (((min(key + 31, pages.keys - 1)) >> pages.shift) - pages.first >= 64) from.hold(pages, key);
            };
            if (shared) {
                // stages of a tile (K, then V); a wave loads 32 / W of the keys
                constexpr int S = Cfg::kLds / (2 * T::kBytes), kMine = 32 / W, kLoads = 2 * kMine / T::kLoadRows;
                auto load_stage = [&](int n, int at) {
                    const int key = k0 + 32 * n + kMine * wave;
                    holds(key);
#pragma unroll
                    for (int u = 0; u < kMine / 8; u++) {
                        const auto run = from.run(pages, key + 8 * u);
                        const uint32_t to = lds0 + (uint32_t)(at * 2 * T::kBytes + (kMine * wave + 8 * u) * T::kRow);
                        const bool odd = kMine == 8 ? wave & 1 : u & 1;
                        from.template load8<false>(run, odd, to);
                        from.template load8<true>(run, odd, to + T::kBytes);
                    }
                };
                int at = 0, n = 0;
                // all waves have read what the loads after this overwrite
                auto meet = [&] {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                };
                load_stage(0, 0);
                if constexpr (X::kPairs) {
                    // Two tiles a step while the next two load: chains of products side by side,
                    // one maximum, one meeting of the waves.
                    static_assert(S == 4, "two stages of two tiles");
                    load_stage(1, 1);
                    for (; n + 2 <= min(whole, tiles); n += 2, at ^= 2) {
                        wait_vmcnt<0>();
                        meet();
                        load_stage(n + 2, at ^ 2);
                        load_stage(n + 3, (at ^ 2) + 1);
                        const uint8_t* kt = lds + at * 2 * T::kBytes;
                        typename X::Keys keys[2];
                        X::read_keys(keys[0], kt);
                        X::read_keys(keys[1], kt + 2 * T::kBytes);
                        v16f s[2];
                        X::scores(s, keys, q);
                        typename X::Values values;
                        X::read_values(values, kt + T::kBytes);
                        typename X::Weights w[2];
                        X::template softmax<2>(st, w, s, j.c);
                        X::add_values(st, values, w[0]);
                        X::read_values(values, kt + 3 * T::kBytes);
                        X::add_values(st, values, w[1]);
                    }
                    meet();
                    load_stage(n + 2, at ^ 2);
                } else {
#pragma unroll
                    for (int i = 1; i < S - 1; i++) load_stage(i, i);
                }
                // One tile a step.  Every step loads the stage S - 1 on, past the end too (zeros
                // from nowhere), so that the count of those in flight stays the same.
                auto stage = [&](auto edge) {
                    wait_vmcnt<(S - 2) * kLoads>();
                    meet();
                    load_stage(n + S - 1, at == 0 ? S - 1 : at - 1);
                    const uint8_t* kt = lds + at * 2 * T::kBytes;
                    if (!decltype(edge)::value || k0 + 32 * n < high)
                        X::template tile<decltype(edge)::value>(st, q, kt, kt + T::kBytes, k0 + 32 * n, limit, low,
                                                                pages.keys, j.c, [] {});
                    at = at + 1 == S ? 0 : at + 1;
                };
                if constexpr (!X::kPairs)
                    for (; n < min(whole, tiles); n++) stage(std::false_type{});
                for (; n < tiles; n++) stage(std::true_type{});
                wait_vmcnt<0>();
                // the next row tile's loads overwrite what other waves may still read
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            } else {
                uint8_t* kt = lds + wave * 2 * T::kBytes;
                const uint32_t at = lds0 + (uint32_t)wave * 2 * T::kBytes;
                auto load_k = [&](int n) {
                    holds(k0 + 32 * n);
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        from.template load8<false>(from.run(pages, k0 + 32 * n + 8 * u), u & 1, at + 8 * u * T::kRow);
                };
                auto load_v = [&](int n) {
                    holds(k0 + 32 * n);
                    if constexpr (2 * T::kLoads > 63) wait_vmcnt<63 - T::kLoads>();  // the counter's range
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        from.template load8<true>(from.run(pages, k0 + 32 * n + 8 * u), u & 1,
                                                  at + T::kBytes + 8 * u * T::kRow);
                };
                if (wave < tiles) {
                    load_k(wave);
                    load_v(wave);
                }
                auto one = [&](int n, auto edge) {
                    const bool more = n + W < tiles;
                    wait_vmcnt<T::kLoads>();
                    asm volatile("" ::: "memory");
                    X::template tile<decltype(edge)::value>(st, q, kt, kt + T::kBytes, k0 + 32 * n, limit, low, pages.keys,
                                                            j.c, [&] {
                        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                        if (more) {
                            load_k(n + W);
                            wait_vmcnt<T::kLoads>();
                        } else {
                            wait_vmcnt<0>();
                        }
                        asm volatile("" ::: "memory");
                    });
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    if (more) load_v(n + W);
                };
                int n = wave;
                for (; n < min(whole, tiles); n += W) one(n, std::false_type{});
                for (; n < tiles; n += W) one(n, std::true_type{});
            }
        }
        const float2 sums = halves(st.l);
        st.l = sums.x + sums.y;
        const int out_split = prefix ? split : j.prefix_splits + split;
        const int late = late_lane(), late_h = late >> 5;
        if (shared) {
            const int row = r0 + wave * 32 + (late & 31);
            if (row < n_rows) {
#pragma unroll
                for (int db = 0; db < D / 32; db++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int d = 32 * db + 8 * i + 4 * late_h;
                        const v16f& o = st.o[db];
                        if (d < hd)
                            put_row<Q, kUpOf<Q>>(j, out_split, t0 + row / G, kv_head * G + row % G, d,
                                       make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]), st.m, st.l);
                    }
            }
        } else {
            // merge the waves' parts of the same rows, each in its own part of LDS
            float* mine = reinterpret_cast<float*>(lds + wave * 2 * T::kBytes);
            const int row = late & 31;
            asm volatile("" ::: "memory");
#pragma unroll
            for (int db = 0; db < D / 32; db++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int c = (8 * db + 2 * i + late_h) ^ (row & 15);
                    const v16f& o = st.o[db];
                    *reinterpret_cast<float4*>(mine + row * D + 4 * c) =
                        make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
            if (late_h == 0) wave_ml[wave][row] = make_float2(st.m, st.l);
            __syncthreads();
            const int rows = min(32, n_rows - r0);
            for (int e = wave * 64 + late; e < rows * (D / 4); e += W * 64) {
                const int rr = e / (D / 4), c = e % (D / 4);
                if (4 * c >= hd) continue;
                float m = -INFINITY;
#pragma unroll
                for (int w = 0; w < W; w++) m = fmaxf(m, wave_ml[w][rr].x);
                const float base = m == -INFINITY ? 0.0f : m;
                float l = 0.0f;
                float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const float2 ml = wave_ml[w][rr];
                    const float f = __builtin_amdgcn_exp2f((ml.x - base) * j.c);
                    const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(
                                                                          lds + w * 2 * T::kBytes) +
                                                                      rr * D + 4 * (c ^ (rr & 15)));
                    l = fmaf(ml.y, f, l);
                    o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
                }
                put_row<Q, kUpOf<Q>>(j, out_split, t0 + (r0 + rr) / G, kv_head * G + (r0 + rr) % G, 4 * c, o, m, l);
            }
            __syncthreads();
        }
    }
}

}  // namespace

size_t attention_workspace(const vtq_kv_cache& cache, const vtq_kv_batch& batch, int type, int64_t tokens, int heads) {
    return parts_bytes(plan_attention(cache, batch, type, tokens, heads), tokens, heads, cache.head_dim);
}

template <class Q, class C, int D>
hipError_t launch_attention_of(const Job& j, hipStream_t stream) {
    using Cfg = Config<Q, C, D>;
    const void* f = reinterpret_cast<const void*>(&attention_kernel<Q, C, D>);
    if (hipError_t e = allow_dynamic_lds(f, Cfg::kLds + 2048)) return e;
    hipLaunchKernelGGL((attention_kernel<Q, C, D>), dim3(8u * (unsigned)(j.prefix_per_xcd + j.own_per_xcd)),
                       dim3(Cfg::kWaves * 64), Cfg::kLds, stream, j);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_join<Q, D, kUpOf<Q>>(j, stream);
}

hipError_t launch_attention(const Attention& a, int type, hipStream_t stream) {
    Job j{};
    static_cast<AttentionPlan&>(j) = plan_attention(a.cache, a.batch, type, a.tokens, a.heads);
    j.a = a;
    j.c = a.scale * kLog2E;
    place_parts(j);
    return with_type(type, [&](auto q) {
        using Q = decltype(q);
        return with_type(a.cache.type, [&](auto c) {
            using C = decltype(c);
            if constexpr (!std::is_same_v<Q, C> && !std::is_same_v<Q, float>) {
                return hipErrorInvalidValue;
            } else {
                if (a.cache.head_dim <= 64) return launch_attention_of<Q, C, 64>(j, stream);
                if (a.cache.head_dim <= 128) return launch_attention_of<Q, C, 128>(j, stream);
                return launch_attention_of<Q, C, 256>(j, stream);
            }
        });
    });
}

}  // namespace vtq
