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
// and loses nothing (4 significant bits of 8).  Queries of 16 and 32 bits become sums of
// one (bf16), two (f16) or three (f32) bf16 parts, exactly, and weights as many, so that every type
// runs at the 16-bit products' rate.
//
// K: a lane reads 16 elements of its key at once, for two products; the order of a head's
// elements inside them is free as long as the query has the same.  V's transpose is the
// 8-bit transposing read: 16 lanes give 8 keys x 16 elements and get an element of all 8
// each, which are the keys that this half-wave's weights are of.
#include <type_traits>

#include "vtq_attention_rows.h"

namespace vtq {
namespace {

typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i lds_v2i;
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

struct Job8 : Job {
    Scales s;
    int block_shift;
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
        if (kChunks == 4) return c ^ ((row >> 2) & 2);
        return kChunks == 8 ? c ^ ((row & 2) | ((row >> 1) & 4)) : c ^ (((row & 3) | ((row >> 1) & 4)) << 1);
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
    int scale_k, scale_v;  // f32 bits
};

template <int D>
struct Loader8 {
    using T = Tile8<D>;
    const char *k, *v;  // of this KV head
    const uint8_t *k_scale, *v_scale;
    int64_t page_bytes, scale_page;
    uint32_t slot_bytes;
    int row_bytes, n_pages, page_shift, page_mask, block_shift;
    uint32_t k_off[T::kLoads], v_off[T::kLoads];

    __device__ __forceinline__ void init(const Job8& j, int head) {
        const vtq_kv_cache& c = j.a.cache;
        const int64_t at = (int64_t)head * (int64_t)c.head_stride;
        k = static_cast<const char*>(c.k) + at;
        v = static_cast<const char*>(c.v) + at;
        k_scale = j.s.k + head * j.s.head_stride;
        v_scale = j.s.v + head * j.s.head_stride;
        page_bytes = (int64_t)c.page_stride;
        scale_page = j.s.page_stride;
        slot_bytes = (uint32_t)c.slot_stride;
        row_bytes = c.head_dim;
        n_pages = (int)c.n_pages;
        page_shift = j.page_shift;
        page_mask = c.page_size - 1;
        block_shift = j.block_shift;
        const int lane = threadIdx.x & 63, chunk = lane % T::kChunks;
#pragma unroll
        for (int i = 0; i < T::kLoads; i++) {
            const int row = i * T::kLoadRows + lane / T::kChunks;
            // chunks past head_dim read past the end: zeros
            auto at_chunk = [&](int c) {
                return c * 16 < row_bytes ? (uint32_t)row * slot_bytes + (uint32_t)c * 16 : 0x7FFFFFF0u;
            };
            k_off[i] = at_chunk(T::k_chunk(row, chunk));
            v_off[i] = at_chunk(T::v_chunk(row, chunk));
        }
    }
    // Holds the runs from `key`'s on.
    __device__ __forceinline__ void hold(Runs& p, int key) const {
        const int lane = threadIdx.x & 63;
        p.first = key >> 4;
        const int at = min(p.first + lane, (p.keys - 1) >> 4) * 16;
        const int page = p.list[at >> page_shift], slot = at & page_mask;
        const bool there = (uint32_t)page < (uint32_t)n_pages;
        const int64_t byte = there ? (int64_t)page * page_bytes + (int64_t)((uint64_t)(uint32_t)slot * slot_bytes) : -1;
        p.low = (int)(uint32_t)byte;
        p.high = (int)(byte >> 32);
        const int64_t scale = there ? (int64_t)page * scale_page + (slot >> block_shift) : 0;
        p.scale_k = there ? min(max((int)k_scale[scale], 10), 246) << 23 : 0x3F800000;
        p.scale_v = there ? min(max((int)v_scale[scale], 10), 246) << 23 : 0x3F800000;
        // waited for here: left to its use, the wait would stand in every tile, and be one for
        // all loads to LDS in flight as well
        asm volatile("" : "+v"(p.low), "+v"(p.high), "+v"(p.scale_k), "+v"(p.scale_v));
    }
    // the lane of `key`'s 16 keys (those past the end have any)
    __device__ __forceinline__ int lane_of(const Runs& p, int key) const { return ((key >> 4) - p.first) & 63; }
    __device__ __forceinline__ TileScales scales(const Runs& p, int key) const {
        const int a = lane_of(p, key), b = lane_of(p, key + 16);
        TileScales s;
        s.k0 = __int_as_float(__builtin_amdgcn_readlane(p.scale_k, a));
        s.k1 = __int_as_float(__builtin_amdgcn_readlane(p.scale_k, b));
        s.v0 = __int_as_float(__builtin_amdgcn_readlane(p.scale_v, a));
        s.v1 = __int_as_float(__builtin_amdgcn_readlane(p.scale_v, b));
        return s;
    }
    // 16 keys from `key` on: K to lds, V to lds + v_at.
    __device__ __forceinline__ void load16(const Runs& p, int key, uint32_t lds, uint32_t v_at) const {
        const int lane = lane_of(p, key);
        const uint32_t low = (uint32_t)__builtin_amdgcn_readlane(p.low, lane);
        const int high = __builtin_amdgcn_readlane(p.high, lane);
        const int64_t at = (int64_t)(((uint64_t)(uint32_t)high << 32) | low);
        const int rows = min(16, p.keys - key);
        int bytes = (rows - 1) * (int)slot_bytes + row_bytes;
        bytes = rows > 0 ? bytes : 0;
        bytes = high >= 0 ? bytes : 0;  // nothing is read at an address of no bytes
        const __amdgpu_buffer_rsrc_t rk =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(k + at), (short)0, bytes, kWord3);
        const __amdgpu_buffer_rsrc_t rv =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(v + at), (short)0, bytes, kWord3);
#pragma unroll
        for (int i = 0; i < T::kLoads; i++) load_to_lds<16>(rk, k_off[i], lds + 1024u * i);
#pragma unroll
        for (int i = 0; i < T::kLoads; i++) load_to_lds<16>(rv, v_off[i], lds + v_at + 1024u * i);
    }
};

// ------------------------------------------------ one tile of 32 keys

template <class Q, int D>
struct Compute8 {
    using T = Tile8<D>;
    static constexpr int P = std::is_same_v<Q, float> ? 3 : std::is_same_v<Q, _Float16> ? 2 : 1;  // parts
    static constexpr bool kPairs = D <= 128;  // two tiles at a time, where registers allow
    // q of row lane & 31: element d of 32 c + 16 h + 8 s + 0..7 is v[part][2 c + s]
    struct Query {
        v8bf v[P][D / 16];
    };
    struct Weights {
        v8bf v[P][2];
    };

    // x as a sum of P bf16 numbers (exact for a query's type)
    __device__ __forceinline__ static void split(float x, __bf16 (&out)[P]) {
#pragma unroll
        for (int i = 0; i < P; i++) {
            out[i] = (__bf16)x;
            // an infinity's remainder would be no number: the first part has it all
            if (i + 1 < P) x = fabsf(x) < INFINITY ? x - (float)out[i] : 0.0f;
        }
    }

    __device__ static void load_query(Query& q, const Q* p, bool valid, int head_dim) {
        const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int s = 0; s < D / 16; s++) {
            const int d = 32 * (s / 2) + 16 * h + 8 * (s & 1);
            const bool in = valid && d < head_dim;
            typedef Q v8q __attribute__((ext_vector_type(8)));
            v8q x = {};
            if (in) x = *reinterpret_cast<const v8q*>(p + d);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if constexpr (P == 1) {
                    q.v[0][s][e] = x[e];
                } else {
                    __bf16 part[P];
                    split((float)x[e], part);
#pragma unroll
                    for (int i = 0; i < P; i++) q.v[i][s][e] = part[i];
                }
            }
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
    __device__ __forceinline__ static v16f mma(v8bf a, v8bf b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }

    // scores of 32 keys: register 4i + e is key 8i + 4h + e, row lane & 31
    __device__ static v16f scores(const uint8_t* k, const Query& q, TileScales sc) {
        const int lane = threadIdx.x & 63, row = lane & 31, h = lane >> 5;
        const float scale = row & 16 ? sc.k1 : sc.k0;
        v16f s = {};
#pragma unroll
        for (int c = 0; c < D / 32; c++) {
            const v4u x = *reinterpret_cast<const v4u*>(k + row * T::kRow + T::k_chunk(row, 2 * c + h) * 16);
            const v8bf a = widen(x[0], x[1], scale), b = widen(x[2], x[3], scale);
#pragma unroll
            for (int i = P - 1; i >= 0; i--) {  // small parts first
                s = mma(a, q.v[i][2 * c], s);
                s = mma(b, q.v[i][2 * c + 1], s);
            }
        }
        return s;
    }

    // elements 32 db + (lane & 31) of keys 16 i + 4 h + {0..3, 8..11}
    __device__ __forceinline__ static v8bf values(const uint8_t* v, int db, int i, TileScales sc) {
        const int lane = threadIdx.x & 63, h = lane >> 5, n = lane & 15, r = n >> 1;
        const int row = 16 * i + 4 * h + (r & 3) + 8 * (r >> 2), c = 2 * db + ((lane >> 4) & 1);
        const uint8_t* at = v + row * T::kRow + T::v_chunk(row, c) * 16 + (n & 1) * 8;
        const v2i x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)(at));
        return widen((uint32_t)x[0], (uint32_t)x[1], i ? sc.v1 : sc.v0);
    }

    __device__ __forceinline__ static Weights weights(const v16f& p) {
        Weights w;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            // As many parts as the query has: off by 2^-8 (bf16), 2^-16 (f16) or 2^-24 (f32) of each
            // at most.  The sum is of the unrounded ones, in f32.
            __bf16 part[P];
            split(p[r], part);
#pragma unroll
            for (int i = 0; i < P; i++) w.v[i][r / 8][r & 7] = part[i];
        }
        return w;
    }

    __device__ __forceinline__ static void add_values(State<D>& st, const uint8_t* v, const Weights& w,
                                                      TileScales sc) {
#pragma unroll
        for (int b = 0; b < D / 32; b++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const v8bf x = values(v, b, i, sc);
#pragma unroll
                for (int p = P - 1; p >= 0; p--) st.o[b] = mma(x, w.v[p][i], st.o[b]);
            }
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
        for (int i = 0; i < T::kBytes / 1024; i++) {
            const v4u x = *reinterpret_cast<const v4u*>(at + 1024 * i);
#pragma unroll
            for (int e = 0; e < 4; e++) any |= (x[e] & 0x7F7F7F7Fu) + 0x01010101u;
        }
        return __ballot((any & 0x80808080u) != 0) == 0;
    }

    // The values of a tile that some row does not see whole.  low: the keys that the wave's
    // rows see at least; there: keys that exist (later ones are zeros in LDS).
    __device__ __forceinline__ static void add_edge(State<D>& st, const Weights& w, const uint8_t* v, int key, int limit,
                                                    int low, int there, TileScales sc) {
        if (low >= there) {
            add_values(st, v, w, sc);
            return;
        }
        // Some row sees less than what is there, and a weight of 0 does not silence a NaN: NaNs
        // count as zeros here, and the rows that see one get it on top.
        const int h = (threadIdx.x & 63) >> 5;
        v8bf seen[2];
#pragma unroll
        for (int r = 0; r < 16; r++)
            seen[r / 8][r & 7] = (__bf16)(key + 8 * (r / 4) + 4 * h + r % 4 < limit ? 1.0f : 0.0f);
#pragma unroll
        for (int b = 0; b < D / 32; b++) {
            v16f bad = {};
#pragma unroll
            for (int i = 0; i < 2; i++) {
                v8bf x = values(v, b, i, sc), none;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const bool number = (float)x[e] == (float)x[e];
                    none[e] = number ? (__bf16)0.0f : (__bf16)1.0f;
                    x[e] = number ? x[e] : (__bf16)0.0f;
                }
#pragma unroll
                for (int p = P - 1; p >= 0; p--) st.o[b] = mma(x, w.v[p][i], st.o[b]);
                bad = mma(none, seen[i], bad);
            }
#pragma unroll
            for (int r = 0; r < 16; r++) st.o[b][r] += bad[r] > 0.0f ? __uint_as_float(0x7FC00000u) : 0.0f;
        }
    }

    // Two tiles that every row sees whole: chains of products side by side, one maximum.
    __device__ __forceinline__ static void pair(State<D>& st, const Query& q, const uint8_t* k, const uint8_t* v,
                                                TileScales s0, TileScales s1, float c) {
        v16f s[2] = {scores(k, q, s0), scores(k + T::kBytes, q, s1)};
        Weights w[2];
        softmax<2>(st, w, s, c);
        add_values(st, v, w[0], s0);
        add_values(st, v + T::kBytes, w[1], s1);
    }

    // A tile from its keys to its values.  EDGE: some row may not see all of the 32 keys from
    // `key` on; limit: keys that this lane's row sees.
    template <bool EDGE>
    __device__ __forceinline__ static void tile(State<D>& st, const Query& q, const uint8_t* k, const uint8_t* v,
                                                TileScales sc, int key, int limit, int low, int there, float c) {
        v16f s[1] = {scores(k, q, sc)};
        if constexpr (EDGE) {
            if (low < there && all_numbers(v)) low = there;
            const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
            for (int r = 0; r < 16; r++)
                if (key + 8 * (r / 4) + 4 * h + r % 4 >= limit) s[0][r] = -INFINITY;
        }
        Weights w[1];
        softmax<1>(st, w, s, c);
        if constexpr (EDGE) add_edge(st, w[0], v, key, limit, low, there, sc);
        else add_values(st, v, w[0], sc);
    }
};

// ------------------------------------------------ workgroups

constexpr int kWaves8 = 4;

template <class Q, int D>
struct Config8 {
    static constexpr int kTile = Tile8<D>::kBytes;
    // two stages: of a tile of K and V a wave, or of two tiles shared.  The merge of the waves' rows
    // takes 32 x D x 4 bytes of each.
    static constexpr int kLds = kWaves8 * 4 * kTile;
    static constexpr int kPerCu = kLds <= 80 * 1024 && !(std::is_same_v<Q, float> && D > 64) ? 2 : 1;
};

template <class Q, int D>
__global__ __launch_bounds__((kWaves8 * 64), (Config8<Q, D>::kPerCu)) void kv8_attention_kernel(Job8 j) {
    using T = Tile8<D>;
    using X = Compute8<Q, D>;
    constexpr int W = kWaves8;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ float2 wave_ml[W][32];
    const Attention& a = j.a;
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int hd = a.cache.head_dim, G = j.group, kv_heads = a.cache.kv_heads;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8*)lds;

    // Which part of the work: as in cache_attention.hip.  Workgroups go to the 8 XCDs in
    // turn; the row tiles of the same keys follow each other on one.
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
    Runs runs;
    int k0, k1, unseen = 0;  // row of token t sees keys below  t - t0 + 1 + unseen  (own keys)
    if (prefix) {
        runs.list = a.batch.prefix_pages;
        runs.keys = a.batch.prefix_len;
        k0 = split * j.prefix_chunk;
        k1 = min(runs.keys, k0 + j.prefix_chunk);
    } else {
        t0 = min(max((int64_t)uniform(a.batch.q_start[seq]), (int64_t)0), all);
        t1 = min(max((int64_t)uniform(a.batch.q_start[seq + 1]), t0), all);
        runs.list = a.batch.pages + (int64_t)seq * a.batch.max_pages;
        const int len = uniform(min(max(a.batch.len[seq], -(1 << 29)), 1 << 30));
        runs.keys = min(max(len, 0), a.batch.max_pages << j.page_shift);
        unseen = len - (int)(t1 - t0);
        const int chunk = own_chunk(runs.keys, splits, j.own_grain);
        k0 = (int)min((int64_t)split * chunk, (int64_t)runs.keys);
        k1 = min(runs.keys, k0 + chunk);
    }
    const int n_rows = (int)min((t1 - t0) * G, (int64_t)INT32_MAX);
    const int tile_rows = shared ? W * 32 : 32;
    Loader8<D> from;
    from.init(j, kv_head);

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
            runs.keys = end;  // past the last row's sight nothing is read
            from.hold(runs, k0);
            auto holds = [&](int key, int keys) {
                if ((min(key + keys, runs.keys) - 1) / 16 - runs.first >= 64) from.hold(runs, key);
            };
            if (shared) {
                // stages of two tiles (K, then V); a wave loads 16 of the 64 keys
                constexpr int kStage = 4 * T::kBytes;
                TileScales ahead0, ahead1;
                auto load_stage = [&](int n, int at) {
                    const int key = k0 + 64 * n;
                    holds(key, 64);
                    from.load16(runs, key + 16 * wave, lds0 + (uint32_t)(at * kStage + 16 * wave * T::kRow), 2 * T::kBytes);
                    ahead0 = from.scales(runs, key);
                    ahead1 = from.scales(runs, key + 32);
                };
                load_stage(0, 0);
                const int stages = (tiles + 1) / 2;
                int n = 0;
                TileScales here0, here1;
                // the stage that n is, and the next one's loads
                auto next_stage = [&] {
                    wait_vmcnt<0>();
                    // all waves have read what the loads after this overwrite
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                    here0 = ahead0, here1 = ahead1;
                    load_stage(n + 1, (n & 1) ^ 1);  // past the end: zeros from nowhere
                    return lds + (n & 1) * kStage;
                };
                if constexpr (X::kPairs) {
                    for (; 2 * n + 2 <= min(whole, tiles); n++) {
                        const uint8_t* k = next_stage();
                        X::pair(st, q, k, k + 2 * T::kBytes, here0, here1, j.c);
                    }
                }
                for (; n < stages; n++) {
                    const uint8_t* k = next_stage();
#pragma unroll 1
                    for (int i = 0; i < 2; i++, k += T::kBytes) {
                        const int key = k0 + 64 * n + 32 * i;
                        const TileScales sc = i ? here1 : here0;
                        if (!X::kPairs && 2 * n + i < whole)
                            X::template tile<false>(st, q, k, k + 2 * T::kBytes, sc, key, limit, low, runs.keys, j.c);
                        else if (2 * n + i < tiles && key < high)
                            X::template tile<true>(st, q, k, k + 2 * T::kBytes, sc, key, limit, low, runs.keys, j.c);
                    }
                }
                wait_vmcnt<0>();
                // the next row tile's loads overwrite what other waves may still read
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            } else {
                // a wave's two stages of a tile
                uint8_t* mine8 = lds + wave * 4 * T::kBytes;
                const uint32_t to = lds0 + (uint32_t)wave * 4 * T::kBytes;
                auto load = [&](int n, int at) {
                    const int key = k0 + 32 * n;
                    holds(key, 32);
                    from.load16(runs, key, to + at * 2 * T::kBytes, T::kBytes);
                    from.load16(runs, key + 16, to + at * 2 * T::kBytes + 16 * T::kRow, T::kBytes);
                    return from.scales(runs, key);
                };
                if (wave < tiles) {
                    TileScales here = load(wave, 0), next = load(wave + W, 1);
                    int n = wave, at = 0;
                    // Every step loads the tile two steps on, past the end too (zeros from nowhere), so
                    // that the count of those in flight stays the same.
                    auto one = [&](auto edge) {
                        const uint8_t* k = mine8 + at * 2 * T::kBytes;
                        wait_vmcnt<4 * T::kLoads>();
                        asm volatile("" ::: "memory");
                        X::template tile<decltype(edge)::value>(st, q, k, k + T::kBytes, here, k0 + 32 * n, limit, low,
                                                                runs.keys, j.c);
                        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                        here = next;
                        next = load(n + 2 * W, at);
                        n += W, at ^= 1;
                    };
                    while (n < min(whole, tiles)) one(std::false_type{});
                    while (n < tiles) one(std::true_type{});
                    wait_vmcnt<0>();
                    asm volatile("" ::: "memory");
                }
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
                            put_row<Q, 0>(j, out_split, t0 + row / G, kv_head * G + row % G, d,
                                          make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]), st.m, st.l);
                    }
            }
        } else {
            // merge the waves' parts of the same rows, each in its own part of LDS
            float* mine = reinterpret_cast<float*>(lds + wave * 4 * T::kBytes);
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
                    const float4 x = *reinterpret_cast<const float4*>(
                        reinterpret_cast<const float*>(lds + w * 4 * T::kBytes) + rr * D + 4 * (c ^ (rr & 15)));
                    l = fmaf(ml.y, f, l);
                    o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
                }
                put_row<Q, 0>(j, out_split, t0 + (r0 + rr) / G, kv_head * G + (r0 + rr) % G, 4 * c, o, m, l);
            }
            __syncthreads();
        }
    }
}

template <class Q, int D>
hipError_t launch_of(const Job8& j, hipStream_t stream) {
    constexpr int kLds = Config8<Q, D>::kLds;
    const void* f = reinterpret_cast<const void*>(&kv8_attention_kernel<Q, D>);
    if (hipError_t e = allow_dynamic_lds(f, kLds + 2048)) return e;
    hipLaunchKernelGGL((kv8_attention_kernel<Q, D>), dim3(8u * (unsigned)(j.prefix_per_xcd + j.own_per_xcd)),
                       dim3(kWaves8 * 64), kLds, stream, j);
    if (hipError_t e = hipGetLastError()) return e;
    return launch_join<Q, D, 0>(j, stream);
}

}  // namespace

size_t kv8_attention_workspace(const vtq_kv_cache& cache, const vtq_kv_batch& batch, int type, int64_t tokens,
                               int heads) {
    return parts_bytes(plan_kv8_attention(cache, batch, type, tokens, heads), tokens, heads, cache.head_dim);
}

hipError_t launch_kv8_attention(const Attention& a, const Scales& s, int type, hipStream_t stream) {
    Job8 j{};
    static_cast<AttentionPlan&>(j) = plan_kv8_attention(a.cache, a.batch, type, a.tokens, a.heads);
    j.a = a;
    j.c = a.scale * kLog2E;
    j.s = s;
    j.block_shift = __builtin_ctz((unsigned)s.block);
    place_parts(j);
    return with_type(type, [&](auto q) {
        using Q = decltype(q);
        if (a.cache.head_dim <= 64) return launch_of<Q, 64>(j, stream);
        if (a.cache.head_dim <= 128) return launch_of<Q, 128>(j, stream);
        return launch_of<Q, 256>(j, stream);
    });
}

}  // namespace vtq
