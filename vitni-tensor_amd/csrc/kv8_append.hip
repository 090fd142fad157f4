// kv8_append.hip -- appending rotated keys and plain values to a paged cache of 8-bit
// floats with a scale to each block of tokens and head (gfx950).
//
//   e = least exponent with max |x| <= 448 * 2^e over a block's new elements, and at
//   least that of the tokens before them;  stored: x / 2^e, rounded to e4m3.
//
// Scales are powers of two, so the quotient is exact but for the one rounding, and a
// block whose scale grows as it fills has its earlier elements shifted, not
// requantized: only what drops below e4m3's smallest normal value rounds again.  A scale
// of more bits would gain little: e4m3 is a float, its rounding relative to the element.
//
// A workgroup takes a block of a sequence and some of its heads, a wave a head's keys or
// values.  What the wave's lanes hold at once, four tokens of 128 elements, stays in
// registers between the maximum and the stores; longer blocks are read again, from the
// caches near by.  Queries are rotated by workgroups of their own in the same launch.
//
// A step of 32 sequences, 8 KV heads of 128 and 32 query heads in bf16, takes 6.5 us in a graph:
// the launch and three reads that wait for each other (lengths, page, scale; 8.3 where the row
// and the angles wait for the page too).  Prompts of 4,500 tokens in f32 (121 MB to read and
// write, 23.4 us at a large copy's rate) take 26.5; of 4000 in bf16 by blocks of 64 35 (17; 38
// with angles of 16 tokens at a time, worked out twice).
#include "vtq_rope.h"

namespace vtq {
namespace {

constexpr int kAngles = 4096;   // cosines and sines that are held at a time: 64 tokens of 128 rotated elements
constexpr int kMostRows = 32;   // heads' keys and values to a workgroup
constexpr int kQueryTokens = 4;  // tokens at most whose queries a workgroup rotates: one a wave
constexpr int kLeast = -117, kMost = 119;  // exponents of scales: what they scale stays a normal bf16

struct Kv8Job : RopeJob {
    Scales s;
    int64_t kv_work;           // workgroups of keys and values, the longer ones; then those of queries
    int q_tokens, q_groups, q_per;  // tokens to one; groups of heads, and their heads
    int kv_groups, rows_per;   // to a block, and their heads' keys and values
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

// A token's sequence, and its place among the sequence's own tokens.
struct Spot {
    int seq;
    int64_t place;
};

// The first token, of those that the call adds to it, of the index-th block that the batch's
// tokens lie in, and how many they are (0: there is no such block).  Every wave finds it for
// itself; tokens before place 0 have none.
__device__ __forceinline__ int block_tokens(const vtq_kv_batch& b, int64_t tokens, int block_shift, int64_t index,
                                            int64_t& token, Spot& spot) {
    const int lane = threadIdx.x & 63;
    for (int i0 = 0; i0 < b.batch; i0 += 64) {
        const int i = min(i0 + lane, b.batch - 1);
        const int64_t q0 = b.q_start[i], q1 = b.q_start[i + 1], len = b.len[i];
        const int64_t end = min(q1, tokens);  // of the tokens; the newest of all is the one before q1
        const int64_t from = max(len - (q1 - q0), (int64_t)0), to = len - (q1 - end);
        const bool some = i0 + lane < b.batch && q0 >= 0 && to > from && end > q0;
        const int64_t blocks = some ? ((to - 1) >> block_shift) - (from >> block_shift) + 1 : 0;
        int64_t up_to = blocks;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int64_t o = __shfl_up(up_to, d, 64);
            if (lane >= d) up_to += o;
        }
        const uint64_t past = __ballot(up_to > index);
        if (past) {
            const int at = __builtin_ctzll(past);
            const int64_t mine = index - (__shfl(up_to, at, 64) - __shfl(blocks, at, 64));
            const int64_t f = __shfl(from, at, 64), t = __shfl(to, at, 64), q = __shfl(q0, at, 64);
            const int64_t behind = __shfl(len - (q1 - q0), at, 64);  // place of the first token, maybe below 0
            const int64_t block0 = (f >> block_shift) + mine;
            spot.seq = i0 + at;
            spot.place = max(f, block0 << block_shift);
            token = q + (spot.place - behind);
            return (int)(min(t, (block0 + 1) << block_shift) - spot.place);
        }
        index -= __shfl(up_to, 63, 64);
    }
    return 0;
}

// A unit of a row of some tokens to each lane: its elements, rotated.  (Four units to a lane hold
// 16 tokens of 128 elements at once, and 173 registers: prompts of 4,500 tokens in f32 take 35 us
// against 26, which read longer blocks again.  Two take 31.)
template <class T, int N>
struct Held {
    float x[2][N];
    int at[2];  // first element of each part; -1: there is none
    int token;
    Pack<T, N> a, b;
    bool turns;
    int pair;

    // Unit w0 + lane of n tokens' `units` each: its loads
    __device__ __forceinline__ void fetch(const T* src, int64_t token_stride, int w0, int n, int units, int rot, bool half) {
        const int lane = threadIdx.x & 63, per = half || N == 1 ? rot / 2 / N : rot / N, step = half ? rot / 2 : 1;
        const int w = w0 + lane, last = min(w, n * units - 1), unit = last % units;
        token = last / units;
        turns = unit < per;
        const bool two = turns && (half || N == 1);
        // where the unit begins; a pair's elements stand side by side, or half the rotated part apart
        int first;
        if (turns) first = half ? unit * N : N == 1 ? 2 * unit : unit * N;
        else first = (half || N == 1 ? rot : per * N) + (unit - per) * N;
        pair = half || N == 1 ? unit * N : unit * N / 2;
        at[0] = w < n * units ? first : -1;
        at[1] = w < n * units && two ? first + step : -1;
        const T* from = src + token * token_stride + first;
        a = *reinterpret_cast<const Pack<T, N>*>(from);
        b = *reinterpret_cast<const Pack<T, N>*>(two ? from + step : from);
    }
    __device__ __forceinline__ void rotate(const float2* cs, int rot, bool half) {
        const float2* c = cs + token * (rot / 2) + (turns ? pair : 0);
        if (half || N == 1) {
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float2 w = c[e];
                const float p = (float)a.v[e], q = (float)b.v[e];
                x[0][e] = turns ? p * w.x - q * w.y : p;
                x[1][e] = turns ? p * w.y + q * w.x : p;
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const float2 w = c[e / 2];
                const float p = (float)a.v[e], q = (float)a.v[e + 1 < N ? e + 1 : e];
                x[0][e] = turns ? p * w.x - q * w.y : p;
                if (e + 1 < N) x[0][e + 1] = turns ? p * w.y + q * w.x : q;
            }
#pragma unroll
            for (int e = 0; e < N; e++) x[1][e] = x[0][e];
        }
    }
    __device__ __forceinline__ float top() const {
        float most = 0.0f;
#pragma unroll
        for (int p = 0; p < 2; p++)
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float v = fabsf(x[p][e]);
                most = fmaxf(most, v < INFINITY ? v : 0.0f);
            }
        return most;
    }
    __device__ __forceinline__ void put(uint8_t* dst, int64_t slot, int e) const {
#pragma unroll
        for (int p = 0; p < 2; p++)
            if (at[p] >= 0) put8<N>(dst + token * slot + at[p], x[p], e);
    }
};

// SHARE: a row that a wave does not hold is all waves', not one's.
template <class T, int N, bool SHARE>
__global__ __launch_bounds__(kRopeThreads) void kv8_append_kernel(Kv8Job j) {
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int rot = j.rotate ? j.rope.rot_dim : 0;
    const bool half = j.rope.layout == VTQ_ROPE_HALF;
    const int units_rot = rotated_units(j.head_dim, rot, half, N), units_plain = j.head_dim / N;
    __shared__ float2 cs[kAngles];
    const int at_once = rot ? min(kAngles / (rot / 2), 64) : 64;  // tokens
    constexpr int kTops = SHARE ? kRopeThreads / 64 : 1;
    __shared__ float tops[kMostRows][kTops];
    __shared__ int olds[kMostRows];
    // cosine and sine of a pair of the token at `place` (behind the prefix)
    auto turn_pair = [&](int64_t place, int pair) {
        const float2 w = turn_cos_sin((uint64_t)(j.batch.prefix_len + place) * j.rope.turns[pair]);
        return make_float2(w.x * j.rope.magnitude, w.y * j.rope.magnitude);
    };
    auto turn = [&](int64_t from, int n) {  // of n tokens from the place `from` on
        for (int i = threadIdx.x; i < n * (rot / 2); i += kRopeThreads) {
            const int token = i / (rot / 2), pair = i % (rot / 2);
            cs[i] = turn_pair(from + token, pair);
        }
    };
    if ((int64_t)blockIdx.x >= j.kv_work) {
        __shared__ int64_t places[kQueryTokens];
        __shared__ int there[kQueryTokens];
        const int64_t work = blockIdx.x - j.kv_work, t0 = work / j.q_groups * j.q_tokens;
        const int group = (int)(work % j.q_groups), n = (int)min((int64_t)j.q_tokens, j.tokens - t0);
        if (wave < n) {
            const int64_t t = t0 + wave;
            const int seq = sequence_of(j.batch, t);
            if (lane == 0) {
                there[wave] = seq < j.batch.batch;
                places[wave] = seq < j.batch.batch ? (int64_t)j.batch.len[seq] - (j.batch.q_start[seq + 1] - t) : 0;
            }
        }
        __syncthreads();
        if (rot)
            for (int i = threadIdx.x; i < n * (rot / 2); i += kRopeThreads)
                cs[i] = turn_pair(places[i / (rot / 2)], i % (rot / 2));
        __syncthreads();
        const int h0 = group * j.q_per, heads = min(j.x_heads, h0 + j.q_per) - h0;
        for (int w = threadIdx.x; w < n * heads * units_rot; w += kRopeThreads) {
            const int u = w % units_rot, h = h0 + w / units_rot % heads, i = w / units_rot / heads;
            if (!there[i]) continue;
            rotate_unit<T, T, N>(static_cast<const T*>(j.x.p) + (t0 + i) * j.x.token_stride + h * j.x.head_stride,
                                 static_cast<T*>(j.y) + (t0 + i) * j.y_token_stride + h * j.y_head_stride, cs + i * (rot / 2), u, rot, half);
        }
        return;
    }
    const int64_t work = blockIdx.x;
    int64_t t;
    Spot spot;
    const int block = j.s.block;
    const int count = block_tokens(j.batch, j.tokens, __builtin_ctz(block), work / j.kv_groups, t, spot);
    if (!count) return;
    const int group = (int)(work % j.kv_groups);
    const int r0 = group * j.rows_per, r1 = min(2 * j.kv_heads, r0 + j.rows_per);
    const bool keys = r0 < j.kv_heads && rot;
    if (spot.place / j.cache.page_size >= j.batch.max_pages) return;
    const int page = j.batch.pages[(int64_t)spot.seq * j.batch.max_pages + spot.place / j.cache.page_size];
    // One pass where a row of all tokens is held at once, else one for the maxima and one for the stores.
    const int most_units = max(units_rot, units_plain);
    const bool once = count <= at_once && count * most_units <= 64;
    Held<T, N> held;
    auto row_of = [&](int r, int c0) {  // from token c0 of the block on
        const HeadRows& in = r >= j.kv_heads ? j.v : j.k;
        return static_cast<const T*>(in.p) + (t + c0) * in.token_stride + (r % j.kv_heads) * in.head_stride;
    };
    auto fetch = [&](int r, int c0, int w0, int n) {
        const bool is_v = r >= j.kv_heads;
        held.fetch(row_of(r, c0), (is_v ? j.v : j.k).token_stride, w0, n, is_v ? units_plain : units_rot, is_v ? 0 : rot, half);
    };
    // the page, the first row and the angles on their way together
    if (once && r0 + wave < r1) fetch(r0 + wave, 0, 0, count);
    if (keys && once) turn(spot.place, count);
    if (page < 0 || page >= (int64_t)j.cache.n_pages) return;
    const int64_t at = page * (int64_t)j.cache.page_stride +
                       (spot.place & (j.cache.page_size - 1)) * (int64_t)j.cache.slot_stride;
    const int before = (int)(spot.place & (block - 1));
    const int64_t scale_at = page * j.s.page_stride + (spot.place & (j.cache.page_size - 1)) / block;
    const bool shared = SHARE && !once;
    const int first = shared ? wave * 64 : 0, step = shared ? kRopeThreads : 64;  // units
    for (int pass = once ? 1 : 0; pass < 2; pass++)
        for (int c0 = 0; c0 < count; c0 += at_once) {
            const int n = min(at_once, count - c0);
            if (keys && !once && (pass == 0 || count > at_once)) {
                if (pass || c0) __syncthreads();
                turn(spot.place + c0, n);
            }
            if (keys || (shared && pass)) __syncthreads();  // the angles, and the maxima of the first pass
            for (int r = r0 + (shared ? 0 : wave); r < r1; r += shared ? 1 : 4) {
                const bool is_v = r >= j.kv_heads;
                const int h = is_v ? r - j.kv_heads : r, units = is_v ? units_plain : units_rot;
                uint8_t* scale = (is_v ? j.s.v : j.s.k) + scale_at + h * j.s.head_stride;
                float top = 0.0f;
                int old;
                if (pass == 0 || once) {
                    old = before && c0 == 0 ? min(max((int)*scale - 127, kLeast), kMost) : kLeast;
                    for (int w0 = first; w0 < n * units; w0 += step) {
                        if (!once || r != r0 + wave) fetch(r, c0, w0, n);
                        held.rotate(cs, rot, half);
                        top = fmaxf(top, held.top());
                    }
#pragma unroll
                    for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x, 64));
                    if (!once) {
                        if (lane == 0) {
                            float& t = tops[r - r0][SHARE ? wave : 0];
                            t = c0 ? fmaxf(t, top) : top;
                            if (c0 == 0 && (!SHARE || wave == 0)) olds[r - r0] = old;
                        }
                        continue;
                    }
                } else {
#pragma unroll
                    for (int w = 0; w < kTops; w++) top = fmaxf(top, tops[r - r0][w]);
                    old = olds[r - r0];
                }
                const int e = max(exponent_for(top), old);
                const int slot = (int)j.cache.slot_stride;
                uint8_t* dst = static_cast<uint8_t*>(is_v ? j.cache.v : j.cache.k) + at + h * (int64_t)j.cache.head_stride;
                if (c0 == 0) {
                    const int words = j.head_dim / 4;
                    if (before && e > old)
                        for (int w = first + lane; w < before * words; w += step) {
                            uint32_t* x = reinterpret_cast<uint32_t*>(dst - (int64_t)(before - w / words) * slot) + w % words;
                            *x = shifted4(*x, old - e);
                        }
                    if (first + lane == 0) *scale = (uint8_t)(e + 127);
                }
                dst += (int64_t)c0 * slot;
                if (once) {
                    held.put(dst, slot, e);
                } else {
                    for (int w0 = first; w0 < n * units; w0 += step) {
                        fetch(r, c0, w0, n);
                        held.rotate(cs, rot, half);
                        held.put(dst, slot, e);
                    }
                }
            }
        }
}

}  // namespace

hipError_t launch_kv8_append(const RopeJob& job, const Scales& s, int type, hipStream_t stream) {
    Kv8Job j{};
    static_cast<RopeJob&>(j) = job;
    j.s = s;
    const int n = rope_access(j, type_bytes(type));
    // Queries: a workgroup takes up to four tokens of a long call, a token a wave to find and four
    // tokens' angles at once, and some heads of a short one, so that they keep the chip busy.  The
    // keys and values, which take longer, go first.  (Prompts of 4,500 tokens in f32, with four units
    // to a lane: a token each 49 us, four 42.5, the keys and values first 35.6.)
    const int64_t units = (int64_t)j.x_heads * (j.head_dim / n);
    j.q_tokens = (int)std::max<int64_t>(1, std::min<int64_t>(kQueryTokens, j.tokens / 1024));
    j.q_groups = (int)std::max<int64_t>(1, std::min<int64_t>({(units + kRopeThreads - 1) / kRopeThreads, 1024 / j.tokens,
                                                              (int64_t)j.x_heads}));
    j.q_per = (j.x_heads + j.q_groups - 1) / j.q_groups;
    j.q_groups = j.q_per ? (j.x_heads + j.q_per - 1) / j.q_per : 1;
    const int64_t q_work = j.x_heads ? (j.tokens + j.q_tokens - 1) / j.q_tokens * j.q_groups : 0;
    // Keys and values: a row a wave where blocks are few, up to 8 where cosines of a block's
    // tokens would be worked out by many workgroups.  Where that leaves most of the chip idle, and by
    // the hint a wave does not hold a row, a row is all waves' and up to all of a workgroup (11
    // prompts of up to 180, 4 KV heads of 128 by blocks of 64: 14 us against 26; where it does not, the
    // angles worked out again cost more: prompts of 4,500 tokens 41 against 26).
    const int64_t blocks = std::min<int64_t>(j.tokens, j.tokens / s.block + 2 * (int64_t)j.batch.batch);
    const int rows = 2 * j.kv_heads;
    const int most = j.batch.max_q > 0 ? std::min(j.batch.max_q, s.block) : s.block;
    const bool share = blocks * ((rows + 3) / 4) < 256 && (int64_t)most * (j.head_dim / n) > 256;
    const int64_t wanted = std::max<int64_t>((rows + kMostRows - 1) / kMostRows,
                                             share ? std::min<int64_t>(rows, 512 / blocks)
                                                   : std::min<int64_t>((rows + 3) / 4, 2048 / blocks));
    j.rows_per = (int)((rows + wanted - 1) / wanted);
    j.kv_groups = (rows + j.rows_per - 1) / j.rows_per;
    j.kv_work = blocks * j.kv_groups;
    const dim3 grid((unsigned)(j.kv_work + q_work));
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        auto launch = [&](auto n_of) {
            constexpr int N = decltype(n_of)::value;
            if (share) hipLaunchKernelGGL((kv8_append_kernel<T, N, true>), grid, dim3(kRopeThreads), 0, stream, j);
            else hipLaunchKernelGGL((kv8_append_kernel<T, N, false>), grid, dim3(kRopeThreads), 0, stream, j);
        };
        if (n == 8) launch(std::integral_constant<int, 8>{});
        if constexpr (sizeof(T) == 4)
            if (n == 4) launch(std::integral_constant<int, 4>{});
        if (n == 1) launch(std::integral_constant<int, 1>{});
        return hipGetLastError();
    });
}

}  // namespace vtq
