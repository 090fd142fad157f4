// beam_select.hip -- the best continuations of beams over their vocabulary (gfx950).
//
//   s(row, token) = score(row) + x(row, token) - ln sum_v exp x(row, v)
//
// and the n greatest s of a group of rows.  The logits are read once: a workgroup has
// up to 8192 of a row in its registers, sums their exponentials below their maximum, and
// leaves its n greatest.  A second launch, a workgroup a group, joins sums and lists.
//
// Which of two sums is greater decides about tokens, so s and a row's sum of exponentials
// are f64 (f32 would leave s wrong by 2^-20 of itself and more, and equal where it is
// not); f64 additions and products run at the f32 rate here.
//
// The n greatest of a workgroup: with T the n-th greatest of the 64 lanes' maxima of a
// wave, n elements at least reach T, so only those that do are looked at (a few times
// n): gathered in LDS and ranked by counting.  T's first 16 bits do.
//
// 512 rows of 128000 bf16 logits (116 MB, 22 us at a large copy's rate), 16 of each group of 8:
// 58 us, of which 24 are memory's, 27 exponentials' (10 f64 operations and an LDS read each) and
// 9 the lists'; 13 to join.  Twice the elements to a workgroup take 56 and 17; a workgroup that
// goes through parts with the next one's loads ahead, 100 (its registers).  Four rows of 32000 in
// f32: 5.9 and 5.1, two launches; 8 of 128000, 16 of each kept, whose lists the join does not hold: 7.2
// and 10.4, places of a list read one after the other.
#include <algorithm>
#include <type_traits>

#include "vtq_device.h"
#include "vtq_serve.h"

namespace vtq {
namespace {

constexpr int kThreads = 256;
constexpr int kGather = 192;     // candidates that a wave gathers to be ranked by counting
constexpr int kJoinGather = 1024;

struct Part {
    double sum;  // of exp(x - top); no number: the row holds +infinity or NaN
    float top;
};

struct BeamJob : BeamSelect {
    int splits;      // workgroups of a row
    uint2* lists;    // [rows][n_out][splits], falling: logit (f32 bits) and token; token -1: no more
    Part* parts;     // [rows][splits]
};

// Order of floats as that of unsigned numbers (both zeros alike).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ (uint32_t)((int32_t)b >> 31 | (int32_t)0x80000000);
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

// exp(y), y <= 0, to 2^-34 of itself; below -700, exp(-700).  Two to the nearest whole number of
// y log2 e, times the polynomial through e^z at the 8 Chebyshev points of |z| <= ln 2 / 2.
__device__ __forceinline__ double exp_of(double y) {
    const double round = 6755399441055744.0;  // 1.5 * 2^52: the sum's last bits are the nearest whole number
    y = fmax(y, -700.0);
    const double shifted = fma(y, 1.4426950408889634074, round);
    const double z = fma(shifted - round, -0.69314718055994530942, y);
    double p = 0.00019907569324043077;
    p = fma(p, z, 0.0013948578338415058);
    p = fma(p, z, 0.008333283538688762);
    p = fma(p, z, 0.041666218319112464);
    p = fma(p, z, 0.16666666786308657);
    p = fma(p, z, 0.500000010772923);
    p = fma(p, z, 0.999999999995509);
    p = fma(p, z, 0.9999999999595617);
    // times two to that number
    return __hiloint2double(__double2hiint(p) + (__double2loint(shifted) << 20), __double2loint(p));
}

// 2^(i / 64)
__device__ const double kPowers[64] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,
};
// sum + exp(y), y <= 0, exp to 2^-37 of itself; below -700, exp(-700).  Two to the nearest 64th of
// y log2 e, a whole number's from its bits and the rest's from the powers in LDS, times
// 1 + z + z^2 / 2 + z^3 / 6 for what is left, |z| <= h = ln 2 / 128, where z^4 / 24 has become its
// nearest parabola, h^2 z^2 / 24 - h^4 / 192.  10 f64 operations; 14 with a polynomial alone.
__device__ __forceinline__ double add_exp(double sum, double y, const double* powers) {
    const double round = 6755399441055744.0;
    y = fmax(y, -700.0);
    const double shifted = fma(y, 92.33248261689366, round);
    const double z = fma(shifted - round, -0.010830424696249145, y);
    const int n = __double2loint(shifted);
    const double power = powers[n & 63];
    double p = fma(1.0 / 6, z, 0.500001221855199);
    p = fma(p, z, 1.0);
    p = fma(p, z, 0.9999999999955212);
    return fma(__hiloint2double(__double2hiint(power) + ((n & ~63) << 14), __double2loint(power)), p, sum);
}

// The greater number; NaN if one is none.
__device__ __forceinline__ float greater(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d, 64);
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x = greater(x, __shfl_xor(x, d, 64));
    return x;
}

// Greatest T, of BITS bits and zeros, that n of the wave's K x 64 keys reach (0: fewer do).
template <int K, int BITS>
__device__ __forceinline__ uint32_t reached_by(const uint32_t (&key)[K], int n) {
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = 31; bit > 31 - BITS; bit--) {
        const uint32_t c = t | 1u << bit;
        int count = 0;
#pragma unroll
        for (int k = 0; k < K; k++) count += __popcll(__ballot(key[k] >= c));
        if (count >= n) t = c;
    }
    return t;
}

// ------------------------------------------------ lists of a row's parts

template <class T, int E>
__global__ __launch_bounds__(kThreads) void list_kernel(BeamJob j) {
    constexpr int V = 16 / sizeof(T), L = E / V;  // elements of a load, loads
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int row = blockIdx.y, split = blockIdx.x, n = j.n_out;
    if (j.done && j.done[row]) return;
    const T* x0 = static_cast<const T*>(j.logits) + row * j.ld;
    const int first = split * kThreads * E;
    // element l V + e of this thread is token first + (l 256 + tid) V + e
    // Rows start at any element.  (Loads from the next multiple of 16 bytes on would give a
    // row's sum another order for each start, and rows of the same logits another sum.)
    typedef T vec __attribute__((ext_vector_type(V)));
    typedef T vec_anywhere __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    vec raw[L];
#pragma unroll
    for (int l = 0; l < L; l++) {
        const int at = first + (l * kThreads + tid) * V;
        if (at + V <= j.vocab) {
            raw[l] = *reinterpret_cast<const vec_anywhere*>(x0 + at);
        } else {
            // past the row: below every number, so that only a comparison by token tells it from -infinity
#pragma unroll
            for (int e = 0; e < V; e++) raw[l][e] = at + e < j.vocab ? x0[at + e] : (T)-INFINITY;
        }
    }
    auto x = [&](int i) { return (float)raw[i / V][i % V]; };
    auto token_of = [&](int i) { return first + (i / V * kThreads + tid) * V + i % V; };
    auto in_row = [&](int token) { return token < j.vocab; };

    // maxima of 4 parts of this thread's elements
    float part[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        part[k] = x(k);
#pragma unroll
        for (int i = k + 4; i < E; i += 4) part[k] = greater(part[k], x(i));
    }
    float top = greater(greater(part[0], part[1]), greater(part[2], part[3]));  // NaN if a logit is
    uint32_t reach;
    if (n <= 16) {
        const uint32_t key[1] = {ordered(top)};
        reach = reached_by<1, 16>(key, n);
    } else {
        const uint32_t key[4] = {ordered(part[0]), ordered(part[1]), ordered(part[2]), ordered(part[3])};
        reach = reached_by<4, 16>(key, n);
    }
    top = wave_max(top);
    __shared__ float tops[4];
    __shared__ uint32_t reaches[4];
    __shared__ int counts[4];  // candidates that a wave gathered; more than kGather: too many
    __shared__ double sums[4];
    __shared__ __attribute__((aligned(16))) uint64_t keys[4][kGather];
    __shared__ double powers[64];
    if (lane == 0) tops[wave] = top, reaches[wave] = reach;
    if (tid < 64) powers[tid] = kPowers[tid];
    __syncthreads();
    top = greater(greater(tops[0], tops[1]), greater(tops[2], tops[3]));
    reach = max(max(reaches[0], reaches[1]), max(reaches[2], reaches[3]));
    const int64_t list = (int64_t)row * j.splits + split;
    if (!(top < INFINITY)) {
        // the row's candidates are all alike: its lists are not read
        if (tid == 0) j.parts[list] = Part{__longlong_as_double(0x7FF8000000000000ll), 0.0f};
        return;
    }
    const double base = top == -INFINITY ? 0.0 : (double)top;
    // T; no number, or -infinity, where fewer than n lanes hold any: then all that is finite
    const float limit = from_ordered(reach);
    const bool masks = !(limit > -INFINITY);
    const float least = masks ? -3.402823466e38f : limit;
    auto below = [&](uint64_t mask) {
        return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    };
    // a candidate as a number: greater logits, then lower tokens are greater
    auto key_of = [&](float v, int token) { return (uint64_t)ordered(v) << 32 | (uint32_t)~token; };
    double sum = 0.0;
    uint32_t reaching = 0;  // of this thread's elements, the first in bit E - 1
#pragma unroll
    for (int i = 0; i < E; i++) {
        const float v = x(i);
        sum = add_exp(sum, (double)v - base, powers);
        reaching = 2 * reaching + (v >= least ? 1 : 0);
        if (i % 4 == 3) asm volatile("" : "+v"(sum));  // more at once would not fit the registers
    }
    // What is rare reads the logits again, where they are near by, and keeps no registers: a lane has
    // one or two that reach T.
    auto again = [&](int token) { return token < j.vocab ? (float)x0[token] : -INFINITY; };
    int n_reach = 0;
    for (uint64_t turn = __ballot(reaching != 0); turn && n_reach <= kGather; turn = __ballot(reaching != 0)) {
        const int i = E - 32 + __builtin_clz(reaching | 1), token = token_of(i);
        const int to = n_reach + below(turn);
        if (reaching && to < kGather) keys[wave][to] = key_of(again(token), token);
        reaching &= ~(1u << (E - 1 - i));
        n_reach += __popcll(turn);
    }
    // Of masked tokens, of which there may be many, n will do that come first: n of the wave's
    // first n + n_reach tokens are masked.
    const int window = n + n_reach;
    if (masks && n_reach + window <= kGather) {
        for (int i0 = 0; i0 < window; i0 += 64) {
            const int i = i0 + lane, token = first + (i / (64 * V) * kThreads + wave * 64) * V + i % (64 * V);
            const bool takes = i < window && i < 64 * E && token < j.vocab && again(token) == -INFINITY;
            const uint64_t taking = __ballot(takes);
            if (takes) keys[wave][n_reach + below(taking)] = key_of(-INFINITY, token);
            n_reach += __popcll(taking);
        }
    } else if (masks) {
        n_reach = kGather + 1;
    }
    sum = wave_sum(sum);
    if (lane == 0) {
        counts[wave] = min(n_reach, kGather + 1);
        sums[wave] = sum;
    }
    __syncthreads();
    const int at1 = counts[0], at2 = at1 + counts[1], at3 = at2 + counts[2], c = at3 + counts[3];
    const bool fits = max(max(counts[0], counts[1]), max(counts[2], counts[3])) <= kGather;
    // (-infinities alone add up to nothing)
    if (tid == 0) j.parts[list] = Part{top > -INFINITY ? (sums[0] + sums[1]) + (sums[2] + sums[3]) : 0.0, top};
    uint2* out = j.lists + (int64_t)row * n * j.splits + split;
    auto put = [&](int at, float v, int token) {
        out[at * j.splits] = make_uint2(__float_as_uint(v), (uint32_t)token);
    };
    if (fits) {
        for (int i = tid; i < c; i += kThreads) {
            const int w0 = (i >= at1) + (i >= at2) + (i >= at3);
            const uint64_t mine = keys[w0][i - (w0 > 2 ? at3 : w0 > 1 ? at2 : w0 > 0 ? at1 : 0)];
            int above = 0;
            for (int w = 0; w < 4; w++) {
                const int m = counts[w];
                int k = 0;
                // LDS's latency is what this costs: 8 numbers at a time
                for (; k + 8 <= m; k += 8) {
                    uint64_t other[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) other[e] = keys[w][k + e];
#pragma unroll
                    for (int e = 0; e < 8; e++) above += other[e] > mine;
                }
                for (; k < m; k++) above += keys[w][k] > mine;
            }
            if (above < n) put(above, from_ordered((uint32_t)(mine >> 32)), ~(int)(uint32_t)mine);
        }
        for (int i = c + tid; i < n; i += kThreads) put(i, -INFINITY, -1);
        return;
    }
    // Many alike: the greatest, n times.
    float last_x = INFINITY;
    int last_at = -1;
    __shared__ float round_x[2][4];
    __shared__ int round_at[2][4];
    for (int k = 0; k < n; k++) {
        float best = -INFINITY;
        int best_at = INT32_MAX;
#pragma unroll 1
        for (int i = 0; i < E; i++) {
            const int token = token_of(i);
            const float v = again(token);
            const bool after = v < last_x || (v == last_x && token > last_at);
            if (in_row(token) && after && (v > best || (v == best && token < best_at))) best = v, best_at = token;
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const float ox = __shfl_xor(best, d, 64);
            const int oa = __shfl_xor(best_at, d, 64);
            if (ox > best || (ox == best && oa < best_at)) best = ox, best_at = oa;
        }
        if (lane == 0) round_x[k & 1][wave] = best, round_at[k & 1][wave] = best_at;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float ox = round_x[k & 1][w];
            const int oa = round_at[k & 1][w];
            if (w == 0 || ox > best || (ox == best && oa < best_at)) best = ox, best_at = oa;
        }
        last_x = best, last_at = best_at;
        if (tid == 0) put(k, best, best_at == INT32_MAX ? -1 : best_at);
    }
}

// ------------------------------------------------ the join

// A candidate's place in the order: greater sums, of equal ones greater logits, of these
// lower numbers (row and token).
struct Candidate {
    double s;
    float x;
    int row, token;  // row in the group
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
    if (a.s != b.s) return a.s > b.s;
    if (a.x != b.x) return a.x > b.x;
    return a.row != b.row ? a.row < b.row : a.token < b.token;
}

// The number that e^y is, to 2^-33 of it: one step of Newton's from f32's.
__device__ __forceinline__ double log_of(double x) {
    const double y = (double)(__builtin_amdgcn_logf((float)x) * 0.69314718055994530942f);
    return y + (x * exp_of(-y) - 1.0);
}

// HELD entries of a list to a thread, in registers: a power of two of threads, 2^list_bits,
// have the lists side by side, and the next as many their next places.  HELD 0: any number of
// lists, read as far as they matter.  (A group is one workgroup, which goes through its code
// once: what it waits for is memory, and the code is part of that.)
template <int HELD, int THREADS>
__global__ __launch_bounds__(THREADS) void join_kernel(BeamJob j, int list_bits) {
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int n = j.n_out, beams = j.beams, splits = j.splits, lists = beams * splits;
    const int64_t row0 = (int64_t)blockIdx.x * beams;
    const uint2* entries = j.lists + row0 * splits * n;
    constexpr int W = THREADS / 64;
    __shared__ double norm[64];  // ln of a row's sum
    __shared__ float score[64];
    __shared__ int kind[64];     // 0 lists, 1 one candidate, 2 all alike
    __shared__ uint32_t reaches[W];
    __shared__ int count;
    __shared__ __attribute__((aligned(16))) double got_s[kJoinGather];
    __shared__ float got_x[kJoinGather];
    __shared__ int got_at[kJoinGather], got_row[kJoinGather];
    // heads first: many lanes have a great one, and few entries reach what n lanes do
    const int own_list = tid & ((1 << list_bits) - 1), own_row = min(own_list, lists - 1) / splits;
    const int own_split = min(own_list, lists - 1) - own_row * splits;
    uint2 held[HELD ? HELD : 1];
    auto place_of = [&](int i) { return (tid >> list_bits) + i * (THREADS >> list_bits); };
#pragma unroll
    for (int i = 0; i < HELD; i++) held[i] = entries[(own_row * n + min(place_of(i), n - 1)) * splits + own_split];
    if (tid == 0) count = 0;
    // `width` lanes to a row
    int width_bits = 0;
    while (width_bits < 6 && 1 << width_bits < splits) width_bits++;
    const int width = 1 << width_bits;
    for (int r0 = 0; r0 < beams; r0 += THREADS >> width_bits) {
        const int r = r0 + (tid >> width_bits), s0 = tid & (width - 1);
        const bool there = r < beams;
        // all loads at once (of an ended row's parts too, which nobody wrote)
        const int64_t row = row0 + (there ? r : 0);
        const Part* parts = j.parts + row * splits;
        const Part own = parts[min(s0, splits - 1)];
        const bool ended = j.done && j.done[row];
        const float cum = j.score[row];
        float top = s0 < splits ? own.top : -INFINITY;
        for (int s = s0 + width; s < splits; s += width) top = greater(top, parts[s].top);
        for (int d = 1; d < width; d *= 2) top = greater(top, __shfl_xor(top, d, 64));
        double sum = 0.0;
        for (int s = s0; s < splits; s += width) {
            const Part p = s == s0 ? own : parts[s];
            sum += p.sum == p.sum ? p.sum * exp_of((double)p.top - (double)top) : p.sum;
        }
        for (int d = 1; d < width; d *= 2) sum += __shfl_xor(sum, d, 64);
        if (there && s0 == 0) {
            // a row of -infinities alone, or of no numbers, has no logarithm
            const double ln = sum > 0.0 ? (double)top + log_of(sum) : __longlong_as_double(0x7FF8000000000000ll);
            norm[r] = ln;
            score[r] = cum;
            kind[r] = ended ? 1 : ln == ln && fabsf(cum) < INFINITY ? 0 : 2;
        }
    }
    __syncthreads();
    // entry `pos` of a row's list of `split`; false: there is none
    auto candidate = [&](int row, int split, int pos, uint2 entry, Candidate& c) {
        const int what = kind[row];
        const float cum = score[row];
        c.row = row;
        c.token = what == 0 ? (int)entry.y : what == 1 ? j.end_token : pos;
        const bool is = what == 0 ? c.token >= 0 : split == 0 && (what == 1 ? pos == 0 : pos < j.vocab);
        const bool counts = what == 0 || (what == 1 && fabsf(cum) < INFINITY);
        c.x = what == 0 ? __uint_as_float(entry.x) : counts ? 0.0f : -INFINITY;
        c.s = counts ? (double)cum + (what == 0 ? (double)c.x - norm[row] : 0.0) : -INFINITY;
        return is;
    };
    auto load = [&](int l, int pos, Candidate& c) {
        const int r = l / splits, split = l - r * splits;
        return candidate(r, split, pos, entries[(r * n + pos) * splits + split], c);
    };
    auto gather = [&](const Candidate& c) {
        const int at = atomicAdd(&count, 1);
        if (at < kJoinGather) got_s[at] = c.s, got_x[at] = c.x, got_row[at] = c.row, got_at[at] = c.token;
    };
    // a thread's greatest, and what n threads of a wave reach
    uint32_t key[1] = {0};
    Candidate mine[HELD ? HELD : 1];
    uint32_t keys[HELD ? HELD : 1];
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const bool is = own_list < lists && place_of(i) < n && candidate(own_row, own_split, place_of(i), held[i], mine[i]);
            keys[i] = is ? ordered((float)mine[i].s) : 0;
            key[0] = max(key[0], keys[i]);
        }
    } else {
        for (int l = tid; l < max(lists, THREADS); l += THREADS) {
            Candidate c;
            if (l / lists < n && load(l % lists, l / lists, c)) key[0] = max(key[0], ordered((float)c.s));
        }
    }
    const uint32_t reached = reached_by<1, 24>(key, n);
    if (lane == 0) reaches[wave] = reached;
    __syncthreads();
    uint32_t reach = 1;
#pragma unroll
    for (int w = 0; w < W; w++) reach = max(reach, reaches[w]);
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++)
            if (keys[i] >= reach) gather(mine[i]);
    } else {
        for (int l = tid; l < lists; l += THREADS) {
            Candidate c;
            for (int pos = 0; pos < n && load(l, pos, c) && ordered((float)c.s) >= reach; pos++) gather(c);
        }
    }
    __syncthreads();
    auto put = [&](int at, const Candidate& c) {
        const int64_t o = (int64_t)blockIdx.x * n + at;
        j.out_score[o] = (float)c.s;
        j.out_token[o] = c.token;
        j.out_parent[o] = (int32_t)(row0 + c.row);
        if (j.out_done) j.out_done[o] = kind[c.row] == 1 || (j.end_token >= 0 && c.token == j.end_token);
    };
    auto put_none = [&](int at) {
        const int64_t o = (int64_t)blockIdx.x * n + at;
        j.out_score[o] = -INFINITY;
        j.out_token[o] = j.out_parent[o] = -1;
        if (j.out_done) j.out_done[o] = 1;
    };
    if (count <= kJoinGather) {
        const int c = count;
        for (int i = tid; i < c; i += THREADS) {
            const Candidate a{got_s[i], got_x[i], got_row[i], got_at[i]};
            // by the sums, 4 at a time; where some are equal, by the rest too
            int above = 0, equal = 0, k = 0;
            for (; k + 4 <= c; k += 4) {
                double other[4];
#pragma unroll
                for (int e = 0; e < 4; e++) other[e] = got_s[k + e];
#pragma unroll
                for (int e = 0; e < 4; e++) above += other[e] > a.s, equal += other[e] == a.s;
            }
            for (; k < c; k++) above += got_s[k] > a.s, equal += got_s[k] == a.s;
            if (equal > 1 && above < n)
                for (k = 0; k < c; k++)
                    above += got_s[k] == a.s && before(Candidate{a.s, got_x[k], got_row[k], got_at[k]}, a);
            if (above < n) put(above, a);
        }
        for (int i = c + tid; i < n; i += THREADS) put_none(i);
        return;
    }
    // Many alike: the first of all, n times.
    Candidate last{INFINITY, INFINITY, -1, -1};
    for (int k = 0; k < n; k++) {
        Candidate best{-INFINITY, -INFINITY, INT32_MAX, INT32_MAX};
        for (int l = tid; l < lists; l += THREADS) {
            // the first of the list after the last one taken: a list falls
            Candidate c;
            int lo = 0, hi = n;
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (!load(l, mid, c) || before(last, c)) hi = mid;
                else lo = mid + 1;
            }
            if (lo < n && load(l, lo, c) && before(c, best)) best = c;
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const Candidate o{__shfl_xor(best.s, d, 64), __shfl_xor(best.x, d, 64), __shfl_xor(best.row, d, 64),
                              __shfl_xor(best.token, d, 64)};
            if (before(o, best)) best = o;
        }
        const int slot = (k & 1) * W;
        if (lane == 0) got_s[slot + wave] = best.s, got_x[slot + wave] = best.x, got_row[slot + wave] = best.row,
                       got_at[slot + wave] = best.token;
        __syncthreads();
        for (int w = 0; w < W; w++) {
            const Candidate o{got_s[slot + w], got_x[slot + w], got_row[slot + w], got_at[slot + w]};
            if (before(o, best)) best = o;
        }
        last = best;
        if (tid == 0) {
            if (best.row == INT32_MAX) put_none(k);
            else put(k, best);
        }
    }
}

// Elements of a thread: 32, or 8 where that leaves most of the chip idle.
int elements_of(int64_t rows, int64_t vocab) { return rows * ((vocab + 8191) / 8192) >= 512 ? 32 : 8; }
int64_t splits_of(int64_t rows, int64_t vocab) {
    const int64_t chunk = kThreads * elements_of(rows, vocab);
    return (vocab + chunk - 1) / chunk;
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace

size_t beam_select_workspace(int64_t groups, int64_t beams, int64_t vocab, int64_t n_out) {
    const size_t lists = (size_t)(groups * beams * splits_of(groups * beams, vocab));
    return up256(lists * n_out * sizeof(uint2)) + up256(lists * sizeof(Part));
}

hipError_t launch_beam_select(const BeamSelect& a, int type, hipStream_t stream) {
    BeamJob j{};
    static_cast<BeamSelect&>(j) = a;
    const int64_t rows = (int64_t)a.groups * a.beams;
    j.splits = (int)splits_of(rows, a.vocab);
    const size_t lists = (size_t)(rows * j.splits);
    j.lists = static_cast<uint2*>(a.ws);
    j.parts = reinterpret_cast<Part*>(static_cast<char*>(a.ws) + up256(lists * a.n_out * sizeof(uint2)));
    const bool wide = elements_of(rows, a.vocab) == 32;
    const hipError_t e = with_type(type, [&](auto t) {
        using T = decltype(t);
        // rows in the grid's y, up to 65535 at a time
        for (int64_t r = 0; r < rows; r += 65535) {
            BeamJob part = j;
            part.logits = static_cast<const T*>(a.logits) + r * a.ld;
            if (a.done) part.done = a.done + r;
            part.lists += r * j.splits * a.n_out;
            part.parts += r * j.splits;
            const dim3 grid((unsigned)j.splits, (unsigned)std::min<int64_t>(65535, rows - r));
            if (wide) hipLaunchKernelGGL((list_kernel<T, 32>), grid, dim3(kThreads), 0, stream, part);
            else hipLaunchKernelGGL((list_kernel<T, 8>), grid, dim3(kThreads), 0, stream, part);
            if (hipError_t e = hipGetLastError()) return e;
        }
        return hipSuccess;
    });
    if (e != hipSuccess) return e;
    const int lists_of = a.beams * j.splits;
    int bits = 0;
    while (1 << bits < lists_of) bits++;
    const dim3 grid((unsigned)a.groups);
    // places of a list that THREADS have at once, `held` to each
    auto holds = [&](int threads, int held) { return 1 << bits <= threads && a.n_out <= held * (threads >> bits); };
    if (holds(256, 2)) hipLaunchKernelGGL((join_kernel<2, 256>), grid, dim3(256), 0, stream, j, bits);
    else if (holds(1024, 4)) hipLaunchKernelGGL((join_kernel<4, 1024>), grid, dim3(1024), 0, stream, j, bits);
    else hipLaunchKernelGGL((join_kernel<0, 256>), grid, dim3(256), 0, stream, j, 0);
    return hipGetLastError();
}

}  // namespace vtq
