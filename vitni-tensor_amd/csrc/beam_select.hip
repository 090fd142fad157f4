// beam_select.hip -- the best continuations of beams over their vocabulary (gfx950).
//
//   s(row, token) = score(row) + x(row, token) - ln sum_v exp x(row, v)
//
// and the n greatest s of a group of rows.  The logits are read once: a workgroup has
// up to 8192 of a row in its registers, sums their exponentials below their maximum, and
// leaves its n greatest.  A second launch, a workgroup a group, joins sums and lists.
//
// Which of two sums is greater decides about tokens, so s is f64, and a row's sum of
// exponentials right to some 2^-30 (f32 would leave s wrong by 2^-20 of itself and more,
// and equal where it is not).  The few logits near the maximum go through a polynomial in
// f64, gathered so that all lanes have some; the many below, which count for little, through
// f32.  Where many are near, all go through f64.
//
// The n greatest of a workgroup: with T the n-th greatest of the 64 lanes' maxima of a
// wave, n elements at least reach T, so only those that do are looked at (a few times
// n): gathered in LDS and ranked by counting.  T's first 16 bits do.
#include <algorithm>
#include <type_traits>

#include "vtq_device.h"
#include "vtq_serve.h"

namespace vtq {
namespace {

constexpr int kThreads = 256;
constexpr int kNear = 1024;      // logits near the maximum that are gathered
constexpr int kGather = 512;     // candidates that a workgroup ranks by counting
constexpr int kJoinGather = 1024;

struct Part {
    double sum;  // of exp(x - top); no number: the row holds +infinity or NaN
    float top;
};

struct BeamJob : BeamSelect {
    int splits;      // workgroups of a row
    uint2* lists;    // [rows][splits][n_out], falling: logit (f32 bits) and token; token -1: no more
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

// exp(y), y <= 0, to 2^-40 of itself; 0 below -80.
__device__ __forceinline__ double exp_of(double y) {
    const double t = y * 1.4426950408889634074;
    const double round = 6755399441055744.0;  // 1.5 * 2^52: the sum's last bits are the nearest whole number
    const double shifted = t + round;
    const double z = (t - (shifted - round)) * 0.69314718055994530942;
    double p = 1.0 / 3628800.0;
    p = fma(p, z, 1.0 / 362880.0);
    p = fma(p, z, 1.0 / 40320.0);
    p = fma(p, z, 1.0 / 5040.0);
    p = fma(p, z, 1.0 / 720.0);
    p = fma(p, z, 1.0 / 120.0);
    p = fma(p, z, 1.0 / 24.0);
    p = fma(p, z, 1.0 / 6.0);
    p = fma(p, z, 0.5);
    p = fma(p, z, 1.0);
    p = fma(p, z, 1.0);
    const uint64_t bits = (uint64_t)__double_as_longlong(p) + ((uint64_t)(uint32_t)__double_as_longlong(shifted) << 52);
    return y < -80.0 ? 0.0 : __longlong_as_double((long long)bits);
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d, 64);
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x = fmaxf(x, __shfl_xor(x, d, 64));
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

// Calls put(place, key) for each of the n greatest of c different numbers in LDS.
template <class Put>
__device__ __forceinline__ void rank_keys(const uint64_t* keys, int c, int n, Put put) {
    for (int i = threadIdx.x; i < c; i += kThreads) {
        const uint64_t mine = keys[i];
        int above = 0, k = 0;
        // LDS's latency is what this costs: 8 numbers at a time
        for (; k + 8 <= c; k += 8) {
            uint64_t other[8];
#pragma unroll
            for (int e = 0; e < 8; e++) other[e] = keys[k + e];
#pragma unroll
            for (int e = 0; e < 8; e++) above += other[e] > mine;
        }
        for (; k < c; k++) above += keys[k] > mine;
        if (above < n) put(above, mine);
    }
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
    float x[E];
#pragma unroll
    for (int l = 0; l < L; l++) {
        const int at = first + (l * kThreads + tid) * V;
        // Rows start at any element.  (Loads from the next multiple of 16 bytes on would give a
        // row's sum another order for each start, and rows of the same logits another sum.)
        typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
        if (at + V <= j.vocab) {
            const vec v = *reinterpret_cast<const vec*>(x0 + at);
#pragma unroll
            for (int e = 0; e < V; e++) x[l * V + e] = (float)v[e];
        } else {
            // past the row: below every number, so that only a comparison by token tells it from -infinity
#pragma unroll
            for (int e = 0; e < V; e++)
                x[l * V + e] = at + e < j.vocab ? (float)x0[at + e] : -INFINITY;
        }
    }
    auto token_of = [&](int i) { return first + (i / V * kThreads + tid) * V + i % V; };
    auto in_row = [&](int token) { return token < j.vocab; };

    // maxima of 4 parts of this thread's elements
    float part[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        part[k] = x[k];
#pragma unroll
        for (int i = k + 4; i < E; i += 4) part[k] = fmaxf(part[k], x[i]);
    }
    float top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
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
    __shared__ int nears[4], reachings[4], more;
    __shared__ double sums[4];
    __shared__ float near[kNear];
    __shared__ __attribute__((aligned(16))) uint64_t keys[kGather];
    if (lane == 0) tops[wave] = top, reaches[wave] = reach;
    if (tid == 0) more = 0;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    reach = max(max(reaches[0], reaches[1]), max(reaches[2], reaches[3]));
    const int64_t list = (int64_t)row * j.splits + split;
    const float base = top == -INFINITY ? 0.0f : top;
    // T; no number, or -infinity, where fewer than n lanes hold any: then all that is finite
    const float limit = from_ordered(reach);
    const bool masks = !(limit > -INFINITY);
    const float least = masks ? -3.402823466e38f : limit;
    // Near the top: within 5, where the exponential's own error of 2^-24 is what an element's
    // below is off by; of f32 logits, whose differences round, within 8.
    const float close = base - (sizeof(T) == 4 ? 8.0f : 5.0f);
    uint64_t is_near[E], reaches_t[E];
    int n_near = 0, n_reach = 0;
    float small = 0.0f;  // sum of the others; no number if a logit is none
#pragma unroll
    for (int i = 0; i < E; i++) {
        const bool in = x[i] >= close;
        is_near[i] = __ballot(in);
        reaches_t[i] = __ballot(x[i] >= least);
        n_near += __popcll(is_near[i]);
        n_reach += __popcll(reaches_t[i]);
        const float y = in ? -INFINITY : x[i] - base;
        // 2^(y log2 e), the product's rounding and the constant's put back
        const float t = y * 1.44269504088896340736f;
        const float rest = fmaf(y, 1.44269504088896340736f, -t) + y * 1.92596299112661746e-8f;
        const float p = __builtin_amdgcn_exp2f(t);
        small += y > -200.0f ? fmaf(p, rest * 0.69314718055994530942f, p) : y == y ? 0.0f : y;
    }
    // places in the order of waves, so that sums have one order
    if (lane == 0) nears[wave] = n_near, reachings[wave] = n_reach;
    __syncthreads();
    int near_at = 0, reach_at = 0;
    n_near = n_reach = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        near_at += w < wave ? nears[w] : 0, reach_at += w < wave ? reachings[w] : 0;
        n_near += nears[w], n_reach += reachings[w];
    }
    const bool few_near = n_near <= kNear, few = n_reach <= kGather;
    auto below = [&](uint64_t mask) {
        return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    };
    // a candidate as a number: greater logits, then lower tokens are greater
    auto key_of = [&](float v, int token) { return (uint64_t)ordered(v) << 32 | (uint32_t)~token; };
#pragma unroll
    for (int i = 0; i < E; i++) {
        if (few_near && is_near[i]) {
            if (is_near[i] >> lane & 1) near[near_at + below(is_near[i])] = x[i];
            near_at += __popcll(is_near[i]);
        }
        if (few && reaches_t[i]) {
            if (reaches_t[i] >> lane & 1) keys[reach_at + below(reaches_t[i])] = key_of(x[i], token_of(i));
            reach_at += __popcll(reaches_t[i]);
        }
    }
    // Of masked tokens, of which there may be many, n will do that come first: n of the first
    // n + n_reach tokens are masked.
    const int window = masks ? min(n + n_reach, min(kThreads * E, j.vocab - first)) : 0;
    const bool fits = few && n_reach + window <= kGather;
    if (fits && window) {
#pragma unroll
        for (int i = 0; i < E; i++)
            if (x[i] == -INFINITY && token_of(i) < first + window) keys[n_reach + atomicAdd(&more, 1)] = key_of(x[i], token_of(i));
    }
    __syncthreads();
    double sum = (double)(few_near ? small : small * 0.0f);
    if (few_near) {
        for (int i = tid; i < n_near; i += kThreads) sum += exp_of((double)near[i] - (double)base);
    } else {
#pragma unroll
        for (int i = 0; i < E; i++) sum += exp_of((double)x[i] - (double)base);
    }
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    uint2* out = j.lists + list * n;
    auto put = [&](int at, float v, int token) { out[at] = make_uint2(__float_as_uint(v), (uint32_t)token); };
    const int c = n_reach + more;
    if (fits) rank_keys(keys, c, n, [&](int at, uint64_t key) { put(at, from_ordered((uint32_t)(key >> 32)), ~(int)(uint32_t)key); });
    __syncthreads();
    if (tid == 0)
        j.parts[list] = Part{top < INFINITY ? (sums[0] + sums[1]) + (sums[2] + sums[3])
                                            : __longlong_as_double(0x7FF8000000000000ll), top};
    if (fits) {
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
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int token = token_of(i);
            const bool after = x[i] < last_x || (x[i] == last_x && token > last_at);
            if (in_row(token) && after && (x[i] > best || (x[i] == best && token < best_at))) best = x[i], best_at = token;
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

// HELD entries of the lists to a thread, in registers, all at once; 0: any number of lists,
// read as far as they matter.
template <int HELD>
__global__ __launch_bounds__(kThreads) void join_kernel(BeamJob j) {
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int n = j.n_out, beams = j.beams, splits = j.splits, lists = beams * splits;
    const int64_t row0 = (int64_t)blockIdx.x * beams;
    const uint2* entries = j.lists + row0 * splits * n;
    __shared__ double norm[64];  // ln of a row's sum
    __shared__ float score[64];
    __shared__ int kind[64];     // 0 lists, 1 one candidate, 2 all alike
    __shared__ uint32_t reaches[4];
    __shared__ int count;
    __shared__ __attribute__((aligned(16))) double got_s[kJoinGather];
    __shared__ float got_x[kJoinGather];
    __shared__ int got_at[kJoinGather], got_row[kJoinGather];
    uint2 held[HELD ? HELD : 1];
#pragma unroll
    for (int i = 0; i < HELD; i++) held[i] = entries[min(i * kThreads + tid, lists * n - 1)];
    if (tid == 0) count = 0;
    // `width` lanes to a row
    int width = 1;
    while (width < 64 && width < splits) width *= 2;
    for (int r0 = 0; r0 < beams; r0 += kThreads / width) {
        const int r = r0 + tid / width;
        const bool there = r < beams, ended = there && j.done && j.done[row0 + r];
        const Part* parts = j.parts + (row0 + (there ? r : 0)) * splits;
        float top = -INFINITY;
        if (there && !ended)
            for (int s = tid % width; s < splits; s += width) top = fmaxf(top, parts[s].top);
        for (int d = 1; d < width; d *= 2) top = fmaxf(top, __shfl_xor(top, d, 64));
        double sum = 0.0;
        if (there && !ended)
            for (int s = tid % width; s < splits; s += width) {
                // (a part of -infinities alone: its sum is 0)
                const Part p = parts[s];
                sum += p.sum == p.sum ? p.sum * exp_of((double)p.top - (double)top) : p.sum;
            }
        for (int d = 1; d < width; d *= 2) sum += __shfl_xor(sum, d, 64);
        if (there && tid % width == 0) {
            const double ln = (double)top + log(sum);
            const float cum = j.score[row0 + r];
            norm[r] = ln;
            score[r] = cum;
            kind[r] = ended ? 1 : isfinite(ln) && isfinite(cum) ? 0 : 2;
        }
    }
    __syncthreads();
    // entry `pos` of list l of the group; false: there is none
    auto candidate = [&](int l, int pos, uint2 entry, Candidate& c) {
        c.row = l / splits;
        const int split = l - c.row * splits, what = kind[c.row];
        if (what == 0) {
            c.token = (int)entry.y;
            c.x = __uint_as_float(entry.x);
            c.s = (double)score[c.row] + ((double)c.x - norm[c.row]);
            return c.token >= 0;
        }
        c.x = -INFINITY;
        if (what == 1) {
            c.token = j.end_token;
            c.s = (double)score[c.row];
            if (!isfinite(c.s)) c.s = -INFINITY;
            else c.x = 0.0f;
            return split == 0 && pos == 0;
        }
        c.token = pos;
        c.s = -INFINITY;
        return split == 0 && pos < j.vocab;
    };
    auto load = [&](int l, int pos, Candidate& c) { return candidate(l, pos, entries[(int64_t)l * n + pos], c); };
    auto gather = [&](const Candidate& c) {
        const int at = atomicAdd(&count, 1);
        if (at < kJoinGather) got_s[at] = c.s, got_x[at] = c.x, got_row[at] = c.row, got_at[at] = c.token;
    };
    // a thread's greatest, and what n threads of a wave reach
    uint32_t key[1] = {0};
    Candidate mine[HELD ? HELD : 1];
    bool is[HELD ? HELD : 1];
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++) {
            const int e = i * kThreads + tid, l = e / n;
            is[i] = e < lists * n && candidate(l, e - l * n, held[i], mine[i]);
            if (is[i]) key[0] = max(key[0], ordered((float)mine[i].s));
        }
    } else {
        for (int l = tid; l < max(lists, kThreads); l += kThreads) {
            Candidate c;
            if (l / lists < n && load(l % lists, l / lists, c)) key[0] = max(key[0], ordered((float)c.s));
        }
    }
    const uint32_t reached = reached_by<1, 32>(key, n);
    if (lane == 0) reaches[wave] = reached;
    __syncthreads();
    const uint32_t reach = max(max(reaches[0], reaches[1]), max(reaches[2], reaches[3]));
    if constexpr (HELD > 0) {
#pragma unroll
        for (int i = 0; i < HELD; i++)
            if (is[i] && ordered((float)mine[i].s) >= reach) gather(mine[i]);
    } else {
        for (int l = tid; l < lists; l += kThreads) {
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
        for (int i = tid; i < c; i += kThreads) {
            const Candidate a{got_s[i], got_x[i], got_row[i], got_at[i]};
            // by the sums, 8 at a time; where some are equal, by the rest too
            int above = 0, equal = 0, k = 0;
            for (; k + 8 <= c; k += 8) {
                double other[8];
#pragma unroll
                for (int e = 0; e < 8; e++) other[e] = got_s[k + e];
#pragma unroll
                for (int e = 0; e < 8; e++) above += other[e] > a.s, equal += other[e] == a.s;
            }
            for (; k < c; k++) above += got_s[k] > a.s, equal += got_s[k] == a.s;
            if (equal > 1 && above < n)
                for (k = 0; k < c; k++)
                    above += got_s[k] == a.s && before(Candidate{a.s, got_x[k], got_row[k], got_at[k]}, a);
            if (above < n) put(above, a);
        }
        for (int i = c + tid; i < n; i += kThreads) put_none(i);
        return;
    }
    // Many alike: the first of all, n times.
    Candidate last{INFINITY, INFINITY, -1, -1};
    for (int k = 0; k < n; k++) {
        Candidate best{-INFINITY, -INFINITY, INT32_MAX, INT32_MAX};
        for (int l = tid; l < lists; l += kThreads) {
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
        const int slot = (k & 1) * 4;
        if (lane == 0) got_s[slot + wave] = best.s, got_x[slot + wave] = best.x, got_row[slot + wave] = best.row,
                       got_at[slot + wave] = best.token;
        __syncthreads();
        for (int w = 0; w < 4; w++) {
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
    const int64_t entries = (int64_t)a.beams * j.splits * a.n_out;
    const dim3 grid((unsigned)a.groups), block(kThreads);
    if (entries <= 2 * kThreads) hipLaunchKernelGGL((join_kernel<2>), grid, block, 0, stream, j);
    else if (entries <= 8 * kThreads) hipLaunchKernelGGL((join_kernel<8>), grid, block, 0, stream, j);
    else hipLaunchKernelGGL((join_kernel<0>), grid, block, 0, stream, j);
    return hipGetLastError();
}

}  // namespace vtq
