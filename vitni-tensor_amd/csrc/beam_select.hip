// beam_select.hip -- the best continuations of beams over their vocabulary (gfx950).
//
//   s(row, token) = score(row) + x(row, token) - ln sum_v exp x(row, v)
//
// and the n greatest s of a group of rows.  The logits are read once: a workgroup has
// up to 8192 of a row in its registers, sums their exponentials below their maximum, and
// leaves its n greatest.  A second launch, a workgroup a group, joins sums and lists.
//
// Which of two sums is greater decides about tokens, so a row's sum of exponentials and
// s itself are f64 (f32 would leave s wrong by 2^-20 of itself and more, and equal where it is
// not).  The exponential is a polynomial in f64, 17 operations at the f32 rate.
//
// The n greatest of a workgroup: with T the n-th greatest of the 64 lanes' maxima of a
// wave, n elements at least reach T, so only those that do are looked at (a few times n): gathered in LDS
// in any order and ranked by counting, which leaves one order.  T's first 16 bits do.
#include <algorithm>
#include <type_traits>

#include "vtq_device.h"
#include "vtq_serve.h"

namespace vtq {
namespace {

constexpr int kThreads = 256;
constexpr int kGather = 512;     // elements that a workgroup ranks by counting
constexpr int kJoinGather = 1024;

struct BeamJob : BeamSelect {
    int splits;        // workgroups of a row
    float* list_x;     // [rows][splits][n_out], falling
    int32_t* list_at;  // tokens; -1: no more
    double* sums;      // [rows][splits]: of exp(x - top); no number: the row holds +infinity or NaN
    float* tops;       // [rows][splits]
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

// ------------------------------------------------ lists of a row's parts

template <class T, int E>
__global__ __launch_bounds__(kThreads) void list_kernel(BeamJob j) {
    constexpr int V = 16 / sizeof(T), L = E / V;  // elements of a load, loads
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int row = blockIdx.y, split = blockIdx.x, n = j.n_out;
    if (j.done && j.done[row]) return;
    const T* x0 = static_cast<const T*>(j.logits) + row * j.ld;
    // loads start at multiples of 16 bytes, the first one maybe before the row
    const int ahead = (int)(reinterpret_cast<uintptr_t>(x0) / sizeof(T) % V);
    const int first = split * kThreads * E - ahead;
    // element l V + e of this thread is token first + (l 256 + tid) V + e
    float x[E];
    bool bad = false;
#pragma unroll
    for (int l = 0; l < L; l++) {
        const int at = first + (l * kThreads + tid) * V;
        typedef T vec __attribute__((ext_vector_type(V)));
        if (at >= 0 && at + V <= j.vocab) {
            const vec v = *reinterpret_cast<const vec*>(x0 + at);
#pragma unroll
            for (int e = 0; e < V; e++) {
                x[l * V + e] = (float)v[e];
                bad |= !(x[l * V + e] < INFINITY);
            }
        } else {
            // past the row: below every number, so that only a comparison by token tells it from -infinity
#pragma unroll
            for (int e = 0; e < V; e++) {
                const bool in = at + e >= 0 && at + e < j.vocab;
                x[l * V + e] = in ? (float)x0[at + e] : -INFINITY;
                bad |= !(x[l * V + e] < INFINITY);
            }
        }
    }
    auto token_of = [&](int i) { return first + (i / V * kThreads + tid) * V + i % V; };
    auto in_row = [&](int token) { return token >= 0 && token < j.vocab; };

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
    __shared__ int bads[4], count, finite;
    __shared__ double sums[4];
    __shared__ float got_x[kGather];
    __shared__ int got_at[kGather];
    const bool any_bad = __ballot(bad) != 0;
    if (lane == 0) tops[wave] = top, reaches[wave] = reach, bads[wave] = any_bad;
    if (tid == 0) count = 0, finite = 0;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    reach = max(max(reaches[0], reaches[1]), max(reaches[2], reaches[3]));
    bad = bads[0] | bads[1] | bads[2] | bads[3];
    const int64_t list = (int64_t)row * j.splits + split;
    if (bad) {
        // the row's candidates are all alike: its lists are not read
        if (tid == 0) j.sums[list] = __longlong_as_double(0x7FF8000000000000ll), j.tops[list] = 0.0f;
        return;
    }

    // the sum, -infinity being 0 (and 0 below a top of -infinity)
    double sum = 0.0;
    const double base = top == -INFINITY ? 0.0 : (double)top;
#pragma unroll
    for (int i = 0; i < E; i++) sum += exp_of((double)x[i] - base);
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;

    // -infinities stand for masked tokens, of which there may be many: of these, the first n
    // tokens that are none of the finite ones will do
    const float least = from_ordered(reach);  // no number where fewer than n lanes hold any
    const bool masks = !(least > -INFINITY);
    int mine = 0;
#pragma unroll
    for (int i = 0; i < E; i++) mine += masks ? x[i] > -INFINITY : x[i] >= least;
    int of_wave = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) of_wave += __shfl_xor(of_wave, d, 64);
    if (lane == 0 && of_wave) atomicAdd(&finite, of_wave);
    __syncthreads();
    if (tid == 0) j.sums[list] = (sums[0] + sums[1]) + (sums[2] + sums[3]), j.tops[list] = top;
    const int reaching = finite;  // elements to gather, masked ones apart
    float* out_x = j.list_x + list * n;
    int32_t* out_at = j.list_at + list * n;
    const int start = max(first, 0);
    if (reaching + (masks ? n : 0) <= kGather) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            const int token = token_of(i);
            const bool take = masks ? x[i] > -INFINITY || (in_row(token) && token < start + reaching + n && x[i] == -INFINITY)
                                    : x[i] >= least;
            if (take) {
                // (at most n + reaching masked tokens lie before that bound, reaching of them at
                // most are too many)
                const int at = atomicAdd(&count, 1);
                if (at < kGather) got_x[at] = x[i], got_at[at] = token;
            }
        }
        __syncthreads();
        if (count <= kGather) {
            const int c = count;
            for (int i = tid; i < c; i += kThreads) {
                const float xi = got_x[i];
                const int ti = got_at[i];
                int rank = 0;
                for (int k = 0; k < c; k++) rank += got_x[k] > xi || (got_x[k] == xi && got_at[k] < ti);
                if (rank < n) out_x[rank] = xi, out_at[rank] = ti;
            }
            for (int i = c + tid; i < n; i += kThreads) out_x[i] = -INFINITY, out_at[i] = -1;
            return;
        }
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
        if (tid == 0) out_x[k] = best, out_at[k] = best_at == INT32_MAX ? -1 : best_at;
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

__global__ __launch_bounds__(kThreads) void join_kernel(BeamJob j) {
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int n = j.n_out, beams = j.beams, splits = j.splits;
    const int64_t row0 = (int64_t)blockIdx.x * beams;
    __shared__ double norm[64];  // ln of a row's sum
    __shared__ float score[64];
    __shared__ int kind[64];     // 0 lists, 1 one candidate, 2 all alike
    __shared__ uint32_t reaches[4];
    __shared__ int count;
    __shared__ double got_s[kJoinGather];
    __shared__ float got_x[kJoinGather];
    __shared__ int got_at[kJoinGather], got_row[kJoinGather];
    if (tid == 0) count = 0;
    for (int r = wave; r < beams; r += 4) {
        const int64_t row = row0 + r;
        const bool ended = j.done && j.done[row];
        double sum = 0.0;
        float top = -INFINITY;
        if (!ended) {
            for (int s = lane; s < splits; s += 64) top = fmaxf(top, j.tops[row * splits + s]);
            top = wave_max(top);
            for (int s = lane; s < splits; s += 64) {
                // a part of -infinities alone has a sum without meaning
                const float t = j.tops[row * splits + s];
                const double part = j.sums[row * splits + s];
                if (t > -INFINITY) sum += part == part ? part * exp_of((double)t - (double)top) : part;
            }
            sum = wave_sum(sum);
        }
        if (lane == 0) {
            const double ln = (double)top + log(sum);
            const float cum = j.score[row];
            norm[r] = ln;
            score[r] = cum;
            kind[r] = ended ? 1 : isfinite(ln) && isfinite(cum) ? 0 : 2;
        }
    }
    __syncthreads();
    // candidate `pos` of list `l` of the group; false: there is none
    auto candidate = [&](int l, int pos, Candidate& c) {
        c.row = l / splits;
        const int split = l % splits;
        if (kind[c.row] == 0) {
            const int64_t at = ((row0 + c.row) * splits + split) * n + pos;
            c.token = j.list_at[at];
            c.x = j.list_x[at];
            c.s = (double)score[c.row] + ((double)c.x - norm[c.row]);
            return c.token >= 0;
        }
        c.x = -INFINITY;
        if (kind[c.row] == 1) {
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
    const int lists = beams * splits;
    // a thread's greatest: of the heads of its lists, or, where lists are fewer than threads,
    // of one candidate further down
    float top = -INFINITY;
    bool some = false;
    for (int l = tid; l < max(lists, kThreads); l += kThreads) {
        Candidate c;
        if (l / lists < n && candidate(l % lists, l / lists, c)) top = fmaxf(top, (float)c.s), some = true;
    }
    const uint32_t key[1] = {some ? ordered(top) : 0u};
    const uint32_t mine = reached_by<1, 32>(key, n);
    if (lane == 0) reaches[wave] = mine;
    __syncthreads();
    const uint32_t reach = max(max(reaches[0], reaches[1]), max(reaches[2], reaches[3]));
    for (int l = tid; l < lists; l += kThreads) {
        Candidate c;
        for (int pos = 0; pos < n && candidate(l, pos, c) && ordered((float)c.s) >= reach; pos++) {
            const int at = atomicAdd(&count, 1);
            if (at < kJoinGather) got_s[at] = c.s, got_x[at] = c.x, got_row[at] = c.row, got_at[at] = c.token;
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
            int rank = 0;
            for (int k = 0; k < c; k++) rank += before(Candidate{got_s[k], got_x[k], got_row[k], got_at[k]}, a);
            if (rank < n) put(rank, a);
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
            int from = 0, to = n;
            while (from < to) {
                const int mid = (from + to) / 2;
                if (!candidate(l, mid, c) || before(last, c)) to = mid;
                else from = mid + 1;
            }
            if (from < n && candidate(l, from, c) && before(c, best)) best = c;
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
    return (vocab + 7 + chunk - 1) / chunk;  // a row may start up to 7 elements into its first load
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace

size_t beam_select_workspace(int64_t groups, int64_t beams, int64_t vocab, int64_t n_out) {
    const size_t lists = (size_t)(groups * beams * splits_of(groups * beams, vocab));
    return up256(lists * n_out * 4) * 2 + up256(lists * 8) + up256(lists * 4);
}

hipError_t launch_beam_select(const BeamSelect& a, int type, hipStream_t stream) {
    BeamJob j{};
    static_cast<BeamSelect&>(j) = a;
    const int64_t rows = (int64_t)a.groups * a.beams;
    j.splits = (int)splits_of(rows, a.vocab);
    const size_t lists = (size_t)(rows * j.splits);
    char* at = static_cast<char*>(a.ws);
    j.list_x = reinterpret_cast<float*>(at);
    at += up256(lists * a.n_out * 4);
    j.list_at = reinterpret_cast<int32_t*>(at);
    at += up256(lists * a.n_out * 4);
    j.sums = reinterpret_cast<double*>(at);
    at += up256(lists * 8);
    j.tops = reinterpret_cast<float*>(at);
    const bool wide = elements_of(rows, a.vocab) == 32;
    const hipError_t e = with_type(type, [&](auto t) {
        using T = decltype(t);
        // rows in the grid's y up to 65535 at a time
        for (int64_t r = 0; r < rows; r += 65535) {
            BeamJob part = j;
            part.logits = static_cast<const T*>(a.logits) + r * a.ld;
            if (a.done) part.done = a.done + r;
            part.list_x += r * j.splits * a.n_out;
            part.list_at += r * j.splits * a.n_out;
            part.sums += r * j.splits;
            part.tops += r * j.splits;
            const dim3 grid((unsigned)j.splits, (unsigned)std::min<int64_t>(65535, rows - r));
            if (wide) hipLaunchKernelGGL((list_kernel<T, 32>), grid, dim3(kThreads), 0, stream, part);
            else hipLaunchKernelGGL((list_kernel<T, 8>), grid, dim3(kThreads), 0, stream, part);
            if (hipError_t e = hipGetLastError()) return e;
        }
        return hipSuccess;
    });
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(join_kernel, dim3((unsigned)a.groups), dim3(kThreads), 0, stream, j);
    return hipGetLastError();
}

}  // namespace vtq
