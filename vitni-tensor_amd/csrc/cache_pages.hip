// cache_pages.hip -- who holds a cache's pages: the next batch's page tables from the
// sequences that it goes on with, the pages in use closed up, and copies of pages (gfx950).
//
// The lists are small (a table of 256 x 256 pages is 256 KB) and each step needs the one
// before, so time is launches and latency: two kernels for a reorder, one or three to close
// up, over all pages at once, with counts of 1024 pages that every workgroup adds up for
// itself.  Free pages are taken lowest first and in the order of sequences, and counts change by
// atomic additions of whole numbers, whose order changes nothing: the same lists every time.
//
// Kernel times beside the copies that they are for: 32 sequences of 64 places on 1400 pages 3.3 and
// 5.8 us; 256 of 256 on 40000 3.6 and 7.3; 1000 and 4096 pages closed up 9.7 and 12.1, as the copies
// before have taken the caches (7.3 and 8.6 without them, 6.9 and 7.0 in a graph).  Copies are
// memory's: 4096 pages of 8 layers, 1.05 GB, 204 us (5.1 TB/s; 222 where a workgroup finds its place by
// dividing one index).
#include <algorithm>

#include "vtq_device.h"
#include "vtq_serve.h"

namespace vtq {
namespace {

constexpr int kSegment = 1024;  // pages to a workgroup
constexpr int kThreads = 256;
constexpr int kOwnScan = 1024;  // new sequences whose counts every workgroup scans for itself

struct ReorderJob : PagesReorder {
    int segments;
    int32_t *begin, *fresh, *to_copy;     // [batch_out]: first place of free pages, how many, whether a page is copied
    int32_t* free_in;                     // [segments]
    int64_t* fresh_before;                // [batch_out + 1]; these two above kOwnScan sequences
    int32_t* copies_before;               // [batch_out + 1]
};

__device__ __forceinline__ int pages_of(int64_t tokens, int page_size) {
    return (int)((tokens + page_size - 1) / page_size);
}
__device__ __forceinline__ bool is_page(int32_t p, int64_t n_pages) { return p >= 0 && p < n_pages; }
__device__ __forceinline__ int length_of(const ReorderJob& j, int seq) {
    return min(max(j.len[seq], 0), j.max_pages * j.page_size);
}

// Counts the segment's free pages (or, without new_refs, those in use); the new counts
// begin as the old ones.
__device__ __forceinline__ void count_segment(const int32_t* refs, int32_t* new_refs, int64_t n_pages, int segment,
                                              int32_t* counts) {
    const int64_t p0 = (int64_t)segment * kSegment;
    int mine = 0;
    for (int k = threadIdx.x; k < kSegment && p0 + k < n_pages; k += kThreads) {
        const int r = refs[p0 + k];
        if (new_refs) new_refs[p0 + k] = r;
        mine += new_refs ? r == 0 : r > 0;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) mine += __shfl_xor(mine, d, 64);
    __shared__ int part[kThreads / 64];
    if ((threadIdx.x & 63) == 0) part[wave_id()] = mine;
    __syncthreads();
    if (threadIdx.x == 0) counts[segment] = part[0] + part[1] + part[2] + part[3];
}

// Workgroups below `segments` count their free pages, the others (one to a new sequence) find
// what it shares and keeps.
__global__ __launch_bounds__(kThreads) void reorder_share_kernel(ReorderJob j) {
    if ((int64_t)blockIdx.x < j.segments) {
        count_segment(j.refs, j.new_refs, j.n_pages, (int)blockIdx.x, j.free_in);
        return;
    }
    const int i = (int)(blockIdx.x - j.segments), tid = threadIdx.x;
    const int parent = j.parent[i];
    const bool has = parent >= 0 && parent < j.batch;
    __shared__ int earlier, stop;
    if (tid == 0) earlier = 0, stop = INT32_MAX;
    __syncthreads();
    if (has) {
        bool any = false;
        for (int k = tid; k < i; k += kThreads) any |= j.parent[k] == parent;
        if (any) earlier = 1;  // all write the same
    }
    const int len = has ? length_of(j, parent) : 0;
    const int64_t grown = (int64_t)len + (j.grow ? max(j.grow[i], 0) : 0);
    const int whole = len / j.page_size, needed = min(pages_of(grown, j.page_size), j.max_pages);
    const int32_t* row = has ? j.pages + (int64_t)parent * j.max_pages : nullptr;
    __syncthreads();
    const bool eldest = has && !earlier;
    // the eldest keeps the pages from `whole` on up to the first that it may not
    if (eldest) {
        int mine = INT32_MAX;
        for (int p = whole + tid; p < needed; p += kThreads)
            if (!(is_page(row[p], j.n_pages) && j.refs[row[p]] == 1)) {
                mine = p;
                break;
            }
        if (mine < INT32_MAX) atomicMin(&stop, mine);
    }
    __syncthreads();
    const int begin = eldest ? min(stop, max(needed, whole)) : whole;
    int32_t* out = j.new_pages + (int64_t)i * j.max_pages;
    for (int p = tid; p < j.max_pages; p += kThreads)
        out[p] = has && p < begin && is_page(row[p], j.n_pages) ? row[p] : -1;
    if (tid == 0) {
        j.new_len[i] = len;
        j.begin[i] = begin;
        j.fresh[i] = max(needed - begin, 0);
        j.to_copy[i] = begin == whole && len % j.page_size && whole < needed && is_page(row[whole], j.n_pages);
        j.copies[3 * (int64_t)i] = j.copies[3 * (int64_t)i + 1] = j.copies[3 * (int64_t)i + 2] = -1;
    }
}

// Sum over a workgroup of THREADS.
template <int THREADS, class S>
__device__ __forceinline__ S sum_of(S x) {
    __shared__ S part[THREADS / 64];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) x += __shfl_xor(x, d, 64);
    __syncthreads();  // the last sum's parts are read
    if ((threadIdx.x & 63) == 0) part[wave_id()] = x;
    __syncthreads();
    S all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; w++) all += part[w];
    return all;
}

// before[i] = sum of value(k) for k below i, i up to n, by a workgroup of THREADS; returns the sum.
template <int THREADS, class S, class Value>
__device__ __forceinline__ S scan(int64_t n, S* before, Value value) {
    __shared__ S waves[THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    S carry = 0;
    for (int64_t i0 = 0; i0 < n; i0 += THREADS) {
        const S own = i0 + tid < n ? (S)value(i0 + tid) : (S)0;
        S up_to = own;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const S o = __shfl_up(up_to, d, 64);
            if (lane >= d) up_to += o;
        }
        if (lane == 63) waves[wave] = up_to;
        __syncthreads();
        S ahead = carry, all = carry;
#pragma unroll
        for (int w = 0; w < THREADS / 64; w++) {
            if (w < wave) ahead += waves[w];
            all += waves[w];
        }
        if (i0 + tid < n) before[i0 + tid] = ahead + up_to - own;
        carry = all;
        __syncthreads();
    }
    if (tid == 0) before[n] = carry;
    __syncthreads();
    return carry;
}

// Pages that a sequence's growth would take beyond max_pages.
__device__ __forceinline__ int64_t beyond(const ReorderJob& j, int i) {
    if (!j.grow) return 0;
    return max(pages_of((int64_t)j.new_len[i] + max(j.grow[i], 0), j.page_size) - j.max_pages, 0);
}

// Scans of the new sequences' counts: free pages that go to those before each, and copies.  A
// sequence's copy has a page while pages last, from the first sequence on.  One workgroup
// alone tells the counts.
template <int THREADS>
__device__ __forceinline__ void scan_sequences(const ReorderJob& j, int64_t free, int64_t* fresh_before,
                                               int32_t* copies_before, bool tells) {
    const int64_t fresh = scan<THREADS>(j.batch_out, fresh_before, [&](int64_t i) { return j.fresh[i]; });
    const int copies = scan<THREADS>(j.batch_out, copies_before, [&](int64_t i) {
        return j.to_copy[i] && fresh_before[i] < free ? 1 : 0;
    });
    if (!tells) return;
    int64_t over = 0;
    for (int i = threadIdx.x; i < j.batch_out; i += THREADS) over += beyond(j, i);
    over = sum_of<THREADS>(over);
    if (threadIdx.x == 0) {
        j.info[0] = copies;
        j.info[1] = (int32_t)min(max(fresh - free, (int64_t)0) + over, (int64_t)INT32_MAX);
    }
}

__global__ __launch_bounds__(1024) void reorder_scan_kernel(ReorderJob j) {
    int64_t free = 0;
    for (int s = threadIdx.x; s < j.segments; s += 1024) free += j.free_in[s];
    scan_sequences<1024>(j, sum_of<1024>(free), j.fresh_before, j.copies_before, true);
}

// Workgroups below `segments` hand out their free pages, the others (one to an old sequence, and
// the last) take its pages' holders off and its children on.
template <bool OWN>
__global__ __launch_bounds__(kThreads) void reorder_apply_kernel(ReorderJob j) {
    const int tid = threadIdx.x, lane = tid & 63;
    const bool tells = (int64_t)blockIdx.x == (int64_t)j.segments + j.batch;
    if ((int64_t)blockIdx.x >= j.segments && !tells) {
        const int old = (int)(blockIdx.x - j.segments);
        __shared__ int children, eldest;
        if (tid == 0) children = 0, eldest = INT32_MAX;
        __syncthreads();
        for (int i = tid; i < j.batch_out; i += kThreads)
            if (j.parent[i] == old) {
                atomicAdd(&children, 1);
                atomicMin(&eldest, i);
            }
        __syncthreads();
        const int whole = length_of(j, old) / j.page_size, keeps = children ? j.begin[eldest] : 0;
        for (int p = tid; p < j.max_pages; p += kThreads) {
            const int32_t page = j.pages[(int64_t)old * j.max_pages + p];
            if (!is_page(page, j.n_pages)) continue;
            const int change = (p < whole ? children : p < keeps ? 1 : 0) - 1;
            if (change) atomicAdd(&j.new_refs[page], change);
        }
        return;
    }
    __shared__ int64_t own_fresh[OWN ? kOwnScan + 1 : 1];
    __shared__ int32_t own_copies[OWN ? kOwnScan + 1 : 1];
    int64_t before = 0, all = 0;
    for (int s = tid; s < j.segments; s += kThreads) {
        const int n = j.free_in[s];
        all += n;
        before += s < (int)blockIdx.x ? n : 0;
    }
    int64_t rank = sum_of<kThreads>(before);
    if constexpr (OWN) scan_sequences<kThreads>(j, sum_of<kThreads>(all), own_fresh, own_copies, tells);
    if (tells) return;
    auto fresh_before = [&](int i) { return OWN ? own_fresh[i] : j.fresh_before[i]; };
    const int64_t total = fresh_before(j.batch_out);
    for (int k0 = 0; k0 < kSegment && rank < total; k0 += kThreads) {
        const int64_t page = (int64_t)blockIdx.x * kSegment + k0 + tid;
        const bool free = page < j.n_pages && j.refs[page] == 0;
        const uint64_t mask = __ballot(free);
        __shared__ int waves[kThreads / 64];
        if (lane == 0) waves[wave_id()] = __popcll(mask);
        __syncthreads();
        int64_t mine = rank + __popcll(mask & ((1ull << lane) - 1));
        for (int w = 0; w < kThreads / 64; w++) {
            if (w < wave_id()) mine += waves[w];
            rank += waves[w];
        }
        __syncthreads();
        if (free && mine < total) {
            // the sequence whose free pages hold this rank
            int lo = 0, hi = j.batch_out;
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (fresh_before(mid) <= mine) lo = mid;
                else hi = mid;
            }
            const int at = (int)(mine - fresh_before(lo));
            j.new_pages[(int64_t)lo * j.max_pages + j.begin[lo] + at] = (int32_t)page;
            atomicAdd(&j.new_refs[page], 1);
            if (at == 0 && j.to_copy[lo]) {
                const int parent = j.parent[lo], len = j.new_len[lo];
                int32_t* c = j.copies + 3 * (int64_t)(OWN ? own_copies[lo] : j.copies_before[lo]);
                c[0] = j.pages[(int64_t)parent * j.max_pages + len / j.page_size];
                c[1] = (int32_t)page;
                c[2] = len % j.page_size;
            }
        }
    }
}

// ------------------------------------------------ pages closed up

struct CompactJob : PagesCompact {
    int segments;
    int32_t* live_in;     // [segments]
    int32_t *low, *high;  // [n_pages / 2]: free pages below the count of those in use, and pages in use past it
    int32_t* rank;        // [n_pages]: of a page among the latter
};

__global__ __launch_bounds__(kThreads) void compact_count_kernel(CompactJob j) {
    count_segment(j.refs, nullptr, j.n_pages, (int)blockIdx.x, j.live_in);
}

__global__ __launch_bounds__(kThreads) void compact_rank_kernel(CompactJob j) {
    const int tid = threadIdx.x, lane = tid & 63;
    int64_t all = 0, up_to = 0;
    for (int s = tid; s < j.segments; s += kThreads) {
        const int n = j.live_in[s];
        all += n;
        up_to += s < (int)blockIdx.x ? n : 0;
    }
    const int64_t n_live = sum_of<kThreads>(all);
    int64_t before = sum_of<kThreads>(up_to);
    // pages in use below n_live: those of whole segments, and of the one that it lies in
    const int64_t edge = n_live / kSegment;
    int64_t mine = 0;
    for (int s = tid; s < edge; s += kThreads) mine += j.live_in[s];
    for (int64_t p = edge * kSegment + tid; p < n_live; p += kThreads) mine += j.refs[p] > 0;
    const int64_t below = sum_of<kThreads>(mine);
    if (blockIdx.x == 0 && tid == 0) {
        j.info[0] = (int32_t)(n_live - below);
        j.info[1] = (int32_t)n_live;
    }
    __shared__ int waves[kThreads / 64];
    for (int k0 = 0; k0 < kSegment; k0 += kThreads) {
        const int64_t p = (int64_t)blockIdx.x * kSegment + k0 + tid;
        const bool there = p < j.n_pages;
        const int refs = there ? j.refs[p] : 0;
        const uint64_t mask = __ballot(refs > 0);
        if (lane == 0) waves[wave_id()] = __popcll(mask);
        __syncthreads();
        int64_t at = before + __popcll(mask & ((1ull << lane) - 1));  // pages in use before this one
        for (int w = 0; w < kThreads / 64; w++) {
            if (w < wave_id()) at += waves[w];
            before += waves[w];
        }
        __syncthreads();
        if (!there) continue;
        if (p < n_live) {
            if (refs > 0) j.new_refs[p] = refs;
            else j.low[p - at] = (int32_t)p;  // (its new count comes with the page that moves there)
        } else {
            j.new_refs[p] = 0;
            if (refs > 0) {
                j.high[at - below] = (int32_t)p;
                j.rank[p] = (int32_t)(at - below);
            }
        }
    }
}

__global__ __launch_bounds__(kThreads) void compact_apply_kernel(CompactJob j) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t n_live = j.info[1], moves = j.info[0];
    if (i < j.n_pages / 2) {
        const bool is = i < moves;
        const int32_t from = is ? j.high[i] : -1, to = is ? j.low[i] : -1;
        j.copies[3 * i] = from;
        j.copies[3 * i + 1] = to;
        j.copies[3 * i + 2] = is ? j.page_size : -1;
        if (is) j.new_refs[to] = j.refs[from];
    }
    auto moved = [&](int32_t p) {
        if (!is_page(p, j.n_pages)) return -1;
        return p >= n_live && j.refs[p] > 0 ? j.low[j.rank[p]] : p;
    };
    if (i < j.n_entries) j.new_pages[i] = moved(j.pages[i]);
    if (i < j.n_prefix) j.new_prefix_pages[i] = moved(j.prefix_pages[i]);
}

// All of it in one launch where pages are few: every workgroup makes a bit to each page in use
// for itself, and finds ranks, and pages of a rank, by counting bits.  One launch / three, us, both in
// a graph of calls alone: 256 pages in 200 places 5.7 / 6.9, 1000 in 960 6.8 / 8.7, 4096 in 5120 7.0 / 9.5
// and in 65536 7.0 / 9.3 (eager 7.4 / 12.4 throughout); 4096 in 2^20, where the search in bits costs more
// than launches, 20.8 / 11.0, and 8192 in 65536 10.8 / 10.
constexpr int kMaskWords = 64, kMaskPages = 64 * kMaskWords, kFewEntries = 1 << 16;

struct PageBits {
    uint64_t word[kMaskWords];
    int before[kMaskWords + 1];  // pages in use before a word's

    __device__ __forceinline__ void make(const int32_t* refs, int n_pages) {
        const int lane = threadIdx.x & 63, wave = wave_id();
        constexpr int kWords = kMaskWords / (kThreads / 64);  // a wave's
        int r[kWords];
#pragma unroll
        for (int k = 0; k < kWords; k++) {
            const int p = (wave * kWords + k) * 64 + lane;
            r[k] = p < n_pages ? refs[p] : 0;
        }
#pragma unroll
        for (int k = 0; k < kWords; k++) {
            const uint64_t used = __ballot(r[k] > 0);
            if (lane == 0) word[wave * kWords + k] = used;
        }
        __syncthreads();
        if (wave == 0) {
            const int own = __popcll(word[lane]);
            int up_to = own;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int o = __shfl_up(up_to, d, 64);
                if (lane >= d) up_to += o;
            }
            before[lane] = up_to - own;
            if (lane == 63) before[64] = up_to;
        }
        __syncthreads();
    }
    __device__ __forceinline__ int in_use() const { return before[kMaskWords]; }
    __device__ __forceinline__ bool used(int p) const { return word[p >> 6] >> (p & 63) & 1; }
    // pages in use below p, which may be the count of pages
    __device__ __forceinline__ int below(int p) const {
        return before[p >> 6] + ((p & 63) ? __popcll(word[p >> 6] << (64 - (p & 63))) : 0);
    }
    // the page of a rank among those in use, or among the free ones
    template <bool USED>
    __device__ __forceinline__ int page_of(int rank) const {
        auto ahead = [&](int w) { return USED ? before[w] : 64 * w - before[w]; };
        int lo = 0, hi = kMaskWords;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (ahead(mid) <= rank) lo = mid;
            else hi = mid;
        }
        uint64_t bits = USED ? word[lo] : ~word[lo];
        int left = rank - ahead(lo), at = 0;
#pragma unroll
        for (int half = 32; half; half /= 2) {
            const int n = __popcll(bits & ((1ull << half) - 1));
            if (left >= n) left -= n, at += half, bits >>= half;
        }
        return 64 * lo + at;
    }
};

__global__ __launch_bounds__(kThreads) void compact_few_kernel(CompactJob j) {
    __shared__ PageBits bits;
    const int n_pages = (int)j.n_pages;
    bits.make(j.refs, n_pages);
    const int n_live = bits.in_use(), below = bits.below(n_live), moves = n_live - below;
    if (blockIdx.x == 0 && threadIdx.x == 0) j.info[0] = moves, j.info[1] = n_live;
    auto moved = [&](int32_t p) {
        if (!is_page(p, n_pages)) return -1;
        return p >= n_live && bits.used(p) ? bits.page_of<false>(bits.below(p) - below) : p;
    };
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i < n_pages) {
        const int p = (int)i;
        if (p < n_pages / 2) {
            const bool is = p < moves;
            j.copies[3 * i] = is ? bits.page_of<true>(below + p) : -1;
            j.copies[3 * i + 1] = is ? bits.page_of<false>(p) : -1;
            j.copies[3 * i + 2] = is ? j.page_size : -1;
        }
        if (p >= n_live) j.new_refs[p] = 0;
        else j.new_refs[p] = j.refs[bits.used(p) ? p : bits.page_of<true>(below + p - bits.below(p))];
    }
    if (i < j.n_entries) j.new_pages[i] = moved(j.pages[i]);
    if (i < j.n_prefix) j.new_prefix_pages[i] = moved(j.prefix_pages[i]);
}

// ------------------------------------------------ copies

struct CopyJob : PagesCopy {
    int elem;
    int row_chunks;  // of 16 bytes, of a head's row
    int units;       // of a copy: layers x 2
    int share;       // XCDs to a unit, where units are few
    int pieces;      // workgroups to a unit
};

// (as the runtime's uint4 the four would be put in LDS, by numbers from the dispatch packet,
// which is host memory: 13 us)
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
constexpr int kPiece = 4 * kThreads;  // chunks to a workgroup, in flight at once

// A workgroup takes up to 16 KB of a copy's keys or values of a layer.  Pages lie anywhere, and
// address translation is what a short list of copies waits for: workgroups go to the 8 XCDs
// in turn, and a layer's keys (or values) stay on one of them, or on some where layers are few
// (240 pages of 256 KB on one layer, with the lists: 55 us against 137).
__global__ __launch_bounds__(kThreads) void copy_kernel(CopyJob j) {
    const int tid = threadIdx.x;
    const int64_t n = j.count ? min(max((int64_t)*j.count, (int64_t)0), j.max_copies) : j.max_copies;
    const vtq_kv_cache& c = j.cache;
    const int xcd = (int)(blockIdx.x & 7), of = j.share > 1 ? xcd / j.units : 0;
    const int unit = j.share > 1 ? xcd % j.units : (int)blockIdx.x;
    if (unit >= j.units || of >= j.share) return;
    for (int64_t copy = blockIdx.z; copy < n; copy += gridDim.z) {
        const int32_t from = j.copies[3 * copy], to = j.copies[3 * copy + 1];
        const int slots = min(max(j.copies[3 * copy + 2], 0), c.page_size);
        if (!is_page(from, (int64_t)c.n_pages) || !is_page(to, (int64_t)c.n_pages)) continue;
        const bool is_v = unit & 1;
        const int64_t layer = unit / 2;
        char* base = static_cast<char*>(is_v ? c.v : c.k) + layer * j.layer_stride * j.elem;
        const char* src = base + from * (int64_t)c.page_stride * j.elem;
        char* dst = base + to * (int64_t)c.page_stride * j.elem;
        const uint32_t of_head = (uint32_t)slots * j.row_chunks, chunks = of_head * c.kv_heads;  // below 2^31
        for (int piece = (int)blockIdx.y * j.share + of; piece < j.pieces; piece += (int)gridDim.y * j.share) {
            const uint32_t first = (uint32_t)piece * kPiece + tid;
            if ((uint32_t)piece * kPiece < chunks) {
                // (past the end the last chunk again, which is not stored: every load stands alone)
                v4u x[4];
                int64_t where[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t chunk = min(first + k * kThreads, chunks - 1);
                    const uint32_t head = chunk / of_head, rest = chunk - head * of_head;
                    const uint32_t slot = rest / (uint32_t)j.row_chunks;
                    where[k] = (head * (int64_t)c.head_stride + slot * (int64_t)c.slot_stride) * j.elem +
                               (rest - slot * j.row_chunks) * 16;
                    x[k] = *reinterpret_cast<const v4u*>(src + where[k]);
                }
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (first + k * kThreads < chunks) *reinterpret_cast<v4u*>(dst + where[k]) = x[k];
            }
            if (piece == 0 && j.scales.k) {
                uint8_t* scale = (is_v ? j.scales.v : j.scales.k) + layer * j.scale_layer_stride;
                const int blocks = (slots + j.scales.block - 1) / j.scales.block;
                for (int k = tid; k < blocks * c.kv_heads; k += kThreads) {
                    uint8_t* s = scale + (k / blocks) * j.scales.head_stride + k % blocks;
                    s[to * j.scales.page_stride] = s[from * j.scales.page_stride];
                }
            }
        }
    }
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Hands out parts of a workspace; from null it measures them.
struct Parts {
    char* base;
    size_t used = 0;
    template <class T>
    void take(T*& p, int64_t n) {
        p = reinterpret_cast<T*>(base + used);
        used += up256((size_t)n * sizeof(T));
    }
};

size_t reorder_parts(ReorderJob& j, int64_t n_pages, int64_t batch_out, void* ws) {
    Parts p{static_cast<char*>(ws)};
    j.segments = (int)((n_pages + kSegment - 1) / kSegment);
    p.take(j.begin, batch_out);
    p.take(j.fresh, batch_out);
    p.take(j.to_copy, batch_out);
    p.take(j.free_in, j.segments);
    p.take(j.fresh_before, batch_out > kOwnScan ? batch_out + 1 : 0);
    p.take(j.copies_before, batch_out > kOwnScan ? batch_out + 1 : 0);
    return p.used;
}

size_t compact_parts(CompactJob& j, int64_t n_pages, void* ws) {
    Parts p{static_cast<char*>(ws)};
    j.segments = (int)((n_pages + kSegment - 1) / kSegment);
    p.take(j.live_in, j.segments);
    p.take(j.low, n_pages / 2);
    p.take(j.high, n_pages / 2);
    p.take(j.rank, n_pages);
    return p.used;
}

unsigned groups_of(int64_t n) { return (unsigned)((n + kThreads - 1) / kThreads); }

}  // namespace

size_t pages_reorder_workspace(int64_t n_pages, int64_t batch_out) {
    ReorderJob j{};
    return reorder_parts(j, n_pages, batch_out, nullptr);
}

size_t pages_compact_workspace(int64_t n_pages) {
    CompactJob j{};
    return compact_parts(j, n_pages, nullptr);
}

hipError_t launch_pages_reorder(const PagesReorder& a, hipStream_t stream) {
    ReorderJob j{};
    static_cast<PagesReorder&>(j) = a;
    reorder_parts(j, a.n_pages, a.batch_out, a.ws);
    if (j.segments + a.batch_out)
        hipLaunchKernelGGL(reorder_share_kernel, dim3((unsigned)(j.segments + a.batch_out)), dim3(kThreads), 0, stream, j);
    const dim3 grid((unsigned)(j.segments + a.batch + 1));
    if (a.batch_out > kOwnScan) {
        hipLaunchKernelGGL(reorder_scan_kernel, dim3(1), dim3(1024), 0, stream, j);
        hipLaunchKernelGGL((reorder_apply_kernel<false>), grid, dim3(kThreads), 0, stream, j);
    } else {
        hipLaunchKernelGGL((reorder_apply_kernel<true>), grid, dim3(kThreads), 0, stream, j);
    }
    return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesCompact& a, hipStream_t stream) {
    CompactJob j{};
    static_cast<PagesCompact&>(j) = a;
    const int64_t listed = std::max(a.n_entries, a.n_prefix);
    if (a.n_pages <= kMaskPages && listed <= kFewEntries) {
        const int64_t most = std::max({a.n_pages, listed, (int64_t)1});
        hipLaunchKernelGGL(compact_few_kernel, dim3(groups_of(most)), dim3(kThreads), 0, stream, j);
        return hipGetLastError();
    }
    compact_parts(j, a.n_pages, a.ws);
    if (j.segments)
        hipLaunchKernelGGL(compact_count_kernel, dim3((unsigned)j.segments), dim3(kThreads), 0, stream, j);
    // (a workgroup at least: it tells the counts)
    hipLaunchKernelGGL(compact_rank_kernel, dim3((unsigned)std::max(j.segments, 1)), dim3(kThreads), 0, stream, j);
    const int64_t most = std::max({a.n_pages / 2, a.n_entries, a.n_prefix});
    hipLaunchKernelGGL(compact_apply_kernel, dim3(groups_of(most)), dim3(kThreads), 0, stream, j);
    return hipGetLastError();
}

hipError_t launch_pages_copy(const PagesCopy& a, hipStream_t stream) {
    CopyJob j{};
    static_cast<PagesCopy&>(j) = a;
    j.elem = a.cache.type == VTQ_TYPE_E4M3 ? 1 : (int)type_bytes(a.cache.type);
    j.row_chunks = a.cache.head_dim * j.elem / 16;
    j.units = a.layers * 2;
    j.pieces = (int)(((int64_t)a.cache.kv_heads * a.cache.page_size * j.row_chunks + kPiece - 1) / kPiece);
    j.share = j.units <= 4 ? 8 / j.units : 1;
    // units (in eights: XCDs in turn), pieces, copies; the last two in strides where there are many
    const unsigned x = (unsigned)(j.units + 7) / 8 * 8;
    const unsigned y = (unsigned)std::min<int64_t>((j.pieces + j.share - 1) / j.share, std::max<int64_t>(1, 65536 / x));
    const unsigned z = (unsigned)std::min<int64_t>(a.max_copies, std::max<int64_t>(1, 131072 / ((int64_t)x * y)));
    hipLaunchKernelGGL(copy_kernel, dim3(x, y, std::min(z, 65535u)), dim3(kThreads), 0, stream, j);
    return hipGetLastError();
}

}  // namespace vtq
