// cache_pages.hip -- who holds a cache's pages: the next batch's page tables from the
// sequences that it goes on with, the pages in use closed up, and copies of pages (gfx950).
//
// The lists are small (a table of 256 x 256 pages is 256 KB) and each step needs the
// one before, so time is launches and latency: a few kernels over all pages at once, with
// counts of 4096 pages, a scan of the counts by one workgroup, and ranks from both.
// Free pages are taken lowest first and in the order of sequences, and counts change by
// atomic additions of whole numbers, whose order changes nothing: the same lists every time.
#include <algorithm>

#include "vtq_device.h"
#include "vtq_serve.h"

namespace vtq {
namespace {

constexpr int kSegment = 4096;  // pages to a workgroup
constexpr int kThreads = 256;

struct ReorderJob : PagesReorder {
    int segments;
    int32_t *begin, *fresh, *to_copy;     // [batch_out]: first place of free pages, how many, whether a page is copied
    int64_t* fresh_before;                // [batch_out + 1]
    int32_t* copies_before;               // [batch_out]
    int32_t* free_in;                     // [segments]
    int64_t* free_before;                 // [segments + 1]
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

// before[i] = sum of values below i, for i up to n, by one workgroup of 1024.
template <class T, class S>
__device__ __forceinline__ S scan(const T* values, int64_t n, S* before, bool total_too) {
    __shared__ S waves[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    S carry = 0;
    for (int64_t i0 = 0; i0 < n; i0 += 1024) {
        const S own = i0 + tid < n ? (S)values[i0 + tid] : (S)0;
        S up_to = own;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const S o = __shfl_up(up_to, d, 64);
            if (lane >= d) up_to += o;
        }
        if (lane == 63) waves[wave] = up_to;
        __syncthreads();
        S ahead = carry, all = carry;
        for (int w = 0; w < 16; w++) {
            if (w < wave) ahead += waves[w];
            all += waves[w];
        }
        if (i0 + tid < n) before[i0 + tid] = ahead + up_to - own;
        carry = all;
        __syncthreads();
    }
    if (total_too && tid == 0) before[n] = carry;
    return carry;
}

__global__ __launch_bounds__(1024) void reorder_scan_kernel(ReorderJob j) {
    const int64_t free = scan(j.free_in, j.segments, j.free_before, true);
    const int64_t fresh = scan(j.fresh, j.batch_out, j.fresh_before, true);
    __syncthreads();
    // a sequence's copy has a page while pages last, from the first sequence on
    for (int i = threadIdx.x; i < j.batch_out; i += 1024)
        if (j.to_copy[i] && j.fresh_before[i] >= free) j.to_copy[i] = 0;
    __syncthreads();
    const int copies = scan(j.to_copy, j.batch_out, j.copies_before, false);
    // places beyond max_pages
    int64_t beyond = 0;
    for (int i = threadIdx.x; i < j.batch_out; i += 1024)
        if (j.grow) beyond += max(pages_of((int64_t)j.new_len[i] + max(j.grow[i], 0), j.page_size) - j.max_pages, 0);
    __shared__ int64_t part[16];
#pragma unroll
    for (int d = 1; d < 64; d *= 2) beyond += __shfl_xor(beyond, d, 64);
    if ((threadIdx.x & 63) == 0) part[wave_id()] = beyond;
    __syncthreads();
    if (threadIdx.x == 0) {
        int64_t missing = max(fresh - free, (int64_t)0);
        for (int w = 0; w < 16; w++) missing += part[w];
        j.info[0] = copies;
        j.info[1] = (int32_t)min(missing, (int64_t)INT32_MAX);
    }
}

// Workgroups below `segments` hand out their free pages, the others (one to an old sequence)
// take its pages' holders off and its children on.
__global__ __launch_bounds__(kThreads) void reorder_apply_kernel(ReorderJob j) {
    const int tid = threadIdx.x, lane = tid & 63;
    if ((int64_t)blockIdx.x >= j.segments) {
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
    const int64_t total = j.fresh_before[j.batch_out];
    int64_t rank = j.free_before[blockIdx.x];
    if (rank >= total) return;
    __shared__ int waves[kThreads / 64];
    for (int k0 = 0; k0 < kSegment; k0 += kThreads) {
        const int64_t page = (int64_t)blockIdx.x * kSegment + k0 + tid;
        const bool free = page < j.n_pages && j.refs[page] == 0;
        const uint64_t mask = __ballot(free);
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
                if (j.fresh_before[mid] <= mine) lo = mid;
                else hi = mid;
            }
            const int at = (int)(mine - j.fresh_before[lo]);
            j.new_pages[(int64_t)lo * j.max_pages + j.begin[lo] + at] = (int32_t)page;
            atomicAdd(&j.new_refs[page], 1);
            if (at == 0 && j.to_copy[lo]) {
                const int parent = j.parent[lo], len = j.new_len[lo];
                int32_t* c = j.copies + 3 * (int64_t)j.copies_before[lo];
                c[0] = j.pages[(int64_t)parent * j.max_pages + len / j.page_size];
                c[1] = (int32_t)page;
                c[2] = len % j.page_size;
            }
        }
        if (rank >= total) return;
    }
}

// ------------------------------------------------ pages closed up

struct CompactJob : PagesCompact {
    int segments;
    int32_t* live_in;      // [segments]
    int64_t* live_before;  // [segments + 1]
    int32_t *low, *high;   // [n_pages / 2]: free pages below the count of those in use, and pages in use past it
    int32_t* rank;         // [n_pages]: of a page among the latter
};

__global__ __launch_bounds__(kThreads) void compact_count_kernel(CompactJob j) {
    count_segment(j.refs, nullptr, j.n_pages, (int)blockIdx.x, j.live_in);
}

__global__ __launch_bounds__(1024) void compact_scan_kernel(CompactJob j) {
    const int64_t live = scan(j.live_in, j.segments, j.live_before, true);
    if (threadIdx.x == 0) j.info[0] = 0, j.info[1] = (int32_t)live;
}

__global__ __launch_bounds__(kThreads) void compact_rank_kernel(CompactJob j) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t n_live = j.live_before[j.segments];
    // pages in use below n_live: those of whole segments, and of the one that it lies in
    const int64_t edge = n_live / kSegment;
    __shared__ int waves[kThreads / 64];
    int64_t below = 0;
    if ((int64_t)blockIdx.x >= edge) {
        int mine = 0;
        for (int64_t p = edge * kSegment + tid; p < n_live; p += kThreads) mine += j.refs[p] > 0;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) mine += __shfl_xor(mine, d, 64);
        if (lane == 0) waves[wave_id()] = mine;
        __syncthreads();
        below = j.live_before[edge] + waves[0] + waves[1] + waves[2] + waves[3];
        __syncthreads();
    }
    int64_t before = j.live_before[blockIdx.x];
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
    if ((int64_t)blockIdx.x == j.segments - 1 && tid == 0) {
        // the last segment knows how many are past n_live
        j.info[0] = n_live < j.n_pages ? (int32_t)(j.live_before[j.segments] - below) : 0;
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

// ------------------------------------------------ copies

struct CopyJob : PagesCopy {
    int elem;
    int row_chunks;   // 16 bytes of a head's row
    int64_t units;    // of a copy: layers x heads x 2
};

// A wave takes a copy's keys or values of one head and layer at a time.
__global__ __launch_bounds__(kThreads) void copy_kernel(CopyJob j) {
    const int lane = threadIdx.x & 63;
    const int64_t n = j.count ? min(max((int64_t)*j.count, (int64_t)0), j.max_copies) : j.max_copies;
    const vtq_kv_cache& c = j.cache;
    const int64_t waves = (int64_t)gridDim.x * (kThreads / 64);
    for (int64_t w = (int64_t)blockIdx.x * (kThreads / 64) + wave_id(); w < n * j.units; w += waves) {
        const int64_t copy = w / j.units;
        int unit = (int)(w % j.units);  // below 2^25
        const int32_t from = j.copies[3 * copy], to = j.copies[3 * copy + 1];
        const int slots = min(max(j.copies[3 * copy + 2], 0), c.page_size);
        if (!is_page(from, (int64_t)c.n_pages) || !is_page(to, (int64_t)c.n_pages)) continue;
        const bool is_v = unit & 1;
        unit /= 2;
        const int head = unit % c.kv_heads, layer = unit / c.kv_heads;
        char* base = static_cast<char*>(is_v ? c.v : c.k) +
                     (layer * j.layer_stride + head * (int64_t)c.head_stride) * j.elem;
        const char* src = base + from * (int64_t)c.page_stride * j.elem;
        char* dst = base + to * (int64_t)c.page_stride * j.elem;
        const int64_t slot = (int64_t)c.slot_stride * j.elem;
        const int chunks = slots * j.row_chunks;
        // four loads in flight
        for (int i0 = lane; i0 < chunks; i0 += 256) {
            uint4 x[4];
            int64_t at[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int i = i0 + 64 * k;
                at[k] = (i / j.row_chunks) * slot + (i % j.row_chunks) * 16;
                if (i < chunks) x[k] = *reinterpret_cast<const uint4*>(src + at[k]);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i0 + 64 * k < chunks) *reinterpret_cast<uint4*>(dst + at[k]) = x[k];
        }
        if (j.scales.k) {
            uint8_t* scale = (is_v ? j.scales.v : j.scales.k) + layer * j.scale_layer_stride + head * j.scales.head_stride;
            const int blocks = (slots + j.scales.block - 1) / j.scales.block;
            for (int i = lane; i < blocks; i += 64)
                scale[to * j.scales.page_stride + i] = scale[from * j.scales.page_stride + i];
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
    p.take(j.fresh_before, batch_out + 1);
    p.take(j.copies_before, batch_out);
    p.take(j.free_in, j.segments);
    p.take(j.free_before, j.segments + 1);
    return p.used;
}

size_t compact_parts(CompactJob& j, int64_t n_pages, void* ws) {
    Parts p{static_cast<char*>(ws)};
    j.segments = (int)((n_pages + kSegment - 1) / kSegment);
    p.take(j.live_in, j.segments);
    p.take(j.live_before, j.segments + 1);
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
    hipLaunchKernelGGL(reorder_scan_kernel, dim3(1), dim3(1024), 0, stream, j);
    if (j.segments + a.batch)
        hipLaunchKernelGGL(reorder_apply_kernel, dim3((unsigned)(j.segments + a.batch)), dim3(kThreads), 0, stream, j);
    return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesCompact& a, hipStream_t stream) {
    CompactJob j{};
    static_cast<PagesCompact&>(j) = a;
    compact_parts(j, a.n_pages, a.ws);
    if (j.segments)
        hipLaunchKernelGGL(compact_count_kernel, dim3((unsigned)j.segments), dim3(kThreads), 0, stream, j);
    hipLaunchKernelGGL(compact_scan_kernel, dim3(1), dim3(1024), 0, stream, j);
    if (j.segments) hipLaunchKernelGGL(compact_rank_kernel, dim3((unsigned)j.segments), dim3(kThreads), 0, stream, j);
    const int64_t most = std::max({a.n_pages / 2, a.n_entries, a.n_prefix});
    if (most) hipLaunchKernelGGL(compact_apply_kernel, dim3(groups_of(most)), dim3(kThreads), 0, stream, j);
    return hipGetLastError();
}

hipError_t launch_pages_copy(const PagesCopy& a, hipStream_t stream) {
    CopyJob j{};
    static_cast<PagesCopy&>(j) = a;
    j.elem = a.cache.type == VTQ_TYPE_E4M3 ? 1 : (int)type_bytes(a.cache.type);
    j.row_chunks = a.cache.head_dim * j.elem / 16;
    j.units = (int64_t)a.layers * a.cache.kv_heads * 2;
    const int64_t waves = a.max_copies * j.units;
    const int64_t groups = std::min<int64_t>((waves + 3) / 4, 256 * 16);
    hipLaunchKernelGGL(copy_kernel, dim3((unsigned)groups), dim3(kThreads), 0, stream, j);
    return hipGetLastError();
}

}  // namespace vtq
