// vtq_attention_plan.h -- how an attention call's work is split: rules on sizes, host
// code without a kernel, so that tests can ask them (libvtq_probe.so).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "../../include/vtq.h"
#include "vtq_serve_checks.h"

namespace vtq {

struct AttentionPlan {
    int group;        // query heads of a KV head
    int page_shift;
    int prefix_rows;  // row tiles of the prefix
    int prefix_splits, prefix_chunk;  // key ranges, and keys to one (a multiple of 32; of 128 where waves share rows)
    int own_rows, own_splits;         // row tiles of a sequence (a workgroup may take several), key ranges
    int own_grain;                    // which are multiples of this: 32, or 128 where waves share rows
    int shared_prefix, shared_own;    // whether the waves share tiles (else they share rows)
    int prefix_per_xcd, own_per_xcd;  // workgroups
};

// Parts that the join takes of a row: two a lane.
constexpr int kMostParts = 128;

// Keys to each of a sequence's own ranges.
__host__ __device__ inline int own_chunk(int keys, int splits, int grain) {
    return ((keys + splits - 1) / splits + grain - 1) & -grain;
}

inline int attention_waves(int cache_type, int head_dim) {
    const int d = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    return 32 * d * (int)type_bytes(cache_type) > 16384 ? 2 : 4;
}

// What the split asks of a kernel.
struct TileCost {
    int waves;     // of a workgroup
    bool f32;      // products in f32
    bool slow;     // tiles that take long: parts of less than four
    double tile;   // 32 keys against 32 rows, us
};

inline TileCost attention_cost(int type, int cache_type, int head_dim) {
    const int d = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    return {attention_waves(cache_type, head_dim), type == VTQ_TYPE_F32, type == VTQ_TYPE_F32 || d > 128,
            type == VTQ_TYPE_F32 ? 3.6 * d / 128 : d > 128 ? 2.4 : 0.18 + 0.0025 * d};
}

// A part of the rows on its way through memory and the join, us.
inline double part_cost(int64_t tokens, int heads, int head_dim) {
    return 0.08 + 2.3e-6 * (double)(tokens * heads * head_dim);
}

// The arguments are what the checks let through: tokens, heads and batch above 0.
inline AttentionPlan plan_attention(const vtq_kv_cache& cache, const vtq_kv_batch& batch, const TileCost& cost,
                                    int64_t tokens, int heads) {
    AttentionPlan p{};
    const int W = cost.waves;
    auto up = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    const int64_t slots = 512;
    p.group = heads / cache.kv_heads;
    p.page_shift = __builtin_ctz((unsigned)cache.page_size);
    const int64_t prefix_rows = tokens * p.group;
    const int64_t own_rows = std::min<int64_t>(std::max(1, batch.max_q), tokens) * p.group;
    p.shared_prefix = prefix_rows > 32;
    p.shared_own = own_rows > 32;
    p.prefix_rows = p.prefix_splits = 0;
    p.prefix_chunk = 128;
    const int64_t most = (int64_t)batch.max_pages << p.page_shift;
    const int64_t len = batch.max_len ? std::min<int64_t>(batch.max_len, most) : most;
    p.own_rows = (int)up(own_rows, p.shared_own ? 32 * W : 32);
    const int64_t own_units = (int64_t)cache.kv_heads * p.own_rows * batch.batch;
    const bool slow = cost.slow;
    const int grain = slow ? 32 : 128;
    p.own_grain = p.shared_own ? grain : 128;
    auto least_keys = [&](int64_t keys) {
        const double part = part_cost(tokens, heads, cache.head_dim);
        return (1 + (int64_t)std::sqrt(32.0 * keys * part / cost.tile) / grain) * grain;
    };
    if (batch.prefix_len) {
        p.prefix_rows = (int)up(prefix_rows, p.shared_prefix ? 32 * W : 32);
        const int64_t units = (int64_t)cache.kv_heads * p.prefix_rows;
        // A workgroup a CU beside the own ones, two where those have little to do, and keys
        // enough to each: n keys take n / 32 tiles one after the other, and each part costs
        // its rows' way through memory and the join, so n = sqrt(32 keys part / tile) (us); of
        // f32 256 at least where fewer would make more than a workgroup a CU.  Where the waves
        // share rows a part is near free: n lets 192 workgroups have all.  Against 512 keys
        // (768 beside own work, 256 or 128 of f32 and 256 elements; 128 for shared rows), 8 KV
        // heads of 128, us: 12 x 1003 22.1 / 16.1, 64 x 8192 29.7 / 28, 2 x 60 tokens x 8192
        // 50 / 42, 1 x 8192 23.7 / 15.9, f32 43.4 / 28.8; over 654 shapes 3 % less in the mean.
        // Multiples of 32 keys, not 128, where a tile takes long: 8 % less again (f32 20 x 1721
        // on 2 KV heads 54 / 25; the worst 16 x 6 x 30000 of 256 elements, 203 / 235, 516
        // workgroups for 256 CUs).
        const int64_t own_keys = own_units * len, prefix_keys = units * batch.prefix_len;
        const bool alone = own_keys * 4 < prefix_keys;
        int64_t least;
        if (p.shared_prefix) {
            least = least_keys(batch.prefix_len);
            if (cost.f32 && units * up(batch.prefix_len, least) + own_units > slots / 2)
                least = std::max<int64_t>(least, 256);
        } else {
            least = std::min<int64_t>(512, up(prefix_keys, 192 * 128) * 128);
        }
        const int64_t splits =
            std::min<int64_t>({up(alone ? slots : slots / 2, units), up(batch.prefix_len, least), 64});
        const int64_t by = p.shared_prefix ? grain : 128;
        p.prefix_chunk = (int)(up(up(batch.prefix_len, splits), by) * by);
        p.prefix_splits = (int)up(batch.prefix_len, p.prefix_chunk);
    }
    // As many parts as run at once beside the prefix: one workgroup more than the chip holds
    // costs a round (8 KV heads of 128, rounded up / down, us: 48 sequences of 600 keys 28.3 /
    // 21.6, 24 of 5 x 600 behind 8192 42.9 / 36.7, 8 of 4000 behind 8192 36.1 / 33.9; the worst
    // of 80 shapes 40 of 600 behind 8192, 32.7 / 34.2).
    const int64_t beside = slots - (int64_t)cache.kv_heads * p.prefix_splits * p.prefix_rows;
    p.own_splits = (int)std::max<int64_t>(1, std::min<int64_t>({beside / own_units, up(len, p.shared_own && slow ? least_keys(len) : 128), 64}));
    p.prefix_per_xcd = (int)up((int64_t)cache.kv_heads * p.prefix_splits, 8) * p.prefix_rows;
    p.own_per_xcd = (int)(up((int64_t)cache.kv_heads * p.own_splits * batch.batch, 8) * p.own_rows);
    return p;
}

inline AttentionPlan plan_attention(const vtq_kv_cache& cache, const vtq_kv_batch& batch, int type, int64_t tokens,
                                    int heads) {
    return plan_attention(cache, batch, attention_cost(type, cache.type, cache.head_dim), tokens, heads);
}

// Over 8-bit caches: products of one, two or three 16-bit parts; heads of more than 128
// elements in two parts, each a workgroup's, so twice as many of both.
inline TileCost kv8_attention_cost(int type, int head_dim) {
    const int d = head_dim <= 64 ? 64 : 128;
    const int parts = type == VTQ_TYPE_F32 ? 3 : type == VTQ_TYPE_F16 ? 2 : 1;
    return {4, false, head_dim > 128, (0.18 + 0.0025 * d) * (1 + parts) / 2};
}
// Units of keys (KV heads, ranges, sequences) go to the 8 XCDs in turn, each with its row tiles; the
// last ones, fewer than 8, to as many XCDs each as leave the fewest without work (one prompt of 2048,
// 32 heads on 4 of 64: 43 us against 59).
__host__ __device__ inline int xcds_of(int last_units) { return last_units ? 8 / last_units : 1; }
inline int per_xcd(int64_t units, int rows) {
    const int last = (int)(units % 8), share = xcds_of(last);
    return (int)(units / 8 * rows + (last ? (rows + share - 1) / share : 0));
}
// Whether the sequences' own workgroups take the prefix too: their rows then leave once, not as two parts
// in f32 to be joined, but each walks all of the prefix, which rows of all sequences packed would in
// fewer, and fuller, workgroups.  `with` and `without` are the plans with prefix workgroups and of the
// own keys alone; the estimate, in us, is what walks the most keys or, above a workgroup a CU, all
// walks, and what a part of the rows costs (plan_attention's least_keys).  Measured inside / outside (bf16,
// 32 heads on 8 of 128): 12 prompts of up to 218 behind 161 keys, of 96, 41 / 70; 64 drafts of 9
// behind 300 31 / 41, behind 1000 55 / 48 and taken outside; one of 60 behind 1000 35 / 19 and behind 4096
// 96 / 24, outside.  Beyond 4096 keys the parts are the least of it (40 x 100, 64 heads, 8000:
// 1324 / 1230).
inline bool kv8_prefix_inside(const vtq_kv_cache& part, const vtq_kv_batch& batch, const TileCost& cost, int64_t tokens,
                              int heads, bool joined, const AttentionPlan& without, const AttentionPlan& with) {
    if (!batch.prefix_len || !without.shared_own || without.own_splits != 1) return false;
    // Rows that are joined anyway (heads of more than 128 elements) save workgroups only: 10 and 62 prompts
    // of 64, f16, 8 heads on 4 of 256, behind 64 keys 23.3 / 22.7 and 84 / 76, behind 200 31 / 27 and 115 / 91.
    if (batch.prefix_len > (joined ? 64 : 4096)) return false;
    const double rows = (double)tokens * without.group, tiles = (double)without.own_rows * batch.batch;
    // One long sequence among short ones: most of the others' tiles have no rows, and the rest few (63
    // tokens of 900 keys beside a chunk of 512 behind 300 204 / 172, behind 1000 287 / 181).
    if (128 * tiles > 5 * rows) return false;
    const double packed = std::ceil(rows / 128), filled = std::min(tiles, rows / 128 + batch.batch);
    const int64_t most = (int64_t)batch.max_pages << without.page_shift;
    const double own = (batch.max_len ? std::min<int64_t>(batch.max_len, most) : most) / 32.0;
    const double prefix = batch.prefix_len / 32.0, range = std::min(prefix, with.prefix_chunk / 32.0);
    // a lone workgroup takes longer to a tile than one of several on a CU do
    auto walk = [&](double longest, double all) { return cost.tile * std::max(1.28 * longest, all * part.kv_heads / 256); };
    const double in = walk(prefix + own, filled * (prefix + own)) + 3;  // (the second page list's latency)
    const double out = walk(std::max(range, own), packed * prefix + filled * own) + 2 +
                       (with.prefix_splits + with.own_splits) * part_cost(tokens, heads, part.head_dim);
    return in <= out;
}
inline AttentionPlan plan_kv8_attention(const vtq_kv_cache& cache, const vtq_kv_batch& batch, int type, int64_t tokens,
                                        int heads, bool* inside = nullptr) {
    const int parts = cache.head_dim > 128 ? 2 : 1;
    vtq_kv_cache part = cache;
    part.kv_heads *= parts;
    part.head_dim = cache.head_dim / parts;
    vtq_kv_batch own = batch;
    own.prefix_len = 0;
    const TileCost cost = kv8_attention_cost(type, cache.head_dim);
    AttentionPlan p = plan_attention(part, batch, cost, tokens, heads * parts);
    const AttentionPlan without = plan_attention(part, own, cost, tokens, heads * parts);
    const bool in = kv8_prefix_inside(part, batch, cost, tokens, heads * parts, parts > 1, without, p);
    if (in) p = without;
    if (inside) *inside = in;
    // y may be q: no part writes rows that the other still reads, so they are joined even if alone
    if (parts > 1 && p.prefix_splits + p.own_splits == 1) p.own_splits = 2;
    // a part's workgroups follow the other's on its XCD, where its L2 has the keys
    p.prefix_per_xcd = per_xcd((int64_t)cache.kv_heads * p.prefix_splits, p.prefix_rows * parts);
    p.own_per_xcd = per_xcd((int64_t)cache.kv_heads * p.own_splits * batch.batch, p.own_rows * parts);
    return p;
}

}  // namespace vtq
