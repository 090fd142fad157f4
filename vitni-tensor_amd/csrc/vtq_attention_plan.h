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

// The arguments are what the checks let through: tokens, heads and batch above 0.
inline AttentionPlan plan_attention(const vtq_kv_cache& cache, const vtq_kv_batch& batch, int type, int64_t tokens,
                                    int heads) {
    AttentionPlan p{};
    const int W = attention_waves(cache.type, cache.head_dim);
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
    const int d = cache.head_dim <= 64 ? 64 : cache.head_dim <= 128 ? 128 : 256;
    const bool slow = type == VTQ_TYPE_F32 || d > 128;  // tiles that take long: parts of less than four
    const int grain = slow ? 32 : 128;
    p.own_grain = p.shared_own ? grain : 128;
    auto least_keys = [&](int64_t keys) {
        const double tile = type == VTQ_TYPE_F32 ? 3.6 * d / 128 : d > 128 ? 2.4 : 0.18 + 0.0025 * d;
        const double part = 0.08 + 2.3e-6 * (double)(tokens * heads * cache.head_dim);
        return (1 + (int64_t)std::sqrt(32.0 * keys * part / tile) / grain) * grain;
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
            if (type == VTQ_TYPE_F32 && units * up(batch.prefix_len, least) + own_units > slots / 2)
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

}  // namespace vtq
