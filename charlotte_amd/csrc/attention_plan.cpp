// How a step of attention runs (attention.hpp), on the host alone.
#include <algorithm>

#include "formats.hpp"
#include "serving.hpp"

namespace chm {

namespace {

// Tiles a split takes at least: of wide binary16 heads two, but four once that
// makes more than 64 splits (126 tiles of one head: 12.9 us in 63, 14.5 in 32; 501
// tiles: 23.3 in 250, 19.3 in 126).
uint64_t least_tiles(const CacheShape& cache, uint64_t tiles) {
    return cache.format == kF16 && cache.head_dim > 128 && tiles <= 128 ? 2 : 4;
}

// Waves of 32 rows a workgroup of attend_rows holds.
uint32_t row_waves(uint32_t head_dim) { return head_dim <= 128 ? 8 : 4; }

uint64_t groups_of(uint64_t rows, uint64_t group) { return (rows + group - 1) / group; }

// A workgroup for each compute unit, while each split has least_tiles.
uint64_t splits_of(const CacheShape& cache, uint64_t row_groups, uint64_t tiles, uint32_t compute_units) {
    const uint64_t wanted = compute_units / (uint64_t{cache.sequences} * cache.kv_heads * row_groups);
    return std::max<uint64_t>(1, std::min(wanted, groups_of(tiles, least_tiles(cache, tiles))));
}

}  // namespace

// `load`: the step's blocks of 16 or 32 rows by a tile, for each compute unit.
//
// Workgroups of 16 rows (attend) have the shorter chain of products, and read
// the cache once for every 16 rows; they are taken while load16 <= 24 and none
// has to wait for another's compute unit. 8 key heads of 128, 20 rows over 8,000
// in Q8_0: 15.2 us, by 32 rows 16.8; in binary16 over 500 9.7 and 11.8, 48 rows
// over 8,000 (load16 = 24) 23.4 and 21.2; 128 rows of 8 sequences with none before
// (twice as many workgroups as compute units) 13.9 and 11.2. Quantized
// heads past 64, whose codes cost more to widen than to read, up to 64: 84 rows
// over 8,000 (48) 28.2 and 32.5, over 60,000 (352) 140 and 140 - 145.
//
// A tile's codes laid out once for 128 or 256 rows (attend_rows) pay where each
// compute unit has many products to feed: 1,024 rows of 8 key heads of 128 over
// 16,000 in Q8_0 (load32 = 531) 173 us, by 32 rows 325; over 1,400 (44) 39.3
// and 41.2; over 1,000 (32) 34.2 and 31.1. Heads of 64, over 8,000 (250) 60 and 69,
// 512 rows over 8,000 (125) 42 and 42. Heads of 256 hold 4 waves' rows, too
// few to pay for laying codes out (Q8_0, 1,024 over 8,000: 387 and 308), but in
// binary16 there is little to lay out: 184 and 408, 192 over 2,000 (11) 33 and 44,
// 1,024 over 300 (10) 34 and 29.
//
// Few tiles are not split: the launch that joins them costs 2.5 us. One token, 2
// rows of 8 heads, in one and in splits of four tiles: heads of 64, 19 tiles 8.3
// and 8.7 us, 26 tiles 9.5 and 8.7; of 128, 11 tiles 7.9 and 9.1, 15 tiles 9.4
// and 9.2; of 256, 8 tiles 13.8 and 13.4 (binary16 14.6 and 13.2, in splits of
// two tiles 11.3). 512 tokens with none before, attend_rows: 47.1 and 33.8.
AttentionPlan plan_attention(const CacheShape& cache, uint32_t query_heads, uint32_t tokens, uint32_t longest,
                             uint32_t window, uint32_t compute_units) {
    const uint64_t rows = uint64_t{tokens} * (query_heads / cache.kv_heads);
    uint64_t reach = std::min(longest ? longest : cache.capacity, cache.capacity);
    if (window) reach = std::min<uint64_t>(reach, uint64_t{window} + tokens + 31);
    const uint64_t tiles = groups_of(reach, 32), heads = uint64_t{cache.sequences} * cache.kv_heads;

    const bool quantized = cache.format != kF16;
    const uint64_t most16 = quantized && cache.head_dim > 64 ? 64 : 24;
    const uint64_t load16 = groups_of(rows, 16) * heads * tiles, load32 = groups_of(rows, 32) * heads * tiles;
    const uint32_t waves = row_waves(cache.head_dim);
    const uint64_t least32 = cache.head_dim <= 64 ? 112 : cache.head_dim <= 128 ? 44 : quantized ? UINT64_MAX : 11;
    AttentionPlan plan{1, 1, 0, 0};
    if (rows > 16 * waves && load32 / compute_units >= least32)
        plan.octets = 2, plan.waves = waves;
    else if (rows > 16 && (load16 > most16 * compute_units || groups_of(rows, 16) * heads > compute_units))
        plan.octets = 2;
    plan.row_groups = static_cast<uint32_t>(groups_of(rows, 16ull * plan.octets * plan.waves));
    const uint64_t one = plan.waves > 1 || cache.head_dim > 128 ? least_tiles(cache, tiles) : cache.head_dim > 64 ? 12 : 24;
    plan.splits = tiles <= one ? 1 : static_cast<uint32_t>(splits_of(cache, plan.row_groups, tiles, compute_units));
    return plan;
}

uint64_t attention_partial_bytes(const CacheShape& cache, uint32_t query_heads, uint32_t tokens, uint32_t splits) {
    if (splits < 2) return 0;
    return uint64_t{cache.sequences} * query_heads * tokens * splits * (uint64_t{cache.head_dim} * 4 + 8);
}

// Over every number of tokens up to `tokens` and every `longest`: most splits
// come of the fewest workgroups and of all the tiles, or the 128 that are still
// split by two; of the tokens that make as many groups the last needs most.
uint64_t attention_workspace_bytes(const CacheShape& cache, uint32_t query_heads, uint32_t tokens, uint32_t compute_units) {
    const uint64_t tiles = groups_of(cache.capacity, 32), shared = query_heads / cache.kv_heads;
    const uint32_t waves = row_waves(cache.head_dim);
    uint64_t most = 0;
    for (uint64_t t = 1; t <= tokens; ++t) {
        const uint64_t rows = t * shared, group = rows <= 16 ? 16 : rows <= 16 * waves ? 32 : 32 * waves;
        const uint64_t row_groups = groups_of(rows, group);
        const uint64_t last = std::min<uint64_t>(row_groups * group, rows <= 16 * waves ? 16 * waves : UINT64_MAX);
        t = std::max(t, std::min<uint64_t>(tokens, last / shared));
        const uint64_t splits = std::max(splits_of(cache, row_groups, tiles, compute_units),
                                         splits_of(cache, row_groups, std::min<uint64_t>(tiles, 128), compute_units));
        most = std::max(most, attention_partial_bytes(cache, query_heads, static_cast<uint32_t>(t),
                                                      static_cast<uint32_t>(splits)));
        if (group == 32 * waves && splits < 2) break;
    }
    return most;
}

}  // namespace chm
