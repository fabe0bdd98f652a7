// How a step of attention runs (attention.hpp), on the host alone.
#include <algorithm>

#include "serving.hpp"

namespace chm {

// Up to 128 rows a key head take workgroups of 16 or 32 rows whose waves split
// the tiles, more take eight (or four) waves of 32 rows each; then splits until
// each compute unit has a workgroup, of at least kLeast tiles, but one while
// the tiles are few: the launch that joins them would cost more.
AttentionPlan plan_attention(const CacheShape& cache, uint32_t query_heads, uint32_t tokens, uint32_t longest,
                             uint32_t window, uint32_t compute_units) {
    const uint64_t rows = uint64_t{tokens} * (query_heads / cache.kv_heads);
    AttentionPlan plan{};
    plan.octets = rows <= 16 ? 1 : 2;
    plan.waves = rows <= 128 ? 1 : cache.head_dim <= 128 ? 8 : 4;
    const uint64_t group = 16ull * plan.octets * plan.waves;
    plan.row_groups = static_cast<uint32_t>((rows + group - 1) / group);
    const uint64_t workgroups = uint64_t{cache.sequences} * cache.kv_heads * plan.row_groups;
    uint64_t reach = std::min(longest ? longest : cache.capacity, cache.capacity);
    if (window) reach = std::min<uint64_t>(reach, uint64_t{window} + tokens + 31);
    const uint64_t tiles = (reach + 31) / 32;
    const uint64_t wanted = compute_units / workgroups;
    constexpr uint64_t kLeast = 4, kOne = 16;
    plan.splits = static_cast<uint32_t>(
        tiles <= kOne ? 1 : std::max<uint64_t>(1, std::min(wanted, (tiles + kLeast - 1) / kLeast)));
    return plan;
}

uint64_t attention_partial_bytes(const CacheShape& cache, uint32_t query_heads, uint32_t tokens, uint32_t splits) {
    if (splits < 2) return 0;
    return uint64_t{cache.sequences} * query_heads * tokens * splits * (uint64_t{cache.head_dim} * 4 + 8);
}

// Steps of every number of tokens up to `tokens`: of those in one number of
// row groups the last needs most, and past the first that does not split none does.
uint64_t attention_workspace_bytes(const CacheShape& cache, uint32_t query_heads, uint32_t tokens, uint32_t compute_units) {
    uint64_t most = 0;
    const uint64_t group = query_heads / cache.kv_heads;
    for (uint32_t t = 1; t <= tokens; ++t) {
        AttentionPlan plan = plan_attention(cache, query_heads, t, 0, 0, compute_units);
        const uint64_t rows = 16ull * plan.octets * plan.waves * plan.row_groups;
        t = static_cast<uint32_t>(std::min<uint64_t>(tokens, std::max<uint64_t>(t, rows / group)));
        plan = plan_attention(cache, query_heads, t, 0, 0, compute_units);
        most = std::max(most, attention_partial_bytes(cache, query_heads, t, plan.splits));
        if (plan.waves > 1 && plan.splits < 2) break;
    }
    return most;
}

}  // namespace chm
