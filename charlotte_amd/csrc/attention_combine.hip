// The splits of a step's attention joined (attention.hpp): a row's splits hold
// outputs and a sum relative to their own offsets, o_s and l_s; the row is
//   sum_s 2^(c - c_s) o_s / sum_s 2^(c - c_s) l_s,  c the least offset,
// added in split order. And the step's plan.
//
// A wave a row: head_dim / 4 lanes hold the row's values, and as many such
// groups as fit the wave take its splits in turn.
#include <algorithm>

#include "serving.hpp"

namespace chm {

template <uint32_t LANES>
__global__ __launch_bounds__(256) void attention_combine(Attention a) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t id = static_cast<uint64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    const uint64_t sequence_head = id / a.rows;
    const uint32_t row = static_cast<uint32_t>(id % a.rows);
    if (sequence_head >= static_cast<uint64_t>(a.cache.sequences) * a.cache.kv_heads) return;
    const uint32_t sequence = static_cast<uint32_t>(sequence_head / a.cache.kv_heads);
    const uint32_t head = static_cast<uint32_t>(sequence_head % a.cache.kv_heads);
    const float2* stats = a.stats + id * a.splits;

    float least = INFINITY;
    for (uint32_t s = lane; s < a.splits; s += 64) {
        const float c = stats[s].x;
        least = c < least || c != c ? c : least;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float c = __shfl_xor(least, o);
        least = c < least || c != c ? c : least;
    }

    constexpr uint32_t kGroups = 64 / LANES;
    const uint32_t part = lane % LANES, group = lane / LANES;
    float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float total = 0.0f;
    if (4 * part < a.cache.head_dim) {
        for (uint32_t s = group; s < a.splits; s += kGroups) {
            const float2 st = stats[s];
            if (st.x == INFINITY) continue;  // nothing seen: its outputs were not written
            const float w = __builtin_amdgcn_exp2f(least - st.x);
            const float4 v = *reinterpret_cast<const float4*>(a.partial + (id * a.splits + s) * a.cache.head_dim + 4 * part);
            total = __builtin_fmaf(w, st.y, total);
            sum = {__builtin_fmaf(w, v.x, sum.x), __builtin_fmaf(w, v.y, sum.y), __builtin_fmaf(w, v.z, sum.z),
                   __builtin_fmaf(w, v.w, sum.w)};
        }
    }
#pragma unroll
    for (uint32_t o = LANES; o < 64; o <<= 1) {
        sum.x += __shfl_xor(sum.x, o);
        sum.y += __shfl_xor(sum.y, o);
        sum.z += __shfl_xor(sum.z, o);
        sum.w += __shfl_xor(sum.w, o);
        total += __shfl_xor(total, o);
    }
    if (group != 0 || 4 * part >= a.cache.head_dim) return;
    const float inverse = least == INFINITY ? 0.0f : 1.0f / total;
    float* to = a.output + (static_cast<uint64_t>(sequence) * a.tokens + row / a.group) * a.output_stride +
                static_cast<uint64_t>(head * a.group + row % a.group) * a.cache.head_dim + 4 * part;
    *reinterpret_cast<float4*>(to) = make_float4(sum.x * inverse, sum.y * inverse, sum.z * inverse, sum.w * inverse);
}

hipError_t launch_attention_combine(const Attention& a, hipStream_t stream) {
    const uint64_t rows = uint64_t{a.cache.sequences} * a.cache.kv_heads * a.rows;
    const dim3 grid(static_cast<uint32_t>((rows + 3) / 4));
    if (a.cache.head_dim <= 32)
        hipLaunchKernelGGL(attention_combine<8>, grid, dim3(256), 0, stream, a);
    else if (a.cache.head_dim <= 64)
        hipLaunchKernelGGL(attention_combine<16>, grid, dim3(256), 0, stream, a);
    else if (a.cache.head_dim <= 128)
        hipLaunchKernelGGL(attention_combine<32>, grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(attention_combine<64>, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

// The least rows a workgroup that hold the step's, at most 32 RT; then splits
// until each compute unit has eight waves, a split of at least four tiles.
AttentionPlan plan_attention(const CacheShape& cache, uint32_t query_heads, uint32_t tokens, uint32_t longest,
                             uint32_t window, uint32_t compute_units) {
    const uint64_t rows = uint64_t{tokens} * (query_heads / cache.kv_heads);
    const uint32_t wide = cache.head_dim <= 128 ? 2 : 1;  // 16-row tiles a wave's registers hold
    AttentionPlan plan{};
    plan.waves = rows <= 16 * wide ? 1 : rows <= 64 * wide ? 4 : 8;
    plan.row_tiles = rows <= 16 || (plan.waves == 4 && rows <= 64) ? 1 : wide;
    const uint64_t group = 16ull * plan.row_tiles * plan.waves;
    plan.row_groups = static_cast<uint32_t>((rows + group - 1) / group);
    const uint64_t workgroups = uint64_t{cache.sequences} * cache.kv_heads * plan.row_groups;
    uint64_t reach = std::min(longest ? longest : cache.capacity, cache.capacity);
    if (window) reach = std::min<uint64_t>(reach, uint64_t{window} + tokens + 31);
    const uint64_t tiles = (reach + 31) / 32;
    const uint64_t wanted = (plan.waves == 8 ? 1ull : 2ull) * compute_units / workgroups;
    plan.splits = static_cast<uint32_t>(std::max<uint64_t>(1, std::min(wanted, (tiles + 3) / 4)));
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
        const uint64_t rows = 16ull * plan.row_tiles * plan.waves * plan.row_groups;
        t = static_cast<uint32_t>(std::min<uint64_t>(tokens, std::max<uint64_t>(t, rows / group)));
        plan = plan_attention(cache, query_heads, t, 0, 0, compute_units);
        most = std::max(most, attention_partial_bytes(cache, query_heads, t, plan.splits));
        if (plan.waves == 8 && plan.splits < 2) break;
    }
    return most;
}

}  // namespace chm
