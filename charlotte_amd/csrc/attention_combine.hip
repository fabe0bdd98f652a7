// The splits of a step's attention joined (attention.hpp): a row's splits hold
// outputs o_s and sums l_s relative to their own offsets c_s; the row is
//   sum_s 2^(c - c_s) o_s / sum_s 2^(c - c_s) l_s,  c the least offset,
// added in an order that their number alone fixes.
//
// As many lanes as hold a row's values, four each, are a group; where the rows
// are few a row's splits are shared among several groups of a workgroup and
// added through LDS. A group has its first splits' outputs on their way while
// its lanes find c and the sum from all of the row's stats, a lane a split; then
// no output waits for another. Bound by the latency of a launch and of two
// dependent reads: 3 - 5 us, 8 for 16,384 rows of 128 in 4 splits (34 MB).
#include "serving.hpp"

namespace chm {

typedef float float4_t __attribute__((ext_vector_type(4)));

// SHARES groups a row.
template <uint32_t LANES, uint32_t SHARES>
__global__ __launch_bounds__(256) void attention_combine(Attention a) {
    constexpr uint32_t kGroups = 256 / LANES;
    __shared__ float4_t sums[SHARES > 1 ? 256 : 1];
    const uint32_t part = threadIdx.x % LANES, group = threadIdx.x / LANES, share = group % SHARES;
    const uint32_t row_of_all = blockIdx.x * (kGroups / SHARES) + group / SHARES;
    const uint32_t sequence_head = row_of_all / a.rows, row = row_of_all % a.rows;
    const bool known = sequence_head < a.cache.sequences * a.cache.kv_heads, live = known && 4 * part < a.cache.head_dim;
    const uint64_t place = static_cast<uint64_t>(row_of_all) * a.splits;
    const uint32_t splits = known ? a.splits : 0u;

    // A batch of this share's splits: c_s and outputs.
    constexpr uint32_t kBatch = SHARES > 1 ? 8 : 4;
    float offset[kBatch];
    float4_t out[kBatch];
    auto load = [&](uint32_t first) {
#pragma unroll
        for (uint32_t u = 0; u < kBatch; ++u) {
            const uint32_t s = first + SHARES * u;
            offset[u] = INFINITY;
            if (s < splits && live) {
                offset[u] = a.stats[place + s].x;
                out[u] = *reinterpret_cast<const float4_t*>(a.partial + (place + s) * a.cache.head_dim + 4 * part);
            }
        }
    };
    load(share);

    // c: the least offset, a NaN if any is one (INFINITY: nothing seen); and the sum relative to it
    auto lesser = [](float x, float y) { return x < y || x != x ? x : y; };
    float least = INFINITY;
    for (uint32_t s = part; s < splits; s += LANES) least = lesser(a.stats[place + s].x, least);
#pragma unroll
    for (uint32_t o = LANES / 2; o > 0; o >>= 1) least = lesser(__shfl_xor(least, o, LANES), least);
    auto weight = [&](float x) { return x == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(least - x); };
    float total = 0.0f;
    for (uint32_t s = part; s < splits; s += LANES) {
        const float2 st = a.stats[place + s];
        total = __builtin_fmaf(weight(st.x), st.y, total);
    }
#pragma unroll
    for (uint32_t o = LANES / 2; o > 0; o >>= 1) total += __shfl_xor(total, o, LANES);

    float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t first = share;;) {
#pragma unroll
        for (uint32_t u = 0; u < kBatch; ++u) {
            if (offset[u] == INFINITY) continue;  // nothing seen: its outputs were not written
            const float w = weight(offset[u]);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(w, out[u][e], sum[e]);
        }
        first += SHARES * kBatch;
        if (first >= splits) break;
        load(first);
    }
    if constexpr (SHARES > 1) {
        sums[threadIdx.x] = sum;
        __syncthreads();
        if (share != 0) return;
#pragma unroll
        for (uint32_t x = 1; x < SHARES; ++x) sum += sums[threadIdx.x + x * LANES];
    }
    if (!live) return;
    const uint32_t sequence = sequence_head / a.cache.kv_heads, head = sequence_head % a.cache.kv_heads;
    const float inverse = least == INFINITY ? 0.0f : 1.0f / total;
    float* to = a.output + (static_cast<uint64_t>(sequence) * a.tokens + row / a.group) * a.output_stride +
                static_cast<uint64_t>(head * a.group + row % a.group) * a.cache.head_dim + 4 * part;
    *reinterpret_cast<float4_t*>(to) = sum * inverse;
}

template <uint32_t LANES>
static hipError_t launch_lanes(const Attention& a, hipStream_t stream) {
    constexpr uint32_t kGroups = 256 / LANES;
    const uint64_t rows = uint64_t{a.cache.sequences} * a.cache.kv_heads * a.rows;
    // a workgroup a row while that is at most three a compute unit; a step's time so
    // and with a group a row: of 32 rows in 32 splits 10.2 and 12.9 us, of 672 16.4
    // and 17.2, of 1,024 18.0 and 17.1, of 2,048 26.3 and 24.6
    if (rows <= 768)
        hipLaunchKernelGGL((attention_combine<LANES, kGroups>), dim3(static_cast<uint32_t>(rows)), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((attention_combine<LANES, 1>), dim3(static_cast<uint32_t>((rows + kGroups - 1) / kGroups)),
                           dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_attention_combine(const Attention& a, hipStream_t stream) {
    if (a.cache.head_dim <= 32) return launch_lanes<8>(a, stream);
    if (a.cache.head_dim <= 64) return launch_lanes<16>(a, stream);
    if (a.cache.head_dim <= 128) return launch_lanes<32>(a, stream);
    return launch_lanes<64>(a, stream);
}

}  // namespace chm
