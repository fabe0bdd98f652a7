// The splits of a step's attention joined (attention.hpp): a row's splits hold
// outputs o_s and sums l_s relative to their own offsets c_s; the row is
//   sum_s 2^(c - c_s) o_s / sum_s 2^(c - c_s) l_s,  c the least offset,
// added in an order that their number alone fixes.
//
// As many lanes as hold a row's values, four each, are a group; where the rows
// are few a row's splits are shared among several groups of a workgroup and
// added through LDS, so that all of its loads are on their way at once. Bound by
// the latency of a launch and of two dependent reads: 3 - 5 us, 8 for 16,384 rows
// of 128 in 4 splits (34 MB).
#include "serving.hpp"

namespace chm {

typedef float float4_t __attribute__((ext_vector_type(4)));

// SHARES groups a row.
template <uint32_t LANES, uint32_t SHARES>
__global__ __launch_bounds__(256) void attention_combine(Attention a) {
    constexpr uint32_t kGroups = 256 / LANES;
    __shared__ float4_t sums[SHARES > 1 ? 256 : 1];
    __shared__ float totals[kGroups];
    const uint32_t part = threadIdx.x % LANES, group = threadIdx.x / LANES, share = group % SHARES;
    const uint32_t row_of_all = blockIdx.x * (kGroups / SHARES) + group / SHARES;
    const uint32_t sequence_head = row_of_all / a.rows, row = row_of_all % a.rows;
    const bool live = sequence_head < static_cast<uint64_t>(a.cache.sequences) * a.cache.kv_heads &&
                      4 * part < a.cache.head_dim;
    const uint64_t place = static_cast<uint64_t>(row_of_all) * a.splits;

    // This share's splits relative to its own least offset, then all of them to the row's.
    float least = INFINITY, total = 0.0f;
    float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) {
#pragma unroll 4
        for (uint32_t s = share; s < a.splits; s += SHARES) {
            const float2 st = a.stats[place + s];
            const float4_t v = *reinterpret_cast<const float4_t*>(a.partial + (place + s) * a.cache.head_dim + 4 * part);
            if (st.x == INFINITY) continue;  // nothing seen: its outputs were not written
            const float to = st.x < least || st.x != st.x ? st.x : least;
            const float old = least == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(to - least);
            const float w = __builtin_amdgcn_exp2f(to - st.x);
            least = to;
            total = __builtin_fmaf(w, st.y, total * old);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(w, v[e], sum[e] * old);
        }
    }
    if constexpr (SHARES > 1) {
        __shared__ float leasts[kGroups];
        sums[threadIdx.x] = sum;
        if (part == 0) totals[group] = total, leasts[group] = least;
        __syncthreads();
        if (share != 0) return;
        for (uint32_t x = 1; x < SHARES; ++x) {
            const float c = leasts[group + x];
            least = c < least || c != c ? c : least;
        }
        sum = {0.0f, 0.0f, 0.0f, 0.0f};
        total = 0.0f;
        for (uint32_t x = 0; x < SHARES; ++x) {
            const float c = leasts[group + x];
            if (c == INFINITY) continue;
            const float w = __builtin_amdgcn_exp2f(least - c);
            total = __builtin_fmaf(w, totals[group + x], total);
            sum += sums[threadIdx.x + x * LANES] * w;
        }
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
    // a workgroup a row while that is at most four a compute unit; a step's time so
    // and with a group a row: of 32 rows in 32 splits 10.3 and 21.3 us, of 672 17.1
    // and 19.9, of 1,024 17.1 and 19.1, of 2,048 25.0 and 25.2
    if (rows <= 1024)
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
