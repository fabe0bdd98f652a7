// Softmax of the head's logits at a temperature: p = exp((x - m) / T) / sum.
// Two passes over chunks of the rows: each chunk's maximum and sum in one read
// (the sum kept relative to the running maximum), then, from all of a row's
// chunks, its probabilities. The second read of the logits comes from cache
// where a step's rows fit it. Few rows are cut into as many chunks as fill
// the card. At temperature 0 the chunks keep the largest's first index.
//
// Bound by bytes: 4 read and 4 written a logit, and 4 more read from cache.
#include <algorithm>

#include "rows.hpp"
#include "serving.hpp"

namespace chm {

constexpr float kPerOctave = 1.44269504088896340736f;  // log2(e)
constexpr uint32_t kNowhere = 0xFFFFFFFFu;

__device__ __forceinline__ RowStats join_stats(const RowStats& a, const RowStats& b, float rate) {
    RowStats r;
    r.largest = fmaxf(a.largest, b.largest);
    // sums relative to the larger maximum; a side without one has the sum 0, or a NaN
    const float fa = a.largest == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((a.largest - r.largest) * rate);
    const float fb = b.largest == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((b.largest - r.largest) * rate);
    r.sum = a.sum * fa + b.sum * fb;
    r.at = a.largest > b.largest ? a.at : b.largest > a.largest ? b.at : min(a.at, b.at);
    return r;
}

__device__ __forceinline__ RowStats shuffled(const RowStats& s, int o) {
    return {__shfl_xor(s.largest, o), __shfl_xor(s.sum, o), static_cast<uint32_t>(__shfl_xor(static_cast<int>(s.at), o))};
}

// A chunk: `share` entries from the row's boundary (rows.hpp), a multiple of 4.
__device__ __forceinline__ uint32_t share_of(const Probabilities& a) {
    return ((a.vocabulary + 3 + a.chunks - 1) / a.chunks + 3) / 4 * 4;
}

__global__ __launch_bounds__(256) void row_stats(Probabilities a) {
    __shared__ RowStats parts[4];
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const float* x = a.logits + row * a.logit_stride;
    const uint32_t lead = lead_of(x), share = share_of(a);
    const float rate = a.temperature > 0.0f ? kPerOctave / a.temperature : 0.0f;
    RowStats s = {-INFINITY, 0.0f, kNowhere};
    const uint32_t end = min((chunk + 1) * share, lead + a.vocabulary);
    for (uint32_t at = chunk * share + 4 * threadIdx.x; at < end; at += 1024) {
        const float4 q = read4(x, lead, a.vocabulary, at, -INFINITY);
        const float v[4] = {q.x, q.y, q.z, q.w};
        const float top = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        if (top > s.largest) {
            s.sum *= s.largest == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((s.largest - top) * rate);
            s.largest = top;
            s.at = at - lead + (v[0] == top ? 0 : v[1] == top ? 1 : v[2] == top ? 2 : 3);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            s.sum += v[e] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((v[e] - s.largest) * rate);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s = join_stats(s, shuffled(s, o), rate);
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        a.stats[blockIdx.x] = join_stats(join_stats(parts[0], parts[1], rate), join_stats(parts[2], parts[3], rate), rate);
}

__global__ __launch_bounds__(256) void row_probabilities(Probabilities a) {
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const float* x = a.logits + row * a.logit_stride;
    float* y = a.output + row * a.output_stride;
    const uint32_t lead = lead_of(x), share = share_of(a);
    const float rate = a.temperature > 0.0f ? kPerOctave / a.temperature : 0.0f;
    // every wave joins the row's chunks, in one order
    RowStats s = {-INFINITY, 0.0f, kNowhere};
    for (uint32_t c = threadIdx.x & 63u; c < a.chunks; c += 64)
        s = join_stats(s, a.stats[static_cast<uint64_t>(row) * a.chunks + c], rate);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s = join_stats(s, shuffled(s, o), rate);
    // nothing but -inf: zeros, where 1 / 0 would make NaNs
    const float inverse = s.sum == 0.0f ? 0.0f : 1.0f / s.sum;
    const float largest = s.largest == -INFINITY ? 0.0f : s.largest;
    const uint32_t end = min((chunk + 1) * share, lead + a.vocabulary);
    for (uint32_t at = chunk * share + 4 * threadIdx.x; at < end; at += 1024) {
        float4 v;
        if (a.temperature > 0.0f) {
            const float4 q = read4(x, lead, a.vocabulary, at, -INFINITY);
            v = {__builtin_amdgcn_exp2f((q.x - largest) * rate) * inverse, __builtin_amdgcn_exp2f((q.y - largest) * rate) * inverse,
                 __builtin_amdgcn_exp2f((q.z - largest) * rate) * inverse, __builtin_amdgcn_exp2f((q.w - largest) * rate) * inverse};
        } else {
            const uint32_t hit = s.at == kNowhere ? kNowhere : s.at + lead - at;
            v = {hit == 0 ? 1.0f : 0.0f, hit == 1 ? 1.0f : 0.0f, hit == 2 ? 1.0f : 0.0f, hit == 3 ? 1.0f : 0.0f};
        }
        write4(y, lead, a.vocabulary, at, v);
    }
}

// About a thousand workgroups, a chunk of at least 2,048 logits.
uint32_t probabilities_chunks(uint32_t rows, uint32_t vocabulary) {
    return std::max(1u, std::min((1024 + rows - 1) / rows, (vocabulary + 2047) / 2048));
}

hipError_t launch_probabilities(const Probabilities& a, hipStream_t stream) {
    const dim3 grid(a.rows * a.chunks);
    hipLaunchKernelGGL(row_stats, grid, dim3(256), 0, stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    hipLaunchKernelGGL(row_probabilities, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace chm
