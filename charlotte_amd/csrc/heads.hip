// Norms of queries and keys for each head, with the position rotation in the
// same pass:
//   y = x / sqrt(mean(x^2) + epsilon) * w,  then for each rotated pair (a, b)
//   (a c - b s, b c + a s), c and s read from the tables at the token's row.
//
// Mapping: a head is 8 .. 64 lanes of four consecutive values each (the least
// power of two that holds head_dim / 4), so a wave takes one to eight heads, a
// load or store of a head is one contiguous run, and the sum of squares is one
// shuffle a doubling. Values 4l .. 4l + 3 and their partners rope_dims / 2
// further on are in two lanes of the same head (whole fours, as rope_dims is
// whole eights), exchanged by shuffle; neighbours are in one lane.
//
// Bound by bytes, each value read and written once; a token's table rows are
// read by every head of it, from cache. 2,048 tokens of 32 + 8 heads of 128 (85
// MB): 17.9 us, 4.7 TB/s, where a large copy moves 5.1. A decode is one launch's
// latency, 3 us.
#include "serving.hpp"

#include "charlotte_hip_matmul.h"

namespace chm {

template <uint32_t LANES>
__global__ __launch_bounds__(256) void head_norm_rope(HeadNormRope a) {
    const uint32_t all = a.part[0].heads + (a.parts > 1 ? a.part[1].heads : 0u);
    const uint32_t row = (blockIdx.x * 256 + threadIdx.x) / LANES;  // a launch has below 2^32 threads
    const uint32_t lane = threadIdx.x % LANES;
    const uint64_t token = row / all;
    uint32_t head = row % all;
    const bool second = head >= a.part[0].heads;
    if (second) head -= a.part[0].heads;
    const HeadPart& p = a.part[second ? 1 : 0];
    const bool live = token < a.tokens && 4 * lane < a.head_dim;
    const uint64_t at = static_cast<uint64_t>(head) * a.head_dim + 4 * lane;

    float4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) x = *reinterpret_cast<const float4*>(p.input + token * p.input_stride + at);
    if (p.weight) {
        float sum = (x.x * x.x + x.y * x.y) + (x.z * x.z + x.w * x.w);
#pragma unroll
        for (uint32_t o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, LANES);
        const float inverse = 1.0f / sqrtf(sum / static_cast<float>(a.head_dim) + a.epsilon);
        if (live) {
            const float4 w = *reinterpret_cast<const float4*>(p.weight + 4 * lane);
            x = {x.x * inverse * w.x, x.y * inverse * w.y, x.z * inverse * w.z, x.w * inverse * w.w};
        }
    }
    if (a.rope != CHARLOTTE_HIP_MATMUL_ROPE_NONE) {
        const uint32_t half = a.rope_dims / 2;
        const bool turned = live && 4 * lane < a.rope_dims;
        const uint32_t position = token < a.tokens ? a.positions[token] : 0u;
        const bool inside = position < a.table_rows;
        const uint64_t entry = static_cast<uint64_t>(inside ? position : 0u) * half;
        const float nan = __builtin_nanf("");
        if (a.rope == CHARLOTTE_HIP_MATMUL_ROPE_HALVES) {
            const bool upper = 4 * lane >= half;
            // every lane shuffles; one that is not rotated reads itself
            const uint32_t partner = !turned ? lane : upper ? lane - half / 4 : lane + half / 4;
            const float4 y = {__shfl(x.x, partner, LANES), __shfl(x.y, partner, LANES), __shfl(x.z, partner, LANES),
                              __shfl(x.w, partner, LANES)};
            if (turned) {
                const uint64_t pair = entry + 4 * lane - (upper ? half : 0u);
                float4 c = {nan, nan, nan, nan}, s = c;
                if (inside) {
                    c = *reinterpret_cast<const float4*>(a.cosines + pair);
                    s = *reinterpret_cast<const float4*>(a.sines + pair);
                }
                const float sign = upper ? 1.0f : -1.0f;
                x = {__builtin_fmaf(x.x, c.x, sign * (y.x * s.x)), __builtin_fmaf(x.y, c.y, sign * (y.y * s.y)),
                     __builtin_fmaf(x.z, c.z, sign * (y.z * s.z)), __builtin_fmaf(x.w, c.w, sign * (y.w * s.w))};
            }
        } else if (turned) {
            const uint64_t pair = entry + 2 * lane;
            float2 c = {nan, nan}, s = c;
            if (inside) {
                c = *reinterpret_cast<const float2*>(a.cosines + pair);
                s = *reinterpret_cast<const float2*>(a.sines + pair);
            }
            x = {__builtin_fmaf(x.x, c.x, -(x.y * s.x)), __builtin_fmaf(x.y, c.x, x.x * s.x),
                 __builtin_fmaf(x.z, c.y, -(x.w * s.y)), __builtin_fmaf(x.w, c.y, x.z * s.y)};
        }
    }
    if (live) *reinterpret_cast<float4*>(p.output + token * p.output_stride + at) = x;
}

template <uint32_t LANES>
static hipError_t launch_lanes(const HeadNormRope& a, hipStream_t stream) {
    const uint64_t heads = uint64_t{a.part[0].heads} + (a.parts > 1 ? a.part[1].heads : 0u);
    const uint64_t groups = (heads * a.tokens * LANES + 255) / 256;
    hipLaunchKernelGGL(head_norm_rope<LANES>, dim3(static_cast<uint32_t>(groups)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_head_norm_rope(const HeadNormRope& a, hipStream_t stream) {
    if (a.head_dim <= 32) return launch_lanes<8>(a, stream);
    if (a.head_dim <= 64) return launch_lanes<16>(a, stream);
    if (a.head_dim <= 128) return launch_lanes<32>(a, stream);
    return launch_lanes<64>(a, stream);
}

}  // namespace chm
