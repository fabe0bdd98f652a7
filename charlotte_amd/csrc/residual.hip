// Norms before and after a block, with its gate and scales, in one pass:
//   r = a x + b g z, z = y or y / sqrt(mean(y^2) + epsilon) * w,
//   n = r / sqrt(mean(r^2) + epsilon) * v.
//
// Mapping: a workgroup a row, its values in registers from the one read to the
// one write, FOURS fours a thread; both sums of squares are shuffles in a wave
// and, over its waves, one pass through LDS. The weights and the gate are read
// with the row, ahead of the sums that they wait for.
//
// Bound by bytes, 16 a value with both results: 2,048 rows of 4,096 (134 MB) out of memory
// 26.7 - 28 us, 4.7 - 5.0 TB/s; 20.8 where the card's last cache has half of it. One row of
// 1,024 2.4 us, latency; 333 gated ones of 1,155, at addresses that are no fours', 5.1 - 6.3.
#include "requests.hpp"

namespace chm {

constexpr uint32_t kMostWaves = 16;

// The workgroup's sum, in every thread. `parts`: kMostWaves floats of this sum's own.
__device__ __forceinline__ float sum_all(float x, float* parts) {
#pragma unroll
    for (uint32_t o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    const uint32_t waves = blockDim.x / 64;
    if (waves == 1) return x;
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = x;
    __syncthreads();
    float sum = parts[0];
    for (uint32_t w = 1; w < waves; ++w) sum += parts[w];
    return sum;
}

// A thread's values of a row: whole fours, or (ALIGNED false: an odd width, stride
// or address) single ones a workgroup apart.
template <uint32_t FOURS, bool ALIGNED>
struct Row {
    float v[FOURS][4];

    __device__ __forceinline__ static uint32_t place(uint32_t f, uint32_t e) {
        return ALIGNED ? 4 * (f * blockDim.x + threadIdx.x) + e : (4 * f + e) * blockDim.x + threadIdx.x;
    }
    __device__ __forceinline__ void read(const float* row, uint32_t width) {
#pragma unroll
        for (uint32_t f = 0; f < FOURS; ++f) {
            if constexpr (ALIGNED) {
                float4 x = {0.0f, 0.0f, 0.0f, 0.0f};
                if (place(f, 0) < width) x = *reinterpret_cast<const float4*>(row + place(f, 0));
                v[f][0] = x.x, v[f][1] = x.y, v[f][2] = x.z, v[f][3] = x.w;
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) v[f][e] = place(f, e) < width ? row[place(f, e)] : 0.0f;
            }
        }
    }
    __device__ __forceinline__ void write(float* row, uint32_t width) const {
#pragma unroll
        for (uint32_t f = 0; f < FOURS; ++f) {
            if constexpr (ALIGNED) {
                if (place(f, 0) < width)
                    *reinterpret_cast<float4*>(row + place(f, 0)) = make_float4(v[f][0], v[f][1], v[f][2], v[f][3]);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e)
                    if (place(f, e) < width) row[place(f, e)] = v[f][e];
            }
        }
    }
    __device__ __forceinline__ float squares() const {
        float sum = 0.0f;
#pragma unroll
        for (uint32_t f = 0; f < FOURS; ++f)
            sum += (v[f][0] * v[f][0] + v[f][1] * v[f][1]) + (v[f][2] * v[f][2] + v[f][3] * v[f][3]);
        return sum;
    }
};

template <uint32_t FOURS, bool ALIGNED>
__global__ __launch_bounds__(64 * kMostWaves) void residual_norm(ResidualNorm a) {
    __shared__ float parts[2][kMostWaves];
    const uint64_t row = blockIdx.x;
    using Values = Row<FOURS, ALIGNED>;
    constexpr bool kEarly = FOURS <= 4;  // more than that the registers of 16 waves do not hold
    Values x, y, w, g, v;
    x.read(a.residual + row * a.residual_stride, a.width);
    if (a.branch) y.read(a.branch + row * a.branch_stride, a.width);
    if (kEarly && a.branch_weight) w.read(a.branch_weight, a.width);
    if (kEarly && a.gate) g.read(a.gate + row * a.gate_stride, a.width);
    if (kEarly && a.normed) v.read(a.weight, a.width);
    const float mean = 1.0f / static_cast<float>(a.width);
    if (a.branch) {
        if (a.branch_weight) {
            const float inverse = 1.0f / sqrtf(__builtin_fmaf(sum_all(y.squares(), parts[0]), mean, a.epsilon));
            if (!kEarly) w.read(a.branch_weight, a.width);
#pragma unroll
            for (uint32_t f = 0; f < FOURS; ++f)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) y.v[f][e] = y.v[f][e] * inverse * w.v[f][e];
        }
        if (a.gate) {
            if (!kEarly) g.read(a.gate + row * a.gate_stride, a.width);
#pragma unroll
            for (uint32_t f = 0; f < FOURS; ++f)
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) y.v[f][e] *= g.v[f][e];
        }
#pragma unroll
        for (uint32_t f = 0; f < FOURS; ++f)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                x.v[f][e] = __builtin_fmaf(a.branch_scale, y.v[f][e], a.residual_scale * x.v[f][e]);
    } else {
#pragma unroll
        for (uint32_t f = 0; f < FOURS; ++f)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) x.v[f][e] *= a.residual_scale;
    }
    if (a.residual_out) x.write(a.residual_out + row * a.residual_out_stride, a.width);
    if (a.normed) {
        const float inverse = 1.0f / sqrtf(__builtin_fmaf(sum_all(x.squares(), parts[1]), mean, a.epsilon));
        if (!kEarly) v.read(a.weight, a.width);
#pragma unroll
        for (uint32_t f = 0; f < FOURS; ++f)
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) x.v[f][e] = x.v[f][e] * inverse * v.v[f][e];
        x.write(a.normed + row * a.normed_stride, a.width);
    }
}

template <uint32_t FOURS>
static hipError_t launch_fours(const ResidualNorm& a, uint32_t threads, hipStream_t stream) {
    if (a.fours)
        hipLaunchKernelGGL((residual_norm<FOURS, true>), dim3(a.rows), dim3(threads), 0, stream, a);
    else
        hipLaunchKernelGGL((residual_norm<FOURS, false>), dim3(a.rows), dim3(threads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_residual_norm(const ResidualNorm& a, hipStream_t stream) {
    // A four a thread while the card holds all rows' threads about at once, else four of
    // them: the same row in a quarter of the waves. With a branch and both results, out of
    // memory, one and four: rows of 4,096, 1 row 3.0 us and 3.2, 333 7.6 and 7.7, 512 8.2 and
    // 8.2, 513 10.2 and 8.5, 1,024 15.9 and 11.8, 2,048 28.3 and 26.7; of 2,048, 513 5.7 and 5.8,
    // 2,048 15.1 and 12.1; of 1,024 (always one), 2,048 8.1 and 8.2. 333 gated of 1,155 6.3 and 7.2.
    const uint32_t fours = (a.width + 3) / 4;
    auto threads = [&](uint32_t each) { return (fours + 64 * each - 1) / (64 * each) * 64; };
    if (threads(1) <= 256 || (threads(1) <= 64 * kMostWaves && a.rows <= 512)) return launch_fours<1>(a, threads(1), stream);
    if (threads(4) <= 64 * kMostWaves) return launch_fours<4>(a, threads(4), stream);
    return launch_fours<8>(a, threads(8), stream);
}

}  // namespace chm
