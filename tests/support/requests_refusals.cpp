// The host checks of a step's operators over several requests (requests.cpp),
// with launches that only count themselves: what is refused before any kernel
// runs, without a device (tests/test_requests_refusals.py). Test infrastructure only.
#include <cstdio>
#include <cstdlib>

#include "context.hpp"
#include "requests.hpp"

static int launches = 0;

namespace chm {
uint64_t cache_bytes(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 0; }
hipError_t launch_page_plan(const PagePlan&, hipStream_t) { return ++launches, hipSuccess; }
hipError_t launch_page_append(const CacheRows&, hipStream_t) { return ++launches, hipSuccess; }
hipError_t launch_page_read(const CacheRows&, hipStream_t) { return ++launches, hipSuccess; }
hipError_t launch_paged_f16(const PagedAttention&, uint32_t, hipStream_t) { return ++launches, hipSuccess; }
hipError_t launch_paged_q4_0(const PagedAttention&, uint32_t, hipStream_t) { return ++launches, hipSuccess; }
hipError_t launch_paged_q8_0(const PagedAttention&, uint32_t, hipStream_t) { return ++launches, hipSuccess; }
hipError_t launch_residual_norm(const ResidualNorm&, hipStream_t) { return ++launches, hipSuccess; }
hipError_t launch_sample(const Sample&, hipStream_t) { return ++launches, hipSuccess; }
uint64_t sample_bytes(uint32_t, uint32_t) { return 0; }
}  // namespace chm

extern "C" {
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipMalloc(void**, size_t) { return hipErrorOutOfMemory; }
hipError_t hipFree(void*) { return hipSuccess; }
hipError_t hipMemset(void*, int, size_t) { return hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return ""; }
}

static charlotte_hip_matmul_context context;
static int failed = 0;

static void expect(const char* what, bool accepted, const charlotte_hip_matmul_residual_norm_desc& d) {
    launches = 0;
    const auto status = charlotte_hip_matmul_residual_norm(&context, &d, 5, nullptr);
    const bool good = accepted ? status == CHARLOTTE_HIP_MATMUL_OK && launches == 1
                               : status == CHARLOTTE_HIP_MATMUL_INVALID_ARGUMENT && launches == 0;
    if (!good) std::printf("%s: status %d, %d launches: %s\n", what, status, launches, context.error.c_str()), ++failed;
}

// Results over inputs: with each input's own stride, two of which may be one memory.
static void results_over_inputs() {
    static float memory[8][4096];
    charlotte_hip_matmul_residual_norm_desc good{};
    good.residual = memory[0], good.branch = memory[1], good.gate = memory[2], good.weight = memory[3];
    good.residual_out = memory[4], good.normed = memory[5];
    good.width = 64, good.gate_stride = 64, good.residual_scale = good.branch_scale = 1.0f;
    expect("apart", true, good);
    for (int result = 0; result < 2; ++result) {
        auto over = [&](charlotte_hip_matmul_residual_norm_desc d, const float* input) {
            (result ? d.normed : d.residual_out) = const_cast<float*>(input);
            return d;
        };
        for (int input = 0; input < 3; ++input) {
            auto d = over(good, memory[input]);
            expect("over an input", true, d);
            uint64_t& stride = input == 0 ? d.residual_stride : input == 1 ? d.branch_stride : d.gate_stride;
            stride = 128;
            expect("over an input of another stride", false, d);
        }
        auto d = good;
        d.branch = good.residual;
        expect("over two inputs of one memory", true, over(d, d.residual));
        d.branch_stride = 128;
        expect("over a branch of the residual's memory and another stride", false, over(d, d.residual));
        d = good, d.gate = good.residual;
        expect("over a gate of the residual's memory", true, over(d, d.residual));
        d.gate_stride = 0;
        expect("over one gate of all rows, the residual's memory", false, over(d, d.residual));
        d = good, d.gate = good.branch, d.gate_stride = 128;
        expect("over a gate of the branch's memory and another stride", false, over(d, d.branch));
    }
}

int main() {
    context.compute_units = 256;
    results_over_inputs();
    if (failed) return 1;
    std::puts("refused as they should be");
    return 0;
}
