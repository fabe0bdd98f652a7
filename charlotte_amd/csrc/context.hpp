// What the C ABI's files share: the context behind its handle, and how an
// entry point reports. Nothing throws across the ABI: a status and a message.
#pragma once

#include <hip/hip_runtime_api.h>

#include <new>
#include <string>

#include "charlotte_hip_matmul.h"

struct charlotte_hip_matmul_context {
    int device = 0;
    uint32_t compute_units = 0;
    float* scratch = nullptr;   // this device's copy of the static range sums
    charlotte_hip_matmul_gemm_path gemm_path = CHARLOTTE_HIP_MATMUL_GEMM_AUTO;
    charlotte_hip_matmul_gemv_path gemv_path = CHARLOTTE_HIP_MATMUL_GEMV_CANONICAL;
    void* workspace = nullptr;  // the matrix-core path's, the caller's memory
    uint64_t workspace_bytes = 0;
    uint32_t patience = CHARLOTTE_HIP_MATMUL_PATIENCE;
    std::string error;
};

namespace chm {

inline charlotte_hip_matmul_status fail(charlotte_hip_matmul_context* ctx, charlotte_hip_matmul_status s,
                                        const std::string& message) {
    if (ctx) ctx->error = message;
    return s;
}

inline charlotte_hip_matmul_status ok(charlotte_hip_matmul_context* ctx) {
    if (ctx) ctx->error.clear();
    return CHARLOTTE_HIP_MATMUL_OK;
}

inline charlotte_hip_matmul_status hip_fail(charlotte_hip_matmul_context* ctx, hipError_t e, const char* what) {
    return fail(ctx, e == hipErrorOutOfMemory ? CHARLOTTE_HIP_MATMUL_OUT_OF_MEMORY : CHARLOTTE_HIP_MATMUL_HIP_ERROR,
                std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace chm
