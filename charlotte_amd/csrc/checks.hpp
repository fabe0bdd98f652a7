// How the entry points of serving.cpp and requests.cpp check their arguments
// and report: a failed check is thrown to `guarded`, which makes it a status
// and a message.
#pragma once

#include <hip/hip_runtime_api.h>

#include <string>

#include "context.hpp"

namespace chm {

using Status = charlotte_hip_matmul_status;

constexpr uint64_t kGrid = 0x7FFFFFull;  // workgroups a launch may have: of up to 512 threads, below 2^32 of them

// A failed check, thrown to `guarded` in the same call.
struct Refused {
    Status status;
    std::string message;
};

[[noreturn]] inline void refuse(std::string message, Status status = CHARLOTTE_HIP_MATMUL_INVALID_ARGUMENT) {
    throw Refused{status, std::move(message)};
}

// Runs `body`, whose every failure becomes a status and a message beginning
// with `who`: nothing is thrown across the ABI.
template <typename Body>
Status guarded(charlotte_hip_matmul_context* ctx, const char* who, Body body) noexcept {
    if (!ctx) return CHARLOTTE_HIP_MATMUL_INVALID_ARGUMENT;
    try {
        try {
            const hipError_t e = body();
            return e == hipSuccess ? ok(ctx) : hip_fail(ctx, e, who);
        } catch (const Refused& r) {
            return fail(ctx, r.status, std::string(who) + ": " + r.message);
        }
    } catch (...) {  // no memory for a message
        return CHARLOTTE_HIP_MATMUL_OUT_OF_MEMORY;
    }
}

inline bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// A required device pointer.
inline void need(const void* p, const char* name, uintptr_t to) {
    if (!p) refuse(std::string("no ") + name);
    if (!aligned(p, to)) refuse(std::string(name) + " not " + std::to_string(to) + "-byte aligned");
}

// A row stride in floats: 0 means `width`; else at least it, in whole `step`s.
inline uint64_t stride_of(uint64_t stride, uint64_t width, uint64_t step, const char* name) {
    if (stride == 0) stride = width;
    if (stride < width) refuse(std::string(name) + " below a row's " + std::to_string(width) + " floats");
    if (stride % step != 0) refuse(std::string(name) + " not whole " + std::to_string(step) + "s");
    if (stride > (1ull << 40)) refuse(std::string(name) + " past 2^40");
    return stride;
}

inline void need_grid(uint64_t workgroups) {
    if (workgroups > kGrid) refuse("too many rows a step");
}

}  // namespace chm
