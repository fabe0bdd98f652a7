// Rows of floats of any length at any 4-byte alignment, read and written four
// at a time: a row is seen from the 16-byte boundary at or before its first
// float, `lead` floats ahead of it, so that every four is aligned; entries
// outside the row are neither read nor written.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace chm {

__device__ __forceinline__ uint32_t lead_of(const float* row) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) >> 2) & 3u;
}

// Entries at .. at + 3 counted from the boundary, `at` a multiple of 4;
// `outside` for those not of the row's `length`. ONCE: not kept in the caches.
template <bool ONCE = false>
__device__ __forceinline__ float4 read4(const float* row, uint32_t lead, uint32_t length, uint32_t at, float outside) {
    if (at >= lead && at + 4 <= lead + length) {
        typedef float vector_t __attribute__((ext_vector_type(4)));
        const auto* from = reinterpret_cast<const vector_t*>(row - lead + at);
        const vector_t v = ONCE ? __builtin_nontemporal_load(from) : *from;
        return {v.x, v.y, v.z, v.w};
    }
    float v[4];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) v[e] = at + e >= lead && at + e < lead + length ? row[at + e - lead] : outside;
    return {v[0], v[1], v[2], v[3]};
}

// Entry i of the row is to[i]; `to` may have another lead than the entries were read with.
__device__ __forceinline__ void write4(float* to, uint32_t lead, uint32_t length, uint32_t at, const float4& v) {
    if (at >= lead && at + 4 <= lead + length && lead_of(to) == lead) {
        *reinterpret_cast<float4*>(to - lead + at) = v;
        return;
    }
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
        if (at + e >= lead && at + e < lead + length) to[at + e - lead] = x[e];
}

}  // namespace chm
