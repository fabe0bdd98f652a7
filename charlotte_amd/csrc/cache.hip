// The quantized cache (its layout: cache.hpp): tokens written as they are
// quantized, slots read back, an accepted path's slots moved together.
//
// append and read: eight lanes a block of 32 values, four values a lane, so
// the f32 side is read or written in whole 128-byte runs; the block's largest
// magnitude is three shuffles. A key's four codes of a lane are neighbours in
// the record, a value's are in four lanes' operands.
#include "cache.hpp"

namespace chm {

uint64_t cache_bytes(uint32_t format, uint32_t sequences, uint32_t kv_heads, uint32_t head_dim, uint32_t capacity) {
    const uint64_t tiles = (uint64_t{capacity} + kTile - 1) / kTile;
    return tiles * sequences * kv_heads * cache_record(format, head_dim / 32);
}

// Which block of which row a thread's eight lanes hold.
struct Piece {
    uint32_t sequence, head, block, lane;  // lane: 0 .. 7 within the block
    uint64_t row;                          // sequence * tokens + token
    uint64_t slot;
    bool values, live;
};

__device__ __forceinline__ Piece piece_of(const CacheRows& a) {
    Piece p;
    const uint64_t id = (static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x) / 8;
    const uint32_t blocks = a.cache.head_dim / 32, row_blocks = blocks * a.cache.kv_heads;
    p.lane = threadIdx.x & 7u;
    p.values = blockIdx.y != 0;
    p.row = id / row_blocks;
    const uint32_t in_row = static_cast<uint32_t>(id % row_blocks);
    p.head = in_row / blocks;
    p.block = in_row % blocks;
    const uint64_t sequence = p.row / a.tokens;
    p.live = sequence < a.cache.sequences;
    p.sequence = p.live ? static_cast<uint32_t>(sequence) : 0u;
    p.slot = static_cast<uint64_t>(a.first[p.sequence]) + p.row % a.tokens;
    p.live = p.live && p.slot < a.cache.capacity;
    return p;
}

__device__ __forceinline__ uint32_t pack4(const uint32_t c[4]) { return c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24; }
__device__ __forceinline__ uint32_t half_bits(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
}

constexpr uint32_t kNanHalf = 0x7E00u;

// A lane's four codes, raised to be unsigned, and its block's scale as f16
// bits; every lane of the block calls it. F16's codes are the halves.
template <uint32_t F>
__device__ __forceinline__ uint32_t quantize(const float4& v, uint32_t lane, bool values, uint32_t code[4]) {
    const float x[4] = {v.x, v.y, v.z, v.w};
    if constexpr (F == kF16) {
        uint32_t bad = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            code[e] = half_bits(x[e]);
            bad |= (code[e] & 0x7C00u) == 0x7C00u ? 1u : 0u;
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) bad |= __shfl_xor(bad, o, 8);
        if (bad)
#pragma unroll
            for (int e = 0; e < 4; ++e) code[e] = values ? 0u : kNanHalf;
        return bad ? kNanHalf : 0x3C00u;
    } else {
        // the largest magnitude, the first of equals; a NaN's bits rank above every magnitude's
        uint32_t largest = 0, at = 0;
        float extreme = 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t bits = __float_as_uint(x[e]) & 0x7FFFFFFFu;
            if (e == 0 || bits > largest) largest = bits, at = 4 * lane + e, extreme = x[e];
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            const uint32_t theirs = __shfl_xor(largest, o, 8), their_at = __shfl_xor(at, o, 8);
            const float their_extreme = __shfl_xor(extreme, o, 8);
            if (theirs > largest || (theirs == largest && their_at < at))
                largest = theirs, at = their_at, extreme = their_extreme;
        }
        const uint32_t d = half_bits(F == kQ8_0 ? fabsf(extreme) / 127.0f : extreme / -8.0f);
        const bool bad = (d & 0x7C00u) == 0x7C00u;
        const float step = half_to_float(d);
        constexpr float kLow = F == kQ8_0 ? -127.0f : -8.0f, kHigh = F == kQ8_0 ? 127.0f : 7.0f;
        constexpr int kRaise = F == kQ8_0 ? 128 : 8;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // the code nearest to x / d, ties to even; the division is rounded once
            const float q = step == 0.0f || bad ? 0.0f : fminf(fmaxf(rintf(x[e] / step), kLow), kHigh);
            code[e] = static_cast<uint32_t>(static_cast<int>(q) + kRaise);
        }
        return bad ? kNanHalf : d;
    }
}

template <uint32_t F>
__global__ __launch_bounds__(256) void cache_append(CacheRows a) {
    const Piece p = piece_of(a);
    const uint32_t blocks = a.cache.head_dim / 32;
    const float* from = (p.values ? a.values + p.row * a.value_stride : a.keys + p.row * a.key_stride) +
                        static_cast<uint64_t>(p.head) * a.cache.head_dim + 32 * p.block + 4 * p.lane;
    float4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.live) x = *reinterpret_cast<const float4*>(from);
    uint32_t code[4];
    const uint32_t d = quantize<F>(x, p.lane, p.values, code);
    // Q4_0: a byte holds values 4 apart of a key, 16 apart of a value: the
    // lower lane of the two takes the other's nibbles
    uint32_t theirs[4] = {0, 0, 0, 0};
    if constexpr (F == kQ4_0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) theirs[e] = __shfl_xor(code[e], p.values ? 4 : 1, 8);
    }
    if (!p.live) return;

    uint8_t* record = record_of(a.cache, F, p.sequence, p.head, p.slot / kTile);
    const Slot s = slot_of(static_cast<uint32_t>(p.slot % kTile));
    if (!p.values) {
        uint8_t* unit = record + p.block * cache_unit(F);
        const uint32_t lane = (p.lane / 2) * 16 + s.column, odd = p.lane & 1u;
        if constexpr (F == kQ8_0) {
            *reinterpret_cast<uint32_t*>(unit + 16 * lane + 8 * s.half + 4 * odd) = pack4(code);
        } else if constexpr (F == kQ4_0) {
            if (!odd) *reinterpret_cast<uint32_t*>(unit + 8 * lane + 4 * s.half) = pack4(code) | pack4(theirs) << 4;
        } else {
            *reinterpret_cast<uint2*>(unit + 1024 * s.half + 16 * lane + 8 * odd) =
                make_uint2(code[0] | code[1] << 16, code[2] | code[3] << 16);
        }
    } else {
        uint8_t* unit = record + values_at(F, blocks) + p.block * cache_unit(F);
        const uint32_t lane = s.group * 16 + 4 * (p.lane & 3u), u = p.lane / 4;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            if constexpr (F == kQ8_0) {
                unit[16 * (lane + e) + 8 * u + s.index] = static_cast<uint8_t>(code[e]);
            } else if constexpr (F == kQ4_0) {
                if (u == 0) unit[8 * (lane + e) + s.index] = static_cast<uint8_t>(code[e] | theirs[e] << 4);
            } else {
                *reinterpret_cast<uint16_t*>(unit + 1024 * u + 16 * (lane + e) + 2 * s.index) =
                    static_cast<uint16_t>(code[e]);
            }
        }
    }
    if (p.lane == 0 && (p.values || key_scales(F))) {
        uint8_t* scales = record + (p.values ? value_scales_at(F, blocks) : key_scales_at(F, blocks)) + 64 * p.block;
        reinterpret_cast<uint16_t*>(scales)[8 * s.group + s.index] = static_cast<uint16_t>(d);
    }
}

template <uint32_t F>
__global__ __launch_bounds__(256) void cache_read(CacheRows a) {
    const Piece p = piece_of(a);
    if (!p.live) return;
    const uint32_t blocks = a.cache.head_dim / 32;
    const uint8_t* record = record_of(a.cache, F, p.sequence, p.head, p.slot / kTile);
    const Slot s = slot_of(static_cast<uint32_t>(p.slot % kTile));
    uint32_t code[4];
    if (!p.values) {
        const uint8_t* unit = record + p.block * cache_unit(F);
        const uint32_t lane = (p.lane / 2) * 16 + s.column, odd = p.lane & 1u;
        if constexpr (F == kF16) {
            const uint2 w = *reinterpret_cast<const uint2*>(unit + 1024 * s.half + 16 * lane + 8 * odd);
            code[0] = w.x & 0xFFFFu, code[1] = w.x >> 16, code[2] = w.y & 0xFFFFu, code[3] = w.y >> 16;
        } else {
            const uint32_t w = F == kQ8_0
                                   ? *reinterpret_cast<const uint32_t*>(unit + 16 * lane + 8 * s.half + 4 * odd)
                                   : *reinterpret_cast<const uint32_t*>(unit + 8 * lane + 4 * s.half) >> (4 * odd);
#pragma unroll
            for (int e = 0; e < 4; ++e) code[e] = w >> (8 * e) & (F == kQ8_0 ? 0xFFu : 0xFu);
        }
    } else {
        const uint8_t* unit = record + values_at(F, blocks) + p.block * cache_unit(F);
        const uint32_t lane = s.group * 16 + 4 * (p.lane & 3u), u = p.lane / 4;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            if constexpr (F == kQ8_0)
                code[e] = unit[16 * (lane + e) + 8 * u + s.index];
            else if constexpr (F == kQ4_0)
                code[e] = unit[8 * (lane + e) + s.index] >> (4 * u) & 0xFu;
            else
                code[e] = *reinterpret_cast<const uint16_t*>(unit + 1024 * u + 16 * (lane + e) + 2 * s.index);
        }
    }
    float d = 1.0f;
    if (p.values || key_scales(F)) {
        const uint8_t* scales = record + (p.values ? value_scales_at(F, blocks) : key_scales_at(F, blocks)) + 64 * p.block;
        d = half_to_float(reinterpret_cast<const uint16_t*>(scales)[8 * s.group + s.index]);
    }
    float x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (F == kF16)
            x[e] = half_to_float(code[e]) * d;
        else
            x[e] = static_cast<float>(static_cast<int>(code[e]) - (F == kQ8_0 ? 128 : 8)) * d;
    }
    float* to = const_cast<float*>(p.values ? a.values + p.row * a.value_stride : a.keys + p.row * a.key_stride) +
                static_cast<uint64_t>(p.head) * a.cache.head_dim + 32 * p.block + 4 * p.lane;
    *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
}

// keep: a workgroup a head of a sequence, a thread a byte run of a token
// (four codes of a key, a byte or half of a value, a scale), 16 path entries
// at a time: all of them read, then all written. An entry's destination lies
// at or before its own source, and before every later entry's, so a batch's
// writes reach no later batch's source.
constexpr uint32_t kKeepBatch = 16;

// The path's entries a sequence moves: rising, inside the step and the capacity.
__device__ __forceinline__ uint32_t path_length(const CacheKeep& a, uint32_t sequence) {
    uint32_t most = a.count[sequence];
    if (most > a.tokens) most = a.tokens;
    const uint64_t past = a.past[sequence];
    const int32_t* path = a.path + static_cast<uint64_t>(sequence) * a.tokens;
    int32_t before = -1;
    for (uint32_t j = 0; j < most; ++j) {
        if (path[j] <= before || past + static_cast<uint32_t>(path[j]) >= a.cache.capacity) return j;
        before = path[j];
    }
    return most;
}

template <uint32_t F>
__global__ __launch_bounds__(256) void cache_keep(CacheKeep a) {
    const uint32_t sequence = blockIdx.x / a.cache.kv_heads, head = blockIdx.x % a.cache.kv_heads;
    const uint32_t blocks = a.cache.head_dim / 32;
    __shared__ uint32_t length;
    if (threadIdx.x == 0) length = path_length(a, sequence);
    __syncthreads();
    const uint64_t past = a.past[sequence];
    const int32_t* path = a.path + static_cast<uint64_t>(sequence) * a.tokens;

    // A block's parts: 8 key words (4 codes of Q8_0; 8 of Q4_0, 4 words; half
    // pairs of F16, 16), 16 or 32 value units, 1 or 2 scales.
    constexpr uint32_t kKeyWords = F == kQ8_0 ? 8u : F == kQ4_0 ? 4u : 16u;
    constexpr uint32_t kValueUnits = F == kQ4_0 ? 16u : 32u;
    constexpr uint32_t kScales = key_scales(F) ? 2u : 1u;
    constexpr uint32_t kParts = kKeyWords + kValueUnits + kScales;

    // the address of part `part` of block `block` for a slot, and its width
    auto place = [&](uint64_t slot, uint32_t block, uint32_t part, uint32_t* width) -> uint8_t* {
        uint8_t* record = record_of(a.cache, F, sequence, head, slot / kTile);
        const Slot s = slot_of(static_cast<uint32_t>(slot % kTile));
        if (part < kKeyWords) {
            uint8_t* unit = record + block * cache_unit(F);
            *width = 4;
            if constexpr (F == kQ8_0)
                return unit + 16 * ((part / 2) * 16 + s.column) + 8 * s.half + 4 * (part & 1u);
            else if constexpr (F == kQ4_0)
                return unit + 8 * (part * 16 + s.column) + 4 * s.half;
            else
                return unit + 1024 * s.half + 16 * ((part / 4) * 16 + s.column) + 4 * (part & 3u);
        }
        part -= kKeyWords;
        if (part < kValueUnits) {
            uint8_t* unit = record + values_at(F, blocks) + block * cache_unit(F);
            const uint32_t lane = s.group * 16 + (part & 15u), u = part / 16;
            *width = F == kF16 ? 2 : 1;
            if constexpr (F == kQ8_0)
                return unit + 16 * lane + 8 * u + s.index;
            else if constexpr (F == kQ4_0)
                return unit + 8 * lane + s.index;
            else
                return unit + 1024 * u + 16 * lane + 2 * s.index;
        }
        part -= kValueUnits;
        *width = 2;
        const uint32_t scales = part == 0 ? value_scales_at(F, blocks) : key_scales_at(F, blocks);
        return record + scales + 64 * block + 2 * (8 * s.group + s.index);
    };

    for (uint32_t j0 = 0; j0 < length; j0 += kKeepBatch) {
        const uint32_t batch = min(kKeepBatch, length - j0);
        // blocks x parts threads' worth of columns: whole passes, every thread in each barrier
        for (uint32_t c0 = 0; c0 < blocks * kParts; c0 += 256) {
            const uint32_t c = c0 + threadIdx.x;
            const bool mine = c < blocks * kParts;
            const uint32_t block = mine ? c / kParts : 0u, part = mine ? c % kParts : 0u;
            uint32_t held[kKeepBatch];
#pragma unroll
            for (uint32_t j = 0; j < kKeepBatch; ++j) {
                held[j] = 0;
                if (!mine || j >= batch) continue;
                uint32_t width;
                const uint8_t* from = place(past + static_cast<uint32_t>(path[j0 + j]), block, part, &width);
                held[j] = width == 4   ? *reinterpret_cast<const uint32_t*>(from)
                          : width == 2 ? *reinterpret_cast<const uint16_t*>(from)
                                       : *from;
            }
            // a column is one thread's alone: its reads are before its writes
#pragma unroll
            for (uint32_t j = 0; j < kKeepBatch; ++j) {
                if (!mine || j >= batch) continue;
                uint32_t width;
                uint8_t* to = place(past + j0 + j, block, part, &width);
                if (width == 4)
                    *reinterpret_cast<uint32_t*>(to) = held[j];
                else if (width == 2)
                    *reinterpret_cast<uint16_t*>(to) = static_cast<uint16_t>(held[j]);
                else
                    *to = static_cast<uint8_t>(held[j]);
            }
        }
    }
}

template <typename A>
static dim3 rows_grid(const A& a) {
    const uint64_t blocks = uint64_t{a.cache.sequences} * a.tokens * a.cache.kv_heads * (a.cache.head_dim / 32);
    return dim3(static_cast<uint32_t>((blocks * 8 + 255) / 256), 2);
}

hipError_t launch_cache_append(const CacheRows& a, hipStream_t stream) {
    switch (a.cache.format) {
        case kF16: hipLaunchKernelGGL(cache_append<kF16>, rows_grid(a), dim3(256), 0, stream, a); break;
        case kQ4_0: hipLaunchKernelGGL(cache_append<kQ4_0>, rows_grid(a), dim3(256), 0, stream, a); break;
        case kQ8_0: hipLaunchKernelGGL(cache_append<kQ8_0>, rows_grid(a), dim3(256), 0, stream, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_cache_read(const CacheRows& a, hipStream_t stream) {
    switch (a.cache.format) {
        case kF16: hipLaunchKernelGGL(cache_read<kF16>, rows_grid(a), dim3(256), 0, stream, a); break;
        case kQ4_0: hipLaunchKernelGGL(cache_read<kQ4_0>, rows_grid(a), dim3(256), 0, stream, a); break;
        case kQ8_0: hipLaunchKernelGGL(cache_read<kQ8_0>, rows_grid(a), dim3(256), 0, stream, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_cache_keep(const CacheKeep& a, hipStream_t stream) {
    const dim3 grid(a.cache.sequences * a.cache.kv_heads);
    switch (a.cache.format) {
        case kF16: hipLaunchKernelGGL(cache_keep<kF16>, grid, dim3(256), 0, stream, a); break;
        case kQ4_0: hipLaunchKernelGGL(cache_keep<kQ4_0>, grid, dim3(256), 0, stream, a); break;
        case kQ8_0: hipLaunchKernelGGL(cache_keep<kQ8_0>, grid, dim3(256), 0, stream, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace chm
