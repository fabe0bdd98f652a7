// The quantized cache (its layout: cache.hpp): tokens written as they are
// quantized, slots read back, an accepted path's slots moved together.
//
// A few tokens (cache_append, cache_read): eight lanes a block of 32 values,
// four values a lane, so the f32 side is read or written in whole 128-byte
// runs and the block's largest magnitude is three shuffles. A key's four codes
// of a lane are neighbours in the record, a value's are in four lanes' operands,
// each stored alone.
//
// From half a tile's worth of tokens on (append_units; read_units from a whole
// one): a wave a unit - a block's 32 values of a tile's 32 tokens - each lane
// with the codes that the unit has at its place, so that the record is read and
// written in whole runs too; the largest magnitudes are over 4 lanes (keys) or 16
// (values). A unit that the step covers in part keeps its other tokens' codes.
//
// Bound by bytes: 4 a value on the f32 side and the codes. 2 sequences of 2,048
// tokens, 8 heads of 128, keys and values: into Q8_0 (42 MB) 9.6 us by units, 20.3
// by tokens; Q4_0 9.4 and 15.9; F16 9.4 and 31.1; read back 9.2 - 10.6 and 14.4 -
// 23.3 (a copy of as many bytes 6.5 - 7.3). 32 sequences of 16 tokens: 4.9 and 5.7,
// 5.1 and 5.2, 4.7 and 7.0; read back 4.4 - 5.2 by units, 4.4 - 4.5 by tokens. Up to
// 256 tokens of one sequence either is a launch's latency (3 us).
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
    const uint32_t id = (blockIdx.x * 256 + threadIdx.x) / 8;  // a launch has below 2^32 threads
    const uint32_t blocks = a.cache.head_dim / 32, row_blocks = blocks * a.cache.kv_heads;
    p.lane = threadIdx.x & 7u;
    p.values = blockIdx.y != 0;
    const uint32_t in_row = id % row_blocks;
    p.head = in_row / blocks;
    p.block = in_row % blocks;
    const uint32_t row = id / row_blocks, sequence = row / a.tokens;
    p.row = row;
    p.live = sequence < a.cache.sequences;
    p.sequence = p.live ? sequence : 0u;
    p.slot = static_cast<uint64_t>(a.first[p.sequence]) + row % a.tokens;
    p.live = p.live && p.slot < a.cache.capacity;
    return p;
}

__device__ __forceinline__ uint32_t pack4(const uint32_t c[4]) { return c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24; }
__device__ __forceinline__ uint32_t half_bits(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
}

constexpr uint32_t kNanHalf = 0x7E00u;

// A block's scale as f16 bits, from its largest magnitude's bits (a NaN's rank
// above every number's) and whether the first value of it is negative. F16:
// one, or a NaN.
template <uint32_t F>
__device__ __forceinline__ uint32_t scale_of(uint32_t largest, bool negative) {
    const float most = __uint_as_float(largest);
    if constexpr (F == kF16) return (half_bits(most) & 0x7C00u) == 0x7C00u ? kNanHalf : 0x3C00u;
    const uint32_t d = half_bits(F == kQ8_0 ? most / 127.0f : (negative ? most : -most) / 8.0f);
    return (d & 0x7C00u) == 0x7C00u ? kNanHalf : d;
}

// A scale as the codes are found by it: d and 1 / d, both 0 where every code is.
// 1 / d, rounded to nearest, is one Newton step on the reciprocal instruction
// (for every one of binary16's scales; the tests go through them all).
struct Step {
    float d, inverse;
};
__device__ __forceinline__ Step step_of(uint32_t scale) {
    const float d = half_to_float(scale);
    if (d == 0.0f || scale == kNanHalf) return {0.0f, 0.0f};
    const float y = __builtin_amdgcn_rcpf(d);
    return {d, __builtin_fmaf(__builtin_fmaf(-d, y, 1.0f), y, y)};
}

// The code nearest to x / d, ties to even, raised to be unsigned; F16's is the
// half. The quotient is rounded once: with 1 / d rounded to nearest, q = x (1 /
// d) corrected by its exact remainder is x / d rounded to nearest (Markstein).
// It is rounded to a whole number, and raised, as the last bits of a float of
// 1.5 * 2^23 (the bounds are whole, so the clamp may come first).
template <uint32_t F>
__device__ __forceinline__ uint32_t code_of(float x, const Step& step, uint32_t scale, bool values) {
    if constexpr (F == kF16) return scale != kNanHalf ? half_bits(x) : values ? 0u : kNanHalf;
    constexpr float kLow = F == kQ8_0 ? -127.0f : -8.0f, kHigh = F == kQ8_0 ? 127.0f : 7.0f;
    const float y = step.d == 0.0f ? 0.0f : x;  // what a block that is not held has may be a NaN
    const float guess = y * step.inverse;
    const float q = __builtin_fmaf(__builtin_fmaf(-guess, step.d, y), step.inverse, guess);
    constexpr float kRaise = 12582912.0f + (F == kQ8_0 ? 128.0f : 8.0f);
    return __float_as_uint(__builtin_amdgcn_fmed3f(q, kLow, kHigh) + kRaise) & (F == kQ8_0 ? 0xFFu : 0xFu);
}

template <uint32_t F>
__device__ __forceinline__ float value_of(uint32_t code, float d) {
    return F == kF16 ? half_to_float(code) * d : static_cast<float>(static_cast<int>(code) - (F == kQ8_0 ? 128 : 8)) * d;
}

__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// What the block's lanes find the sign of its largest magnitude by: the least of
// twice the place of a value of it plus whether it is negative.
__device__ __forceinline__ uint32_t place_of(float x, uint32_t largest, uint32_t place) {
    return magnitude(x) == largest ? 2 * place + (__float_as_uint(x) >> 31) : 0xFFu;
}

// A lane's four codes and its block's scale; every lane of the block calls it.
template <uint32_t F>
__device__ __forceinline__ uint32_t quantize(const float4& v, uint32_t lane, bool values, uint32_t code[4]) {
    const float x[4] = {v.x, v.y, v.z, v.w};
    uint32_t largest = max(max(magnitude(x[0]), magnitude(x[1])), max(magnitude(x[2]), magnitude(x[3])));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), o, 8)));
    uint32_t place = 0;
    if constexpr (F == kQ4_0) {
        place = 0xFFu;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) place = min(place, place_of(x[e], largest, 4 * lane + e));
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) place = min(place, static_cast<uint32_t>(__shfl_xor(static_cast<int>(place), o, 8)));
    }
    const uint32_t d = scale_of<F>(largest, place & 1u);
    const Step step = step_of(d);
#pragma unroll
    for (int e = 0; e < 4; ++e) code[e] = code_of<F>(x[e], step, d, values);
    return d;
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
    for (int e = 0; e < 4; ++e) x[e] = value_of<F>(code[e], d);
    float* to = const_cast<float*>(p.values ? a.values + p.row * a.value_stride : a.keys + p.row * a.key_stride) +
                static_cast<uint64_t>(p.head) * a.cache.head_dim + 32 * p.block + 4 * p.lane;
    *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
}

// ---- whole units ---------------------------------------------------------------

// Over the 16 lanes of a row (values) or the four lanes 16 apart (keys).
template <bool VALUES>
__device__ __forceinline__ uint32_t most_of_block(uint32_t x) {
    if constexpr (VALUES) {
        x = max(x, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x121, 0xF, 0xF, true)));
        x = max(x, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x122, 0xF, 0xF, true)));
        x = max(x, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x124, 0xF, 0xF, true)));
        return max(x, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x128, 0xF, 0xF, true)));
    } else {
        const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = max(a[0], a[1]);
        const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return max(b[0], b[1]);
    }
}

// Lane t of each row of 16, in all of its lanes.
__device__ __forceinline__ uint32_t of_lane(uint32_t x, uint32_t t) {
    const int v = static_cast<int>(x);
    switch (t) {  // (an operand of the instruction)
        case 0: return __builtin_amdgcn_mov_dpp(v, 0x150, 0xF, 0xF, true);
        case 1: return __builtin_amdgcn_mov_dpp(v, 0x151, 0xF, 0xF, true);
        case 2: return __builtin_amdgcn_mov_dpp(v, 0x152, 0xF, 0xF, true);
        case 3: return __builtin_amdgcn_mov_dpp(v, 0x153, 0xF, 0xF, true);
        case 4: return __builtin_amdgcn_mov_dpp(v, 0x154, 0xF, 0xF, true);
        case 5: return __builtin_amdgcn_mov_dpp(v, 0x155, 0xF, 0xF, true);
        case 6: return __builtin_amdgcn_mov_dpp(v, 0x156, 0xF, 0xF, true);
        default: return __builtin_amdgcn_mov_dpp(v, 0x157, 0xF, 0xF, true);
    }
}

// A wave's unit, its lane's 16 values in it and which of them the step holds.
// Value e of token part p: keys - value 8 (lane / 16) + e of token 16p + lane % 16
// (in memory, `exchange`, 4 (lane / 16) + e, and 16 further on for e >= 4, so that
// a wave's load or store has 64 bytes of each token); values - value 16p + lane %
// 16 of the token of slot e of group lane / 16.
template <bool VALUES>
struct Unit {
    uint32_t sequence, head, block, lane;
    uint64_t tile;
    int32_t ahead;    // the tile's first slot, counted from the step's first
    uint32_t limit;   // the step's tokens that have slots
    bool live, whole;
    float* first;     // the lane's first value at the tile's first token
    uint64_t stride;

    __device__ __forceinline__ explicit Unit(const CacheRows& a, uint32_t tiles) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t id = blockIdx.x * 4 + wave;
        const uint32_t blocks = a.cache.head_dim / 32, units = blocks * a.cache.kv_heads;
        lane = threadIdx.x & 63u;
        const uint32_t at = id / units;  // sequence, tile
        head = id % units / blocks;
        block = id % units % blocks;
        live = at / tiles < a.cache.sequences;
        sequence = live ? at / tiles : 0u;
        const uint32_t past = a.first[sequence];
        tile = uint64_t{past / kTile} + at % tiles;
        limit = past < a.cache.capacity ? min(a.tokens, a.cache.capacity - past) : 0u;
        const int64_t from = static_cast<int64_t>(tile * kTile) - past;
        live = live && limit > 0 && from < limit;  // a step past the capacity has no unit at all
        ahead = static_cast<int32_t>(from);
        whole = ahead >= 0 && ahead + static_cast<int32_t>(kTile) <= static_cast<int32_t>(limit);
        stride = VALUES ? a.value_stride : a.key_stride;
        const int64_t row = static_cast<int64_t>(static_cast<uint64_t>(sequence) * a.tokens) + ahead +
                            (VALUES ? 4 * (lane >> 4) : lane & 15u);
        first = const_cast<float*>(VALUES ? a.values : a.keys) + row * static_cast<int64_t>(stride) +
                static_cast<uint64_t>(head) * a.cache.head_dim + 32 * block + (VALUES ? lane & 15u : 4 * (lane >> 4));
    }
    // a token of the tile: past the lane's first one
    __device__ __forceinline__ static uint32_t token(uint32_t part, uint32_t e) { return VALUES ? 16 * (e >> 2) + (e & 3) : 16 * part; }
    __device__ __forceinline__ bool inside(uint32_t part, uint32_t e) const {
        const uint32_t mine = VALUES ? 4 * (lane >> 4) : lane & 15u;
        return static_cast<uint32_t>(ahead + static_cast<int32_t>(mine + token(part, e))) < limit;
    }
    // where it is one of the step's
    __device__ __forceinline__ float* row(uint32_t part, uint32_t e) const {
        return first + token(part, e) * stride + (VALUES ? 16 * part : 0u);
    }
};

// Of four lanes 16 apart, g their number: values 8g .. 8g + 7 (a, then b) to and
// from values 4g .. 4g + 3 (a) and 16 + 4g .. 16 + 4g + 3 (b).
__device__ __forceinline__ void exchange(float4& a, float4& b, bool to_memory) {
    float x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t u = __float_as_uint(x[e]), v = __float_as_uint(y[e]);
        auto swap16 = [&] {
            const auto s = __builtin_amdgcn_permlane16_swap(u, v, false, false);
            u = s[0], v = s[1];
        };
        auto swap32 = [&] {
            const auto s = __builtin_amdgcn_permlane32_swap(u, v, false, false);
            u = s[0], v = s[1];
        };
        if (to_memory)
            swap16(), swap32();
        else
            swap32(), swap16();
        x[e] = __uint_as_float(u), y[e] = __uint_as_float(v);
    }
    a = {x[0], x[1], x[2], x[3]}, b = {y[0], y[1], y[2], y[3]};
}

// A lane's codes as its unit holds them: Q8_0 16 bytes, 8 a part; Q4_0 8 bytes;
// F16 16 bytes a part, 1,024 apart. And a mask of those that a code covers.
template <uint32_t F, bool VALUES>
__device__ __forceinline__ void pack(const uint32_t (&code)[2][8], uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (F == kQ8_0)
                w[2 * p + (e >> 2)] |= code[p][e] << (8 * (e & 3));
            else if constexpr (F == kF16)
                w[4 * p + (e >> 1)] |= code[p][e] << (16 * (e & 1));
            else if constexpr (VALUES)
                w[e >> 2] |= code[p][e] << (8 * (e & 3) + 4 * p);
            else
                w[p] |= code[p][e] << (8 * (e & 3) + 4 * (e >> 2));
        }
}
template <uint32_t F, bool VALUES>
__device__ __forceinline__ void unpack(const uint32_t (&w)[8], uint32_t (&code)[2][8]) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (F == kQ8_0)
                code[p][e] = w[2 * p + (e >> 2)] >> (8 * (e & 3)) & 0xFFu;
            else if constexpr (F == kF16)
                code[p][e] = w[4 * p + (e >> 1)] >> (16 * (e & 1)) & 0xFFFFu;
            else if constexpr (VALUES)
                code[p][e] = w[e >> 2] >> (8 * (e & 3) + 4 * p) & 0xFu;
            else
                code[p][e] = w[p] >> (8 * (e & 3) + 4 * (e >> 2)) & 0xFu;
        }
}
template <uint32_t F>
__device__ __forceinline__ void load_unit(const uint8_t* unit, uint32_t lane, uint32_t (&w)[8]) {
    if constexpr (F == kQ4_0) {
        const uint2 v = *reinterpret_cast<const uint2*>(unit + 8 * lane);
        w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
        for (int p = 0; p < (F == kF16 ? 2 : 1); ++p) {
            const uint4 v = *reinterpret_cast<const uint4*>(unit + 1024 * p + 16 * lane);
            w[4 * p] = v.x, w[4 * p + 1] = v.y, w[4 * p + 2] = v.z, w[4 * p + 3] = v.w;
        }
    }
}
template <uint32_t F>
__device__ __forceinline__ void store_unit(uint8_t* unit, uint32_t lane, const uint32_t (&w)[8]) {
    if constexpr (F == kQ4_0) {
        *reinterpret_cast<uint2*>(unit + 8 * lane) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int p = 0; p < (F == kF16 ? 2 : 1); ++p)
            *reinterpret_cast<uint4*>(unit + 1024 * p + 16 * lane) = make_uint4(w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]);
    }
}

template <uint32_t F, bool VALUES>
__device__ __forceinline__ void append_unit(const CacheRows& a, uint32_t tiles) {
    const Unit<VALUES> u(a, tiles);
    if (!u.live) return;
    float x[2][8];
#pragma unroll
    for (uint32_t p = 0; p < 2; ++p) {
        if constexpr (VALUES) {
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) x[p][e] = u.whole || u.inside(p, e) ? *u.row(p, e) : 0.0f;
        } else {
            float4 v = {0.0f, 0.0f, 0.0f, 0.0f}, w = v;
            if (u.whole || u.inside(p, 0)) {
                const float4* from = reinterpret_cast<const float4*>(u.row(p, 0));
                v = from[0], w = from[4];
            }
            exchange(v, w, false);
            x[p][0] = v.x, x[p][1] = v.y, x[p][2] = v.z, x[p][3] = v.w;
            x[p][4] = w.x, x[p][5] = w.y, x[p][6] = w.z, x[p][7] = w.w;
        }
    }
    // A block is a token's: for the keys a part, over its eight values here and
    // three more lanes'; for the values a slot, over both parts and 15 more lanes'.
    constexpr uint32_t kBlocks = VALUES ? 8 : 2, kHere = VALUES ? 2 : 8;
    auto value = [&](uint32_t t, uint32_t i) { return VALUES ? x[i][t] : x[t][i]; };
    // Twice the largest magnitude, plus, Q4_0, whether the first value of it is
    // negative: where only one sign has it, the largest of the values' bits with
    // the sign put last. (Both signs' is as rare as +m and -m in a block; ~0 is a
    // NaN, in a block that is not held.)
    uint32_t most[kBlocks];
    bool both = false;
#pragma unroll
    for (uint32_t t = 0; t < kBlocks; ++t) {
        uint32_t largest = 0;
#pragma unroll
        for (uint32_t i = 0; i < kHere; ++i) {
            const uint32_t bits = __float_as_uint(value(t, i));
            largest = max(largest, F == kQ4_0 ? __builtin_amdgcn_alignbit(bits, bits, 31) : bits & 0x7FFFFFFFu);
        }
        largest = most_of_block<VALUES>(largest);
        most[t] = F == kQ4_0 ? largest : largest << 1;
        if constexpr (F == kQ4_0) {
            const uint32_t other = largest & 1u ? largest >> 1 : ~0u;
#pragma unroll
            for (uint32_t i = 0; i < kHere; ++i) both |= __float_as_uint(value(t, i)) == other;
        }
    }
    if (F == kQ4_0 && __any(both)) {
#pragma unroll
        for (uint32_t t = 0; t < kBlocks; ++t) {
            uint32_t place = 0;
#pragma unroll
            for (uint32_t i = 0; i < kHere; ++i)
                place = max(place, 0xFFu - place_of(value(t, i), most[t] >> 1, VALUES ? 16 * i + (u.lane & 15u) : 8 * (u.lane >> 4) + i));
            most[t] = (most[t] & ~1u) | ((0xFFu - most_of_block<VALUES>(place)) & 1u);
        }
    }
    // Their scales: of the values lane t of a row of 16 finds token t's, for all of it.
    constexpr uint32_t kOwn = VALUES ? 1 : 2;
    uint32_t own_scale[kOwn];
    Step own[kOwn];
#pragma unroll
    for (uint32_t t = 0; t < kOwn; ++t) {
        uint32_t mine = most[t];
        if constexpr (VALUES)
#pragma unroll
            for (uint32_t e = 1; e < 8; ++e) mine = (u.lane & 7u) == e ? most[e] : mine;
        own_scale[t] = scale_of<F>(mine >> 1, mine & 1u);
        own[t] = step_of(own_scale[t]);
    }
    uint32_t code[2][8];
#pragma unroll
    for (uint32_t t = 0; t < kBlocks; ++t) {
        Step step;
        uint32_t scale;
        if constexpr (VALUES) {
            step.d = __uint_as_float(of_lane(__float_as_uint(own[0].d), t));
            step.inverse = __uint_as_float(of_lane(__float_as_uint(own[0].inverse), t));
            scale = of_lane(own_scale[0], t);
        } else {
            step = own[t], scale = own_scale[t];
        }
#pragma unroll
        for (uint32_t i = 0; i < kHere; ++i) (VALUES ? code[i][t] : code[t][i]) = code_of<F>(value(t, i), step, scale, VALUES);
    }

    const uint32_t blocks = a.cache.head_dim / 32;
    uint8_t* record = record_of(a.cache, F, u.sequence, u.head, u.tile);
    uint8_t* unit = record + (VALUES ? values_at(F, blocks) : 0u) + u.block * cache_unit(F);
    uint32_t w[8];
    pack<F, VALUES>(code, w);
    if (!u.whole) {  // other tokens' codes stay
        uint32_t old[8], old_code[2][8];
        load_unit<F>(unit, u.lane, old);
        unpack<F, VALUES>(old, old_code);
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int e = 0; e < 8; ++e) code[p][e] = u.inside(p, e) ? code[p][e] : old_code[p][e];
        pack<F, VALUES>(code, w);
    }
    store_unit<F>(unit, u.lane, w);

    if constexpr (VALUES) {
        const uint32_t e = u.lane & 15u;
        if (e < 8 && (u.whole || u.inside(0, e)))  // a group's eight tokens
            reinterpret_cast<uint16_t*>(record + value_scales_at(F, blocks) + 64 * u.block)[8 * (u.lane >> 4) + e] =
                static_cast<uint16_t>(own_scale[0]);
    } else if constexpr (key_scales(F)) {
        if (u.lane < 16) {
            uint16_t* scales = reinterpret_cast<uint16_t*>(record + key_scales_at(F, blocks) + 64 * u.block);
#pragma unroll
            for (int p = 0; p < 2; ++p)
                if (u.whole || u.inside(p, 0)) scales[8 * (u.lane >> 2) + 4 * p + (u.lane & 3u)] = static_cast<uint16_t>(own_scale[p]);
        }
    }
}

template <uint32_t F, bool VALUES>
__device__ __forceinline__ void read_unit(const CacheRows& a, uint32_t tiles) {
    const Unit<VALUES> u(a, tiles);
    if (!u.live) return;
    const uint32_t blocks = a.cache.head_dim / 32;
    const uint8_t* record = record_of(a.cache, F, u.sequence, u.head, u.tile);
    uint32_t w[8], code[2][8];
    load_unit<F>(record + (VALUES ? values_at(F, blocks) : 0u) + u.block * cache_unit(F), u.lane, w);
    uint16_t d[8];
    if constexpr (VALUES || key_scales(F)) {
        const uint16_t* scales = reinterpret_cast<const uint16_t*>(
            record + (VALUES ? value_scales_at(F, blocks) : key_scales_at(F, blocks)) + 64 * u.block);
        if constexpr (VALUES) {
            const uint4 v = *reinterpret_cast<const uint4*>(scales + 8 * (u.lane >> 4));
            d[0] = v.x, d[1] = v.x >> 16, d[2] = v.y, d[3] = v.y >> 16, d[4] = v.z, d[5] = v.z >> 16, d[6] = v.w, d[7] = v.w >> 16;
        } else {
            const uint32_t token = u.lane & 15u;
            d[0] = scales[8 * (token >> 2) + (token & 3u)], d[1] = scales[8 * (token >> 2) + 4 + (token & 3u)];
        }
    }
    unpack<F, VALUES>(w, code);
#pragma unroll
    for (uint32_t p = 0; p < 2; ++p) {
        if constexpr (VALUES) {
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e)
                if (u.whole || u.inside(p, e)) *u.row(p, e) = value_of<F>(code[p][e], half_to_float(d[e]));
        } else {
            const float by = key_scales(F) ? half_to_float(d[p]) : 1.0f;
            float4 v = make_float4(value_of<F>(code[p][0], by), value_of<F>(code[p][1], by), value_of<F>(code[p][2], by),
                                   value_of<F>(code[p][3], by));
            float4 w = make_float4(value_of<F>(code[p][4], by), value_of<F>(code[p][5], by), value_of<F>(code[p][6], by),
                                   value_of<F>(code[p][7], by));
            exchange(v, w, true);
            if (!u.whole && !u.inside(p, 0)) continue;
            float4* to = reinterpret_cast<float4*>(u.row(p, 0));
            to[0] = v, to[4] = w;
        }
    }
}

template <uint32_t F>
__global__ __launch_bounds__(256) void append_units(CacheRows a, uint32_t tiles) {
    if (blockIdx.y == 0)
        append_unit<F, false>(a, tiles);
    else
        append_unit<F, true>(a, tiles);
}
template <uint32_t F>
__global__ __launch_bounds__(256) void read_units(CacheRows a, uint32_t tiles) {
    if (blockIdx.y == 0)
        read_unit<F, false>(a, tiles);
    else
        read_unit<F, true>(a, tiles);
}

// keep: a workgroup a head of a sequence, a thread a byte run of a token
// (four codes of a key, a byte or half of a value, a scale), 16 path entries
// at a time: all of them read, then all written. An entry's destination lies
// at or before its own source, and before every later entry's, so a batch's
// writes reach no later batch's source.
constexpr uint32_t kKeepBatch = 16;

// The path's entries a sequence moves: rising, their slots inside the capacity.
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

// From how many tokens on (both sides' times: above).
constexpr uint32_t kAppendUnits = 16, kReadUnits = 32;

template <uint32_t F>
static void launch_rows(const CacheRows& a, bool read, hipStream_t stream) {
    const uint64_t units = uint64_t{a.cache.kv_heads} * (a.cache.head_dim / 32);
    if (a.tokens < (read ? kReadUnits : kAppendUnits)) {
        const uint64_t blocks = uint64_t{a.cache.sequences} * a.tokens * units;
        const dim3 grid(static_cast<uint32_t>((blocks * 8 + 255) / 256), 2);
        if (read)
            hipLaunchKernelGGL(cache_read<F>, grid, dim3(256), 0, stream, a);
        else
            hipLaunchKernelGGL(cache_append<F>, grid, dim3(256), 0, stream, a);
        return;
    }
    const uint32_t tiles = a.tokens / kTile + (a.tokens % kTile > 1 ? 2 : 1);  // touched at the most
    const dim3 grid(static_cast<uint32_t>((a.cache.sequences * uint64_t{tiles} * units + 3) / 4), 2);
    if (read)
        hipLaunchKernelGGL(read_units<F>, grid, dim3(256), 0, stream, a, tiles);
    else
        hipLaunchKernelGGL(append_units<F>, grid, dim3(256), 0, stream, a, tiles);
}

static hipError_t launch_rows(const CacheRows& a, bool read, hipStream_t stream) {
    switch (a.cache.format) {
        case kF16: launch_rows<kF16>(a, read, stream); break;
        case kQ4_0: launch_rows<kQ4_0>(a, read, stream); break;
        case kQ8_0: launch_rows<kQ8_0>(a, read, stream); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_cache_append(const CacheRows& a, hipStream_t stream) { return launch_rows(a, false, stream); }
hipError_t launch_cache_read(const CacheRows& a, hipStream_t stream) { return launch_rows(a, true, stream); }

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
