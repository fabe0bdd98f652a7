// The cache's layout: what the attention's matrix instructions read as their
// operands, in the order in which a lane reads it.
//
// A head of a sequence is whole 32-token tiles, a tile one record:
//   keys' codes    [blocks][UNIT]   UNIT: 32 tokens x 32 values - 512 bytes of
//   values' codes  [blocks][UNIT]   Q4_0, 1,024 of Q8_0, 2,048 of F16
//   keys' scales   [blocks][32 f16]   (quantized formats only)
//   values' scales [blocks][32 f16]
//
// v_mfma_f32_16x16x32_f16 takes, in lane 16g + m, row (or column) m's eight
// operands 8g .. 8g + 7 along the sum. For the keys (rows: 16 tokens, sum: a
// block's 32 values) lane 16g + m reads token m's values 8g .. 8g + 7, for
// the tile's two halves of 16 tokens. Its results give a lane of group g the
// tokens 4g .. 4g + 3 of each half: eight of the tile's tokens, which are its
// operands along the sum when the values are weighted by them. So lane 16g +
// m of the values holds value m (and 16 + m) of a block for the tokens 4g + r
// and 16 + 4g + r, and probabilities never move between lanes. A block's
// scales stand in that same order of tokens, eight a group.
//
//   token t of a tile: half h = t / 16, group g = t % 16 / 4, r = t % 4
//   keys, value v of a block (k = v / 8, e = v % 8), lane 16k + t % 16:
//     Q8_0  byte 16 lane + 8h + e
//     Q4_0  byte 8 lane + 4h + e % 4, the high nibble for e >= 4
//     F16   half 512h + 8 lane + e
//   values, value v (u = v / 16), lane 16g + v % 16, slot i = 4h + r:
//     Q8_0  byte 16 lane + 8u + i
//     Q4_0  byte 8 lane + i, the high nibble for u = 1
//     F16   half 512u + 8 lane + i
//   scales: half 8g + i
// so every load of a wave is one contiguous run, and each byte belongs to one
// token alone. Codes are stored raised to be unsigned (Q8_0 + 128, Q4_0 + 8).
//
// A block that its format cannot hold has the scale NaN and codes of zero; F16
// keys hold the NaNs themselves (a key reaches its own token's scores alone),
// F16 values zeros under a NaN scale (1 otherwise), so that no operand of the
// weighted sum is ever other than finite.
#pragma once

#include "formats.hpp"
#include "serving.hpp"

namespace chm {

constexpr uint32_t kTile = 32;  // tokens a record

__host__ __device__ constexpr uint32_t cache_unit(uint32_t format) {
    return format == kF16 ? 2048u : format == kQ8_0 ? 1024u : 512u;
}
__host__ __device__ constexpr bool key_scales(uint32_t format) { return format != kF16; }
__host__ __device__ constexpr uint32_t cache_record(uint32_t format, uint32_t blocks) {
    return blocks * (2 * cache_unit(format) + (key_scales(format) ? 128u : 64u));
}
__host__ __device__ constexpr uint32_t values_at(uint32_t format, uint32_t blocks) { return blocks * cache_unit(format); }
__host__ __device__ constexpr uint32_t key_scales_at(uint32_t format, uint32_t blocks) {
    return 2 * blocks * cache_unit(format);
}
__host__ __device__ constexpr uint32_t value_scales_at(uint32_t format, uint32_t blocks) {
    return key_scales_at(format, blocks) + (key_scales(format) ? 64u * blocks : 0u);
}

// A token's place in its tile.
struct Slot {
    uint32_t column;  // t % 16: the keys' lane within a group of 16
    uint32_t half;    // h
    uint32_t group;   // g
    uint32_t index;   // i = 4h + r
};
__device__ __forceinline__ Slot slot_of(uint32_t t) {
    return {t & 15u, (t >> 4) & 1u, (t >> 2) & 3u, ((t >> 4) & 1u) * 4 + (t & 3u)};
}

// The record of a slot's tile. The product of sequences, heads, tiles and the
// record passes 32 bits.
__device__ __forceinline__ uint8_t* record_of(const CacheShape& c, uint32_t format, uint32_t sequence, uint32_t head,
                                              uint64_t tile) {
    const uint64_t heads = static_cast<uint64_t>(sequence) * c.kv_heads + head;
    return c.base + (heads * c.tiles + tile) * cache_record(format, c.head_dim / 32);
}

}  // namespace chm
