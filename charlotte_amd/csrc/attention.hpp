// Attention over the quantized cache (its layout: cache.hpp), for one token, a
// tree or a chain of drafted ones, or a prompt's block:
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m)
// in one pass over the visible tokens, m the running maximum: when it grows, the
// sum and the outputs so far are multiplied by exp(m_old - m_new).
//
// The rows of a key head - its queries, of every token of the step - share
// each cached byte: 16 rows by a tile of 32 tokens are two matrix products.
// The scores are taken transposed, tokens as rows, so that a lane's results
// are eight tokens' scores of one query row (row lane % 16), which are its
// operands along the sum of the second product: probabilities stay in the
// lane, and the maximum and the sum of a row are four lanes' (two shuffles).
//
// Precision: activations are f32 and keep their bits. A query, times scale /
// ln 2 and a power of two that puts its largest value in [2^10, 2^11), and a
// probability times a value's scale are each taken as two binary16 parts, hi +
// lo, about 22 bits; a cache's codes are exact in binary16. A block's key scale
// multiplies its product in f32 (F16: none). Sums are f32 throughout.
//
// Range: values' scales, and so the outputs, are held over 2^D, D the exponent
// of the largest scale met; the outputs follow where it grows, as they follow
// the maximum. p is below 2^14 (the offset follows the maximum once a score
// passes it by 2^8, which a tile seldom does) and p d below 2^15, so that the
// parts' steps (2^-24) lie at least 30 bits below the largest.
//
// Split: up to 32 rows of a key head (attend) - the rows one wave holds - a
// workgroup's waves take its tiles in turn, operands straight from the record,
// and are joined in LDS. More rows (attend_rows): each wave has rows of its
// own, and a tile's codes become binary16 operands in LDS once for all of them.
// Where a step has too few rows to fill the card its tiles are split among
// several workgroups, joined by attention_combine.
#pragma once

#include "cache.hpp"
#include "stream.hpp"

namespace chm {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));

typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2E = 1.44269504088896340736f;
// A probability is 2^kHeadroom at the maximum last followed, and a score may go
// kSlack past it; the largest value scale met is 2^kScaleTop to twice it. Their
// product stays below 2^15 (a half ends at 2^16).
constexpr int kHeadroom = 7, kScaleTop = 3;
constexpr float kSlack = 4.0f;

// A lane's codes of one unit (keys or values of a block by 32 tokens).
template <uint32_t F>
struct Codes {
    uint32_t w[F == kQ8_0 ? 4 : F == kQ4_0 ? 2 : 8];
};

template <uint32_t F>
__device__ __forceinline__ Codes<F> load_codes(const uint8_t* unit, uint32_t lane) {
    Codes<F> c;
    if constexpr (F == kQ8_0) {
        const uint4 v = *reinterpret_cast<const uint4*>(unit + 16 * lane);
        c.w[0] = v.x, c.w[1] = v.y, c.w[2] = v.z, c.w[3] = v.w;
    } else if constexpr (F == kQ4_0) {
        const uint2 v = *reinterpret_cast<const uint2*>(unit + 8 * lane);
        c.w[0] = v.x, c.w[1] = v.y;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(unit + 16 * lane);
        const uint4 u = *reinterpret_cast<const uint4*>(unit + 1024 + 16 * lane);
        c.w[0] = v.x, c.w[1] = v.y, c.w[2] = v.z, c.w[3] = v.w;
        c.w[4] = u.x, c.w[5] = u.y, c.w[6] = u.z, c.w[7] = u.w;
    }
    return c;
}

// Four unsigned bytes, each raised by `raise`, as halves: under the high byte
// 0x64 a byte c is 1,024 + c in binary16, and taking 1,024 + raise is exact.
template <int RAISE>
__device__ __forceinline__ void halves_of(uint32_t bytes, half2_t* low, half2_t* high) {
    const half2_t raise = {static_cast<_Float16>(-1024 - RAISE), static_cast<_Float16>(-1024 - RAISE)};
    *low = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, bytes, 0x04010400u)) + raise;
    *high = __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, bytes, 0x04030402u)) + raise;
}

__device__ __forceinline__ half8_t join(half2_t a, half2_t b, half2_t c, half2_t d) {
    return half8_t{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The lane's operand of a key unit's token half h, or of a value unit's 16
// values u (cache.hpp).
template <uint32_t F, bool VALUES>
__device__ __forceinline__ half8_t operand(const Codes<F>& c, int part) {
    if constexpr (F == kF16) {
        const uint4_t w = {c.w[4 * part], c.w[4 * part + 1], c.w[4 * part + 2], c.w[4 * part + 3]};
        return __builtin_bit_cast(half8_t, w);
    } else {
        half2_t a, b, d, e;
        if constexpr (F == kQ8_0) {
            halves_of<128>(c.w[2 * part], &a, &b);
            halves_of<128>(c.w[2 * part + 1], &d, &e);
        } else if constexpr (VALUES) {
            halves_of<8>(c.w[0] >> (4 * part) & 0x0F0F0F0Fu, &a, &b);
            halves_of<8>(c.w[1] >> (4 * part) & 0x0F0F0F0Fu, &d, &e);
        } else {
            halves_of<8>(c.w[part] & 0x0F0F0F0Fu, &a, &b);
            halves_of<8>(c.w[part] >> 4 & 0x0F0F0F0Fu, &d, &e);
        }
        return join(a, b, d, e);
    }
}

__device__ __forceinline__ float4_t multiply(half8_t a, half8_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// A dword's two halves, the dword passed by value: a bit cast straight from a
// vector's element reads its first.
__device__ __forceinline__ half2_t pair_of(uint32_t w) { return __builtin_bit_cast(half2_t, w); }

// Slot i's scale of a lane's eight, i a constant.
__device__ __forceinline__ float scale_at(const uint4_t& s, int i) { return static_cast<float>(pair_of(s[i >> 1])[i & 1]); }

// Two f32 as two binary16 parts of each: hi, and lo what it leaves, both
// rounded to nearest (lo's bias, were it cut, would be every probability's):
// within 2^-22 of the value, or 2^-25.
__device__ __forceinline__ void split2(float a, float b, half2_t* hi, half2_t* lo) {
    *hi = half2_t{static_cast<_Float16>(a), static_cast<_Float16>(b)};
    *lo = half2_t{static_cast<_Float16>(__builtin_fmaf(static_cast<float>(hi->x), -1.0f, a)),
                  static_cast<_Float16>(__builtin_fmaf(static_cast<float>(hi->y), -1.0f, b))};
}

// The larger of two scales' magnitudes as bits, a NaN's as none.
__device__ __forceinline__ uint32_t larger_scale(uint32_t w) {
    const uint32_t lo = w & 0x7FFFu, hi = w >> 16 & 0x7FFFu;
    return max(lo > 0x7C00u ? 0u : lo, hi > 0x7C00u ? 0u : hi);
}
// D: 2^D <= the scale < 2^(D + 1); any below 2^-12 counts as that.
__device__ __forceinline__ int exponent_of(uint32_t bits) { return static_cast<int>(max(bits >> 10, 3u)) - 15; }
// What a scale is multiplied by, a power of two: from 2^(3 - 15) to 2^(3 + 12), which binary16 holds.
__device__ __forceinline__ half2_t over(int exponent) {
    const _Float16 by = static_cast<_Float16>(ldexpf(1.0f, kScaleTop - exponent));
    return half2_t{by, by};
}

// Over the four lanes that share a row (lane % 16).
__device__ __forceinline__ float most_of_row(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_of_row(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// What lies past the last token is no one's, and may be anything: `kept`
// masks dword w of a lane's eight slots (two a dword) to those before `latest`.
__device__ __forceinline__ uint32_t kept_of(uint32_t slot0, uint32_t g, uint32_t w, uint32_t latest) {
    const uint32_t slot = slot0 + w / 2 * 16 + 4 * g + (w & 1) * 2;
    return slot >= latest ? 0u : slot + 1 >= latest ? 0xFFFFu : 0xFFFFFFFFu;
}
// A scale there reads as never met: zero, or F16's one.
template <uint32_t F>
__device__ __forceinline__ uint32_t kept_scale(uint32_t scale, uint32_t kept) {
    return (scale & kept) | ((F == kF16 ? 0x3C003C00u : 0u) & ~kept);
}

// The step's tree as a workgroup's rows see it: for each of its tokens, the
// tokens above it (itself among them) as bits, and its depth; kUnused where it
// or one above it is unused.
constexpr uint32_t kUnused = 0xFFFFFFFFu;
template <uint32_t TOKENS>
struct Tree {
    int32_t parents[kTreeTokens];
    uint32_t above[TOKENS][kTreeTokens / 32];
    uint32_t depth[TOKENS];
};

// `reach`: the most tokens of a line that a window leaves (0: all).
template <uint32_t TOKENS>
__device__ void read_tree(Tree<TOKENS>& tree, const int32_t* parents, uint32_t tokens, uint32_t first, uint32_t count,
                          uint32_t reach) {
    for (uint32_t i = threadIdx.x; i < tokens; i += blockDim.x) tree.parents[i] = parents[i];
    for (uint32_t i = threadIdx.x; i < TOKENS * (kTreeTokens / 32); i += blockDim.x)
        (&tree.above[0][0])[i] = 0;
    __syncthreads();
    if (threadIdx.x < count) {
        // at most `tokens` steps: a parent not below its token ends the line
        uint32_t steps = 0;
        int32_t node = static_cast<int32_t>(first + threadIdx.x);
        bool used = true;
        while (node >= 0) {
            if (reach == 0 || steps < reach) tree.above[threadIdx.x][node >> 5] |= 1u << (node & 31);
            ++steps;
            const int32_t up = tree.parents[node];
            if (up < -1 || up >= node) {
                used = false;
                break;
            }
            node = up;
        }
        tree.depth[threadIdx.x] = used ? steps - 1 : kUnused;
    }
    __syncthreads();
}

// A lane's query row: where it may look.
struct Sight {
    uint32_t first;   // the first slot it sees
    uint32_t last;    // chain: the last; tree: its token's place in the workgroup's Tree
    bool live;        // a row of the step, and used
};

// Bits `from` .. `to` - 1 of a tile's 32 slots, the bounds counted from its
// first and anywhere.
__device__ __forceinline__ uint32_t bits_between(int64_t from, int64_t to) {
    const uint32_t lo = static_cast<uint32_t>(from < 0 ? 0 : from > 32 ? 32 : from);
    const uint32_t hi = static_cast<uint32_t>(to < 0 ? 0 : to > 32 ? 32 : to);
    return static_cast<uint32_t>((1ull << hi) - 1) & ~static_cast<uint32_t>((1ull << lo) - 1);
}

// What a workgroup's rows, row0 .. row_end - 1 of a key head, have in common.
struct Group {
    uint32_t sequence, head, past, latest;
    uint32_t row0, row_end, token0, token_end;
    uint32_t tile_begin, tile_end;  // its split's tiles
    uint32_t all_begin;             // every row sees the slots from here to past
    uint64_t sequence_head;
    uint32_t split;

    // `rows` rows a workgroup, blockIdx.x = (head, row group, split).
    __device__ __forceinline__ Group(const Attention& a, uint32_t rows) {
        split = blockIdx.x % a.splits;
        const uint32_t at = blockIdx.x / a.splits, row_groups = (a.rows + rows - 1) / rows;
        row0 = at % row_groups * rows;
        sequence_head = at / row_groups;
        sequence = static_cast<uint32_t>(sequence_head) / a.cache.kv_heads;
        head = static_cast<uint32_t>(sequence_head) % a.cache.kv_heads;
        past = min(a.past[sequence], a.cache.capacity - a.tokens);
        latest = past + a.tokens;
        row_end = min(row0 + rows, a.rows);
        token0 = row0 / a.group, token_end = (row_end - 1) / a.group + 1;
        // From the window's first to the last token that its rows may see.
        const uint32_t end = a.parents ? latest : past + token_end;
        const uint32_t earliest = past + (a.parents ? 0u : token0) + 1;
        const uint32_t begin = a.window && earliest > a.window ? earliest - a.window : 0u;
        all_begin = a.window && latest > a.window ? latest - a.window : 0u;
        const uint32_t first = begin / kTile, last = (end + kTile - 1) / kTile;
        const uint32_t share = (last - first + a.splits - 1) / a.splits;
        tile_begin = min(first + split * share, last);
        tile_end = min(tile_begin + share, last);
    }

    __device__ __forceinline__ bool masked(uint32_t slot0) const { return slot0 + kTile > past || slot0 < all_begin; }
};

// A wave's RT x 16 rows as they go over the tiles: lane 16g + n holds, of rows
// n, 16 + n, ..., the queries' operands and the outputs' values 4g .. 4g + 3 of
// each 16.
template <uint32_t F, uint32_t NB, uint32_t RT>
struct Rows {
    half8_t high[RT][NB], low[RT][NB];
    float unit[RT];                          // what a raw score stands for, a power of two
    float4_t out[RT][2 * NB];
    float largest[RT], offset[RT], sum[RT];  // the raw maximum; exp2's offset; the lane's part of the sum
    int exponent;                            // D, the same in every lane
    Sight sight[RT];

    // The queries' loads alone, ahead of what the rows wait for: a lane's
    // values 8g .. 8g + 7 of each block. Rows past the group's end repeat its last.
    struct Queries {
        float x[RT][NB][8];
    };
    __device__ __forceinline__ static void fetch(const Attention& a, const Group& group, uint32_t row0, Queries& q) {
        const uint32_t lane = threadIdx.x & 63u, n = lane & 15u, g = lane >> 4;
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) {
            const uint32_t inside = min(row0 + 16 * i + n, group.row_end - 1);
            const float* from = a.queries +
                                (static_cast<uint64_t>(group.sequence) * a.tokens + inside / a.group) * a.query_stride +
                                static_cast<uint64_t>(group.head * a.group + inside % a.group) * (32 * NB) + 8 * g;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const float4 u = *reinterpret_cast<const float4*>(from + 32 * b);
                const float4 v = *reinterpret_cast<const float4*>(from + 32 * b + 4);
                q.x[i][b][0] = u.x, q.x[i][b][1] = u.y, q.x[i][b][2] = u.z, q.x[i][b][3] = u.w;
                q.x[i][b][4] = v.x, q.x[i][b][5] = v.y, q.x[i][b][6] = v.z, q.x[i][b][7] = v.w;
            }
        }
    }

    template <typename TREE>
    __device__ __forceinline__ void begin(const Attention& a, const Group& group, const TREE& tree, uint32_t row0,
                                          Queries& q) {
        const uint32_t lane = threadIdx.x & 63u, n = lane & 15u;
        exponent = F == kF16 ? kScaleTop : -64;
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) {
            const uint32_t row = row0 + 16 * i + n;
            const uint32_t token = min(row, group.row_end - 1) / a.group;
            const uint32_t depth = a.parents ? tree.depth[token - group.token0] : token;
            sight[i].live = row < group.row_end && depth != kUnused;
            const uint32_t place = group.past + (depth != kUnused ? depth : 0u) + 1;  // one past its own place
            sight[i].first = a.window && place > a.window ? place - a.window : 0u;
            sight[i].last = a.parents ? token - group.token0 : group.past + token;

            float most = 0.0f;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    q.x[i][b][e] *= a.scale * kLog2E, most = fmaxf(most, fabsf(q.x[i][b][e]));
            most = most_of_row(most);
            int shift = 0;
            if (most > 0.0f && most <= 3.4e38f) {
                int e;
                (void)frexpf(most, &e);
                shift = min(11 - e, 126);
            }
            unit[i] = ldexpf(1.0f, -shift);
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                half2_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    split2(ldexpf(q.x[i][b][2 * e], shift), ldexpf(q.x[i][b][2 * e + 1], shift), &hi[e], &lo[e]);
                high[i][b] = join(hi[0], hi[1], hi[2], hi[3]);
                low[i][b] = join(lo[0], lo[1], lo[2], lo[3]);
            }
            largest[i] = -INFINITY, offset[i] = INFINITY, sum[i] = 0.0f;
#pragma unroll
            for (uint32_t t = 0; t < 2 * NB; ++t) out[i][t] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }

    // The slots of the tile at slot0 that row i of the lane sees, as bits.
    template <typename TREE>
    __device__ __forceinline__ uint32_t sees(const Attention& a, const Group& group, const TREE& tree, uint32_t slot0,
                                             uint32_t i) const {
        const int64_t at = slot0;
        if (!a.parents) return bits_between(sight[i].first - at, static_cast<int64_t>(sight[i].last) + 1 - at);
        uint32_t seen = bits_between(sight[i].first - at, group.past - at);
        if (slot0 + kTile > group.past) {
            // the tree's tokens from `node` on: two words of the row's bits, shifted
            const int32_t node = static_cast<int32_t>(slot0 - group.past);
            const uint32_t* above = tree.above[sight[i].last];
            uint64_t words = 0;
            if (node < 0) {
                words = static_cast<uint64_t>(above[0]) << -node;
            } else if (node < static_cast<int32_t>(kTreeTokens)) {
                const uint32_t w = static_cast<uint32_t>(node) >> 5;
                words = above[w];
                if (w + 1 < kTreeTokens / 32) words |= static_cast<uint64_t>(above[w + 1]) << 32;
                words >>= node & 31;
            }
            seen |= static_cast<uint32_t>(words);
        }
        return seen;
    }

    // One tile. `source` gives the operands: key(b, h), key_scale(b), value(b, u),
    // value_scale(b); and, PARTED, value_low(b, u), the values being scaled (over
    // 2^D by 2^kScaleTop) and in two parts of their own: their scales are then
    // looked at only where `spoilt`, some of them a NaN, stands.
    template <bool PARTED, typename SOURCE, typename TREE>
    __device__ __forceinline__ void tile(const Attention& a, const Group& group, const TREE& tree, uint32_t slot0,
                                         const SOURCE& source, bool spoilt = false) {
        const uint32_t lane = threadIdx.x & 63u, g = lane >> 4;
        // Scores: s[i][h][r] of token 16h + 4g + r.
        float4_t s[RT][2];
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) s[i][0] = s[i][1] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            uint4_t scale;
            if constexpr (key_scales(F)) scale = source.key_scale(b);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const half8_t k = source.key(b, h);
#pragma unroll
                for (uint32_t i = 0; i < RT; ++i) {
                    if constexpr (key_scales(F)) {
                        float4_t p = multiply(k, high[i][b], float4_t{0.0f, 0.0f, 0.0f, 0.0f});
                        p = multiply(k, low[i][b], p);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            s[i][h][r] = __builtin_fmaf(p[r], scale_at(scale, 4 * h + r), s[i][h][r]);
                    } else {
                        s[i][h] = multiply(k, high[i][b], s[i][h]);
                        s[i][h] = multiply(k, low[i][b], s[i][h]);
                    }
                }
            }
        }

        const bool masked = group.masked(slot0);
        if (masked)
#pragma unroll
            for (uint32_t i = 0; i < RT; ++i) {
                const uint32_t bits = sees(a, group, tree, slot0, i) >> (4 * g);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(bits >> ((e >> 2) * 16 + (e & 3)) & 1u)) s[i][e >> 2][e & 3] = -INFINITY;
            }

        // The value scales: the largest's exponent, and all of them over 2^D.
        uint4_t scale[NB];
        int grown = exponent;
        constexpr bool kScaled = F != kF16 && !PARTED;
        if (kScaled || F == kF16 || spoilt) {
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) scale[b] = source.value_scale(b);
        }
        if constexpr (F == kF16) {
            uint32_t other = 0;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (int w = 0; w < 4; ++w) other |= scale[b][w] ^ 0x3C003C00u;
            spoilt = __any(other != 0);
        }
        if constexpr (kScaled) {
            ushort2_t top = {0, 0};
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t size = F == kQ4_0 ? scale[b][w] & 0x7FFF7FFFu : scale[b][w];
                    top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2_t, size));
                }
            spoilt = __any(max(top.x, top.y) > 0x7C00);
        }
        if (spoilt) spoil(a, group, tree, slot0, masked, scale);
        if constexpr (kScaled) {
            ushort2_t top = {0, 0};
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t size = F == kQ4_0 ? scale[b][w] & 0x7FFF7FFFu : scale[b][w];
                    top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2_t, size));
                }
            // the same in a group's 16 lanes
            const uint32_t mine = max(top.x, top.y);
            const uint32_t most = max(max(__builtin_amdgcn_readlane(mine, 0), __builtin_amdgcn_readlane(mine, 16)),
                                      max(__builtin_amdgcn_readlane(mine, 32), __builtin_amdgcn_readlane(mine, 48)));
            grown = max(exponent, exponent_of(most));
            const half2_t by = over(grown);
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
                for (int w = 0; w < 4; ++w) scale[b][w] = __builtin_bit_cast(uint32_t, pair_of(scale[b][w]) * by);
        }

#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) {
            float top = fmaxf(fmaxf(fmaxf(s[i][0][0], s[i][0][1]), fmaxf(s[i][0][2], s[i][0][3])),
                              fmaxf(fmaxf(s[i][1][0], s[i][1][1]), fmaxf(s[i][1][2], s[i][1][3])));
            top = most_of_row(top);
            // the offset follows once a score passes it by kSlack (the first: -inf + inf is a NaN, no less than)
            const bool follow = top > largest[i] && !((top - largest[i]) * unit[i] <= kSlack);
            if (__any(follow) || grown != exponent) {
                const float most = fmaxf(largest[i], top);
                // the offset as used is what the factor is made of, so that its rounding cancels
                const float to = most == -INFINITY ? INFINITY : __builtin_fmaf(-most, unit[i], static_cast<float>(kHeadroom));
                const float factor = largest[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(to - offset[i]);
                const float down = factor * ldexpf(1.0f, exponent - grown);
                largest[i] = most;
                offset[i] = to;
                sum[i] *= factor;
#pragma unroll
                for (uint32_t t = 0; t < 2 * NB; ++t) out[i][t] *= down;
            }
        }
        exponent = grown;

        half2_t hi[RT][4], lo[RT][4];
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) {
            // rows that have seen nothing: -inf + inf would be a NaN
            const float to = largest[i] == -INFINITY ? 0.0f : offset[i];
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e >> 2][e & 3], unit[i], to));
            sum[i] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
            for (int e = 0; e < 4; ++e) split2(p[2 * e], p[2 * e + 1], &hi[i][e], &lo[i][e]);
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            half8_t v[2], v_low[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                v[u] = source.value(b, u);
                if constexpr (PARTED && F != kF16) v_low[u] = source.value_low(b, u);
            }
#pragma unroll
            for (uint32_t i = 0; i < RT; ++i) {
                half8_t x, y;
                if constexpr (!kScaled) {
                    x = join(hi[i][0], hi[i][1], hi[i][2], hi[i][3]);
                    y = join(lo[i][0], lo[i][1], lo[i][2], lo[i][3]);
                } else {
                    // (hi + lo) d in two parts: hi d rounded, what that leaves
                    // (exact: 22 bits less their first 11) plus lo d
                    half2_t u[4], w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const half2_t d = pair_of(scale[b][e]);
                        u[e] = hi[i][e] * d;
                        w[e] = __builtin_elementwise_fma(lo[i][e], d, __builtin_elementwise_fma(hi[i][e], d, -u[e]));
                    }
                    x = join(u[0], u[1], u[2], u[3]);
                    y = join(w[0], w[1], w[2], w[3]);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float4_t& to = out[i][2 * b + u];
                    to = multiply(v[u], x, to);
                    to = multiply(v[u], y, to);
                    if constexpr (PARTED && F != kF16) to = multiply(v_low[u], x, to);
                }
            }
        }
    }

    // A tile with value scales that are NaNs: a row that sees such a token gets
    // NaNs in its block, and the scale becomes 0, for the rows that do not.
    template <typename TREE>
    __device__ __forceinline__ void spoil(const Attention& a, const Group& group, const TREE& tree, uint32_t slot0,
                                                    bool masked, uint4_t (&scale)[NB]) {
        const uint32_t g = (threadIdx.x & 63u) >> 4;
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            uint32_t nans = 0;  // a bit a slot of the lane's eight
#pragma unroll
            for (int e = 0; e < 8; ++e) nans |= (scale[b][e >> 1] >> (16 * (e & 1)) & 0x7FFFu) > 0x7C00u ? 1u << e : 0u;
#pragma unroll
            for (uint32_t i = 0; i < RT; ++i) {
                const uint32_t bits = (masked ? sees(a, group, tree, slot0, i) : 0xFFFFFFFFu) >> (4 * g);
                const float mine = nans & ((bits & 15u) | (bits >> 12 & 0xF0u)) ? 1.0f : 0.0f;
                const float nan = most_of_row(mine) > 0.0f ? __builtin_nanf("") : 0.0f;
                out[i][2 * b] += nan;
                out[i][2 * b + 1] += nan;
            }
#pragma unroll
            for (int w = 0; w < 4; ++w)
                scale[b][w] &= (nans >> (2 * w) & 1u ? 0u : 0xFFFFu) | (nans >> (2 * w + 1) & 1u ? 0u : 0xFFFF0000u);
        }
    }

    // The last tile is done: the outputs, held over 2^(D - kScaleTop), as the sum is.
    __device__ __forceinline__ void end() {
        const float up = ldexpf(1.0f, exponent - kScaleTop);
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i)
#pragma unroll
            for (uint32_t t = 0; t < 2 * NB; ++t) out[i][t] *= up;
    }
};

// Four values of a row's outputs, its sum `total` and its offset `least`: to
// the step's output, or to the split's place. `stats`: whether this thread
// writes the row's.
template <uint32_t NB>
__device__ __forceinline__ void finish(const Attention& a, const Group& group, uint32_t row, bool live, uint32_t at,
                                       float4_t out, float total, float least, bool stats) {
    // nothing seen: no maximum, and no NaN either
    const bool empty = !live || (least == INFINITY && total == 0.0f);
    if (a.splits == 1) {
        float* to = a.output + (static_cast<uint64_t>(group.sequence) * a.tokens + row / a.group) * a.output_stride +
                    static_cast<uint64_t>(group.head * a.group + row % a.group) * (32 * NB) + at;
        *reinterpret_cast<float4_t*>(to) = empty ? float4_t{0.0f, 0.0f, 0.0f, 0.0f} : out * (1.0f / total);
        return;
    }
    const uint64_t place = (group.sequence_head * a.rows + row) * a.splits + group.split;
    if (!empty) *reinterpret_cast<float4_t*>(a.partial + place * (32 * NB) + at) = out;
    if (stats) {
        const bool spoilt = total != total;
        a.stats[place] = make_float2(empty ? INFINITY : spoilt ? total : least, empty ? 0.0f : total);
    }
}

// ---- few rows: the waves split the tiles ----------------------------------------

// Records copied to LDS as they are, a wave's own ring of them: each copy is
// 64 lanes of 16 bytes straight from memory to LDS, so that a wave's next
// tiles are on their way while it works on one, with no registers for them.
typedef __attribute__((address_space(3))) void* lds_pointer;

template <uint32_t RECORD>
__device__ __forceinline__ void copy_record(const uint8_t* from, uint8_t* to) {
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (uint32_t at = 0; at < RECORD; at += 1024)
        if (at + 1024 <= RECORD || at + 16 * lane < RECORD)
            __builtin_amdgcn_global_load_lds(from + at + 16 * lane, (lds_pointer)(to + at), 16, 0, kStreamPolicy);
}

// Waits until at most `LEFT` of the wave's loads are on their way (they end in
// order), what they write in LDS then being there. LEFT below 64: s_waitcnt's
// vmcnt, its low four bits and its high two, the other counters at no wait.
template <uint32_t LEFT>
__device__ __forceinline__ void wait_loads() {
    static_assert(LEFT < 64, "vmcnt");
    __builtin_amdgcn_s_waitcnt((LEFT & 15u) | (LEFT >> 4) << 14 | 0x7u << 4 | 0xFu << 8);
    __asm__ __volatile__("" ::: "memory");
}

// A tile's operands out of its record in LDS.
template <uint32_t F, uint32_t NB>
struct Record {
    const uint8_t* at;
    uint32_t slot0, latest;  // what lies past the last token is cut: kept_of

    __device__ __forceinline__ half8_t key(uint32_t b, int h) const {
        return operand<F, false>(load_codes<F>(at + b * cache_unit(F), threadIdx.x & 63u), h);
    }
    __device__ __forceinline__ half8_t value(uint32_t b, int u) const {
        const uint32_t lane = threadIdx.x & 63u;
        Codes<F> c = load_codes<F>(at + values_at(F, NB) + b * cache_unit(F), lane);
        if constexpr (F == kF16)
            if (slot0 + kTile > latest)
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) c.w[4 * u + w] &= kept_of(slot0, lane >> 4, w, latest);
        return operand<F, true>(c, u);
    }
    __device__ __forceinline__ uint4_t key_scale(uint32_t b) const {
        return *reinterpret_cast<const uint4_t*>(at + key_scales_at(F, NB) + 64 * b + 16 * ((threadIdx.x & 63u) >> 4));
    }
    __device__ __forceinline__ uint4_t value_scale(uint32_t b) const {
        const uint32_t g = (threadIdx.x & 63u) >> 4;
        uint4_t s = *reinterpret_cast<const uint4_t*>(at + value_scales_at(F, NB) + 64 * b + 16 * g);
        if (slot0 + kTile > latest)
#pragma unroll
            for (uint32_t w = 0; w < 4; ++w) s[w] = kept_scale<F>(s[w], kept_of(slot0, g, w, latest));
        return s;
    }
};

// Waves a workgroup and records a wave's ring: eight waves where two fit a
// SIMD's registers and two records of each fit the LDS, else four, else two.
constexpr uint32_t kRingBytes = 144 * 1024;
template <uint32_t F, uint32_t NB, uint32_t RT>
struct AttendShape {
    static constexpr uint32_t kRecord = cache_record(F, NB);
    static constexpr uint32_t kWaves = NB * RT <= 4 && 16 * kRecord <= kRingBytes ? 8 : 8 * kRecord <= kRingBytes ? 4 : 2;
    static constexpr uint32_t kRing = kRingBytes / (kWaves * kRecord) < 4 ? kRingBytes / (kWaves * kRecord) : 4;
    static constexpr uint32_t kCopies = (kRecord + 1023) / 1024;
};

template <uint32_t F, uint32_t NB, uint32_t RT>
__global__ __launch_bounds__((64 * AttendShape<F, NB, RT>::kWaves)) void attend(Attention a) {
    using Shape = AttendShape<F, NB, RT>;
    constexpr uint32_t kRows = 16 * RT, kRecord = Shape::kRecord, W = Shape::kWaves, D = Shape::kRing;
    constexpr uint32_t kParts = RT * 2 * NB * 64;  // float4s of a wave's outputs
    __shared__ Tree<kRows> tree;
    // The waves' rings; then, all tiles done, their outputs.
    __shared__ __align__(16) uint8_t space[sizeof(uint8_t[W][D][kRecord]) > sizeof(float4_t[W][kParts])
                                               ? sizeof(uint8_t[W][D][kRecord])
                                               : sizeof(float4_t[W][kParts])];
    __shared__ float joined_offset[W][kRows], joined_sum[W][kRows];
    __shared__ uint32_t joined_live[kRows];

    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15u, g = lane >> 4;
    const Group group(a, kRows);
    const uint8_t* base = record_of(a.cache, F, group.sequence, group.head, 0);
    uint8_t* ring = space + wave * (D * kRecord);
    const uint32_t first = group.tile_begin + wave;
    const uint32_t count = first < group.tile_end ? (group.tile_end - first + W - 1) / W : 0;  // the wave's tiles
    auto copy = [&](uint32_t j) {
        copy_record<kRecord>(base + static_cast<uint64_t>(first + j * W) * kRecord, ring + j % D * kRecord);
    };
    // The first copies go out before anything that the rows wait for.
#pragma unroll
    for (uint32_t j = 0; j + 1 < D; ++j)
        if (j < count) copy(j);
    typename Rows<F, NB, RT>::Queries queries;
    Rows<F, NB, RT>::fetch(a, group, group.row0, queries);
    if (a.parents)
        read_tree(tree, a.parents + static_cast<uint64_t>(group.sequence) * a.tokens, a.tokens, group.token0,
                  group.token_end - group.token0, a.window);
    Rows<F, NB, RT> rows;
    rows.begin(a, group, tree, group.row0, queries);
    // Only copies are on their way from here on: the queries' own loads, the
    // youngest, have been waited for.
    for (uint32_t j = 0; j < count; ++j) {
        // tile j + D - 1 into the place of tile j - 1, whose reads are done
        if (j + D - 1 < count) {
            copy(j + D - 1);
            wait_loads<(D - 1) * Shape::kCopies>();
        } else {
            wait_loads<0>();
        }
        const uint32_t slot0 = (first + j * W) * kTile;
        const Record<F, NB> record{ring + j % D * kRecord, slot0, group.latest};
        rows.template tile<false>(a, group, tree, slot0, record);
        __asm__ __volatile__("s_waitcnt lgkmcnt(0)" ::: "memory");  // the record's reads, before its place is copied to
    }
    rows.end();
    __syncthreads();
    float4_t(*joined)[kParts] = reinterpret_cast<float4_t(*)[kParts]>(space);

    // The waves joined: each one's outputs on the least offset's (the largest
    // maximum's) scale, added in wave order, a thread some of the values.
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
        const float mine = sum_of_row(rows.sum[i]);
        if (g == 0) joined_offset[wave][16 * i + n] = rows.offset[i], joined_sum[wave][16 * i + n] = mine;
        if (threadIdx.x < 16) joined_live[16 * i + n] = rows.sight[i].live;
    }
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i)
#pragma unroll
        for (uint32_t t = 0; t < 2 * NB; ++t) joined[wave][(i * 2 * NB + t) * 64 + lane] = rows.out[i][t];
    __syncthreads();
    for (uint32_t x = 0; x < (kParts + 64 * W - 1) / (64 * W); ++x) {
        const uint32_t at = threadIdx.x + 64 * W * x;
        if (at >= kParts) break;
        const uint32_t i = at / (128 * NB), t = at / 64 % (2 * NB), in_row = 16 * i + n;
        if (group.row0 + in_row >= group.row_end) continue;
        float least = INFINITY, total = 0.0f;
        float4_t out = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            const float theirs = joined_offset[w][in_row];
            least = theirs < least || theirs != theirs ? theirs : least;
        }
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            // a wave that saw nothing has zeros, or the NaNs of scores that are
            const float theirs = joined_offset[w][in_row];
            const float factor = theirs == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(least - theirs);
            total = __builtin_fmaf(joined_sum[w][in_row], factor, total);
            out += joined[w][at] * factor;
        }
        finish<NB>(a, group, group.row0 + in_row, joined_live[in_row] != 0, 16 * t + 4 * g, out, total, least,
                   t == 0 && g == 0);
    }
}

// ---- many rows: the waves split the rows -------------------------------------------

// A tile laid out in LDS by the workgroup for all of its waves: the codes as
// binary16 operands, the values' scaled, in two parts (the product of a code
// and a scale is exact in them), so that a wave does no more than read them.
// (A NaN among the scales, which is not every row's, goes in as 0: Rows::spoil.)
template <uint32_t F, uint32_t NB>
struct Stage {
    half8_t keys[2 * NB][64], values[2 * NB][64];    // [2 b + h], [2 b + u]
    half8_t values_low[F == kF16 ? 1 : 2 * NB][64];  // (F16's are exact in one)
    uint4_t key_scales_[NB][4], value_scales_[NB][4];

    __device__ __forceinline__ half8_t key(uint32_t b, int h) const { return keys[2 * b + h][threadIdx.x & 63u]; }
    __device__ __forceinline__ half8_t value(uint32_t b, int u) const { return values[2 * b + u][threadIdx.x & 63u]; }
    __device__ __forceinline__ half8_t value_low(uint32_t b, int u) const { return values_low[2 * b + u][threadIdx.x & 63u]; }
    __device__ __forceinline__ uint4_t key_scale(uint32_t b) const { return key_scales_[b][(threadIdx.x & 63u) >> 4]; }
    __device__ __forceinline__ uint4_t value_scale(uint32_t b) const { return value_scales_[b][(threadIdx.x & 63u) >> 4]; }
};

constexpr uint32_t kRowWaves = 8;

template <uint32_t F, uint32_t NB, uint32_t RT>
__global__ __launch_bounds__(64 * kRowWaves) void attend_rows(Attention a) {
    constexpr uint32_t W = kRowWaves, kRows = 16 * RT * W, kRecord = cache_record(F, NB);
    constexpr uint32_t kTiles = NB <= 4 ? 2 : 1;                                // a stage's
    constexpr uint32_t kUnits = 2 * NB * kTiles, kMine = (kUnits + W - 1) / W;  // units of a stage; a wave's, at most
    constexpr uint32_t kScaleWords = (key_scales(F) ? 32 : 16) * NB;            // a tile's
    static_assert(kScaleWords * kTiles <= 64 * W, "a thread a dword");
    __shared__ Tree<kRows < kTreeTokens ? kRows : kTreeTokens> tree;
    __shared__ Stage<F, NB> stages[2][kTiles];
    __shared__ uint32_t wave_most[W], wave_spoilt[W];

    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Group group(a, kRows);
    const uint32_t row0 = group.row0 + 16 * RT * wave;
    const bool mine = row0 < group.row_end;  // a wave without rows still lays out its share
    typename Rows<F, NB, RT>::Queries queries;
    Rows<F, NB, RT>::fetch(a, group, min(row0, group.row_end - 1), queries);
    // a chain's wave sees nothing past its last row's token
    const uint32_t sees_to =
        a.parents ? group.latest : group.past + (min(row0 + 16 * RT, group.row_end) - 1) / a.group + 1;
    const uint8_t* base = record_of(a.cache, F, group.sequence, group.head, 0);

    // All the tiles' value scales, once: their largest exponent, and whether any is a NaN (F16: other than one).
    uint32_t most = 0, spoilt = 0;
#pragma unroll 4
    for (uint32_t x = threadIdx.x; x < (group.tile_end - group.tile_begin) * 16 * NB; x += 64 * W) {
        const uint32_t t = group.tile_begin + x / (16 * NB), w = x % (16 * NB);
        const uint32_t word = kept_scale<F>(
            reinterpret_cast<const uint32_t*>(base + static_cast<uint64_t>(t) * kRecord + value_scales_at(F, NB))[w],
            kept_of(t * kTile, w / 4 & 3u, w & 3u, group.latest));
        most = max(most, larger_scale(word));
        spoilt |= F == kF16 ? word ^ 0x3C003C00u
                            : static_cast<uint32_t>((word & 0x7FFFu) > 0x7C00u || (word & 0x7FFF0000u) > 0x7C000000u);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), o)));
    spoilt = __any(spoilt != 0);
    if (lane == 0) wave_most[wave] = most, wave_spoilt[wave] = spoilt;
    if (a.parents)
        read_tree(tree, a.parents + static_cast<uint64_t>(group.sequence) * a.tokens, a.tokens, group.token0,
                  group.token_end - group.token0, a.window);
    __syncthreads();
    most = spoilt = 0;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) most = max(most, wave_most[w]), spoilt |= wave_spoilt[w];
    spoilt = __builtin_amdgcn_readfirstlane(spoilt);
    const int exponent = F == kF16 ? kScaleTop : exponent_of(__builtin_amdgcn_readfirstlane(most));
    const half2_t by = over(exponent);

    Rows<F, NB, RT> rows;
    rows.begin(a, group, tree, min(row0, group.row_end - 1), queries);
    rows.exponent = exponent;

    // Unit u of a stage: tile u / 2NB, block u % NB, keys then values.
    Codes<F> codes[kMine];
    uint4_t unit_scale[kMine];  // a value unit's
    uint32_t scale_word = 0;    // of those that the waves read
    auto load = [&](uint32_t tile0) {
#pragma unroll
        for (uint32_t j = 0; j < kMine; ++j) {
            const uint32_t u = wave + W * j, t = tile0 + u / (2 * NB);
            if (u >= kUnits || t >= group.tile_end) continue;
            const uint8_t* record = base + static_cast<uint64_t>(t) * kRecord;
            codes[j] = load_codes<F>(record + u % (2 * NB) * cache_unit(F), lane);
            if (F != kF16 && u % (2 * NB) >= NB)
                unit_scale[j] = *reinterpret_cast<const uint4_t*>(record + value_scales_at(F, NB) + 64 * (u % NB) + 16 * (lane >> 4));
        }
        const uint32_t t = tile0 + threadIdx.x / kScaleWords;
        if (threadIdx.x < kScaleWords * kTiles && t < group.tile_end)
            scale_word = reinterpret_cast<const uint32_t*>(base + static_cast<uint64_t>(t) * kRecord +
                                                           key_scales_at(F, NB))[threadIdx.x % kScaleWords];
    };
    auto lay = [&](uint32_t tile0, Stage<F, NB>* stage) {
#pragma unroll
        for (uint32_t j = 0; j < kMine; ++j) {
            const uint32_t u = wave + W * j, t = u / (2 * NB), b = u % NB, slot0 = (tile0 + t) * kTile;
            if (u >= kUnits || tile0 + t >= group.tile_end) continue;
            if (u % (2 * NB) < NB) {
                stage[t].keys[2 * b][lane] = operand<F, false>(codes[j], 0);
                stage[t].keys[2 * b + 1][lane] = operand<F, false>(codes[j], 1);
                continue;
            }
            // what lies past the last token is no one's, and may be anything
            if (slot0 + kTile > group.latest)
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) {
                    const uint32_t kept = kept_of(slot0, lane >> 4, w, group.latest);
                    if constexpr (F == kF16)
                        codes[j].w[w] &= kept, codes[j].w[4 + w] &= kept;
                    else
                        unit_scale[j][w] &= kept;
                }
            if (F != kF16 && spoilt)
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) {
                    const uint32_t s = unit_scale[j][w];
                    unit_scale[j][w] = ((s & 0x7FFFu) > 0x7C00u ? 0u : s & 0xFFFFu) |
                                       ((s & 0x7FFF0000u) > 0x7C000000u ? 0u : s & 0xFFFF0000u);
                }
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const half8_t code = operand<F, true>(codes[j], part);
                half8_t high = code, low = {0, 0, 0, 0, 0, 0, 0, 0};
                if constexpr (F != kF16) {
                    half2_t hi[4], lo[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const half2_t c = {code[2 * w], code[2 * w + 1]}, d = pair_of(unit_scale[j][w]) * by;
                        hi[w] = c * d;
                        lo[w] = __builtin_elementwise_fma(c, d, -hi[w]);
                    }
                    high = join(hi[0], hi[1], hi[2], hi[3]);
                    low = join(lo[0], lo[1], lo[2], lo[3]);
                    stage[t].values_low[2 * b + part][lane] = low;
                }
                stage[t].values[2 * b + part][lane] = high;
            }
        }
        const uint32_t t = threadIdx.x / kScaleWords, w = threadIdx.x % kScaleWords;
        if (threadIdx.x < kScaleWords * kTiles && tile0 + t < group.tile_end) {
            const bool values = !key_scales(F) || w >= 16 * NB;
            if (values)
                scale_word = kept_scale<F>(scale_word, kept_of((tile0 + t) * kTile, w / 4 & 3u, w & 3u, group.latest));
            uint32_t* to = reinterpret_cast<uint32_t*>(values ? stage[t].value_scales_ : stage[t].key_scales_);
            to[w % (16 * NB)] = scale_word;
        }
    };
    if (group.tile_begin < group.tile_end) {
        load(group.tile_begin);
        lay(group.tile_begin, stages[0]);
    }
    __syncthreads();
    uint32_t turn = 0;
    for (uint32_t tile0 = group.tile_begin; tile0 < group.tile_end; tile0 += kTiles, turn ^= 1) {
        // the next stage's loads are in flight over this one's products
        const bool more = tile0 + kTiles < group.tile_end;
        if (more) load(tile0 + kTiles);
#pragma unroll 1
        for (uint32_t t = 0; t < kTiles; ++t) {
            const uint32_t slot0 = (tile0 + t) * kTile;
            if (mine && tile0 + t < group.tile_end && slot0 < sees_to)
                rows.template tile<true>(a, group, tree, slot0, stages[turn][t], spoilt != 0);
        }
        // the other stage was read before the last barrier
        if (more) lay(tile0 + kTiles, stages[turn ^ 1]);
        __syncthreads();
    }
    if (mine) {
        rows.end();
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) {
            const float total = sum_of_row(rows.sum[i]);
            const uint32_t row = row0 + 16 * i + (lane & 15u);
            if (row >= group.row_end) continue;
#pragma unroll
            for (uint32_t t = 0; t < 2 * NB; ++t)
                finish<NB>(a, group, row, rows.sight[i].live, 16 * t + 4 * (lane >> 4), rows.out[i][t], total,
                           rows.offset[i], t == 0 && lane < 16);
        }
    }
}

template <uint32_t F, uint32_t NB>
static hipError_t launch_blocks(const Attention& a, const AttentionPlan& plan, hipStream_t stream) {
    const dim3 grid(a.cache.sequences * a.cache.kv_heads * plan.row_groups * plan.splits);
    constexpr uint32_t kWide = NB <= 4 ? 2 : 1;  // 16-row tiles a wave's registers hold
    if (plan.waves > 1)
        hipLaunchKernelGGL((attend_rows<F, NB, kWide>), grid, dim3(64 * kRowWaves), 0, stream, a);
    else if (plan.row_tiles == kWide)
        hipLaunchKernelGGL((attend<F, NB, kWide>), grid, dim3(64 * AttendShape<F, NB, kWide>::kWaves), 0, stream, a);
    else
        hipLaunchKernelGGL((attend<F, NB, 1>), grid, dim3(64 * AttendShape<F, NB, 1>::kWaves), 0, stream, a);
    return hipGetLastError();
}

template <uint32_t F>
static hipError_t launch_format(const Attention& a, const AttentionPlan& plan, hipStream_t stream) {
    switch (a.cache.head_dim / 32) {
        case 1: return launch_blocks<F, 1>(a, plan, stream);
        case 2: return launch_blocks<F, 2>(a, plan, stream);
        case 3: return launch_blocks<F, 3>(a, plan, stream);
        case 4: return launch_blocks<F, 4>(a, plan, stream);
        case 5: return launch_blocks<F, 5>(a, plan, stream);
        case 6: return launch_blocks<F, 6>(a, plan, stream);
        case 7: return launch_blocks<F, 7>(a, plan, stream);
        case 8: return launch_blocks<F, 8>(a, plan, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace chm
