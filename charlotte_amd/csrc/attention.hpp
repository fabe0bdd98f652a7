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
// ln 2 and a power of two that puts its largest value in [2^14, 2^15), and a
// probability (attend_rows, F16) or its product with a value's scale are each
// taken as two binary16 parts, hi + lo: 22 bits, but no less than the half of
// binary16's least step, 2^-25. A cache's codes are exact in binary16. A block's
// key scale multiplies its product in f32 (F16: none). Sums are f32 throughout.
//
// Range: a query's parts leave 2^-22 of it, or 2^-39 of the row's largest. p is
// 2^up at the maximum last followed, which follows once a score passes it by
// 2^kSlack, so below 2^(up + kSlack):
//   F16 and attend_rows  up = 11, p below 2^15: its parts leave 2^-22 of it, or
//     2^-36 of the row's largest;
//   attend, quantized    up = 7, and p d over 2^held below 2^15. held is that of
//     the tile's largest scale, and stays while the tiles' scales lie within 2^-8
//     to 2 of it; the outputs are held over it and follow. The parts leave 2^-21 of
//     p d, or 2^-25 of the row's largest p times d. A tile whose own scales lie
//     further apart - whether its rows see the tokens or not - takes p d in f32,
//     and parts them over each row's largest, lo over a step of its own (wide).
// attend_rows lays values out as code times scale over 2^held, in two parts that
// are exact while the scale is 2^-14 or more: while the split's scales lie within
// 2^22. It does so while they lie within 2^16, so that 2^-36 of a row's largest p
// times any value is 2^-20 of the least block's; else its waves take the tiles as
// attend's do.
//
// Split: where there are few products for each compute unit (attend), a
// workgroup has 16 or 32 rows, those one wave holds; its waves take the tiles in
// turn, operands straight from the record, and are joined in LDS. Where there
// are many (attend_rows), each wave has rows of its own, and a tile's codes
// become binary16 operands in LDS once for all of them. Where rows do not fill
// the card, tiles are split among several workgroups, joined by
// attention_combine. attention_plan.cpp chooses, with what each side measured.
//
// Bound and measured (8 key heads; a large copy moves 5.1 TB/s, a large binary16
// product of the library's runs at 1.1 - 1.16 PFLOP/s):
//   one token of 32 heads of 128 over 65,536 in Q8_0, by the cache's 142 MB: 30.8
//   us, 4.6 TB/s, and 4.6 to join its 32 splits; with half of its blocks 2^12 below
//   the others, every tile wide, 44 in all where that is 34;
//   16 heads over 911, by the latency of a launch and its reads: 6.6 and 3.4 us;
//   a tree of 21 tokens of 32 heads of 64 over 8,191 in Q4_0, by latency: the VALU
//   issues 42% of the time (some 500 instructions a tile of 32 rows: codes widened,
//   the probabilities scaled and parted for each block of values), the matrix cores
//   10%; the rest is the tree, read by every split, and 26 tiles over 8 waves: 16.6
//   and 4.0 us;
//   512 tokens of 32 heads of 128 over 15,873 in Q8_0 (attend_rows), by the matrix
//   instructions: 339 GFLOP with queries, probabilities and values in parts (135
//   by the formula), 318 - 340 us, 1.04 PFLOP/s; matrix cores busy 50% and the VALU
//   44% of the time; priorities and the waves of a SIMD half a tile apart changed
//   nothing or cost time. Scales too far apart to lay out (attend_alone): 900 us.
#pragma once

#include "cache.hpp"
#include "stream.hpp"

namespace chm {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef float float16_t __attribute__((ext_vector_type(16)));

typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2E = 1.44269504088896340736f;
// A probability is 2^up at the maximum last followed, and a score may go kSlack
// past it; the largest value scale is held as 2^top to twice that. What is
// parted stays below 2^15 or, a code of at most 7 bits times its scale, 2^16.
constexpr int kSlack = 4;
constexpr int kProductUp = 7, kScaleTop = 3;  // p d, of quantized values in attend
constexpr int kAloneUp = 11, kCodeTop = 8;    // p, and code times scale
static_assert(kProductUp + kSlack + kScaleTop + 1 <= 15 && kAloneUp + kSlack <= 15 && 7 + kCodeTop + 1 <= 16,
              "past binary16");
// How far below the largest, in octaves, scales may lie: of a tile in attend, of a split in attend_rows.
constexpr int kTileSpread = 8, kSplitSpread = 16;

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
template <int RAISE>
__device__ __forceinline__ half8_t halves_of(uint32_t first, uint32_t second) {
    half2_t a, b, c, d;
    halves_of<RAISE>(first, &a, &b);
    halves_of<RAISE>(second, &c, &d);
    return join(a, b, c, d);
}

// Eight codes as an operand: of lane `from` of a unit as cache.hpp lays it
// out, for the keys those of token half `part`, for the values those of value
// 16 part + from % 16.
template <uint32_t F, bool VALUES>
__device__ __forceinline__ half8_t operand(const uint8_t* unit, uint32_t from, uint32_t part) {
    if constexpr (F == kF16) {
        return *reinterpret_cast<const half8_t*>(unit + 1024 * part + 16 * from);
    } else if constexpr (F == kQ8_0) {
        const uint2 w = *reinterpret_cast<const uint2*>(unit + 16 * from + 8 * part);
        return halves_of<128>(w.x, w.y);
    } else if constexpr (VALUES) {
        const uint2 w = *reinterpret_cast<const uint2*>(unit + 8 * from);
        return halves_of<8>(w.x >> (4 * part) & 0x0F0F0F0Fu, w.y >> (4 * part) & 0x0F0F0F0Fu);
    } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(unit + 8 * from + 4 * part);
        return halves_of<8>(w & 0x0F0F0F0Fu, w >> 4 & 0x0F0F0F0Fu);
    }
}

__device__ __forceinline__ float4_t multiply(half8_t a, half8_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ float16_t multiply(half8_t a, half8_t b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
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
    *hi = __builtin_convertvector((float2_t{a, b}), half2_t);
    // a factor the compiler does not know keeps each difference one mixed-precision instruction
    float minus = -1.0f;
    __asm__("" : "+s"(minus));
    *lo = __builtin_convertvector((float2_t{__builtin_fmaf(static_cast<float>(hi->x), minus, a),
                                            __builtin_fmaf(static_cast<float>(hi->y), minus, b)}),
                                  half2_t);
}

// A wave's scales, two a dword: the largest and least magnitudes as bits, of
// those that are neither zero, which weighs nothing, nor a NaN.
struct Scales {
    uint32_t most = 0, least = 0x7FFFu;
    bool nan = false;
    __device__ __forceinline__ void add(uint32_t word) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t size = word >> (16 * h) & 0x7FFFu;
            nan |= size > 0x7C00u;
            most = max(most, size > 0x7C00u ? 0u : size);
            least = min(least, size - 1 < 0x7C00u ? size : 0x7FFFu);
        }
    }
    // The wave's, in every lane.
    __device__ __forceinline__ void join() {
        uint32_t both = most | (0x7FFFu - least) << 16;
        auto more = [&](uint32_t other) {
            both = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, both),
                                                                          __builtin_bit_cast(ushort2_t, other)));
        };
        // within rows of 16 lanes, rotated by 1, 2, 4 and 8, then over the rows
        more(static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(both), 0x121, 0xF, 0xF, true)));
        more(static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(both), 0x122, 0xF, 0xF, true)));
        more(static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(both), 0x124, 0xF, 0xF, true)));
        more(static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(both), 0x128, 0xF, 0xF, true)));
        const auto a = __builtin_amdgcn_permlane16_swap(both, both, false, false);
        both = a[0], more(a[1]);
        const auto b = __builtin_amdgcn_permlane32_swap(both, both, false, false);
        both = b[0], more(b[1]);
        both = __builtin_amdgcn_readfirstlane(both);
        most = both & 0xFFFFu, least = 0x7FFFu - (both >> 16);
        nan = __any(nan);
    }
};
// Where scales up to `most` are held over 2^held: the largest as 2^TOP to twice
// that, but none times more than 2^15, which binary16 holds.
template <int TOP>
__device__ __forceinline__ int held_of(uint32_t most) {
    return static_cast<int>(max(most >> 10, static_cast<uint32_t>(TOP))) - 15 - TOP;
}
// 2^-held, what a scale is multiplied by.
__device__ __forceinline__ half2_t over(int held) {
    const _Float16 by = static_cast<_Float16>(ldexpf(1.0f, -held));
    return half2_t{by, by};
}
// 2^x as binary16's bits; what lies below its least, as that.
__device__ __forceinline__ uint32_t power_bits(int x) {
    return x >= -14 ? static_cast<uint32_t>(x + 15) << 10 : x >= -24 ? 1u << (x + 24) : 1u;
}

// How a tile's values come: as codes and scales (attend), or laid out, scaled, in
// two parts (attend_rows).
enum Values : uint32_t { kCodes, kLaidOut };

// Over the lanes that share a row: lane % 16, four of them, or lane % 32, two.
template <uint32_t X>
__device__ __forceinline__ float most_of_row(float x) {
    if constexpr (X == 1) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    }
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
template <uint32_t X>
__device__ __forceinline__ float sum_of_row(float x) {
    if constexpr (X == 1) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
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
    static constexpr bool kTrees = true;
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

    Group() = default;
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

// A wave's 16 X rows as they go over the tiles. X = 1: the 16 x 16 x 32
// instruction, lane 16g + n row n, its eight tokens those of group g. X = 2: the
// 32 x 32 x 16 one, which does twice the work in little more time; lane 32f + n
// row n, its 16 tokens those of groups f and 2 + f, octets 0 and 1. That takes
// the keys' rows in the order of their slots: row 16 (g / 2) + 8h + 4 (g % 2) + r
// is token 16h + 4g + r, so that a result's octet is a group's eight slots in
// the record's order, and they are the operands along the next sum, 16 tokens
// an instruction.
template <uint32_t X>
__device__ __forceinline__ uint32_t group_of(uint32_t octet) {
    const uint32_t lane = threadIdx.x & 63u;
    return X == 1 ? lane >> 4 : 2 * octet + (lane >> 5);
}

template <uint32_t X>
struct Result {
    typedef float4_t type;
};
template <>
struct Result<2> {
    typedef float16_t type;
};

template <uint32_t F, uint32_t NB, uint32_t X>
struct Rows {
    typedef typename Result<X>::type result_t;
    static constexpr uint32_t kOuts = X == 1 ? 2 * NB : NB;    // results: 16 values of 16 rows, or 32 of 32
    static constexpr uint32_t kQuads = X == 1 ? 2 * NB : 4 * NB;  // a lane's runs of four values

    half8_t high[NB * X], low[NB * X];  // the queries
    float unit;                         // what a raw score stands for, a power of two
    result_t out[kOuts];
    float largest, offset, sum;         // the raw maximum; exp2's offset; the lane's part of the sum
    int held;                           // outputs are over 2^held, the same in every lane
    // The scales that it stays for, each twice in its dword: the least's bits less one, and the largest's.
    uint32_t scale_low, scale_high;
    Sight sight;

    // Where a lane's run of four output values stands in its row.
    __device__ __forceinline__ static uint32_t quad_at(uint32_t quad) {
        const uint32_t lane = threadIdx.x & 63u;
        return X == 1 ? 16 * quad + 4 * (lane >> 4) : 8 * quad + 4 * (lane >> 5);
    }
    __device__ __forceinline__ float4_t quad(uint32_t q) const {
        if constexpr (X == 1) {
            return out[q];
        } else {
            const uint32_t r = 4 * (q & 3u);
            return float4_t{out[q >> 2][r], out[q >> 2][r + 1], out[q >> 2][r + 2], out[q >> 2][r + 3]};
        }
    }

    // The queries' loads alone, ahead of what the rows wait for: eight values an
    // operand. Rows past the group's end repeat its last.
    struct Queries {
        float x[NB * X][8];
    };
    __device__ __forceinline__ static void fetch(const Attention& a, const Group& group, uint32_t row0, Queries& q) {
        const uint32_t lane = threadIdx.x & 63u, n = lane % (16 * X);
        const uint32_t inside = min(row0 + n, group.row_end - 1);
        const float* from = a.queries +
                            (static_cast<uint64_t>(group.sequence) * a.tokens + inside / a.group) * a.query_stride +
                            static_cast<uint64_t>(group.head * a.group + inside % a.group) * (32 * NB) + 8 * (lane / (16 * X));
#pragma unroll
        for (uint32_t b = 0; b < NB * X; ++b) {
            const float4 u = *reinterpret_cast<const float4*>(from + 32 / X * b);
            const float4 v = *reinterpret_cast<const float4*>(from + 32 / X * b + 4);
            q.x[b][0] = u.x, q.x[b][1] = u.y, q.x[b][2] = u.z, q.x[b][3] = u.w;
            q.x[b][4] = v.x, q.x[b][5] = v.y, q.x[b][6] = v.z, q.x[b][7] = v.w;
        }
    }

    template <typename TREE>
    __device__ __forceinline__ void begin(const Attention& a, const Group& group, const TREE& tree, uint32_t row0,
                                          Queries& q) {
        const uint32_t row = row0 + (threadIdx.x & 63u) % (16 * X);
        const uint32_t token = min(row, group.row_end - 1) / a.group;
        const uint32_t depth = a.parents ? tree.depth[token - group.token0] : token;
        sight.live = row < group.row_end && depth != kUnused;
        const uint32_t place = group.past + (depth != kUnused ? depth : 0u) + 1;  // one past its own place
        sight.first = a.window && place > a.window ? place - a.window : 0u;
        sight.last = a.parents ? token - group.token0 : group.past + token;

        float most = 0.0f;
#pragma unroll
        for (uint32_t b = 0; b < NB * X; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e) q.x[b][e] *= a.scale * kLog2E, most = fmaxf(most, fabsf(q.x[b][e]));
        most = most_of_row<X>(most);
        int shift = 0;
        if (most > 0.0f && most <= 3.4e38f) {
            int e;
            (void)frexpf(most, &e);
            shift = min(15 - e, 126);
        }
        unit = ldexpf(1.0f, -shift);
#pragma unroll
        for (uint32_t b = 0; b < NB * X; ++b) {
            half2_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                split2(ldexpf(q.x[b][2 * e], shift), ldexpf(q.x[b][2 * e + 1], shift), &hi[e], &lo[e]);
            high[b] = join(hi[0], hi[1], hi[2], hi[3]);
            low[b] = join(lo[0], lo[1], lo[2], lo[3]);
        }
        held = 0;
        scale_low = 0xFFFEFFFEu, scale_high = 0x7FFF7FFFu;  // zeros alone
        largest = -INFINITY, offset = INFINITY, sum = 0.0f;
#pragma unroll
        for (uint32_t t = 0; t < kOuts; ++t) out[t] = result_t(0.0f);
    }

    // The slots of the tile at slot0 that the lane's row sees, as bits.
    template <typename TREE>
    __device__ __forceinline__ uint32_t sees(const Attention& a, const Group& group, const TREE& tree, uint32_t slot0) const {
        const int64_t at = slot0;
        if (!a.parents) return bits_between(sight.first - at, static_cast<int64_t>(sight.last) + 1 - at);
        uint32_t seen = bits_between(sight.first - at, group.past - at);
        if (slot0 + kTile > group.past) {
            // the tree's tokens from `node` on: two words of the row's bits, shifted
            const int32_t node = static_cast<int32_t>(slot0 - group.past);
            const uint32_t* above = tree.above[sight.last];
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
    // Those of an octet, a bit a slot of its eight.
    __device__ __forceinline__ static uint32_t octet_bits(uint32_t seen, uint32_t octet) {
        const uint32_t bits = seen >> (4 * group_of<X>(octet));
        return (bits & 15u) | (bits >> 12 & 0xF0u);
    }

    // One tile. `source` gives the operands: keys(b, i) and values(b, i), i = 0, 1
    // (X = 1: token half, 16 values; X = 2: 16 dims, 16 tokens), and an octet's
    // scales, key_scale(b, x) and value_scale(b, x), a dword a lane scale_word(i);
    // and, kLaidOut, values_low(b, i): then held is the split's, and `spoilt` says
    // whether some value scale of it is a NaN.
    template <Values HOW, typename SOURCE, typename TREE>
    __device__ __forceinline__ void tile(const Attention& a, const Group& group, const TREE& tree, uint32_t slot0,
                                         const SOURCE& source, bool spoilt = false) {
        constexpr bool kFollowed = F != kF16 && HOW == kCodes;
        // The value scales, each looked at by one lane, ahead of what waits for the products.
        constexpr uint32_t kWords = (16 * NB + 63) / 64;
        [[maybe_unused]] uint32_t word[kWords], outside = 0;
        if constexpr (HOW == kCodes)
#pragma unroll
            for (uint32_t i = 0; i < kWords; ++i) {
                word[i] = source.scale_word(i);
                if constexpr (F == kF16) {
                    outside |= word[i] ^ 0x3C003C00u;
                } else {
                    const auto size = __builtin_bit_cast(ushort2_t, F == kQ4_0 ? word[i] & 0x7FFF7FFFu : word[i]);
                    const auto low = __builtin_bit_cast(ushort2_t, scale_low), high = __builtin_bit_cast(ushort2_t, scale_high);
                    outside |= __builtin_bit_cast(uint32_t, __builtin_elementwise_min(ushort2_t(size - ushort2_t(1)), low)) ^ scale_low;
                    outside |= __builtin_bit_cast(uint32_t, __builtin_elementwise_max(size, high)) ^ scale_high;
                }
            }
        float s[X][8];
        if constexpr (X == 1) {
            float4_t sums[2] = {float4_t(0.0f), float4_t(0.0f)};
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                uint4_t scale;
                if constexpr (key_scales(F)) scale = source.key_scale(b, 0);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const half8_t k = source.keys(b, h);
                    if constexpr (key_scales(F)) {
                        const float4_t p = multiply(k, low[b], multiply(k, high[b], float4_t(0.0f)));
#pragma unroll
                        for (int r = 0; r < 4; ++r) sums[h][r] = __builtin_fmaf(p[r], scale_at(scale, 4 * h + r), sums[h][r]);
                    } else {
                        sums[h] = multiply(k, low[b], multiply(k, high[b], sums[h]));
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) s[0][e] = sums[e >> 2][e & 3];
        } else {
            float16_t sums = float16_t(0.0f), p[2];
            auto product = [&](uint32_t b, float16_t from) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const half8_t k = source.keys(b, y);
                    from = multiply(k, low[2 * b + y], multiply(k, high[2 * b + y], from));
                }
                return from;
            };
            // attend_rows: a block's products are out before those of the one before it
            // are scaled (512 tokens over 15,873: 327 us, else 330)
            constexpr bool kAhead = HOW == kLaidOut && key_scales(F);
            if constexpr (kAhead) p[0] = product(0, float16_t(0.0f));
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                if constexpr (!key_scales(F)) {
                    sums = product(b, sums);
                } else {
                    if constexpr (kAhead) {
                        if (b + 1 < NB) p[(b + 1) & 1] = product(b + 1, float16_t(0.0f));
                        __builtin_amdgcn_sched_barrier(0);
                    } else {
                        p[b & 1] = product(b, float16_t(0.0f));
                    }
#pragma unroll
                    for (uint32_t x = 0; x < 2; ++x) {
                        const uint4_t scale = source.key_scale(b, x);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            sums[8 * x + e] = __builtin_fmaf(p[b & 1][8 * x + e], scale_at(scale, e), sums[8 * x + e]);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e >> 3][e & 7] = sums[e];
        }

        const bool masked = group.masked(slot0);
        if (masked) {
            const uint32_t seen = sees(a, group, tree, slot0);
#pragma unroll
            for (uint32_t x = 0; x < X; ++x) {
                const uint32_t bits = octet_bits(seen, x);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(bits >> e & 1u)) s[x][e] = -INFINITY;
            }
        }

        // Where some scale lies outside what the outputs are held for, all of them say over what.
        int grown = held;
        bool wide = false;
        constexpr int kUp = kFollowed ? kProductUp : kAloneUp;
        if constexpr (HOW == kCodes) {
            spoilt = __any(outside != 0);
            if constexpr (kFollowed)
                if (spoilt) {
                    Scales reach;
#pragma unroll
                    for (uint32_t i = 0; i < kWords; ++i) reach.add(word[i]);
                    reach.join();
                    spoilt = reach.nan;
                    if (reach.most != 0) {
                        grown = held_of<kScaleTop>(reach.most);
                        const uint32_t from = power_bits(grown + kScaleTop - kTileSpread);
                        scale_low = (from - 1) * 0x10001u;
                        scale_high = (power_bits(grown + kScaleTop + 1) - 1) * 0x10001u;
                        wide = reach.least < from;
                    }
                }
        }
        if (__builtin_expect(spoilt, false)) spoil(a, group, tree, slot0, masked, source);

        float top = s[0][0];
#pragma unroll
        for (int e = 1; e < 8 * static_cast<int>(X); ++e) top = fmaxf(top, s[e >> 3][e & 7]);
        top = most_of_row<X>(top);
        // the offset follows once a score passes it by kSlack (the first: -inf + inf is a NaN, no less than)
        const bool follow = top > largest && !((top - largest) * unit <= static_cast<float>(kSlack));
        if (__any(follow) || grown != held) {
            const float most = fmaxf(largest, top);
            // the offset as used is what the factor is made of, so that its rounding cancels
            const float to = most == -INFINITY ? INFINITY : __builtin_fmaf(-most, unit, static_cast<float>(kUp));
            const float factor = largest == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(to - offset);
            const float down = factor * ldexpf(1.0f, held - grown);
            largest = most;
            offset = to;
            sum *= factor;
#pragma unroll
            for (uint32_t t = 0; t < kOuts; ++t) out[t] *= down;
        }
        held = grown;

        // rows that have seen nothing: -inf + inf would be a NaN
        const float to = largest == -INFINITY ? 0.0f : offset;
        float p[X][8];
        auto weigh = [&](uint32_t x) {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[x][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][e], unit, to));
            sum += ((p[x][0] + p[x][1]) + (p[x][2] + p[x][3])) + ((p[x][4] + p[x][5]) + (p[x][6] + p[x][7]));
        };
        if constexpr (kFollowed) {
#pragma unroll
            for (uint32_t x = 0; x < X; ++x) weigh(x);
            if (__builtin_expect(wide, false)) {
                widely(source, p, spoilt);
                return;
            }
        }
        [[maybe_unused]] const half2_t by = over(held);
        half2_t hi[X][4], lo[X][4];
#pragma unroll
        for (uint32_t x = 0; x < X; ++x) {
            if constexpr (!kFollowed) weigh(x);
#pragma unroll
            for (int e = 0; e < 4; ++e) split2(p[x][2 * e], p[x][2 * e + 1], &hi[x][e], &lo[x][e]);
        }
        [[maybe_unused]] uint4_t ahead[X];
        if constexpr (kFollowed)
#pragma unroll
            for (uint32_t x = 0; x < X; ++x) ahead[x] = finite_scale(source, 0, x, spoilt);
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            half8_t first[X], second[X];
            [[maybe_unused]] uint4_t scales[X];
            if constexpr (kFollowed)
#pragma unroll
                for (uint32_t x = 0; x < X; ++x) {
                    scales[x] = ahead[x];
                    if (b + 1 < NB) ahead[x] = finite_scale(source, b + 1, x, spoilt);
                }
#pragma unroll
            for (uint32_t x = 0; x < X; ++x) {
                if constexpr (!kFollowed) {
                    first[x] = join(hi[x][0], hi[x][1], hi[x][2], hi[x][3]);
                    second[x] = join(lo[x][0], lo[x][1], lo[x][2], lo[x][3]);
                } else {
                    // (hi + lo) d in two parts: hi d rounded, what that leaves
                    // (exact: 22 bits less their first 11) plus lo d
                    const uint4_t scale = scales[x];
                    half2_t u[4], w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const half2_t d = pair_of(scale[e]) * by;
                        u[e] = hi[x][e] * d;
                        w[e] = __builtin_elementwise_fma(lo[x][e], d, __builtin_elementwise_fma(hi[x][e], d, -u[e]));
                    }
                    first[x] = join(u[0], u[1], u[2], u[3]);
                    second[x] = join(w[0], w[1], w[2], w[3]);
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                const half8_t v = source.values(b, i);
                result_t& to = out[X == 1 ? 2 * b + i : b];
                to = multiply(v, second[X == 1 ? 0 : i], multiply(v, first[X == 1 ? 0 : i], to));
                if constexpr (HOW == kLaidOut && F != kF16) to = multiply(source.values_low(b, i), first[X == 1 ? 0 : i], to);
            }
            if constexpr (HOW == kLaidOut && F != kF16) {
                // a block's LDS reads among the products of the block before it
                if (b == 0) __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
                if (b + 1 < NB) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x8, 3, 0);
                if (b + 1 < NB) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x8, 3, 0);
            }
        }
    }

    // The outputs of a tile whose scales lie far apart: p d in f32, times the power
    // of two that puts the row's largest in [2^14, 2^15); hi, and lo times 2^11, so
    // that what is 2^-28 of the largest still has 22 bits. The outputs so far go
    // through the same powers, which stay far from f32's ends.
    template <typename SOURCE>
    __device__ __forceinline__ void widely(const SOURCE& source, const float (&p)[X][8], bool nan) {
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            __builtin_amdgcn_sched_barrier(0);  // a block's registers after another's
            float w[X][8], most = 0.0f;
#pragma unroll
            for (uint32_t x = 0; x < X; ++x) {
                const uint4_t scale = finite_scale(source, b, x, nan);
#pragma unroll
                for (int e = 0; e < 8; ++e) w[x][e] = p[x][e] * scale_at(scale, e), most = fmaxf(most, fabsf(w[x][e]));
            }
            const int shift = min(15 - __builtin_amdgcn_frexp_expf(most_of_row<X>(most)), 40);
            half8_t hi[X], lo[X];
#pragma unroll
            for (uint32_t x = 0; x < X; ++x)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y = ldexpf(w[x][e], shift);
                    hi[x][e] = static_cast<_Float16>(y);
                    lo[x][e] = static_cast<_Float16>((y - static_cast<float>(hi[x][e])) * 2048.0f);
                }
            const float there = ldexpf(2048.0f, held + shift), back = ldexpf(1.0f, -held - shift);
#pragma unroll
            for (uint32_t t = 0; t < kOuts / NB; ++t) out[kOuts / NB * b + t] *= there;
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                result_t& to = out[X == 1 ? 2 * b + i : b];
                to = multiply(source.values(b, i), lo[X == 1 ? 0 : i], to);
            }
#pragma unroll
            for (uint32_t t = 0; t < kOuts / NB; ++t) out[kOuts / NB * b + t] *= 1.0f / 2048.0f;
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                result_t& to = out[X == 1 ? 2 * b + i : b];
                to = multiply(source.values(b, i), hi[X == 1 ? 0 : i], to);
            }
#pragma unroll
            for (uint32_t t = 0; t < kOuts / NB; ++t) out[kOuts / NB * b + t] *= back;
        }
    }

    // Bit e: slot e of an octet has a scale that is a NaN.
    __device__ __forceinline__ static uint32_t nans_of(const uint4_t& scale) {
        uint32_t nans = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) nans |= (scale[e >> 1] >> (16 * (e & 1)) & 0x7FFFu) > 0x7C00u ? 1u << e : 0u;
        return nans;
    }
    // An octet's scales, zeros for NaNs where the tile has some: those are in the outputs already.
    template <typename SOURCE>
    __device__ __forceinline__ static uint4_t finite_scale(const SOURCE& source, uint32_t b, uint32_t x, bool nan) {
        uint4_t scale = source.value_scale(b, x);
        if (__builtin_expect(nan, false)) {
            const uint32_t nans = nans_of(scale);
#pragma unroll
            for (int w = 0; w < 4; ++w)
                scale[w] &= (nans >> (2 * w) & 1u ? 0u : 0xFFFFu) | (nans >> (2 * w + 1) & 1u ? 0u : 0xFFFF0000u);
        }
        return scale;
    }

    // A tile with value scales that are NaNs: a row that sees such a token gets NaNs in its block.
    template <typename SOURCE, typename TREE>
    __device__ __forceinline__ void spoil(const Attention& a, const Group& group, const TREE& tree, uint32_t slot0,
                                          bool masked, const SOURCE& source) {
        const uint32_t seen = masked ? sees(a, group, tree, slot0) : 0xFFFFFFFFu;
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            float mine = 0.0f;
#pragma unroll
            for (uint32_t x = 0; x < X; ++x)
                if (nans_of(source.value_scale(b, x)) & octet_bits(seen, x)) mine = 1.0f;
            const float nan = most_of_row<X>(mine) > 0.0f ? __builtin_nanf("") : 0.0f;
#pragma unroll
            for (uint32_t t = 0; t < kOuts / NB; ++t) out[kOuts / NB * b + t] += nan;
        }
    }

    // The last tile is done: the outputs, over 2^held, as the sum is.
    __device__ __forceinline__ void end() {
        const float up = ldexpf(1.0f, held);
#pragma unroll
        for (uint32_t t = 0; t < kOuts; ++t) out[t] *= up;
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

// A tile's operands out of its record in LDS. X = 2 reads them by lanes of its
// own order (Rows).
template <uint32_t F, uint32_t NB, uint32_t X>
struct Record {
    const uint8_t* at;
    uint32_t slot0, latest;  // what lies past the last token is cut: kept_of

    __device__ __forceinline__ half8_t keys(uint32_t b, uint32_t i) const {
        const uint32_t lane = threadIdx.x & 63u;
        const uint8_t* unit = at + b * cache_unit(F);
        if constexpr (X == 1) return operand<F, false>(unit, lane, i);
        // row n = 16 (g / 2) + 8h + 4 (g % 2) + r, values 16i + 8f on
        const uint32_t column = (lane >> 4 & 1u) * 8 + (lane >> 2 & 1u) * 4 + (lane & 3u);
        return operand<F, false>(unit, 16 * (2 * i + (lane >> 5)) + column, lane >> 3 & 1u);
    }
    __device__ __forceinline__ half8_t values(uint32_t b, uint32_t i) const {
        const uint32_t lane = threadIdx.x & 63u, g = group_of<X>(i);
        const uint8_t* unit = at + values_at(F, NB) + b * cache_unit(F);
        half8_t v = X == 1 ? operand<F, true>(unit, lane, i) : operand<F, true>(unit, 16 * g + (lane & 15u), lane >> 4 & 1u);
        if constexpr (F == kF16)
            if (slot0 + kTile > latest) {
                uint4_t w = __builtin_bit_cast(uint4_t, v);
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) w[x] &= kept_of(slot0, g, x, latest);
                v = __builtin_bit_cast(half8_t, w);
            }
        return v;
    }
    __device__ __forceinline__ uint4_t key_scale(uint32_t b, uint32_t x) const {
        return *reinterpret_cast<const uint4_t*>(at + key_scales_at(F, NB) + 64 * b + 16 * group_of<X>(x));
    }
    __device__ __forceinline__ uint4_t value_scale(uint32_t b, uint32_t x) const {
        const uint32_t g = group_of<X>(x);
        uint4_t s = *reinterpret_cast<const uint4_t*>(at + value_scales_at(F, NB) + 64 * b + 16 * g);
        if (slot0 + kTile > latest)
#pragma unroll
            for (uint32_t w = 0; w < 4; ++w) s[w] = kept_scale<F>(s[w], kept_of(slot0, g, w, latest));
        return s;
    }
    // The lane's of the tile's value scales, two; past the last, that.
    __device__ __forceinline__ uint32_t scale_word(uint32_t i) const {
        const uint32_t w = min(64 * i + (threadIdx.x & 63u), 16 * NB - 1);
        uint32_t s = reinterpret_cast<const uint32_t*>(at + value_scales_at(F, NB))[w];
        if (slot0 + kTile > latest) s = kept_scale<F>(s, kept_of(slot0, w / 4 & 3u, w & 3u, latest));
        return s;
    }
};

// Waves a workgroup and records a wave's ring: eight waves where two fit a
// SIMD's registers and two records of each fit the LDS, else four, else two.
constexpr uint32_t kRingBytes = 144 * 1024;
template <uint32_t F, uint32_t NB, uint32_t X>
struct AttendShape {
    static constexpr uint32_t kRecord = cache_record(F, NB);
    static constexpr uint32_t kWaves = NB * X <= 4 && 16 * kRecord <= kRingBytes ? 8 : 8 * kRecord <= kRingBytes ? 4 : 2;
    static constexpr uint32_t kRing = kRingBytes / (kWaves * kRecord) < 4 ? kRingBytes / (kWaves * kRecord) : 4;
    static constexpr uint32_t kCopies = (kRecord + 1023) / 1024;
};

template <uint32_t F, uint32_t NB, uint32_t X>
__global__ __launch_bounds__((64 * AttendShape<F, NB, X>::kWaves)) void attend(Attention a) {
    using Shape = AttendShape<F, NB, X>;
    constexpr uint32_t kRows = 16 * X, kRecord = Shape::kRecord, W = Shape::kWaves, D = Shape::kRing;
    constexpr uint32_t kQuads = Rows<F, NB, X>::kQuads, kParts = kQuads * 64;  // float4s of a wave's outputs
    __shared__ Tree<kRows> tree;
    // The waves' rings; then, all tiles done, their outputs.
    __shared__ __align__(16) uint8_t space[sizeof(uint8_t[W][D][kRecord]) > sizeof(float4_t[W][kParts])
                                               ? sizeof(uint8_t[W][D][kRecord])
                                               : sizeof(float4_t[W][kParts])];
    __shared__ float joined_offset[W][kRows], joined_sum[W][kRows];
    __shared__ uint32_t joined_live[kRows];

    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane % kRows;
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
    typename Rows<F, NB, X>::Queries queries;
    Rows<F, NB, X>::fetch(a, group, group.row0, queries);
    if (a.parents)
        read_tree(tree, a.parents + static_cast<uint64_t>(group.sequence) * a.tokens, a.tokens, group.token0,
                  group.token_end - group.token0, a.window);
    Rows<F, NB, X> rows;
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
        const Record<F, NB, X> record{ring + j % D * kRecord, slot0, group.latest};
        rows.template tile<kCodes>(a, group, tree, slot0, record);
        __asm__ __volatile__("s_waitcnt lgkmcnt(0)" ::: "memory");  // the record's reads, before its place is copied to
    }
    rows.end();
    __syncthreads();
    float4_t(*joined)[kParts] = reinterpret_cast<float4_t(*)[kParts]>(space);

    // The waves joined: each one's outputs on the least offset's (the largest
    // maximum's) scale, added in wave order, a thread some of the values.
    const float mine = sum_of_row<X>(rows.sum);
    if (lane < kRows) joined_offset[wave][n] = rows.offset, joined_sum[wave][n] = mine;
    if (threadIdx.x < kRows) joined_live[n] = rows.sight.live;
#pragma unroll
    for (uint32_t t = 0; t < kQuads; ++t) joined[wave][t * 64 + lane] = rows.quad(t);
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < kParts; at += 64 * W) {
        if (group.row0 + n >= group.row_end) continue;
        float least = INFINITY, total = 0.0f;
        float4_t out = float4_t(0.0f);
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            const float theirs = joined_offset[w][n];
            least = theirs < least || theirs != theirs ? theirs : least;
        }
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            // a wave that saw nothing has zeros, or the NaNs of scores that are
            const float theirs = joined_offset[w][n];
            const float factor = theirs == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(least - theirs);
            total = __builtin_fmaf(joined_sum[w][n], factor, total);
            out += joined[w][at] * factor;
        }
        finish<NB>(a, group, group.row0 + n, joined_live[n] != 0, Rows<F, NB, X>::quad_at(at / 64), out, total, least,
                   at < kRows);
    }
}

// ---- many rows: the waves split the rows -------------------------------------------

// A tile laid out in LDS by the workgroup for all of its waves: the codes as
// binary16 operands in the order of Rows (X = 2), the values' scaled, in two
// parts (the product of a code and a scale is exact in them), so that a wave
// does no more than read them. (A NaN among the scales, which is not every
// row's, goes in as 0: Rows::spoil.)
template <uint32_t F, uint32_t NB>
struct Stage {
    half8_t keys_[2 * NB][64], values_[2 * NB][64];   // [2 b + i]
    half8_t values_low_[F == kF16 ? 1 : 2 * NB][64];  // (F16's are exact in one)
    uint4_t key_scales_[NB][4], value_scales_[NB][4];

    __device__ __forceinline__ half8_t keys(uint32_t b, uint32_t i) const { return keys_[2 * b + i][threadIdx.x & 63u]; }
    __device__ __forceinline__ half8_t values(uint32_t b, uint32_t i) const { return values_[2 * b + i][threadIdx.x & 63u]; }
    __device__ __forceinline__ half8_t values_low(uint32_t b, uint32_t i) const {
        return values_low_[2 * b + i][threadIdx.x & 63u];
    }
    __device__ __forceinline__ uint4_t key_scale(uint32_t b, uint32_t x) const { return key_scales_[b][group_of<2>(x)]; }
    __device__ __forceinline__ uint4_t value_scale(uint32_t b, uint32_t x) const { return value_scales_[b][group_of<2>(x)]; }
};

// Waves of 32 rows a workgroup: two a SIMD where their registers allow.
constexpr uint32_t row_waves(uint32_t blocks) { return blocks <= 4 ? 8 : 4; }

// A wave's rows, their last tile done: `write` takes what `finish` does.
template <uint32_t F, uint32_t NB, uint32_t X, typename WRITE>
__device__ __forceinline__ void write_rows(const Group& group, Rows<F, NB, X>& rows, uint32_t row0, const WRITE& write) {
    rows.end();
    const uint32_t lane = threadIdx.x & 63u, row = row0 + lane % (16 * X);
    const float total = sum_of_row<X>(rows.sum);
    if (row >= group.row_end) return;
#pragma unroll
    for (uint32_t t = 0; t < Rows<F, NB, X>::kQuads; ++t)
        write(row, rows.sight.live, Rows<F, NB, X>::quad_at(t), rows.quad(t), total, rows.offset, t == 0 && lane < 16 * X);
}

// A sequence's records, one after the other: record t.
template <uint32_t BYTES>
struct Records {
    static constexpr bool kGaps = false;  // none is missing
    const uint8_t* base;
    __device__ __forceinline__ const uint8_t* operator()(uint32_t t) const { return base + static_cast<uint64_t>(t) * BYTES; }
    __device__ __forceinline__ const uint8_t* of_wave(uint32_t t) const { return (*this)(t); }  // a t that is the wave's
};

// A wave's 32 rows by themselves, straight from the records, 16 at a time.
template <uint32_t F, uint32_t NB, typename TREE, typename RECORDS, typename WRITE>
__device__ __forceinline__ void attend_alone(const Attention& a, const Group& group, const TREE& tree, const RECORDS& records,
                                             uint32_t row0, const WRITE& write) {
#pragma unroll 1
    for (uint32_t first = row0; first < min(row0 + 32, group.row_end); first += 16) {
        typename Rows<F, NB, 1>::Queries queries;
        Rows<F, NB, 1>::fetch(a, group, first, queries);
        Rows<F, NB, 1> rows;
        rows.begin(a, group, tree, first, queries);
#pragma unroll 1
        for (uint32_t t = group.tile_begin; t < group.tile_end; ++t) {
            const uint8_t* at = records(t);
            if constexpr (RECORDS::kGaps)
                if (!at) {  // NaNs for the rows that see it
                    if (rows.sees(a, group, tree, t * kTile) != 0) rows.sum = __builtin_nanf("");
                    continue;
                }
            const Record<F, NB, 1> record{at, t * kTile, group.latest};
            rows.template tile<kCodes>(a, group, tree, t * kTile, record);
        }
        write_rows(group, rows, first, write);
    }
}

// A workgroup's LDS for them.
template <uint32_t F, uint32_t NB>
struct RowsShape {
    static constexpr uint32_t W = row_waves(NB), kRows = 32 * W;
    static constexpr uint32_t kTiles = NB <= 4 ? 2 : 1;  // a stage's
};
template <uint32_t F, uint32_t NB>
struct RowsSpace {
    Stage<F, NB> stages[2][RowsShape<F, NB>::kTiles];
    uint32_t wave_most[row_waves(NB)], wave_least[row_waves(NB)], wave_spoilt[row_waves(NB)];
};

// A workgroup's rows over its split's tiles; `alone`: some record is missing.
template <uint32_t F, uint32_t NB, typename TREE, typename RECORDS, typename WRITE>
__device__ __forceinline__ void attend_group(Attention a, Group group, TREE& tree, RowsSpace<F, NB>& space,
                                             RECORDS records, WRITE write, bool alone) {
    using Shape = RowsShape<F, NB>;
    constexpr uint32_t W = Shape::W, kUnit = cache_unit(F), kTiles = Shape::kTiles;
    constexpr uint32_t kUnits = 2 * NB * kTiles, kMine = (kUnits + W - 1) / W;  // units of a stage; a wave's, at most
    constexpr uint32_t kScaleWords = (key_scales(F) ? 32 : 16) * NB;            // a tile's
    constexpr uint32_t kLoads = kUnit / 1024 + (kUnit < 1024 ? 1 : 0);          // 16-byte (Q4_0: 8-byte) loads a lane a unit
    static_assert(kScaleWords * kTiles <= 64 * W, "a thread a dword");
    auto& stages = space.stages;
    auto &wave_most = space.wave_most, &wave_least = space.wave_least, &wave_spoilt = space.wave_spoilt;

    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row0 = group.row0 + 32 * wave;
    const bool mine = row0 < group.row_end;  // a wave without rows still lays out its share
    typename Rows<F, NB, 2>::Queries queries;
    Rows<F, NB, 2>::fetch(a, group, min(row0, group.row_end - 1), queries);
    // a chain's wave sees nothing past its last row's token
    const uint32_t sees_to =
        a.parents ? group.latest : group.past + (min(row0 + 32, group.row_end) - 1) / a.group + 1;
    if constexpr (RECORDS::kGaps)
        if (alone) {
            attend_alone<F, NB>(a, group, tree, records, row0, write);
            return;
        }

    // All the tiles' value scales, once: how far they reach, and whether any is a NaN (F16: other than one).
    Scales reach;
    uint32_t spoilt = 0;
#pragma unroll 4
    for (uint32_t x = threadIdx.x; x < (group.tile_end - group.tile_begin) * 16 * NB; x += 64 * W) {
        const uint32_t t = group.tile_begin + x / (16 * NB), w = x % (16 * NB);
        const uint32_t word = kept_scale<F>(
            reinterpret_cast<const uint32_t*>(records(t) + value_scales_at(F, NB))[w],
            kept_of(t * kTile, w / 4 & 3u, w & 3u, group.latest));
        if constexpr (F == kF16)
            spoilt |= word ^ 0x3C003C00u;
        else
            reach.add(word);
    }
    reach.join();
    spoilt = F == kF16 ? __any(spoilt != 0) : reach.nan;
    if (lane == 0) wave_most[wave] = reach.most, wave_least[wave] = reach.least, wave_spoilt[wave] = spoilt;
    if constexpr (TREE::kTrees)
        if (a.parents)
            read_tree(tree, a.parents + static_cast<uint64_t>(group.sequence) * a.tokens, a.tokens, group.token0,
                      group.token_end - group.token0, a.window);
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < W; ++w)
        reach.most = max(reach.most, wave_most[w]), reach.least = min(reach.least, wave_least[w]), spoilt |= wave_spoilt[w];
    spoilt = __builtin_amdgcn_readfirstlane(spoilt);
    const int exponent = F == kF16 ? 0 : held_of<kCodeTop>(__builtin_amdgcn_readfirstlane(reach.most));
    const half2_t by = over(exponent);

    if constexpr (F != kF16)
        if (__builtin_amdgcn_readfirstlane(reach.least) < power_bits(exponent + kCodeTop - kSplitSpread)) {
            // scales further apart than a layout is made for
            attend_alone<F, NB>(a, group, tree, records, row0, write);
            return;
        }
    Rows<F, NB, 2> rows;
    rows.begin(a, group, tree, min(row0, group.row_end - 1), queries);
    rows.held = exponent;

    // Unit u of a stage: tile u / 2NB, block u % NB, keys then values. A lane
    // holds what it will lay out: as the unit has it, lane for lane.
    struct Held {
        uint4_t w[kLoads];
    } held[kMine];
    uint4_t unit_scale[kMine];  // a value unit's
    uint32_t scale_word = 0;    // of those that the waves read
    auto load = [&](uint32_t tile0) {
#pragma unroll
        for (uint32_t j = 0; j < kMine; ++j) {
            const uint32_t u = wave + W * j, t = tile0 + u / (2 * NB);
            if (u >= kUnits || t >= group.tile_end) continue;
            const uint8_t* record = records.of_wave(t);
            const uint8_t* unit = record + u % (2 * NB) * kUnit;
            if constexpr (F == kQ4_0) {
                const uint2 w = *reinterpret_cast<const uint2*>(unit + 8 * lane);
                held[j].w[0][0] = w.x, held[j].w[0][1] = w.y;
            } else {
#pragma unroll
                for (uint32_t x = 0; x < kLoads; ++x) held[j].w[x] = *reinterpret_cast<const uint4_t*>(unit + 1024 * x + 16 * lane);
            }
            if (F != kF16 && u % (2 * NB) >= NB)
                unit_scale[j] = *reinterpret_cast<const uint4_t*>(record + value_scales_at(F, NB) + 64 * (u % NB) + 16 * (lane >> 4));
        }
        const uint32_t t = tile0 + threadIdx.x / kScaleWords;
        if (threadIdx.x < kScaleWords * kTiles && t < group.tile_end)
            scale_word = reinterpret_cast<const uint32_t*>((kScaleWords % 64 ? records(t) : records.of_wave(t)) +
                                                           key_scales_at(F, NB))[threadIdx.x % kScaleWords];
    };
    auto lay = [&](uint32_t tile0, Stage<F, NB>* stage) {
        const uint32_t quarter = lane >> 4, column = lane & 15u;
#pragma unroll
        for (uint32_t j = 0; j < kMine; ++j) {
            const uint32_t u = wave + W * j, t = u / (2 * NB), b = u % NB, slot0 = (tile0 + t) * kTile;
            if (u >= kUnits || tile0 + t >= group.tile_end) continue;
            uint32_t w[8];
#pragma unroll
            for (uint32_t x = 0; x < 4 * kLoads; ++x) w[x] = held[j].w[x >> 2][x & 3];
            if (u % (2 * NB) < NB) {
                // token 16h + column, its row; values 8 quarter on
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    half8_t k;
                    if constexpr (F == kF16)
                        k = __builtin_bit_cast(half8_t, held[j].w[h]);
                    else if constexpr (F == kQ8_0)
                        k = halves_of<128>(w[2 * h], w[2 * h + 1]);
                    else
                        k = halves_of<8>(w[h] & 0x0F0F0F0Fu, w[h] >> 4 & 0x0F0F0F0Fu);
                    const uint32_t row = column / 8 * 16 + 8 * h + column % 8;
                    stage[t].keys_[2 * b + quarter / 2][32 * (quarter & 1u) + row] = k;
                }
                continue;
            }
            // what lies past the last token is no one's, and may be anything
            uint32_t kept[4] = {~0u, ~0u, ~0u, ~0u};
            if (slot0 + kTile > group.latest)
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) kept[x] = kept_of(slot0, quarter, x, group.latest);
            half2_t d[4];
            if constexpr (F != kF16)
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) {
                    uint32_t s = unit_scale[j][x] & kept[x];
                    if (spoilt)
                        s = ((s & 0x7FFFu) > 0x7C00u ? 0u : s & 0xFFFFu) | ((s & 0x7FFF0000u) > 0x7C000000u ? 0u : s & 0xFFFF0000u);
                    d[x] = pair_of(s) * by;
                }
            // tokens of group `quarter`, value 16 part + column
#pragma unroll
            for (uint32_t part = 0; part < 2; ++part) {
                const uint32_t to = 32 * (quarter & 1u) + 16 * part + column, i = 2 * b + quarter / 2;
                if constexpr (F == kF16) {
                    uint4_t v = held[j].w[part];
#pragma unroll
                    for (uint32_t x = 0; x < 4; ++x) v[x] &= kept[x];
                    stage[t].values_[i][to] = __builtin_bit_cast(half8_t, v);
                } else {
                    const half8_t code = F == kQ8_0 ? halves_of<128>(w[2 * part], w[2 * part + 1])
                                                    : halves_of<8>(w[0] >> (4 * part) & 0x0F0F0F0Fu, w[1] >> (4 * part) & 0x0F0F0F0Fu);
                    half2_t hi[4], lo[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const half2_t c = {code[2 * x], code[2 * x + 1]};
                        hi[x] = c * d[x];
                        lo[x] = __builtin_elementwise_fma(c, d[x], -hi[x]);
                    }
                    stage[t].values_[i][to] = join(hi[0], hi[1], hi[2], hi[3]);
                    stage[t].values_low_[i][to] = join(lo[0], lo[1], lo[2], lo[3]);
                }
            }
        }
        const uint32_t t = threadIdx.x / kScaleWords, x = threadIdx.x % kScaleWords;
        if (threadIdx.x < kScaleWords * kTiles && tile0 + t < group.tile_end) {
            const bool values = !key_scales(F) || x >= 16 * NB;
            if (values)
                scale_word = kept_scale<F>(scale_word, kept_of((tile0 + t) * kTile, x / 4 & 3u, x & 3u, group.latest));
            uint32_t* to = reinterpret_cast<uint32_t*>(values ? stage[t].value_scales_ : stage[t].key_scales_);
            to[x % (16 * NB)] = scale_word;
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
                rows.template tile<kLaidOut>(a, group, tree, slot0, stages[turn][t], spoilt != 0);
        }
        // the other stage was read before the last barrier
        if (more) lay(tile0 + kTiles, stages[turn ^ 1]);
        __syncthreads();
    }
    if (mine) write_rows(group, rows, row0, write);
}

template <uint32_t F, uint32_t NB>
__global__ __launch_bounds__(64 * row_waves(NB)) void attend_rows(Attention a) {
    constexpr uint32_t kRows = RowsShape<F, NB>::kRows;
    __shared__ Tree<kRows < kTreeTokens ? kRows : kTreeTokens> tree;
    __shared__ RowsSpace<F, NB> space;
    const Group group(a, kRows);
    const Records<cache_record(F, NB)> records{record_of(a.cache, F, group.sequence, group.head, 0)};
    auto write = [&](uint32_t row, bool live, uint32_t at, float4_t out, float total, float least, bool stats) {
        finish<NB>(a, group, row, live, at, out, total, least, stats);
    };
    attend_group<F, NB>(a, group, tree, space, records, write, false);
}

template <uint32_t F, uint32_t NB>
static hipError_t launch_blocks(const Attention& a, const AttentionPlan& plan, hipStream_t stream) {
    const dim3 grid(a.cache.sequences * a.cache.kv_heads * plan.row_groups * plan.splits);
    if (plan.waves > 1) {
        if constexpr (NB <= 4 || F == kF16)  // wider quantized heads take attend alone: plan_attention
            hipLaunchKernelGGL((attend_rows<F, NB>), grid, dim3(64 * row_waves(NB)), 0, stream, a);
    } else if (plan.octets == 2)
        hipLaunchKernelGGL((attend<F, NB, 2>), grid, dim3(64 * AttendShape<F, NB, 2>::kWaves), 0, stream, a);
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
