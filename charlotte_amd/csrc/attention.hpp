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
// Range: p is at most 2^(10 - D), D the exponent of the largest value scale
// met, so p d stays below 2^12 and its lo part's steps (2^-24) 34 bits below
// the largest: D stands in the exponent's offset as the maximum does, and
// grows as it does.
//
// Split: a workgroup takes up to 16 or 32 rows of a key head and a run of its
// tiles, each wave every fourth tile, and joins its four waves' outputs in
// LDS; where a step has too few rows to fill the card its tiles are split
// among several workgroups, joined by attention_combine.
#pragma once

#include "cache.hpp"

namespace chm {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));

constexpr float kLog2E = 1.44269504088896340736f;
constexpr uint32_t kAttentionWaves = 4;

// A lane's codes of one unit (keys or values of a block by 32 tokens).
template <uint32_t F>
struct Codes;
template <>
struct Codes<kQ8_0> {
    uint32_t w[4];
};
template <>
struct Codes<kQ4_0> {
    uint32_t w[2];
};
template <>
struct Codes<kF16> {
    uint32_t w[8];
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
    half2_t a, b, d, e;
    if constexpr (F == kQ8_0) {
        halves_of<128>(c.w[2 * part], &a, &b);
        halves_of<128>(c.w[2 * part + 1], &d, &e);
    } else if constexpr (F == kQ4_0) {
        if constexpr (VALUES) {
            halves_of<8>(c.w[0] >> (4 * part) & 0x0F0F0F0Fu, &a, &b);
            halves_of<8>(c.w[1] >> (4 * part) & 0x0F0F0F0Fu, &d, &e);
        } else {
            halves_of<8>(c.w[part] & 0x0F0F0F0Fu, &a, &b);
            halves_of<8>(c.w[part] >> 4 & 0x0F0F0F0Fu, &d, &e);
        }
    } else {
        uint4 w = {c.w[4 * part], c.w[4 * part + 1], c.w[4 * part + 2], c.w[4 * part + 3]};
        return __builtin_bit_cast(half8_t, w);
    }
    return join(a, b, d, e);
}

__device__ __forceinline__ float4_t multiply(half8_t a, half8_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Slot i's scale of a lane's eight, i a constant.
__device__ __forceinline__ float scale_at(const uint4& s, int i) {
    const uint32_t w = i < 2 ? s.x : i < 4 ? s.y : i < 6 ? s.z : s.w;
    return static_cast<float>(__builtin_bit_cast(half2_t, w)[i & 1]);
}

// Two f32 as two binary16 parts of each: hi rounded towards zero, lo what it
// leaves, rounded likewise (2^-21 of the value at the most).
__device__ __forceinline__ void split2(float a, float b, half2_t* hi, half2_t* lo) {
    *hi = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    *lo = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf(static_cast<float>(hi->x), -1.0f, a),
                                                                 __builtin_fmaf(static_cast<float>(hi->y), -1.0f, b)));
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
    for (uint32_t i = threadIdx.x; i < tokens; i += 256) tree.parents[i] = parents[i];
    for (uint32_t i = threadIdx.x; i < TOKENS * (kTreeTokens / 32); i += 256)
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

template <uint32_t F, uint32_t NB, uint32_t RT>
__global__ __launch_bounds__(256) void attend(Attention a) {
    constexpr uint32_t kRows = 16 * RT, kRecord = cache_record(F, NB), kUnit = cache_unit(F);
    __shared__ Tree<kRows> tree;
    __shared__ float4_t joined[2][RT * 2 * NB][64];
    __shared__ float joined_offset[kAttentionWaves][kRows], joined_sum[kAttentionWaves][kRows];

    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, n = lane & 15u, g = lane >> 4;
    const uint32_t split = blockIdx.x % a.splits, at = blockIdx.x / a.splits;
    const uint32_t row_groups = (a.rows + kRows - 1) / kRows;
    const uint32_t row0 = at % row_groups * kRows, sequence_head = at / row_groups;
    const uint32_t sequence = sequence_head / a.cache.kv_heads, head = sequence_head % a.cache.kv_heads;
    const uint32_t past = min(a.past[sequence], a.cache.capacity - a.tokens);

    // The workgroup's tokens, and its rows' sight.
    const uint32_t row_end = min(row0 + kRows, a.rows);
    const uint32_t token0 = row0 / a.group, token_end = (row_end - 1) / a.group + 1;
    if (a.parents)
        read_tree(tree, a.parents + static_cast<uint64_t>(sequence) * a.tokens, a.tokens, token0, token_end - token0,
                  a.window);
    Sight sight[RT];
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
        const uint32_t row = row0 + 16 * i + n;
        const uint32_t token = min(row, row_end - 1) / a.group;
        const uint32_t depth = a.parents ? tree.depth[token - token0] : token;
        sight[i].live = row < row_end && depth != kUnused;
        const uint32_t place = past + (sight[i].live ? depth : 0u) + 1;  // one past its own place
        sight[i].first = a.window && place > a.window ? place - a.window : 0u;
        sight[i].last = a.parents ? token - token0 : past + token;
    }

    // Its tiles: from the window's first to the last token its rows may see.
    const uint32_t end = a.parents ? past + a.tokens : past + token_end;
    const uint32_t earliest = past + (a.parents ? 0u : token0) + 1;
    const uint32_t begin = a.window && earliest > a.window ? earliest - a.window : 0u;
    const uint32_t tile_begin = begin / kTile, tile_end = (end + kTile - 1) / kTile;
    const uint32_t share = (tile_end - tile_begin + a.splits - 1) / a.splits;
    const uint32_t my_begin = min(tile_begin + split * share, tile_end), my_end = min(my_begin + share, tile_end);
    // Slots that every row of the workgroup sees: from `all_begin` to `past`.
    const uint32_t latest = past + a.tokens;
    const uint32_t all_begin = a.window && latest > a.window ? latest - a.window : 0u;

    // The rows' queries as operands, 2^(-shift) their power of two.
    half8_t high[RT][NB], low[RT][NB];
    float unit[RT];
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
        const uint32_t row = min(row0 + 16 * i + n, row_end - 1);
        const float* q = a.queries + (static_cast<uint64_t>(sequence) * a.tokens + row / a.group) * a.query_stride +
                         static_cast<uint64_t>(head * a.group + row % a.group) * (32 * NB) + 8 * g;
        float x[NB][8], largest = 0.0f;
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            const float4 u = *reinterpret_cast<const float4*>(q + 32 * b), v = *reinterpret_cast<const float4*>(q + 32 * b + 4);
            x[b][0] = u.x, x[b][1] = u.y, x[b][2] = u.z, x[b][3] = u.w;
            x[b][4] = v.x, x[b][5] = v.y, x[b][6] = v.z, x[b][7] = v.w;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[b][e] *= a.scale * kLog2E, largest = fmaxf(largest, fabsf(x[b][e]));
        }
        largest = fmaxf(largest, __shfl_xor(largest, 16));
        largest = fmaxf(largest, __shfl_xor(largest, 32));
        int shift = 0;
        if (largest > 0.0f && largest <= 3.4e38f) {
            int e;
            (void)frexpf(largest, &e);
            shift = min(11 - e, 126);
        }
        unit[i] = ldexpf(1.0f, -shift);
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            half2_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) split2(ldexpf(x[b][2 * e], shift), ldexpf(x[b][2 * e + 1], shift), &hi[e], &lo[e]);
            high[i][b] = join(hi[0], hi[1], hi[2], hi[3]);
            low[i][b] = join(lo[0], lo[1], lo[2], lo[3]);
        }
    }

    float4_t out[RT][2 * NB];
    float largest[RT], offset[RT], sum[RT];  // the raw maximum; exp2's offset; the lane's part of the sum
    int exponent = -64;                      // D, the same in every lane
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
        largest[i] = -INFINITY, offset[i] = INFINITY, sum[i] = 0.0f;
#pragma unroll
        for (uint32_t t = 0; t < 2 * NB; ++t) out[i][t] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const uint8_t* base = record_of(a.cache, F, sequence, head, 0);
    for (uint32_t tile = my_begin + wave; tile < my_end; tile += kAttentionWaves) {
        const uint8_t* record = base + static_cast<uint64_t>(tile) * kRecord;
        Codes<F> keys[NB], values[NB];
        uint4 key_scale[NB], value_scale[NB];
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            keys[b] = load_codes<F>(record + b * kUnit, lane);
            if constexpr (key_scales(F))
                key_scale[b] = *reinterpret_cast<const uint4*>(record + key_scales_at(F, NB) + 64 * b + 16 * g);
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            values[b] = load_codes<F>(record + values_at(F, NB) + b * kUnit, lane);
            value_scale[b] = *reinterpret_cast<const uint4*>(record + value_scales_at(F, NB) + 64 * b + 16 * g);
        }

        // Scores: s[i][h][r] of token 16h + 4g + r.
        float4_t s[RT][2];
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) s[i][0] = s[i][1] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const half8_t k = operand<F, false>(keys[b], h);
#pragma unroll
                for (uint32_t i = 0; i < RT; ++i) {
                    if constexpr (key_scales(F)) {
                        float4_t p = multiply(k, high[i][b], float4_t{0.0f, 0.0f, 0.0f, 0.0f});
                        p = multiply(k, low[i][b], p);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            s[i][h][r] = __builtin_fmaf(p[r], scale_at(key_scale[b], 4 * h + r), s[i][h][r]);
                    } else {
                        s[i][h] = multiply(k, high[i][b], s[i][h]);
                        s[i][h] = multiply(k, low[i][b], s[i][h]);
                    }
                }
            }
        }

        const uint32_t slot0 = tile * kTile;
        const bool masked = slot0 + kTile > past || slot0 < all_begin;
        bool seen[RT][8];
        if (masked) {
#pragma unroll
            for (uint32_t i = 0; i < RT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const uint32_t slot = slot0 + 16 * h + 4 * g + r;
                        bool sees = slot >= sight[i].first;
                        if (!a.parents) {
                            sees = sees && slot <= sight[i].last;
                        } else if (slot >= past) {
                            const uint32_t node = slot - past;
                            sees = node < a.tokens && (tree.above[sight[i].last][node >> 5] >> (node & 31u) & 1u);
                        }
                        seen[i][4 * h + r] = sees;
                        if (!sees) s[i][h][r] = -INFINITY;
                    }
            // What lies past the last token is no one's, and may be anything:
            // scales as if never met, F16's values zero.
            if (slot0 + kTile > latest) {
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) {
                    constexpr uint32_t kPlain = F == kF16 ? 0x3C003C00u : 0u;
                    uint32_t* const scale[4] = {&value_scale[b].x, &value_scale[b].y, &value_scale[b].z, &value_scale[b].w};
#pragma unroll
                    for (uint32_t w = 0; w < 4; ++w) {
                        const uint32_t slot = slot0 + w / 2 * 16 + 4 * g + (w & 1) * 2;
                        const uint32_t kept = slot >= latest ? 0u : slot + 1 >= latest ? 0xFFFFu : 0xFFFFFFFFu;
                        *scale[w] = (*scale[w] & kept) | (kPlain & ~kept);
                        if constexpr (F == kF16) values[b].w[w] &= kept, values[b].w[4 + w] &= kept;
                    }
                }
            }
        }

        // The largest value scale's exponent.
        bool scaled = true;  // whether value scales are other than one
        int grown = exponent;
        if constexpr (F == kF16) {
            uint32_t other = 0;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b)
                other |= (value_scale[b].x ^ 0x3C003C00u) | (value_scale[b].y ^ 0x3C003C00u) |
                         (value_scale[b].z ^ 0x3C003C00u) | (value_scale[b].w ^ 0x3C003C00u);
            scaled = __any(other != 0);
            grown = 0;
        } else {
            uint32_t most = 0;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const uint32_t w[4] = {value_scale[b].x, value_scale[b].y, value_scale[b].z, value_scale[b].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lo = w[e] & 0x7FFFu, hi = w[e] >> 16 & 0x7FFFu;
                    // a NaN scale spoils its own rows alone
                    most = max(most, max(lo > 0x7C00u ? 0u : lo, hi > 0x7C00u ? 0u : hi));
                }
            }
            most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 16)));
            most = max(most, static_cast<uint32_t>(__shfl_xor(static_cast<int>(most), 32)));
            // 2^grown <= the scale < 2^(grown + 1); subnormals count as the least normal
            grown = max(exponent, static_cast<int>(max(most >> 10, 1u)) - 15);
        }

#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) {
            float top = fmaxf(fmaxf(fmaxf(s[i][0][0], s[i][0][1]), fmaxf(s[i][0][2], s[i][0][3])),
                              fmaxf(fmaxf(s[i][1][0], s[i][1][1]), fmaxf(s[i][1][2], s[i][1][3])));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float most = fmaxf(largest[i], top);
            if (__any(most > largest[i]) || grown != exponent) {
                // the offset as used is what the factor is made of, so that its rounding cancels
                const float to = most == -INFINITY ? INFINITY : __builtin_fmaf(-most, unit[i], static_cast<float>(10 - grown));
                const float factor = largest[i] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(to - offset[i]);
                largest[i] = most;
                offset[i] = to;
                sum[i] *= factor;
#pragma unroll
                for (uint32_t t = 0; t < 2 * NB; ++t) out[i][t] *= factor;
            }
        }
        exponent = grown;

#pragma unroll
        for (uint32_t i = 0; i < RT; ++i) {
            // rows that have seen nothing: -inf + inf would be a NaN
            const float to = largest[i] == -INFINITY ? 0.0f : offset[i];
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][e >> 2][e & 3], unit[i], to));
                sum[i] += p[e];
            }
            half8_t hi8, lo8;
            auto split8 = [&](const float* x) {
                half2_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) split2(x[2 * e], x[2 * e + 1], &hi[e], &lo[e]);
                hi8 = join(hi[0], hi[1], hi[2], hi[3]);
                lo8 = join(lo[0], lo[1], lo[2], lo[3]);
            };
            if (F == kF16 && !scaled) split8(p);
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                if (scaled) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        x[e] = __builtin_fmaf(p[e], scale_at(value_scale[b], e), 0.0f);
                        // a scale that the row does not see may be a NaN
                        if (masked && !seen[i][e]) x[e] = 0.0f;
                    }
                    split8(x);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const half8_t v = operand<F, true>(values[b], u);
                    out[i][2 * b + u] = multiply(v, hi8, out[i][2 * b + u]);
                    out[i][2 * b + u] = multiply(v, lo8, out[i][2 * b + u]);
                }
            }
        }
    }

    // The four waves joined: each one's outputs on the least offset's (the
    // largest maximum's) scale, waves 2 and 3 into 0 and 1, then 1 into 0.
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
        sum[i] += __shfl_xor(sum[i], 16);
        sum[i] += __shfl_xor(sum[i], 32);
        if (g == 0) joined_offset[wave][16 * i + n] = offset[i], joined_sum[wave][16 * i + n] = sum[i];
    }
    __syncthreads();
    float total[RT], least[RT];
#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
        least[i] = INFINITY, total[i] = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kAttentionWaves; ++w) {
            const float theirs = joined_offset[w][16 * i + n];
            least[i] = theirs < least[i] || theirs != theirs ? theirs : least[i];
        }
#pragma unroll
        for (uint32_t w = 0; w < kAttentionWaves; ++w) {
            const float theirs = joined_offset[w][16 * i + n];
            total[i] += joined_sum[w][16 * i + n] * (theirs == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(least[i] - theirs));
        }
        const float factor = offset[i] == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(least[i] - offset[i]);
#pragma unroll
        for (uint32_t t = 0; t < 2 * NB; ++t) out[i][t] *= factor;
    }
    auto give = [&](uint32_t place) {
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i)
#pragma unroll
            for (uint32_t t = 0; t < 2 * NB; ++t) joined[place][i * 2 * NB + t][lane] = out[i][t];
    };
    auto take = [&](uint32_t place) {
#pragma unroll
        for (uint32_t i = 0; i < RT; ++i)
#pragma unroll
            for (uint32_t t = 0; t < 2 * NB; ++t) out[i][t] += joined[place][i * 2 * NB + t][lane];
    };
    if (wave >= 2) give(wave - 2);
    __syncthreads();
    if (wave < 2) take(wave);
    __syncthreads();
    if (wave == 1) give(0);
    __syncthreads();
    if (wave != 0) return;
    take(0);

#pragma unroll
    for (uint32_t i = 0; i < RT; ++i) {
        const uint32_t row = row0 + 16 * i + n;
        if (row >= row_end) continue;
        // nothing seen: no maximum, and no NaN either
        const bool empty = !sight[i].live || (least[i] == INFINITY && total[i] == 0.0f);
        if (a.splits == 1) {
            const float inverse = empty ? 0.0f : 1.0f / total[i];
            float* to = a.output + (static_cast<uint64_t>(sequence) * a.tokens + row / a.group) * a.output_stride +
                        static_cast<uint64_t>(head * a.group + row % a.group) * (32 * NB) + 4 * g;
#pragma unroll
            for (uint32_t t = 0; t < 2 * NB; ++t)
                *reinterpret_cast<float4*>(to + 16 * t) =
                    empty ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                          : make_float4(out[i][t][0] * inverse, out[i][t][1] * inverse, out[i][t][2] * inverse,
                                        out[i][t][3] * inverse);
        } else {
            const uint64_t place = (static_cast<uint64_t>(sequence_head) * a.rows + row) * a.splits + split;
            float* to = a.partial + place * (32 * NB) + 4 * g;
            if (!empty)
#pragma unroll
                for (uint32_t t = 0; t < 2 * NB; ++t)
                    *reinterpret_cast<float4*>(to + 16 * t) = make_float4(out[i][t][0], out[i][t][1], out[i][t][2], out[i][t][3]);
            if (g == 0) {
                const bool spoilt = total[i] != total[i];
                a.stats[place] = make_float2(empty ? INFINITY : spoilt ? total[i] : least[i], empty ? 0.0f : total[i]);
            }
        }
    }
}

template <uint32_t F, uint32_t NB>
static hipError_t launch_blocks(const Attention& a, const AttentionPlan& plan, hipStream_t stream) {
    const dim3 grid(a.cache.sequences * a.cache.kv_heads * plan.row_groups * plan.splits);
    if constexpr (NB <= 4) {
        if (plan.row_tiles == 2) {
            hipLaunchKernelGGL((attend<F, NB, 2>), grid, dim3(256), 0, stream, a);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL((attend<F, NB, 1>), grid, dim3(256), 0, stream, a);
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
