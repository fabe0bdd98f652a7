// Drafted tokens against the target's probabilities, from given uniform
// numbers. The draws are exact, in whole numbers: a probability x counts
// floor(x 2^44) units, a row's units W are summed in 64 bits in any order, and
// the token drawn is the lowest index whose running sum passes W r / 2^31, r =
// floor(u 2^31); so however a row is cut, the token is the same.
//
// Two launches. draw_sums: each row to draw from, in segments of 256 entries, a
// wave a segment at a time, each segment's units summed: the one pass over the
// probabilities. A chain with a draft draws once a sequence, from the row where
// its walk ends; every workgroup walks it anew (a lane a token, three reads
// each), which costs less than a launch. walk_*: a wave a draw sums the
// segments, a lane a run of them, finds the segment, and reads its entries again
// (from cache) for the index: two dependent reads. Without a draft a workgroup a
// sequence draws for every node and its first wave then walks the tree.
//
// Bound by bytes: 4 a probability of the rows drawn from, once. A tree of 21 nodes
// over 151,936 (12.8 MB): 5.1 us, and its walk 6.4: one compute unit reads the 21
// rows' sums, 100 KB (7.8 with each lane's run read where it lies, through no
// LDS). Chains of 6 in 8 sequences over 128,256: 4.1 and 4.4.
#include <algorithm>

#include "rows.hpp"
#include "serving.hpp"

namespace chm {

constexpr uint32_t kWalkWaves = 16;

__device__ __forceinline__ uint32_t length_of(const Verify& a, uint32_t sequence) {
    return a.lengths ? min(a.lengths[sequence], a.tokens) : a.tokens;
}

// The row a draw is from: the target's after `node`, less the draft's where
// the token drafted after it was refused.
struct DrawRow {
    const float* target;
    const float* draft;  // or null
};

// A chain's walk: the last node accepted, by one wave, every lane the same.
__device__ __forceinline__ uint32_t accepted_of(const Verify& a, uint32_t sequence, uint32_t length) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t first = static_cast<uint64_t>(sequence) * a.tokens;
    for (uint32_t i0 = 0; i0 + 1 < length; i0 += 64) {
        const uint32_t i = i0 + lane;
        bool refused = false;
        if (i + 1 < length) {
            const int32_t token = a.node_tokens[first + i + 1];
            refused = true;
            if (token >= 0 && static_cast<uint32_t>(token) < a.vocabulary) {
                const float p = a.target[(first + i) * a.target_stride + token];
                const float q = a.draft[(static_cast<uint64_t>(sequence) * (a.tokens - 1) + i) * a.draft_stride + token];
                refused = !(a.accepts[first + i + 1] * q < p);
            }
        }
        const uint64_t some = __ballot(refused);
        if (some) return i0 + static_cast<uint32_t>(__builtin_ctzll(some));
    }
    return length - 1;
}

__device__ __forceinline__ DrawRow row_of(const Verify& a, uint32_t sequence, uint32_t node, bool refused) {
    DrawRow r;
    r.target = a.target + (static_cast<uint64_t>(sequence) * a.tokens + node) * a.target_stride;
    r.draft = refused ? a.draft + (static_cast<uint64_t>(sequence) * (a.tokens - 1) + node) * a.draft_stride : nullptr;
    return r;
}

// floor(min(max(x, 0), 1) 2^44) as its high and low 22 bits (the high up to
// 2^22); each step exact. A NaN counts 0.
__device__ __forceinline__ void units_of(float x, uint32_t* high, uint32_t* low) {
    const float scaled = fminf(fmaxf(x, 0.0f), 1.0f) * 4194304.0f;
    *high = static_cast<uint32_t>(scaled);
    *low = static_cast<uint32_t>((scaled - static_cast<float>(*high)) * 4194304.0f);
}

__device__ __forceinline__ uint64_t units_of(float x) {
    uint32_t high, low;
    units_of(x, &high, &low);
    return (static_cast<uint64_t>(high) << 22) + low;
}

constexpr uint32_t kSegment = 256;  // entries: four a lane

// Segments of a row, counted from its boundary (rows.hpp).
__host__ __device__ constexpr uint32_t segments_of(uint32_t vocabulary) { return (vocabulary + 3 + kSegment - 1) / kSegment; }

// Entries at .. at + 3 of a draw's row, counted from its target's boundary
// (rows.hpp): a refused draft's taken off. Where the draft's rows lie otherwise
// to theirs, one by one.
__device__ __forceinline__ float4 weights4(const DrawRow& r, uint32_t lead, uint32_t vocabulary, uint32_t at) {
    float4 v = read4(r.target, lead, vocabulary, at, 0.0f);
    if (r.draft) {
        float4 q;
        if (lead_of(r.draft) == lead) {
            q = read4(r.draft, lead, vocabulary, at, 0.0f);
        } else {
            float x[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                x[e] = at + e >= lead && at + e < lead + vocabulary ? r.draft[at + e - lead] : 0.0f;
            q = {x[0], x[1], x[2], x[3]};
        }
        v = {v.x - q.x, v.y - q.y, v.z - q.z, v.w - q.w};
    }
    return v;
}

// The sum over the wave's lanes, in every lane.
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) {
    // within rows of 16 lanes, rotated by 1, 2, 4 and 8
    x += static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x121, 0xF, 0xF, true));
    x += static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x122, 0xF, 0xF, true));
    x += static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x124, 0xF, 0xF, true));
    x += static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), 0x128, 0xF, 0xF, true));
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = a[0] + a[1];
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return b[0] + b[1];
}

__global__ __launch_bounds__(256) void draw_sums(Verify a) {
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const uint32_t sequence = a.draft ? row : row / a.tokens;
    const uint32_t length = length_of(a, sequence);
    uint32_t node = a.draft ? 0 : row % a.tokens;
    if (node >= length) return;
    bool refused = false;
    if (a.draft) {
        node = accepted_of(a, sequence, length);
        refused = node + 1 < length;
        if (chunk == 0 && threadIdx.x == 0) a.drawn[sequence] = static_cast<int32_t>(node);
    }
    const DrawRow r = row_of(a, sequence, node, refused);
    const uint32_t lead = lead_of(r.target), all = segments_of(a.vocabulary);
    const uint32_t end = min((chunk + 1) * a.share, all);
    for (uint32_t segment = chunk * a.share + (threadIdx.x >> 6); segment < end; segment += 4) {
        const float4 v = weights4(r, lead, a.vocabulary, segment * kSegment + 4 * (threadIdx.x & 63u));
        uint32_t high[4], low[4];
        units_of(v.x, &high[0], &low[0]);
        units_of(v.y, &high[1], &low[1]);
        units_of(v.z, &high[2], &low[2]);
        units_of(v.w, &high[3], &low[3]);
        // 256 entries of at most 2^22 each
        const uint32_t h = wave_sum(high[0] + high[1] + high[2] + high[3]), l = wave_sum(low[0] + low[1] + low[2] + low[3]);
        if ((threadIdx.x & 63u) == 0) a.sums[static_cast<uint64_t>(row) * all + segment] = (static_cast<uint64_t>(h) << 22) + l;
    }
}

// The wave's running sum: each lane's, itself included. Within rows of 16 lanes,
// then over the rows.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t x) {
    const int low = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xF, false);
    const int high = __builtin_amdgcn_update_dpp(0, static_cast<int>(x >> 32), CTRL, ROWS, 0xF, false);
    return static_cast<uint64_t>(static_cast<uint32_t>(high)) << 32 | static_cast<uint32_t>(low);
}
__device__ __forceinline__ uint64_t running(uint64_t x) {
    x += moved<0x111, 0xF>(x);  // from 1, 2, 4 and 8 lanes before, in the row
    x += moved<0x112, 0xF>(x);
    x += moved<0x114, 0xF>(x);
    x += moved<0x118, 0xF>(x);
    x += moved<0x142, 0xA>(x);  // the last of rows 0 and 2 to rows 1 and 3
    x += moved<0x143, 0xC>(x);  // the last of the first two to the others
    return x;
}

// The segments a row may have, 2^18 entries at any boundary, and of them a lane's.
constexpr uint32_t kSegments = segments_of(1u << 18), kRun = (kSegments + 63) / 64;

// The token drawn from `r` by uniform number u, its segments' sums at `sums`:
// by one wave, every lane the same. `held` (LDS) is the wave's: a lane's run of
// the sums, read there side by side, is one of neighbours. Runs are odd, so that
// the lanes' places fall on all banks.
__device__ __forceinline__ uint32_t drawn_from(const Verify& a, const DrawRow& r, const uint64_t* sums, float u, uint64_t* held) {
    const uint32_t lane = threadIdx.x & 63u, all = segments_of(a.vocabulary), run = (all + 63) / 64 | 1u;
    uint64_t got[kRun];
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i) got[i] = 64 * i + lane < all ? sums[64 * i + lane] : 0;
#pragma unroll
    for (uint32_t i = 0; i < kRun; ++i)
        if (64 * i + lane < all) held[64 * i + lane] = got[i];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint64_t mine = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < run; ++i)
        if (lane * run + i < all) mine += held[lane * run + i];
    uint64_t to = running(mine);
    const uint64_t total = __shfl(static_cast<unsigned long long>(to), 63);
    if (total == 0) return 0;
    // floor(u 2^31) within 0 .. 2^31 - 1 (a NaN: 0), and floor(W r / 2^31)
    const float scaled = fminf(fmaxf(u, 0.0f), 0.99999994f) * 2147483648.0f;
    const uint64_t by = static_cast<uint32_t>(scaled);
    const uint64_t passed = __umul64hi(total, by) << 33 | (total * by) >> 31;

    // the first run that passes it, a lane a segment of that run (at most 17), and
    // its first segment that does
    const uint32_t owner = static_cast<uint32_t>(__builtin_ctzll(__ballot(to > passed)));
    uint64_t before = __shfl(static_cast<unsigned long long>(to - mine), owner);
    mine = lane < run && owner * run + lane < all ? held[owner * run + lane] : 0;
    to = before + running(mine);
    const uint32_t place = static_cast<uint32_t>(__builtin_ctzll(__ballot(to > passed)));
    before = __shfl(static_cast<unsigned long long>(to - mine), place);
    const uint32_t segment = owner * run + place;

    const uint32_t lead = lead_of(r.target), at = segment * kSegment + 4 * lane;
    const float4 v = weights4(r, lead, a.vocabulary, at);
    const uint64_t w[4] = {units_of(v.x), units_of(v.y), units_of(v.z), units_of(v.w)};
    mine = w[0] + w[1] + w[2] + w[3];
    to = before + running(mine);
    const int first = __builtin_ctzll(__ballot(to > passed));
    before = to - mine;
    uint32_t e = 0;
#pragma unroll
    for (uint32_t i = 0; i < 3; ++i)
        if (e == i && before + w[i] <= passed) before += w[i], ++e;
    return __shfl(at + e - lead, first);
}

// A chain with a draft: a wave a sequence; draw_sums left where its walk ended.
__global__ __launch_bounds__(64) void walk_chain(Verify a) {
    __shared__ uint64_t held[kSegments];
    const uint32_t sequence = blockIdx.x, lane = threadIdx.x;
    const uint32_t length = length_of(a, sequence);
    const uint64_t first = static_cast<uint64_t>(sequence) * a.tokens;
    uint32_t count = 0, token = 0;
    if (length > 0) {
        const uint32_t node = static_cast<uint32_t>(a.drawn[sequence]);
        count = node + 1;
        token = drawn_from(a, row_of(a, sequence, node, count < length),
                           a.sums + static_cast<uint64_t>(sequence) * segments_of(a.vocabulary), a.uniforms[first + node], held);
    }
    for (uint32_t i = lane; i < a.tokens; i += 64) {
        a.path[first + i] = i < count ? static_cast<int32_t>(i) : -1;
        a.emitted[first + i] = i + 1 < count ? a.node_tokens[first + i + 1] : i < count ? static_cast<int32_t>(token) : -1;
    }
    if (lane == 0) a.count[sequence] = count;
}

// Without a draft: every node's draw, a wave a node; then the first wave walks
// from node 0, each step to the first child with the token drawn.
__global__ __launch_bounds__(64 * kWalkWaves) void walk_tree(Verify a) {
    __shared__ int32_t drawn[kVerifyTokens], tokens[kVerifyTokens], parents[kVerifyTokens];
    __shared__ uint64_t held[kWalkWaves][kSegments];
    const uint32_t sequence = blockIdx.x, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t length = length_of(a, sequence);
    const uint64_t first = static_cast<uint64_t>(sequence) * a.tokens;
    for (uint32_t i = threadIdx.x; i < length; i += 64 * kWalkWaves) {
        tokens[i] = a.node_tokens[first + i];
        parents[i] = a.parents ? a.parents[first + i] : static_cast<int32_t>(i) - 1;
    }
    for (uint32_t node = wave; node < length; node += kWalkWaves) {
        const uint32_t token = drawn_from(a, row_of(a, sequence, node, false), a.sums + (first + node) * segments_of(a.vocabulary),
                                          a.uniforms[first + node], held[wave]);
        if (lane == 0) drawn[node] = static_cast<int32_t>(token);
    }
    __syncthreads();
    if (wave != 0) return;
    uint32_t count = 0, node = 0;
    while (count < length) {
        const int32_t token = drawn[node];
        if (lane == 0) {
            a.path[first + count] = static_cast<int32_t>(node);
            a.emitted[first + count] = token;
        }
        ++count;
        uint32_t next = 0;
        for (uint32_t i0 = node + 1; i0 < length; i0 += 64) {
            const uint32_t i = i0 + lane;
            const uint64_t some = __ballot(i < length && tokens[i] == token && parents[i] == static_cast<int32_t>(node));
            if (some) {
                next = i0 + static_cast<uint32_t>(__builtin_ctzll(some));
                break;
            }
        }
        if (next == 0) break;
        node = next;
    }
    for (uint32_t i = count + lane; i < a.tokens; i += 64) a.path[first + i] = a.emitted[first + i] = -1;
    if (lane == 0) a.count[sequence] = count;
}

// Workgroups of at least two segments a wave, about two thousand of them. A
// step by segments a workgroup, 8 / 16 / 32 / 64: one chain's row of 151,936 (by 8)
// 7.1 / 7.8 / 8.9 / 11.3 us; 64 of them (20 by this rule: 18.3) 19.7 / 20.6 / 18.6 /
// 21.8; 8 trees of 21 (48: 28.0) 26.9 / 26.2 / 25.9 / 26.3.
uint32_t verify_share(uint32_t rows, uint32_t vocabulary) {
    const uint64_t all = segments_of(vocabulary);
    return static_cast<uint32_t>(std::max<uint64_t>(8, (rows * all / 2048 + 3) / 4 * 4));
}

uint64_t verify_bytes(uint32_t sequences, uint32_t tokens, uint32_t vocabulary) {
    const uint64_t rows = uint64_t{sequences} * tokens;
    return rows * segments_of(vocabulary) * 8 + uint64_t{sequences} * 4;
}

hipError_t launch_verify(Verify a, hipStream_t stream) {
    const uint32_t rows = a.draft ? a.sequences : a.sequences * a.tokens;
    a.share = verify_share(rows, a.vocabulary);
    a.chunks = (segments_of(a.vocabulary) + a.share - 1) / a.share;
    hipLaunchKernelGGL(draw_sums, dim3(rows * a.chunks), dim3(256), 0, stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (a.draft)
        hipLaunchKernelGGL(walk_chain, dim3(a.sequences), dim3(64), 0, stream, a);
    else
        hipLaunchKernelGGL(walk_tree, dim3(a.sequences), dim3(64 * kWalkWaves), 0, stream, a);
    return hipGetLastError();
}

}  // namespace chm
