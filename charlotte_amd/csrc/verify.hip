// Drafted tokens against the target's probabilities, from given uniform
// numbers. The draws are exact, in whole numbers: a probability x counts
// floor(x 2^44) units, a row's units W are summed in 64 bits in any order, and
// the token drawn is the lowest index whose running sum passes W r / 2^31, r =
// floor(u 2^31); so however a row is cut, the token is the same.
//
// Two launches. draw_sums: each row to draw from, in chunks, a workgroup a
// chunk, each chunk's units summed: the one pass over the probabilities. A
// chain with a draft draws once a sequence, from the row where its walk ends;
// every workgroup walks it anew (a lane a token, three reads each), which
// costs less than a launch. walk: a workgroup a sequence finds the chunk that
// holds the draw from the sums, reads it again (from cache) for the index, and
// writes what was accepted; without a draft, each of its waves draws nodes and
// the first lane then walks the tree.
//
// Bound by bytes: 4 a probability of the rows drawn from, once.
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

__device__ __forceinline__ uint32_t share_of(const Verify& a) {
    return ((a.vocabulary + 3 + a.chunks - 1) / a.chunks + 3) / 4 * 4;
}

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

__global__ __launch_bounds__(256) void draw_sums(Verify a) {
    __shared__ uint64_t parts[4];
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const uint32_t sequence = a.draft ? row : row / a.tokens;
    const uint32_t length = length_of(a, sequence);
    uint32_t node = a.draft ? 0 : row % a.tokens;
    if (node >= length) return;
    bool refused = false;
    if (a.draft) {
        node = accepted_of(a, sequence, length);
        refused = node + 1 < length;
    }
    const DrawRow r = row_of(a, sequence, node, refused);
    const uint32_t lead = lead_of(r.target), share = share_of(a);
    const uint32_t end = min((chunk + 1) * share, lead + a.vocabulary);
    // a thread adds at most 256 entries' 2^22 before it widens: below 2^32
    uint32_t high = 0, low = 0;
    for (uint32_t at = chunk * share + 4 * threadIdx.x; at < end; at += 1024) {
        const float4 v = weights4(r, lead, a.vocabulary, at);
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t h, l;
            units_of(x[e], &h, &l);
            high += h;
            low += l;
        }
    }
    uint64_t sum = (static_cast<uint64_t>(high) << 22) + low;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(static_cast<unsigned long long>(sum), o);
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) a.sums[blockIdx.x] = parts[0] + parts[1] + parts[2] + parts[3];
}

// The wave's running sum: each lane's, itself included.
__device__ __forceinline__ uint64_t running(uint64_t x) {
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint64_t y = __shfl_up(static_cast<unsigned long long>(x), o);
        if (lane >= o) x += y;
    }
    return x;
}

// The token drawn from `r` by uniform number u, its chunks' sums at `sums`: by
// one wave, every lane the same.
__device__ uint32_t drawn_from(const Verify& a, const DrawRow& r, const uint64_t* sums, float u) {
    const uint32_t lane = threadIdx.x & 63u;
    uint64_t total = 0;
    for (uint32_t c = lane; c < a.chunks; c += 64) total += sums[c];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(static_cast<unsigned long long>(total), o);
    if (total == 0) return 0;
    // floor(u 2^31) within 0 .. 2^31 - 1 (a NaN: 0), and floor(W r / 2^31)
    const float scaled = fminf(fmaxf(u, 0.0f), 0.99999994f) * 2147483648.0f;
    const uint64_t by = static_cast<uint32_t>(scaled);
    const uint64_t passed = __umul64hi(total, by) << 33 | (total * by) >> 31;

    // the chunk: the first whose running sum passes it
    uint64_t before = 0;
    uint32_t chunk = a.chunks - 1;
    for (uint32_t c0 = 0; c0 < a.chunks; c0 += 64) {
        const uint64_t mine = c0 + lane < a.chunks ? sums[c0 + lane] : 0;
        const uint64_t run = before + running(mine);
        const uint64_t past = __ballot(run > passed);
        if (past) {
            const int first = __builtin_ctzll(past);
            chunk = c0 + first;
            before = __shfl(static_cast<unsigned long long>(run - mine), first);
            break;
        }
        before = __shfl(static_cast<unsigned long long>(run), 63);
    }
    // within it: 256 entries a step
    const uint32_t lead = lead_of(r.target), share = share_of(a);
    const uint32_t end = min((chunk + 1) * share, lead + a.vocabulary);
    for (uint32_t at0 = chunk * share; at0 < end; at0 += 256) {
        const uint32_t at = at0 + 4 * lane;
        uint64_t w[4] = {0, 0, 0, 0};
        if (at < end) {
            const float4 v = weights4(r, lead, a.vocabulary, at);
            w[0] = units_of(v.x), w[1] = units_of(v.y), w[2] = units_of(v.z), w[3] = units_of(v.w);
        }
        const uint64_t mine = w[0] + w[1] + w[2] + w[3];
        const uint64_t run = before + running(mine);
        const uint64_t past = __ballot(run > passed);
        if (past) {
            const int first = __builtin_ctzll(past);
            uint64_t so_far = run - mine;
            uint32_t e = 0;
            while (e < 3 && so_far + w[e] <= passed) so_far += w[e++];
            return __shfl(at + e - lead, first);
        }
        before = __shfl(static_cast<unsigned long long>(run), 63);
    }
    return a.vocabulary - 1;  // not reached: the chunk's sum passes
}

// A chain with a draft: a wave a sequence.
__global__ __launch_bounds__(64) void walk_chain(Verify a) {
    const uint32_t sequence = blockIdx.x, lane = threadIdx.x;
    const uint32_t length = length_of(a, sequence);
    const uint64_t first = static_cast<uint64_t>(sequence) * a.tokens;
    uint32_t count = 0, token = 0;
    if (length > 0) {
        const uint32_t node = accepted_of(a, sequence, length);
        count = node + 1;
        token = drawn_from(a, row_of(a, sequence, node, count < length), a.sums + static_cast<uint64_t>(sequence) * a.chunks,
                           a.uniforms[first + node]);
    }
    for (uint32_t i = lane; i < a.tokens; i += 64) {
        a.path[first + i] = i < count ? static_cast<int32_t>(i) : -1;
        a.emitted[first + i] = i + 1 < count ? a.node_tokens[first + i + 1] : i < count ? static_cast<int32_t>(token) : -1;
    }
    if (lane == 0) a.count[sequence] = count;
}

// Without a draft: every node's draw, then the walk from node 0, each step by
// the first wave: the first child with the token drawn.
__global__ __launch_bounds__(64 * kWalkWaves) void walk_tree(Verify a) {
    const uint32_t sequence = blockIdx.x, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t length = length_of(a, sequence);
    const uint64_t first = static_cast<uint64_t>(sequence) * a.tokens;
    for (uint32_t node = wave; node < length; node += kWalkWaves) {
        const uint32_t token = drawn_from(a, row_of(a, sequence, node, false), a.sums + (first + node) * a.chunks,
                                          a.uniforms[first + node]);
        if (lane == 0) a.drawn[first + node] = static_cast<int32_t>(token);
    }
    __syncthreads();
    if (wave != 0) return;
    uint32_t count = 0, node = 0;
    while (count < length) {
        const int32_t token = a.drawn[first + node];
        if (lane == 0) {
            a.path[first + count] = static_cast<int32_t>(node);
            a.emitted[first + count] = token;
        }
        ++count;
        uint32_t next = 0;
        for (uint32_t i0 = node + 1; i0 < length; i0 += 64) {
            const uint32_t i = i0 + lane;
            const bool child = i < length && a.node_tokens[first + i] == token &&
                               (a.parents ? a.parents[first + i] == static_cast<int32_t>(node) : i == node + 1);
            const uint64_t some = __ballot(child);
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

// Chunks of 2,048 to 8,192 entries, about a thousand of them where the rows are few.
uint32_t verify_chunks(uint32_t rows, uint32_t vocabulary) {
    const uint64_t share = std::clamp<uint64_t>(uint64_t{rows} * vocabulary / 1024, 2048, 8192);
    return static_cast<uint32_t>((vocabulary + share - 1) / share);
}

uint64_t verify_bytes(uint32_t sequences, uint32_t tokens, uint32_t vocabulary) {
    // the most chunks any number of rows gives; then the draws
    const uint64_t rows = uint64_t{sequences} * tokens;
    return rows * ((vocabulary + 2047) / 2048) * 8 + rows * 4;
}

hipError_t launch_verify(const Verify& a, hipStream_t stream) {
    const uint32_t rows = a.draft ? a.sequences : a.sequences * a.tokens;
    hipLaunchKernelGGL(draw_sums, dim3(rows * a.chunks), dim3(256), 0, stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (a.draft)
        hipLaunchKernelGGL(walk_chain, dim3(a.sequences), dim3(64), 0, stream, a);
    else
        hipLaunchKernelGGL(walk_tree, dim3(a.sequences), dim3(64 * kWalkWaves), 0, stream, a);
    return hipGetLastError();
}

}  // namespace chm
