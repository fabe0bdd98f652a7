// Attention of several requests' new tokens over their pages (attention.hpp's
// arithmetic, few rows' form: a workgroup has 16 or 32 rows of a key head, its
// waves take the tiles in turn through LDS rings, and are joined in LDS).
//
// The requests' lengths are known to the device alone, and are anything: a
// unit - 16 or 32 rows of a request and key head, over the tiles they see - may
// be one tile or thousands. Each wave finds its workgroup's work from all the
// lengths, by sums over the requests, some a lane, with no launch ahead of it. Where units are fewer than
// workgroups, each is cut in pieces of equal length, a workgroup a piece. Where
// that would leave some with much more than others, the units are laid along a line,
// a key head after another, and each workgroup takes an equal part of it: a long
// unit that crosses parts is in pieces, a short one is its first part's.
//
// A unit's pieces leave their outputs, and their rows' offsets and sums, in the
// workspace, past the caches that the workgroups do not share (loads and stores of
// the device's scope); each waits for its own to arrive, then counts itself, and
// the one that finds itself the last (the counter is left at 0) joins them, in the
// pieces' order. No cache is written back or cleared for it.
#pragma once

#include "attention.hpp"
#include "requests.hpp"

namespace chm {

// What a unit costs beside its tiles, in tiles, and up to what length it is whole
// on the line.
constexpr uint32_t kUnitTiles = 8, kWholeTiles = 16;
// Tiles more than on the line that a workgroup may have for units cut in pieces:
// about what a unit's ends cost that the line leaves in two workgroups.
constexpr uint32_t kPieceTiles = 24;

// What is the same in every lane, as the compiler then knows; a lane's.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t of_lane(uint32_t x, uint32_t lane) { return __builtin_amdgcn_readlane(x, lane); }

// What does not fit in 32 bits stays at kTooMuch: of a step's own lengths none does
// (the host refuses one that may not), of starts and counts that are none's it may.
constexpr uint32_t kTooMuch = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t times(uint32_t x, uint32_t y) {
    const uint64_t product = uint64_t{x} * y;
    return product >> 32 ? kTooMuch : static_cast<uint32_t>(product);
}
__device__ __forceinline__ uint32_t plus(uint32_t x, uint32_t y) { return x + y < x ? kTooMuch : x + y; }

// Four floats at the device's scope.
__device__ __forceinline__ void put(float* to, const float4_t& x) {
    auto* words = reinterpret_cast<uint64_t*>(to);
    const auto pair = __builtin_bit_cast(uint64_t __attribute__((ext_vector_type(2))), x);
    __hip_atomic_store(words, pair.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(words + 1, pair.y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float4_t get(const float* from) {
    const auto* words = reinterpret_cast<const uint64_t*>(from);
    uint64_t __attribute__((ext_vector_type(2))) pair;
    pair.x = __hip_atomic_load(words, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    pair.y = __hip_atomic_load(words + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return __builtin_bit_cast(float4_t, pair);
}
// A row's offset and sum.
__device__ __forceinline__ void put(float2* to, float2 x) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(to), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get(const float2* from) {
    return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Another piece's offset and sum, and its outputs, to those so far.
__device__ __forceinline__ void join(float2 side, const float4_t& theirs, float& least, float& total, float4_t& out) {
    const float lower = side.x < least || side.x != side.x ? side.x : least;
    const float down = least == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lower - least);
    const float factor = side.x == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lower - side.x);
    total = total * down + side.y * factor;
    out = out * down + theirs * factor;
    least = lower;
}

struct NoTree {
    uint32_t above[1][kTreeTokens / 32];
    uint32_t depth[1];
};

// A request: its tokens, and the tiles that its rows see some of.
struct Request {
    uint32_t past, count, start;
    uint32_t begin, tiles;  // the first, how many
    uint32_t groups;        // units a key head
    bool over;              // its tokens pass the table's row
};

template <uint32_t ROWS>
__device__ __forceinline__ void place_request(const PagedAttention& a, Request& r) {
    if (uint64_t{r.start} + r.count > a.rows) r.count = 0;
    r.groups = (r.count * a.group + ROWS - 1) / ROWS;  // (rows * group is below 2^32)
    const uint64_t end = uint64_t{r.past} + r.count;
    r.over = end > uint64_t{a.table_stride} * a.pool.capacity;
    if (r.over) {
        r.begin = 0, r.tiles = 1;
        return;
    }
    r.begin = a.window && r.past + 1 > a.window ? (r.past + 1 - a.window) / kTile : 0;
    r.tiles = (static_cast<uint32_t>(end) + kTile - 1) / kTile - r.begin;
}

// A line in equal parts, the first ones a place longer.
struct Parts {
    uint32_t each, more;
    __device__ __forceinline__ uint32_t begin(uint32_t part) const { return part * each + min(part, more); }
    __device__ __forceinline__ uint32_t at(uint32_t place) const {
        const uint32_t wide = more * (each + 1);
        return place < wide ? place / (each + 1) : more + (place - wide) / each;
    }
};

template <uint32_t F, uint32_t NB, uint32_t X>
__global__ __launch_bounds__((64 * AttendShape<F, NB, X>::kWaves)) void attend_pages(PagedAttention a) {
    using Shape = AttendShape<F, NB, X>;
    constexpr uint32_t kRows = 16 * X, kRecord = Shape::kRecord, W = Shape::kWaves, D = Shape::kRing, T = 64 * W;
    constexpr uint32_t kQuads = Rows<F, NB, X>::kQuads, kParts = kQuads * 64;  // float4s of a wave's outputs
    __shared__ __align__(16) uint8_t space[sizeof(uint8_t[W][D][kRecord]) > sizeof(float4_t[W][kParts])
                                               ? sizeof(uint8_t[W][D][kRecord])
                                               : sizeof(float4_t[W][kParts])];
    __shared__ float joined_offset[W][kRows], joined_sum[W][kRows];
    __shared__ uint32_t last_piece;

    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane % kRows;
    // neighbours on the line on one XCD, whose cache then has the tiles that a request's units share
    const uint32_t part = gridDim.x % 8 == 0 ? blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
    const uint32_t share = (a.requests + 63) / 64, first_request = lane * share;
    const uint32_t last_request = min(first_request + share, a.requests);
    const uint32_t tiles_a_page = a.pool.capacity / kTile;
    // a tile's page, exact: tiles are below 2^26, pages of at most 64
    auto page_at = [&](uint32_t tile) { return tiles_a_page == 1 ? tile : __umulhi(tile, a.page_inverse); };

    auto request_of = [&](uint32_t i) {
        Request r{a.past[i], a.counts[i], a.starts[i], 0, 0, 0, false};
        place_request<kRows>(a, r);
        return r;
    };
    Request mine{};
    if (first_request < last_request) mine = request_of(first_request);
    uint32_t tiles = times(mine.groups, mine.tiles);
    uint32_t units = mine.groups, longest = mine.groups ? mine.tiles : 0;
    for (uint32_t i = first_request + 1; i < last_request; ++i) {
        const Request r = request_of(i);
        tiles = plus(tiles, times(r.groups, r.tiles)), units = plus(units, r.groups);
        if (r.groups) longest = max(longest, r.tiles);
    }
#pragma unroll
    for (uint32_t o = 32; o > 0; o >>= 1) {
        tiles = plus(tiles, __shfl_xor(tiles, o)), units = plus(units, __shfl_xor(units, o));
        longest = max(longest, static_cast<uint32_t>(__shfl_xor(longest, o)));
    }
    const uint32_t all_tiles = times(uniform(tiles), a.pool.kv_heads), all_units = times(uniform(units), a.pool.kv_heads);
    if (all_tiles == kTooMuch || all_units == kTooMuch) return;

    // Pieces of at most `piece_tiles`, which are no more than the workgroups; or equal parts of the line.
    const uint32_t even_tiles = all_tiles / gridDim.x;
    uint32_t piece_tiles = 0;
    if (all_units < gridDim.x) piece_tiles = max(all_tiles / (gridDim.x - all_units) + 1, W);
    const bool even = all_units >= gridDim.x || min(piece_tiles, uniform(longest)) > even_tiles + kPieceTiles;
    auto length_of = [&](const Request& r) {
        return even ? r.tiles + kUnitTiles : (r.tiles + piece_tiles - 1) / piece_tiles;
    };
    uint32_t line = mine.groups ? times(mine.groups, length_of(mine)) : 0;
    for (uint32_t i = first_request + 1; i < last_request; ++i) {
        const Request r = request_of(i);
        line = plus(line, times(r.groups, length_of(r)));
    }
    // what is before the lane
    uint32_t line_before = line;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint32_t other = __shfl_up(line_before, o);
        if (lane >= o) line_before = plus(line_before, other);
    }
    const uint32_t head_line = of_lane(line_before, 63u);
    line_before -= line;

    const uint32_t length = times(head_line, a.pool.kv_heads);
    if (length == kTooMuch) return;
    const Parts parts{length / gridDim.x, length % gridDim.x};
    uint32_t place = even ? parts.begin(part) : part;
    const uint32_t end = even ? parts.begin(part + 1) : min(length, part + 1);

    Attention b{};
    b.queries = a.queries, b.output = a.output;
    b.query_stride = a.query_stride, b.output_stride = a.output_stride;
    b.tokens = 1, b.group = a.group, b.window = a.window, b.scale = a.scale, b.splits = 1;
    const NoTree tree{};

    while (place < end) {
        // The unit: its request, of those of the last lane whose line does not begin past the place.
        const uint32_t head = place / head_line;
        const uint32_t on_head = place - head * head_line;
        const uint32_t low = 63u - __builtin_clzll(__ballot(first_request < a.requests && line_before <= on_head));
        uint32_t before = of_lane(line_before, low);
        uint32_t at = low * share;
        Request r{of_lane(mine.past, low), of_lane(mine.count, low), of_lane(mine.start, low), 0, 0, 0, false};
        place_request<kRows>(a, r);
        while (before + r.groups * length_of(r) <= on_head) {
            before += r.groups * length_of(r);
            ++at;
            r.past = uniform(a.past[at]), r.count = uniform(a.counts[at]), r.start = uniform(a.starts[at]);
            place_request<kRows>(a, r);
        }
        const uint32_t unit_length = length_of(r);
        const uint32_t unit = (on_head - before) / unit_length;
        const uint32_t unit_begin = head * head_line + before + unit * unit_length, unit_end = unit_begin + unit_length;

        // The piece: its tiles of the unit's, its number among the unit's, where it is
        // kept. (On the line a part keeps at most the end of one unit and the begin of
        // another.)
        uint32_t tile_begin = 0, tile_end = r.tiles, pieces = 1, piece = 0, kept = 0, counter = 0;
        if (!even) {
            pieces = unit_length, piece = place - unit_begin;
            kept = part, counter = part - piece;
            // equal but for one tile: the first ones have it
            const uint32_t each = r.tiles / pieces, more = r.tiles % pieces;
            tile_begin = piece * each + min(piece, more), tile_end = tile_begin + each + (piece < more);
            place = end;
        } else if (unit_length <= kUnitTiles + kWholeTiles) {
            const bool earlier = unit_begin < parts.begin(part);
            place = unit_end;
            if (earlier) continue;
        } else {
            const uint32_t from = parts.at(unit_begin), to = parts.at(unit_end - 1);
            pieces = to - from + 1, piece = part - from;
            kept = 2 * part + (piece == 0), counter = 2 * from + 1;
            const uint32_t begin = max(parts.begin(part), unit_begin), until = min(end, unit_end);
            tile_begin = max(begin - unit_begin, kUnitTiles) - kUnitTiles;
            tile_end = max(until - unit_begin, kUnitTiles) - kUnitTiles;
            place = until;
        }

        Group group;
        group.sequence = r.start, group.head = head, group.past = r.past, group.latest = r.past + r.count;
        group.row0 = unit * kRows, group.row_end = min(group.row0 + kRows, r.count * a.group);
        group.token0 = group.row0 / a.group, group.token_end = (group.row_end - 1) / a.group + 1;
        group.all_begin = a.window && group.latest > a.window ? group.latest - a.window : 0u;
        // of the tiles, those that its rows see
        const uint32_t sees_from = a.window && r.past + group.token0 + 1 > a.window ? r.past + group.token0 + 1 - a.window : 0u;
        group.tile_begin = max(r.begin + tile_begin, sees_from / kTile);
        group.tile_end = min(r.begin + tile_end, (r.past + group.token_end + kTile - 1) / kTile);
        if (r.over) group.tile_end = group.tile_begin;

        // A tile's record: its page is read from the table by scalar loads, an iteration ahead of its copy.
        typedef const __attribute__((address_space(4))) uint32_t* scalar_pointer;
        const auto entries = (scalar_pointer)(a.table + uint64_t{at} * a.table_stride);
        const uint32_t first = group.tile_begin + wave;
        const uint32_t count = first < group.tile_end ? (group.tile_end - first + W - 1) / W : 0;  // the wave's tiles
        uint8_t* ring = space + wave * (D * kRecord);
        uint32_t gone = 0;  // a bit a place of the ring: its page is none of the pool's
        auto page_of = [&](uint32_t j) { return entries[page_at(first + j * W)]; };
        auto copy = [&](uint32_t j, uint32_t page) {
            const uint32_t tile = first + j * W, bit = 1u << (j % D);
            const bool there = page < a.pool.sequences;
            gone = there ? gone & ~bit : gone | bit;
            const uint64_t record = (uint64_t{there ? page : 0u} * a.pool.kv_heads + head) * tiles_a_page +
                                    (tile - page_at(tile) * tiles_a_page);
            copy_record<kRecord>(a.pool.base + record * kRecord, ring + j % D * kRecord);
        };
#pragma unroll
        for (uint32_t j = 0; j + 1 < D; ++j)
            if (j < count) copy(j, page_of(j));
        uint32_t ahead = D - 1 < count ? page_of(D - 1) : 0;
        typename Rows<F, NB, X>::Queries queries;
        Rows<F, NB, X>::fetch(b, group, group.row0, queries);
        Rows<F, NB, X> rows;
        rows.begin(b, group, tree, group.row0, queries);
        if (r.over) rows.sum = __builtin_nanf("");
        for (uint32_t j = 0; j < count; ++j) {
            if (j + D - 1 < count) {
                copy(j + D - 1, ahead);
                if (j + D < count) ahead = page_of(j + D);
                wait_loads<(D - 1) * Shape::kCopies>();
            } else {
                wait_loads<0>();
            }
            const uint32_t slot0 = (first + j * W) * kTile;
            if (__builtin_expect(gone >> (j % D) & 1u, 0)) {
                if (rows.sees(b, group, tree, slot0) != 0) rows.sum = __builtin_nanf("");
            } else {
                const Record<F, NB, X> record{ring + j % D * kRecord, slot0, group.latest};
                rows.template tile<kCodes>(b, group, tree, slot0, record);
            }
            __asm__ __volatile__("s_waitcnt lgkmcnt(0)" ::: "memory");  // the record's reads, before its place is copied to
        }
        rows.end();
        __syncthreads();

        // The waves joined, as attend joins them.
        float4_t(*joined)[kParts] = reinterpret_cast<float4_t(*)[kParts]>(space);
        const float row_sum = sum_of_row<X>(rows.sum);
        if (lane < kRows) joined_offset[wave][n] = rows.offset, joined_sum[wave][n] = row_sum;
#pragma unroll
        for (uint32_t t = 0; t < kQuads; ++t) joined[wave][t * 64 + lane] = rows.quad(t);
        __syncthreads();
        auto output_of = [&](uint32_t row, uint32_t value) {
            return a.output + (uint64_t{r.start} + row / a.group) * a.output_stride +
                   (uint64_t{head} * a.group + row % a.group) * (32 * NB) + value;
        };
        for (uint32_t i = threadIdx.x; i < kParts; i += T) {
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
                const float theirs = joined_offset[w][n];
                const float factor = theirs == INFINITY ? 0.0f : __builtin_amdgcn_exp2f(least - theirs);
                total = __builtin_fmaf(joined_sum[w][n], factor, total);
                out += joined[w][i] * factor;
            }
            const bool empty = least == INFINITY && total == 0.0f;
            const uint32_t value = Rows<F, NB, X>::quad_at(i / 64);
            if (pieces == 1) {
                *reinterpret_cast<float4_t*>(output_of(group.row0 + n, value)) = empty ? float4_t(0.0f) : out * (1.0f / total);
            } else {
                put(a.partial + (uint64_t{kept} * kRows + n) * (32 * NB) + value, out);
                if (i < kRows) put(a.stats + uint64_t{kept} * kRows + n, make_float2(total != total ? total : least, total));
            }
        }
        wait_loads<0>();
        __syncthreads();  // the LDS is read, and what was written has arrived
        if (pieces == 1) continue;
        if (threadIdx.x == 0) last_piece = atomicInc(a.counters + counter, pieces - 1) == pieces - 1;
        __syncthreads();
        if (!last_piece) continue;

        // The pieces joined: a thread four values of a row, over its share of the pieces; then over the shares.
        const uint32_t quads = 8 * NB, work = (group.row_end - group.row0) * quads;
        const uint32_t shares = max(1u, T / work);
        auto kept_of = [&](uint32_t p) { return even ? 2 * (part - piece + p) + (p == 0) : counter + p; };
        float4_t* sums = reinterpret_cast<float4_t*>(space);
        float2* sides = reinterpret_cast<float2*>(space + T * sizeof(float4_t));
        for (uint32_t i0 = 0; i0 < work; i0 += T) {
            const uint32_t i = i0 + threadIdx.x % min(work, T), mine_of = work <= T ? threadIdx.x / work : 0;
            const bool live = i < work && mine_of < shares;
            const uint32_t row = i / quads, value = i % quads * 4;
            float least = INFINITY, total = 0.0f;
            float4_t out = float4_t(0.0f);
            constexpr uint32_t kBatch = 8;  // on their way together
            for (uint32_t p0 = mine_of; live && p0 < pieces; p0 += kBatch * shares) {
                float2 side[kBatch];
                float4_t theirs[kBatch];
#pragma unroll
                for (uint32_t x = 0; x < kBatch; ++x) {
                    const uint32_t p = p0 + x * shares;
                    side[x] = make_float2(INFINITY, 0.0f), theirs[x] = float4_t(0.0f);
                    if (p >= pieces) continue;
                    const uint64_t from = uint64_t{kept_of(p)} * kRows + row;
                    side[x] = get(a.stats + from), theirs[x] = get(a.partial + from * (32 * NB) + value);
                }
#pragma unroll
                for (uint32_t x = 0; x < kBatch; ++x) join(side[x], theirs[x], least, total, out);
            }
            if (shares > 1) {
                sums[threadIdx.x] = out, sides[threadIdx.x] = make_float2(least, total);
                __syncthreads();
                if (live && mine_of == 0)
                    for (uint32_t x = 1; x < shares; ++x)
                        join(sides[threadIdx.x + x * work], sums[threadIdx.x + x * work], least, total, out);
            }
            if (live && mine_of == 0)
                *reinterpret_cast<float4_t*>(output_of(group.row0 + row, value)) =
                    least == INFINITY ? float4_t(0.0f) : out * (1.0f / total);
        }
        __syncthreads();
    }
}

template <uint32_t F, uint32_t NB>
static hipError_t launch_paged_blocks(const PagedAttention& a, uint32_t octets, hipStream_t stream) {
    if (octets == 2)
        hipLaunchKernelGGL((attend_pages<F, NB, 2>), dim3(a.parts), dim3(64 * AttendShape<F, NB, 2>::kWaves), 0, stream, a);
    else
        hipLaunchKernelGGL((attend_pages<F, NB, 1>), dim3(a.parts), dim3(64 * AttendShape<F, NB, 1>::kWaves), 0, stream, a);
    return hipGetLastError();
}

template <uint32_t F>
static hipError_t launch_paged(const PagedAttention& a, uint32_t octets, hipStream_t stream) {
    switch (a.pool.head_dim / 32) {
        case 1: return launch_paged_blocks<F, 1>(a, octets, stream);
        case 2: return launch_paged_blocks<F, 2>(a, octets, stream);
        case 3: return launch_paged_blocks<F, 3>(a, octets, stream);
        case 4: return launch_paged_blocks<F, 4>(a, octets, stream);
        case 5: return launch_paged_blocks<F, 5>(a, octets, stream);
        case 6: return launch_paged_blocks<F, 6>(a, octets, stream);
        case 7: return launch_paged_blocks<F, 7>(a, octets, stream);
        case 8: return launch_paged_blocks<F, 8>(a, octets, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace chm
