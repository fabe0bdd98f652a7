// Attention of several requests' new tokens over their pages (attention.hpp's
// arithmetic): attend_pages with few rows a workgroup, 16 or 32 of a key head, its
// waves taking the tiles in turn through LDS rings and joined in LDS;
// attend_page_rows, for the requests of a step that bring many_from rows and more,
// with 128 or 256, a tile laid out once for all of them.
//
// The requests' lengths are known to the device alone, and are anything: a
// unit - 16 or 32 rows of a request and key head, over the tiles they see - may
// be one tile or thousands. Each wave finds its workgroup's work from all the
// lengths, by sums over the requests, some a lane, with no launch ahead of it. Where units are fewer than
// workgroups, each is cut in pieces of equal length, a workgroup a piece. Where
// that would leave some with much more than others, the units are laid along a line,
// a key head after another, and each workgroup takes an equal part of it: a
// unit that crosses parts is in pieces.
//
// A unit's pieces leave their outputs, and their rows' offsets and sums, in the
// workspace, past the caches that the workgroups do not share (loads and stores of
// the device's scope); each waits for its own to arrive, then counts itself, and
// the one that finds itself the last (the counter is left at 0) joins them, in the
// pieces' order. No cache is written back or cleared for it: the write-back that a
// release at the device's scope asks for took 4 us. Of many rows, whose pieces are
// MBs, a launch of its own joins them.
//
// Few rows are bound by the cache's bytes: 64 requests of 50 - 32,768 tokens, 8 key
// heads of 128 in Q8_0 (731 MB), 140 - 146 us, 5.0 - 5.2 TB/s, as a large copy. One token over
// 65,536, 8 heads of 64 in Q4_0 (38 MB): 23.8 us, of which 4.5 go before the first tile,
// 11 over the tiles (the VALU: 4-bit codes widened for four rows of 16) and 8 from a
// workgroup's last tile to the units' join. 3 requests of up to 911 tokens: 15 us, of the
// same parts. Many rows are bound by the VALU and the matrix cores in turn (two prompts of
// 512 tokens over up to 8,000, 8 key heads of 64: 212 - 219 us; traced 217 in attend_page_rows,
// matrix cores 35% busy, VALU 48%, beside 32 in the other launches); their requests in
// units of 32 rows took 293. The launches are one after the other: requests of 17 rows up to
// many_from beside single tokens are two chains of 15 - 20 us.
//
// Against one sequence's contiguous cache (attention.hpp), Q8_0, 8 key heads of 128, us:
// 512 tokens over 15,873 368 beside 341, over 2,000 82 and 71, over none 37 and 36; 2,048 over
// 2,048 312 and 314; one over 65,536 39 and 33. What finds the work stays in registers over
// the tiles: every kernel here keeps 23 - 122 scalars in lanes of vector registers (attend_rows
// at most 4), heads of 32 in many rows have 3 waves a SIMD (there 4), and some vector registers
// spill, which none does there: 6 and 4 of attend_page_rows in Q8_0 and Q4_0 with heads of 128, 4, 2
// and 11 in F16 with 160, 224 and 256 (512 over 8,000, one key head of 256 87 - 90 us and 67), 32
// and 29 of attend_pages of 32 rows in Q8_0 and Q4_0 with heads of 256.
// Q8_0 and Q4_0 with heads of 160 - 256 have no form of many rows, as attention has none: 512 over
// 8,000, heads of 256, one key head 110 and 108 us (contiguous 97 and 91), eight 652 and 639 (644 and
// 573; 122 by the formula's operations, 304 with operands in parts); of 160, eight 439 and 416 (410 both).
#pragma once

#include "attention.hpp"
#include "requests.hpp"

namespace chm {

// What a unit costs beside its tiles, in tiles (its queries, its waves' join). One token
// each of 64 requests of 50 - 32,768 tokens, 8 key heads of 128 in Q8_0: 164 - 170 us at none,
// 149 at 8, 144 at 16, 146 at 24; of 200 requests of 50 - 2,000 115, 92, 92 and 92.
constexpr uint32_t kUnitTiles = 16;
// Tiles more than on the line that a workgroup may have for units cut in pieces:
// about what a unit's ends cost that the line leaves in two workgroups. 8 requests of
// 4,000 tokens 25.5 us in pieces, 28.6 on the line; 30 of 50 - 32,768 340 and 81.
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
    static constexpr bool kTrees = false;
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

// `many`: requests of many_from rows and more are the other kernel's.
template <uint32_t ROWS>
__device__ __forceinline__ void place_request(const PagedAttention& a, Request& r, bool many) {
    if (uint64_t{r.start} + r.count > a.rows) r.count = 0;
    const uint32_t rows = r.count * a.group;  // below 2^28
    r.groups = rows > a.above && rows <= a.upto ? (rows + ROWS - 1) / ROWS : 0;
    const uint64_t end = uint64_t{r.past} + r.count;
    r.over = end > uint64_t{a.table_stride} * a.pool.capacity;
    if (r.over) {
        r.begin = 0, r.tiles = 1;
        return;
    }
    if (many && rows >= a.many_from) r.groups = 0;
    r.begin = a.window && r.past + 1 > a.window ? (r.past + 1 - a.window) / kTile : 0;
    r.tiles = (static_cast<uint32_t>(end) + kTile - 1) / kTile - r.begin;
}

// Whether the requests of many_from rows and more are worth their own kernel: 32 rows by
// a tile of theirs number a.many_load a workgroup and more. The same in every kernel
// of the step.
__device__ __forceinline__ bool many_rows(const PagedAttention& a) {
    if (a.many_load == 0) return false;
    const uint32_t lane = threadIdx.x & 63u, share = (a.requests + 63) / 64;
    uint32_t load = 0;
    for (uint32_t i = lane * share; i < min((lane + 1) * share, a.requests); ++i) {
        Request r{a.past[i], a.counts[i], a.starts[i], 0, 0, 0, false};
        if (uint64_t{r.start} + r.count > a.rows || r.count * a.group < a.many_from) continue;
        const uint64_t end = uint64_t{r.past} + r.count;
        if (end > uint64_t{a.table_stride} * a.pool.capacity) continue;
        const uint32_t begin = a.window && r.past + 1 > a.window ? (r.past + 1 - a.window) / kTile : 0;
        load = plus(load, times((r.count * a.group + 31) / 32, (static_cast<uint32_t>(end) + kTile - 1) / kTile - begin));
    }
#pragma unroll
    for (uint32_t o = 32; o > 0; o >>= 1) load = plus(load, __shfl_xor(load, o));
    return times(uniform(load), a.pool.kv_heads) >= a.many_load * a.parts;
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

// A unit's pieces joined, by a thread four values of a row over its share of the
// pieces; then over the shares. `space`: T float4s and T float2s of LDS.
template <uint32_t NB, uint32_t T, typename KEPT, typename OUTPUT>
__device__ __forceinline__ void join_pieces(const PagedAttention& a, uint32_t unit_rows, uint32_t rows, uint32_t pieces,
                                            const KEPT& kept_of, const OUTPUT& output_of, uint8_t* space) {
    const uint32_t quads = 8 * NB, work = rows * quads, shares = max(1u, T / work);
    float4_t* sums = reinterpret_cast<float4_t*>(space);
    float2* sides = reinterpret_cast<float2*>(space + T * sizeof(float4_t));
    for (uint32_t i0 = 0; i0 < work; i0 += T) {
        const uint32_t i = i0 + threadIdx.x % min(work, T), mine = work <= T ? threadIdx.x / work : 0;
        const bool live = i < work && mine < shares;
        const uint32_t row = i / quads, value = i % quads * 4;
        float least = INFINITY, total = 0.0f;
        float4_t out = float4_t(0.0f);
        constexpr uint32_t kBatch = 8;  // on their way together
        for (uint32_t p0 = mine; live && p0 < pieces; p0 += kBatch * shares) {
            float2 side[kBatch];
            float4_t theirs[kBatch];
#pragma unroll
            for (uint32_t x = 0; x < kBatch; ++x) {
                const uint32_t p = p0 + x * shares;
                side[x] = make_float2(INFINITY, 0.0f), theirs[x] = float4_t(0.0f);
                if (p >= pieces) continue;
                const uint64_t from = uint64_t{kept_of(p)} * unit_rows + row;
                side[x] = get(a.stats + from), theirs[x] = get(a.partial + from * (32 * NB) + value);
            }
#pragma unroll
            for (uint32_t x = 0; x < kBatch; ++x) join(side[x], theirs[x], least, total, out);
        }
        if (shares > 1) {
            sums[threadIdx.x] = out, sides[threadIdx.x] = make_float2(least, total);
            __syncthreads();
            if (live && mine == 0)
                for (uint32_t x = 1; x < shares; ++x)
                    join(sides[threadIdx.x + x * work], sums[threadIdx.x + x * work], least, total, out);
        }
        if (live && mine == 0)
            *reinterpret_cast<float4_t*>(output_of(row, value)) = least == INFINITY ? float4_t(0.0f) : out * (1.0f / total);
    }
}

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

    const bool many = many_rows(a);
    auto request_of = [&](uint32_t i) {
        Request r{a.past[i], a.counts[i], a.starts[i], 0, 0, 0, false};
        place_request<kRows>(a, r, many);
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
    if (all_units == 0 || all_tiles == kTooMuch || all_units == kTooMuch) return;

    // Pieces of at most `piece_tiles`, which are no more than the workgroups; or equal parts of the line.
    const uint32_t even_tiles = all_tiles / gridDim.x;
    uint32_t piece_tiles = 0;
    if (all_units < gridDim.x) {
        // as many workgroups as there are have it evenly, if the units' own ends leave them enough
        piece_tiles = max((all_tiles + gridDim.x - 1) / gridDim.x, W);
        uint32_t pieces = 0;
        for (uint32_t i = first_request; i < last_request; ++i) {
            const Request r = i == first_request ? mine : request_of(i);
            pieces += r.groups * ((r.tiles + piece_tiles - 1) / piece_tiles);
        }
#pragma unroll
        for (uint32_t o = 32; o > 0; o >>= 1) pieces += __shfl_xor(pieces, o);
        if (uniform(pieces) * a.pool.kv_heads > gridDim.x) piece_tiles = max(all_tiles / (gridDim.x - all_units) + 1, W);
    }
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
        place_request<kRows>(a, r, many);
        while (before + r.groups * length_of(r) <= on_head) {
            before += r.groups * length_of(r);
            ++at;
            r.past = uniform(a.past[at]), r.count = uniform(a.counts[at]), r.start = uniform(a.starts[at]);
            place_request<kRows>(a, r, many);
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

        join_pieces<NB, T>(a, kRows, group.row_end - group.row0, pieces,
                           [&](uint32_t p) { return even ? 2 * (part - piece + p) + (p == 0) : counter + p; },
                           [&](uint32_t row, uint32_t value) { return output_of(group.row0 + row, value); }, space);
        __syncthreads();
    }
}

// ---- requests of many rows -----------------------------------------------------

// What a unit of many rows costs beside its tiles, and the least tiles of a part. 512
// tokens over 2,000 (8 key heads of 128, Q8_0) 86 us at a cost of 2, 82 at 4, 89 at 6; over
// 8,000 (one of 256, F16) 91, 87 and 89.
constexpr uint32_t kManyUnitTiles = 4, kManyPartTiles = 8;
// Tiles of a piece whose records' places are kept in LDS; past them they are found anew.
constexpr uint32_t kKeptTiles = 1024;

// Where a request's tile is in its pool; kNoRecord where its page is none of the pool's.
constexpr uint64_t kNoRecord = ~0ull;
struct PagePlaces {
    const uint32_t* table;  // the request's row
    uint32_t tiles_a_page, page_inverse, kv_heads, head, pages, record;
    __device__ __forceinline__ uint64_t operator()(uint32_t t) const {
        const uint32_t place = tiles_a_page == 1 ? t : __umulhi(t, page_inverse), page = table[place];
        return page < pages ? ((uint64_t{page} * kv_heads + head) * tiles_a_page + (t - place * tiles_a_page)) * record : kNoRecord;
    }
};
// A piece's records, from its tile `first` on.
struct PagedRecords {
    static constexpr bool kGaps = true;
    const uint8_t* base;
    const uint64_t* kept;  // LDS
    const PagePlaces* far; // LDS
    uint32_t first;
    __device__ __forceinline__ const uint8_t* operator()(uint32_t t) const {
        const uint64_t at = __builtin_expect(t - first < kKeptTiles, true) ? kept[t - first] : (*far)(t);
        return at != kNoRecord ? base + at : nullptr;
    }
    // The wave's t, of a unit that misses no page: an address that is the same in every lane.
    __device__ __forceinline__ const uint8_t* of_wave(uint32_t t) const {
        const uint64_t at = __builtin_expect(t - first < kKeptTiles, true) ? kept[t - first] : (*far)(t);
        return base + (uint64_t{uniform(static_cast<uint32_t>(at >> 32))} << 32 | uniform(static_cast<uint32_t>(at)));
    }
};

// Where piece p of the unit that begins in part `first` is kept.
__device__ __forceinline__ uint64_t kept_at(uint32_t first, uint32_t p) { return 2 * (first + p) + (p == 0); }

// Request i, if it is of many rows: a unit each ROWS of them.
struct Many {
    uint32_t at, past, count, start, groups;
};
// Their units on a line, each as long as the tiles that its rows see and kManyUnitTiles.
template <uint32_t ROWS>
struct ManyLine {
    const PagedAttention& a;
    uint32_t share, line_before, head_line, count;
    Parts parts;

    __device__ __forceinline__ Many many_of(uint32_t i) const {
        Many m{i, a.past[i], a.counts[i], a.starts[i], 0};
        const bool mine = uint64_t{m.start} + m.count <= a.rows && m.count * a.group >= a.many_from &&
                          uint64_t{m.past} + m.count <= uint64_t{a.table_stride} * a.pool.capacity;
        if (mine) m.groups = (m.count * a.group + ROWS - 1) / ROWS;
        return m;
    }
    __device__ __forceinline__ uint32_t begin_of(const Many& m, uint32_t unit) const {
        const uint32_t place = m.past + unit * ROWS / a.group + 1;
        return a.window && place > a.window ? (place - a.window) / kTile : 0u;
    }
    __device__ __forceinline__ uint32_t tiles_of(const Many& m, uint32_t unit) const {
        const uint32_t rows = min((unit + 1) * ROWS, m.count * a.group);
        return (m.past + (rows - 1) / a.group + kTile) / kTile - begin_of(m, unit);
    }
    __device__ __forceinline__ uint32_t length_of(const Many& m, uint32_t unit) const {
        return tiles_of(m, unit) + kManyUnitTiles;
    }
    // All units of the lane's requests, summed up.
    template <typename FN>
    __device__ __forceinline__ uint32_t sum_units(FN f) const {
        const uint32_t first = (threadIdx.x & 63u) * share;
        uint32_t sum = 0;
        for (uint32_t i = first; i < min(first + share, a.requests); ++i) {
            const Many m = many_of(i);
            for (uint32_t g = 0; g < m.groups; ++g) sum = plus(sum, f(m, g));
        }
        return sum;
    }
    // A part's tiles of a unit: of the unit's.
    template <typename UNIT>
    __device__ __forceinline__ void tiles_at(const UNIT& u, uint32_t part, uint32_t* from, uint32_t* to) const {
        *from = max(max(parts.begin(part), u.begin) - u.begin, kManyUnitTiles) - kManyUnitTiles;
        *to = max(min(parts.begin(part + 1), u.end) - u.begin, kManyUnitTiles) - kManyUnitTiles;
    }
    // Laid out by each wave; no parts where there is nothing, or too much.
    __device__ __forceinline__ explicit ManyLine(const PagedAttention& a_) : a(a_), share((a_.requests + 63) / 64), count(0) {
        const uint32_t lane = threadIdx.x & 63u;
        const uint32_t line = sum_units([&](const Many& m, uint32_t g) { return length_of(m, g); });
        line_before = line;
#pragma unroll
        for (uint32_t o = 1; o < 64; o <<= 1) {
            const uint32_t other = __shfl_up(line_before, o);
            if (lane >= o) line_before = plus(line_before, other);
        }
        head_line = of_lane(line_before, 63u);
        line_before -= line;
        const uint32_t length = times(head_line, a.pool.kv_heads);
        if (length == kTooMuch || length == 0) return;
        count = min(a.parts, max(length / kManyPartTiles, 1u));
        parts = {length / count, length % count};
    }
    // The unit at a place: of those of the last lane whose line does not begin past it.
    struct Unit {
        Many m;
        uint32_t head, unit, begin, end;  // on the line
        uint32_t first, pieces;           // its first part, its parts
    };
    __device__ __forceinline__ Unit unit_at(uint32_t place) const {
        const uint32_t lane = threadIdx.x & 63u, head = place / head_line, on_head = place - head * head_line;
        const uint32_t low = 63u - __builtin_clzll(__ballot(lane * share < a.requests && line_before <= on_head));
        uint32_t before = of_lane(line_before, low), at = low * share, unit = 0;
        Many m = many_of(at);
        for (;;) {
            if (unit < m.groups) {
                const uint32_t next = before + length_of(m, unit);
                if (next > on_head) break;
                before = next, ++unit;
            } else {
                m = many_of(++at), unit = 0;
            }
        }
        unit = uniform(unit);
        m = Many{uniform(m.at), uniform(m.past), uniform(m.count), uniform(m.start), uniform(m.groups)};
        Unit u{m, head, unit, head * head_line + uniform(before), 0, 0, 0};
        u.end = u.begin + length_of(m, unit);
        u.first = parts.at(u.begin), u.pieces = parts.at(u.end - 1) - u.first + 1;
        return u;
    }
    // Where piece p of a unit is kept: a part has at most the end of one unit and the begin of another.
    __device__ __forceinline__ static uint64_t kept_of(const Unit& u, uint32_t p) { return kept_at(u.first, p); }
};

template <uint32_t F, uint32_t NB>
__global__ __launch_bounds__(64 * row_waves(NB)) void attend_page_rows(PagedAttention a) {
    constexpr uint32_t kRows = RowsShape<F, NB>::kRows, T = 64 * row_waves(NB);
    __shared__ RowsSpace<F, NB> space;
    __shared__ uint64_t kept_places[kKeptTiles];
    __shared__ PagePlaces far;
    __shared__ uint32_t missing, line_before[64];
    // neighbours on the line on one XCD
    const uint32_t part = gridDim.x % 8 == 0 ? blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
    if (threadIdx.x == 0) a.joins[part].pieces = 0;
    if (!many_rows(a)) return;
    ManyLine<kRows> line(a);
    if (part >= line.count) return;
    if (threadIdx.x < 64) line_before[threadIdx.x] = line.line_before;
    __syncthreads();
    uint32_t place = line.parts.begin(part);
    const uint32_t end = line.parts.begin(part + 1);

    Attention b{};
    b.queries = a.queries, b.output = a.output;
    b.query_stride = a.query_stride, b.output_stride = a.output_stride;
    b.tokens = 1, b.group = a.group, b.window = a.window, b.scale = a.scale, b.splits = 1;
    NoTree tree{};

    while (place < end) {
        line.line_before = line_before[threadIdx.x & 63u];  // no register over the tiles
        const auto u = line.unit_at(place);
        place = min(end, u.end);

        Group group;
        group.sequence = u.m.start, group.head = u.head, group.past = u.m.past, group.latest = u.m.past + u.m.count;
        group.row0 = u.unit * kRows, group.row_end = min(group.row0 + kRows, u.m.count * a.group);
        group.token0 = group.row0 / a.group, group.token_end = (group.row_end - 1) / a.group + 1;
        group.all_begin = a.window && group.latest > a.window ? group.latest - a.window : 0u;
        line.tiles_at(u, part, &group.tile_begin, &group.tile_end);
        group.tile_begin += line.begin_of(u.m, u.unit), group.tile_end += line.begin_of(u.m, u.unit);

        // The piece's records, and whether one has a page that is none of the pool's.
        const PagePlaces places{a.table + uint64_t{u.m.at} * a.table_stride, a.pool.capacity / kTile, a.page_inverse,
                                a.pool.kv_heads, u.head, a.pool.sequences, cache_record(F, NB)};
        if (threadIdx.x == 0) missing = 0, far = places;
        __syncthreads();
        bool gone = false;
        for (uint32_t t = group.tile_begin + threadIdx.x; t < group.tile_end; t += T) {
            const uint64_t at = places(t);
            if (t - group.tile_begin < kKeptTiles) kept_places[t - group.tile_begin] = at;
            gone |= at == kNoRecord;
        }
        if (gone) missing = 1;
        __syncthreads();
        const PagedRecords records{a.pool.base, kept_places, &far, group.tile_begin};
        // (the part's one unit that goes on past it)
        if (threadIdx.x == 0 && u.pieces > 1 && u.first == part)
            a.joins[part] = {u.m.start, u.head, group.row0, group.row_end - group.row0, u.pieces, 0};
        const uint64_t kept = line.kept_of(u, part - u.first) * kRows;
        auto write = [&](uint32_t row, bool live, uint32_t value, float4_t out, float total, float least, bool stats) {
            if (u.pieces == 1) {
                finish<NB>(b, group, row, live, value, out, total, least, false);
                return;
            }
            const bool empty = !live || (least == INFINITY && total == 0.0f);
            const uint64_t to = kept + (row - group.row0);
            *reinterpret_cast<float4_t*>(a.partial + to * (32 * NB) + value) = empty ? float4_t(0.0f) : out;
            if (stats) a.stats[to] = make_float2(empty ? INFINITY : total != total ? total : least, empty ? 0.0f : total);
        };
        attend_group<F, NB>(b, group, tree, space, records, write, uniform(missing) != 0);
        __syncthreads();  // the LDS is read
    }
}

// The units in pieces joined, in a launch of its own, by all its threads: each finds
// all units (that which begins in a part and goes on past it), and a thread takes
// four values of a row of theirs at a time.
constexpr uint32_t kJoinThreads = 256;
template <uint32_t NB, uint32_t ROWS>
__global__ __launch_bounds__(kJoinThreads) void join_page_rows(PagedAttention a) {
    constexpr uint32_t kQuads = 8 * NB;
    __shared__ uint32_t unit_parts[kJoinThreads], wave_units[kJoinThreads / 64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t part0 = 0; part0 < a.parts; part0 += kJoinThreads) {
        const uint32_t mine = part0 + threadIdx.x;
        const bool in_pieces = mine < a.parts && a.joins[mine].pieces > 1;
        const uint64_t theirs = __ballot(in_pieces);
        if (lane == 0) wave_units[wave] = __builtin_popcountll(theirs);
        __syncthreads();
        uint32_t units = 0, at = 0;
        for (uint32_t w = 0; w < kJoinThreads / 64; ++w) {
            if (w == wave) at = units;
            units += wave_units[w];
        }
        if (in_pieces) unit_parts[at + __builtin_popcountll(theirs & ((1ull << lane) - 1))] = mine;
        __syncthreads();
        for (uint32_t i = blockIdx.x * kJoinThreads + threadIdx.x; i < units * ROWS * kQuads; i += gridDim.x * kJoinThreads) {
            const uint32_t part = unit_parts[i / (ROWS * kQuads)], row = i / kQuads % ROWS, value = i % kQuads * 4;
            const PagedJoin u = a.joins[part];
            if (row >= u.rows) continue;
            float least = INFINITY, total = 0.0f;
            float4_t out = float4_t(0.0f);
            constexpr uint32_t kBatch = 8;  // on their way together
            for (uint32_t p0 = 0; p0 < u.pieces; p0 += kBatch) {
                float2 side[kBatch];
                float4_t theirs[kBatch];
#pragma unroll
                for (uint32_t x = 0; x < kBatch; ++x) {
                    const uint64_t from = kept_at(part, min(p0 + x, u.pieces - 1)) * ROWS + row;
                    side[x] = a.stats[from];
                    theirs[x] = *reinterpret_cast<const float4_t*>(a.partial + from * (32 * NB) + value);
                }
#pragma unroll
                for (uint32_t x = 0; x < kBatch; ++x)
                    if (p0 + x < u.pieces) join(side[x], theirs[x], least, total, out);
            }
            const uint32_t of = u.row0 + row;
            float* to = a.output + (uint64_t{u.start} + of / a.group) * a.output_stride +
                        (uint64_t{u.head} * a.group + of % a.group) * (32 * NB) + value;
            *reinterpret_cast<float4_t*>(to) = least == INFINITY ? float4_t(0.0f) : out * (1.0f / total);
        }
        __syncthreads();  // the list is read
    }
}

template <uint32_t F, uint32_t NB>
static hipError_t launch_paged_blocks(const PagedAttention& a, uint32_t octets, hipStream_t stream) {
    if (octets == 0) {
        if constexpr (many_rows_of(F, 32 * NB)) {
            hipLaunchKernelGGL((attend_page_rows<F, NB>), dim3(a.parts), dim3(64 * row_waves(NB)), 0, stream, a);
            if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
            constexpr uint32_t kRows = RowsShape<F, NB>::kRows;
            hipLaunchKernelGGL((join_page_rows<NB, kRows>), dim3(4 * a.parts), dim3(kJoinThreads), 0, stream, a);
        }
    } else if (octets == 2)
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
