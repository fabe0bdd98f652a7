// The operators of a step over several requests as their kernels receive them,
// built and checked on the host from the C ABI's descriptors (requests.cpp).
#pragma once

#include "serving.hpp"

namespace chm {

// ---- page_plan (pages.hip) ----

struct PagePlan {
    const uint32_t* past;
    const uint32_t* counts;
    const uint32_t* held;
    uint32_t* held_after;
    uint32_t* table;
    uint32_t* free_pages;
    const uint32_t* free_count;
    uint32_t* free_count_after;
    uint32_t* starts;
    uint32_t* granted;
    uint32_t* slots;
    uint32_t* positions;  // or null
    uint32_t requests, rows, table_stride, pages, page_tokens;
};

hipError_t launch_page_plan(const PagePlan& a, hipStream_t stream);

// ---- the pool (cache.hip) ----

// A pool is a cache whose sequences are its pages: `cache.sequences` pages of
// `cache.capacity` tokens; `first` holds a slot a row, `tokens` the rows.
hipError_t launch_page_append(const CacheRows& a, hipStream_t stream);
hipError_t launch_page_read(const CacheRows& a, hipStream_t stream);

// ---- paged attention (paged.hpp, paged_*.hip) ----

// A unit of many rows in pieces, of which the first is a part's.
struct PagedJoin {
    uint32_t start, head, row0, rows, pieces, reserved;
};

struct PagedAttention {
    CacheShape pool;
    const float* queries;
    float* output;
    uint64_t query_stride, output_stride;
    const uint32_t* past;
    const uint32_t* counts;
    const uint32_t* starts;
    const uint32_t* table;
    float* partial;      // a piece's outputs, [piece][row][head_dim]
    float2* stats;       // its rows' offsets and sums, [piece][row]
    PagedJoin* joins;    // many rows: a part's unit in pieces
    uint32_t* counters;  // pieces of a unit that are done; 0 between launches
    uint32_t requests, rows, table_stride, group, window, parts;
    // attend_pages has the requests of more rows of a key head than `above`, up to
    // `upto`; but those of many_from and more are attend_page_rows' where their load
    // is many_load and more (0: never).
    uint32_t above, upto, many_from, many_load;
    uint32_t page_inverse;  // of a page's tiles, where they are two and more: 2^32 over them, rounded up
    float scale;
};

// Pieces of units that a step may leave, a workgroup.
constexpr uint32_t kPieces = 2;
// Rows of a key head from which a request has workgroups of many rows, in the
// formats and widths that attention has them for (attention_plan.cpp). 8 requests over
// 4,000, 8 key heads in Q8_0, so and by units of 32: 128 rows of 128 values 101 us and 109,
// of 64 61 and 44; 256 rows 129 and 200, 78 and 84.
constexpr uint32_t many_from(uint32_t head_dim) { return head_dim <= 64 ? 256 : 128; }
// (Wider quantized heads: 4 waves' rows are too few to pay for laying codes out, 387 us beside 308 of a
// contiguous cache, attention_plan.cpp; by units of 32 here: paged.hpp.)
constexpr bool many_rows_of(uint32_t format, uint32_t head_dim) { return format == 1 /* F16 */ || head_dim <= 128; }
// `octets`: 1 or 2 of attend_pages; 0: attend_page_rows, and what joins its pieces.
hipError_t launch_paged_f16(const PagedAttention& a, uint32_t octets, hipStream_t stream);
hipError_t launch_paged_q4_0(const PagedAttention& a, uint32_t octets, hipStream_t stream);
hipError_t launch_paged_q8_0(const PagedAttention& a, uint32_t octets, hipStream_t stream);

// ---- residual_norm (residual.hip) ----

struct ResidualNorm {
    const float* residual;
    const float* branch;         // or null, as the next two
    const float* branch_weight;
    const float* gate;
    const float* weight;
    float* residual_out;         // or null
    float* normed;               // or null
    uint64_t residual_stride, branch_stride, gate_stride, residual_out_stride, normed_stride;
    uint32_t width, rows;
    float epsilon, residual_scale, branch_scale;
    bool fours;                  // every row is whole, aligned fours
};

hipError_t launch_residual_norm(const ResidualNorm& a, hipStream_t stream);

// ---- sample (sample.hip) ----

struct Sample {
    const float* logits;
    const float* uniforms;
    int32_t* tokens;
    float* chances;             // or null, as the next four
    const float* temperatures;
    const int32_t* top_ks;
    const float* top_ps;
    const float* min_ps;
    uint64_t logit_stride;
    uint32_t rows, vocabulary;
    float temperature;
    int32_t top_k;
    float top_p, min_p;
    void* workspace;
};

uint64_t sample_bytes(uint32_t rows, uint32_t vocabulary);
hipError_t launch_sample(const Sample& a, hipStream_t stream);

}  // namespace chm
