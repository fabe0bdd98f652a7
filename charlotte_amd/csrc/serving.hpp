// The steps between a decoder step's products as their kernels receive them,
// built and checked on the host from the C ABI's descriptors (serving.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace chm {

// ---- head_norm_rope (heads.hip) ----

struct HeadPart {
    const float* input;
    float* output;
    const float* weight;  // or null
    uint64_t input_stride, output_stride;
    uint32_t heads;
};

struct HeadNormRope {
    HeadPart part[2];
    uint32_t parts, head_dim, rope, rope_dims, tokens, table_rows;
    float epsilon;
    const float* cosines;
    const float* sines;
    const uint32_t* positions;
};

hipError_t launch_head_norm_rope(const HeadNormRope& a, hipStream_t stream);

// ---- the cache (cache.hip; its layout: cache.hpp) ----

struct CacheShape {
    uint8_t* base;
    uint64_t tiles;     // 32-token tiles a head of a sequence
    uint32_t format;    // kF16, kQ4_0 or kQ8_0
    uint32_t sequences, kv_heads, head_dim, capacity;
};

struct CacheRows {
    CacheShape cache;
    const float* keys;  // append: read; read: written
    const float* values;
    uint64_t key_stride, value_stride;
    const uint32_t* first;
    uint32_t tokens;
};

struct CacheKeep {
    CacheShape cache;
    const uint32_t* past;
    const int32_t* path;
    const uint32_t* count;
    uint32_t tokens;
};

uint64_t cache_bytes(uint32_t format, uint32_t sequences, uint32_t kv_heads, uint32_t head_dim, uint32_t capacity);
hipError_t launch_cache_append(const CacheRows& a, hipStream_t stream);
hipError_t launch_cache_read(const CacheRows& a, hipStream_t stream);
hipError_t launch_cache_keep(const CacheKeep& a, hipStream_t stream);

// ---- attention (attention.hpp, attention_*.hip, attention_plan.cpp) ----

constexpr uint32_t kTreeTokens = 256;

struct Attention {
    CacheShape cache;
    const float* queries;
    float* output;
    uint64_t query_stride, output_stride;
    const uint32_t* past;
    const int32_t* parents;  // or null: a chain
    float2* stats;           // splits > 1: each row's offset and sum, [head][row][split]
    float* partial;          // and its outputs over neither, [head][row][split][head_dim]
    uint32_t tokens, group, rows;  // rows = tokens x group, of one key head
    uint32_t window, splits;
    float scale;
};

// How a step runs: rows a workgroup, workgroups along its rows and its keys.
struct AttentionPlan {
    uint32_t octets;      // a wave's rows, in 16s
    uint32_t waves;       // waves with rows of their own: 8 or 4 (attend_rows); 1: the waves split the tiles (attend)
    uint32_t row_groups;  // workgroups along the rows of a key head
    uint32_t splits;      // workgroups along the keys
};

AttentionPlan plan_attention(const CacheShape& cache, uint32_t query_heads, uint32_t tokens, uint32_t longest,
                             uint32_t window, uint32_t compute_units);
// The workspace of a step in `splits`: its outputs, then its stats.
uint64_t attention_partial_bytes(const CacheShape& cache, uint32_t query_heads, uint32_t tokens, uint32_t splits);
// What any step of at most `tokens` tokens a sequence may need of it.
uint64_t attention_workspace_bytes(const CacheShape& cache, uint32_t query_heads, uint32_t tokens, uint32_t compute_units);
hipError_t launch_attention_f16(const Attention& a, const AttentionPlan& plan, hipStream_t stream);
hipError_t launch_attention_q4_0(const Attention& a, const AttentionPlan& plan, hipStream_t stream);
hipError_t launch_attention_q8_0(const Attention& a, const AttentionPlan& plan, hipStream_t stream);
hipError_t launch_attention_combine(const Attention& a, hipStream_t stream);

// ---- probabilities (probabilities.hip) ----

struct RowStats {
    float largest, sum;
    uint32_t at;  // the largest's first index
};

struct Probabilities {
    const float* logits;
    float* output;
    uint64_t logit_stride, output_stride;
    uint32_t rows, vocabulary, chunks;  // chunks a row: launch_probabilities'
    float temperature;
    uint32_t looks;   // at a row's other chunks, before a workgroup reads the row itself
    RowStats* stats;  // [rows][chunks], or words of 8 bytes
};

uint64_t probabilities_bytes(uint32_t rows, uint32_t vocabulary);
hipError_t launch_probabilities(Probabilities a, hipStream_t stream);

// ---- verify (verify.hip) ----

struct Verify {
    const int32_t* node_tokens;
    const float* target;
    const float* draft;  // or null: by the target's draws
    const float* uniforms;
    const float* accepts;
    const int32_t* parents;
    const uint32_t* lengths;
    int32_t* path;
    int32_t* emitted;
    uint32_t* count;
    uint64_t target_stride, draft_stride;
    uint32_t vocabulary, sequences, tokens;
    uint32_t share, chunks;  // segments a workgroup, workgroups a row (launch_verify's)
    uint64_t* sums;          // [drawn rows][segments]: a segment's weights summed
    int32_t* drawn;          // [sequences]: with a draft, the last node accepted
};

constexpr uint32_t kVerifyTokens = 1024;  // nodes a sequence

uint64_t verify_bytes(uint32_t sequences, uint32_t tokens, uint32_t vocabulary);
hipError_t launch_verify(Verify a, hipStream_t stream);

}  // namespace chm
