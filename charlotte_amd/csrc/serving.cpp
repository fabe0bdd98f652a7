// The C ABI's steps between the products and after the head
// (include/charlotte_hip_matmul.h): their checks, on the host and before any
// kernel launches, and their launches. Sizes are multiplied in 64 bits, and
// every value a kernel holds in 32 is checked first.
#include <cmath>

#include "checks.hpp"
#include "formats.hpp"
#include "serving.hpp"

struct charlotte_hip_matmul_cache {
    const charlotte_hip_matmul_context* ctx = nullptr;  // compared, never followed: it may be gone before the cache
    int device = 0;
    chm::CacheShape shape{};
    bool owned = false;
};

namespace {

using chm::aligned;
using chm::guarded;
using chm::need;
using chm::need_grid;
using chm::refuse;
using chm::Status;
using chm::stride_of;

bool cache_type(uint32_t type) {
    return type == CHARLOTTE_HIP_MATMUL_F16 || type == CHARLOTTE_HIP_MATMUL_Q4_0 || type == CHARLOTTE_HIP_MATMUL_Q8_0;
}

// Sizes a cache may have: at most 2^40 records, whose bytes stay below 2^56.
bool cache_sizes(uint32_t sequences, uint32_t kv_heads, uint32_t head_dim, uint32_t capacity) {
    return sequences > 0 && sequences <= 65535 && kv_heads > 0 && kv_heads <= 65535 && head_dim >= 32 && head_dim <= 256 &&
           head_dim % 32 == 0 && capacity > 0 && capacity <= 0x7FFFFFFFu &&
           (uint64_t{capacity} + 31) / 32 * sequences * kv_heads <= (1ull << 40);
}

chm::CacheShape shape_of(uint32_t type, uint32_t sequences, uint32_t kv_heads, uint32_t head_dim, uint32_t capacity,
                         void* base) {
    chm::CacheShape s{};
    s.base = static_cast<uint8_t*>(base);
    s.tiles = (uint64_t{capacity} + 31) / 32;
    s.format = type;
    s.sequences = sequences, s.kv_heads = kv_heads, s.head_dim = head_dim, s.capacity = capacity;
    return s;
}

void check_cache(uint32_t type, uint32_t sequences, uint32_t kv_heads, uint32_t head_dim, uint32_t capacity) {
    if (!cache_type(type)) refuse("GGUF type " + std::to_string(type), CHARLOTTE_HIP_MATMUL_UNSUPPORTED_TYPE);
    if (!cache_sizes(sequences, kv_heads, head_dim, capacity))
        refuse("sequences " + std::to_string(sequences) + ", key heads " + std::to_string(kv_heads) + ", head " +
               std::to_string(head_dim) + ", capacity " + std::to_string(capacity));
}

void own_cache(const charlotte_hip_matmul_context* ctx, const charlotte_hip_matmul_cache* cache) {
    if (!cache) refuse("no cache");
    if (cache->ctx != ctx) refuse("a cache of another context");
}

void step_in(const chm::CacheShape& c, uint32_t tokens) {
    if (tokens == 0) refuse("a step of no tokens");
    if (tokens > c.capacity) refuse("more tokens than the cache's capacity");
}

chm::CacheRows rows_of(const charlotte_hip_matmul_context* ctx, const charlotte_hip_matmul_cache* cache,
                       const float* keys, const float* values, uint64_t key_stride, uint64_t value_stride,
                       const uint32_t* first, uint32_t tokens) {
    own_cache(ctx, cache);
    step_in(cache->shape, tokens);
    need(keys, "keys", 16);
    need(values, "values", 16);
    need(first, "slots", 4);
    const chm::CacheShape& c = cache->shape;
    const uint64_t width = uint64_t{c.kv_heads} * c.head_dim;
    chm::CacheRows a{};
    a.cache = c;
    a.keys = keys, a.values = values;
    a.key_stride = stride_of(key_stride, width, 4, "key stride");
    a.value_stride = stride_of(value_stride, width, 4, "value stride");
    a.first = first;
    a.tokens = tokens;
    need_grid((uint64_t{c.sequences} * tokens * (width / 32) * 8 + 255) / 256);
    return a;
}

// Rows of a key head, if a step of them can be.
uint64_t rows_a_head(const chm::CacheShape& c, uint32_t query_heads, uint32_t tokens) {
    if (query_heads == 0 || query_heads % c.kv_heads != 0 || tokens == 0 || tokens > c.capacity) return 0;
    const uint64_t rows = uint64_t{tokens} * (query_heads / c.kv_heads);
    return rows * c.sequences * c.kv_heads <= 16 * chm::kGrid ? rows : 0;
}

}  // namespace

extern "C" {

charlotte_hip_matmul_status charlotte_hip_matmul_head_norm_rope(charlotte_hip_matmul_context* ctx,
                                                                const charlotte_hip_matmul_head_norm_rope_desc* desc,
                                                                uint32_t tokens, void* stream) {
    return guarded(ctx, "head norm rope", [&] {
        if (!desc) refuse("no descriptor");
        const charlotte_hip_matmul_head_norm_rope_desc& d = *desc;
        if (tokens == 0) refuse("a step of no tokens");
        if (d.part_count < 1 || d.part_count > 2) refuse("part_count " + std::to_string(d.part_count));
        if (d.head_dim < 8 || d.head_dim > 256 || d.head_dim % 8 != 0) refuse("head_dim " + std::to_string(d.head_dim));
        if (d.rope > CHARLOTTE_HIP_MATMUL_ROPE_NEIGHBOURS) refuse("rope " + std::to_string(d.rope));
        if (!std::isfinite(d.epsilon) || d.epsilon < 0.0f) refuse("epsilon");
        chm::HeadNormRope a{};
        uint64_t heads = 0;
        for (uint32_t i = 0; i < d.part_count; ++i) {
            const charlotte_hip_matmul_heads& p = d.parts[i];
            if (p.heads == 0 || p.heads > 65535) refuse("heads " + std::to_string(p.heads));
            need(p.input, "input", 16);
            need(p.output, "output", 16);
            if (!aligned(p.weight, 16)) refuse("weight not 16-byte aligned");
            const uint64_t width = uint64_t{p.heads} * d.head_dim;
            a.part[i] = {p.input, p.output, p.weight, stride_of(p.input_stride, width, 4, "input stride"),
                         stride_of(p.output_stride, width, 4, "output stride"), p.heads};
            if (p.input == p.output && a.part[i].input_stride != a.part[i].output_stride)
                refuse("in place with two strides");
            heads += p.heads;
        }
        a.parts = d.part_count;
        a.head_dim = d.head_dim;
        a.rope = d.rope;
        a.epsilon = d.epsilon;
        a.tokens = tokens;
        if (d.rope != CHARLOTTE_HIP_MATMUL_ROPE_NONE) {
            a.rope_dims = d.rope_dims ? d.rope_dims : d.head_dim;
            if (a.rope_dims % 8 != 0 || a.rope_dims > d.head_dim) refuse("rope_dims " + std::to_string(d.rope_dims));
            need(d.cosines, "cosines", 16);
            need(d.sines, "sines", 16);
            need(d.positions, "positions", 4);
            a.table_rows = d.table_rows;
            a.cosines = d.cosines, a.sines = d.sines, a.positions = d.positions;
        }
        need_grid((heads * tokens * 64 + 255) / 256);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_head_norm_rope(a, static_cast<hipStream_t>(stream));
    });
}

uint64_t charlotte_hip_matmul_cache_bytes(uint32_t gguf_type, uint32_t sequences, uint32_t kv_heads, uint32_t head_dim,
                                          uint32_t capacity) {
    if (!cache_type(gguf_type) || !cache_sizes(sequences, kv_heads, head_dim, capacity)) return 0;
    return chm::cache_bytes(gguf_type, sequences, kv_heads, head_dim, capacity);
}

charlotte_hip_matmul_status charlotte_hip_matmul_cache_create(charlotte_hip_matmul_context* ctx, uint32_t gguf_type,
                                                              uint32_t sequences, uint32_t kv_heads, uint32_t head_dim,
                                                              uint32_t capacity, charlotte_hip_matmul_cache** out) {
    if (out) *out = nullptr;
    return guarded(ctx, "cache create", [&] {
        if (!out) refuse("nowhere to put the cache");
        check_cache(gguf_type, sequences, kv_heads, head_dim, capacity);
        const uint64_t bytes = chm::cache_bytes(gguf_type, sequences, kv_heads, head_dim, capacity);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        void* device = nullptr;
        if (hipError_t e = hipMalloc(&device, bytes); e != hipSuccess) return e;
        hipError_t e = hipMemset(device, 0, bytes);
        if (e == hipSuccess) e = hipDeviceSynchronize();
        auto* c = e == hipSuccess ? new (std::nothrow) charlotte_hip_matmul_cache : nullptr;
        if (!c) {
            (void)hipFree(device);
            if (e != hipSuccess) return e;
            refuse("no host memory", CHARLOTTE_HIP_MATMUL_OUT_OF_MEMORY);
        }
        *c = {ctx, ctx->device, shape_of(gguf_type, sequences, kv_heads, head_dim, capacity, device), true};
        *out = c;
        return hipSuccess;
    });
}

charlotte_hip_matmul_status charlotte_hip_matmul_cache_wrap(charlotte_hip_matmul_context* ctx, uint32_t gguf_type,
                                                            uint32_t sequences, uint32_t kv_heads, uint32_t head_dim,
                                                            uint32_t capacity, void* device, uint64_t bytes,
                                                            charlotte_hip_matmul_cache** out) {
    if (out) *out = nullptr;
    return guarded(ctx, "cache wrap", [&] {
        if (!out) refuse("nowhere to put the cache");
        check_cache(gguf_type, sequences, kv_heads, head_dim, capacity);
        need(device, "memory", 16);
        if (bytes < chm::cache_bytes(gguf_type, sequences, kv_heads, head_dim, capacity))
            refuse("memory shorter than the cache");
        auto* c = new (std::nothrow) charlotte_hip_matmul_cache;
        if (!c) refuse("no host memory", CHARLOTTE_HIP_MATMUL_OUT_OF_MEMORY);
        *c = {ctx, ctx->device, shape_of(gguf_type, sequences, kv_heads, head_dim, capacity, device), false};
        *out = c;
        return hipSuccess;
    });
}

charlotte_hip_matmul_status charlotte_hip_matmul_cache_free(charlotte_hip_matmul_cache* cache) {
    if (!cache) return CHARLOTTE_HIP_MATMUL_OK;
    Status s = CHARLOTTE_HIP_MATMUL_OK;
    if (cache->owned) {
        (void)hipSetDevice(cache->device);
        if (hipFree(cache->shape.base) != hipSuccess) s = CHARLOTTE_HIP_MATMUL_HIP_ERROR;
    }
    delete cache;
    return s;
}

charlotte_hip_matmul_status charlotte_hip_matmul_cache_append(charlotte_hip_matmul_context* ctx,
                                                              charlotte_hip_matmul_cache* cache, const float* keys,
                                                              const float* values, uint64_t key_stride,
                                                              uint64_t value_stride, const uint32_t* past,
                                                              uint32_t tokens, void* stream) {
    return guarded(ctx, "cache append", [&] {
        const chm::CacheRows a = rows_of(ctx, cache, keys, values, key_stride, value_stride, past, tokens);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_cache_append(a, static_cast<hipStream_t>(stream));
    });
}

charlotte_hip_matmul_status charlotte_hip_matmul_cache_read(charlotte_hip_matmul_context* ctx,
                                                            const charlotte_hip_matmul_cache* cache, float* keys,
                                                            float* values, uint64_t key_stride, uint64_t value_stride,
                                                            const uint32_t* first, uint32_t tokens, void* stream) {
    return guarded(ctx, "cache read", [&] {
        const chm::CacheRows a = rows_of(ctx, cache, keys, values, key_stride, value_stride, first, tokens);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_cache_read(a, static_cast<hipStream_t>(stream));
    });
}

charlotte_hip_matmul_status charlotte_hip_matmul_cache_keep(charlotte_hip_matmul_context* ctx,
                                                            charlotte_hip_matmul_cache* cache, const uint32_t* past,
                                                            const int32_t* path, const uint32_t* count, uint32_t tokens,
                                                            void* stream) {
    return guarded(ctx, "cache keep", [&] {
        own_cache(ctx, cache);
        step_in(cache->shape, tokens);
        need(past, "past", 4);
        need(path, "path", 4);
        need(count, "count", 4);
        need_grid(uint64_t{cache->shape.sequences} * cache->shape.kv_heads);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_cache_keep({cache->shape, past, path, count, tokens}, static_cast<hipStream_t>(stream));
    });
}

uint64_t charlotte_hip_matmul_attention_workspace_bytes(const charlotte_hip_matmul_context* ctx,
                                                        const charlotte_hip_matmul_cache* cache, uint32_t query_heads,
                                                        uint32_t tokens) {
    if (!ctx || !cache || rows_a_head(cache->shape, query_heads, tokens) == 0) return 0;
    return chm::attention_workspace_bytes(cache->shape, query_heads, tokens, ctx->compute_units);
}

charlotte_hip_matmul_status charlotte_hip_matmul_attention(charlotte_hip_matmul_context* ctx,
                                                           const charlotte_hip_matmul_attention_desc* desc,
                                                           uint32_t tokens, void* stream) {
    return guarded(ctx, "attention", [&] {
        if (!desc) refuse("no descriptor");
        const charlotte_hip_matmul_attention_desc& d = *desc;
        own_cache(ctx, d.cache);
        const chm::CacheShape& c = d.cache->shape;
        step_in(c, tokens);
        if (d.query_heads == 0 || d.query_heads % c.kv_heads != 0)
            refuse("query heads " + std::to_string(d.query_heads) + " over " + std::to_string(c.kv_heads) + " key heads");
        const uint64_t rows = rows_a_head(c, d.query_heads, tokens);
        if (rows == 0) refuse("too many rows a step");
        if (!std::isfinite(d.scale)) refuse("scale not finite");
        if (d.parents && tokens > chm::kTreeTokens)
            refuse("a tree of " + std::to_string(tokens) + " tokens", CHARLOTTE_HIP_MATMUL_UNSUPPORTED);
        need(d.queries, "queries", 16);
        need(d.output, "output", 16);
        need(d.past, "past", 4);
        if (!aligned(d.parents, 4)) refuse("parents not 4-byte aligned");
        const uint64_t width = uint64_t{d.query_heads} * c.head_dim;
        chm::Attention a{};
        a.cache = c;
        a.queries = d.queries, a.output = d.output;
        a.query_stride = stride_of(d.query_stride, width, 4, "query stride");
        a.output_stride = stride_of(d.output_stride, width, 4, "output stride");
        a.past = d.past, a.parents = d.parents;
        a.tokens = tokens;
        a.group = d.query_heads / c.kv_heads;
        a.rows = static_cast<uint32_t>(rows);
        a.window = d.window;
        a.scale = d.scale;
        const chm::AttentionPlan plan =
            chm::plan_attention(c, d.query_heads, tokens, d.longest, d.window, ctx->compute_units);
        a.splits = plan.splits;
        if (plan.splits > 1) {
            const uint64_t bytes = chm::attention_partial_bytes(c, d.query_heads, tokens, plan.splits);
            if (!d.workspace || d.workspace_bytes < bytes)
                refuse("needs a workspace of " + std::to_string(bytes) + " bytes");
            need(d.workspace, "workspace", 16);
            a.partial = static_cast<float*>(d.workspace);
            a.stats = reinterpret_cast<float2*>(a.partial + uint64_t{c.sequences} * d.query_heads * tokens * plan.splits *
                                                                c.head_dim);
        }
        need_grid(uint64_t{c.sequences} * c.kv_heads * plan.row_groups * plan.splits);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        const auto s = static_cast<hipStream_t>(stream);
        hipError_t e = c.format == chm::kF16    ? chm::launch_attention_f16(a, plan, s)
                       : c.format == chm::kQ4_0 ? chm::launch_attention_q4_0(a, plan, s)
                                                : chm::launch_attention_q8_0(a, plan, s);
        if (e == hipSuccess && plan.splits > 1) e = chm::launch_attention_combine(a, s);
        return e;
    });
}

uint64_t charlotte_hip_matmul_probabilities_workspace_bytes(uint32_t rows, uint32_t vocabulary) {
    if (rows == 0 || vocabulary == 0) return 0;
    return chm::probabilities_bytes(rows, vocabulary);
}

charlotte_hip_matmul_status charlotte_hip_matmul_probabilities(charlotte_hip_matmul_context* ctx,
                                                               const charlotte_hip_matmul_probabilities_desc* desc,
                                                               void* stream) {
    return guarded(ctx, "probabilities", [&] {
        if (!desc) refuse("no descriptor");
        const charlotte_hip_matmul_probabilities_desc& d = *desc;
        if (d.rows == 0 || d.vocabulary == 0) refuse("no rows or no vocabulary");
        if (d.vocabulary > 0x7FFFFFF0u) refuse("vocabulary " + std::to_string(d.vocabulary));
        if (!std::isfinite(d.temperature) || d.temperature < 0.0f || (d.temperature > 0.0f && d.temperature < 1e-6f))
            refuse("temperature " + std::to_string(d.temperature));
        need(d.logits, "logits", 4);
        need(d.output, "output", 4);
        chm::Probabilities a{};
        a.logits = d.logits, a.output = d.output;
        a.logit_stride = stride_of(d.logit_stride, d.vocabulary, 1, "logit stride");
        a.output_stride = stride_of(d.output_stride, d.vocabulary, 1, "output stride");
        if (d.logits == d.output && a.logit_stride != a.output_stride) refuse("in place with two strides");
        a.rows = d.rows, a.vocabulary = d.vocabulary;
        a.temperature = d.temperature;
        need_grid(uint64_t{d.rows} * ((uint64_t{d.vocabulary} + 2047) / 2048));
        need(d.workspace, "workspace", 16);
        if (d.workspace_bytes < charlotte_hip_matmul_probabilities_workspace_bytes(d.rows, d.vocabulary))
            refuse("workspace shorter than probabilities_workspace_bytes");
        a.looks = ctx->patience;
        a.stats = static_cast<chm::RowStats*>(d.workspace);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_probabilities(a, static_cast<hipStream_t>(stream));
    });
}

charlotte_hip_matmul_status charlotte_hip_matmul_set_patience(charlotte_hip_matmul_context* ctx, uint32_t looks) {
    return guarded(ctx, "patience", [&] {
        if (looks > CHARLOTTE_HIP_MATMUL_PATIENCE) refuse(std::to_string(looks) + " looks");
        ctx->patience = looks;
        return hipSuccess;
    });
}

uint64_t charlotte_hip_matmul_verify_workspace_bytes(uint32_t sequences, uint32_t tokens, uint32_t vocabulary) {
    if (sequences == 0 || tokens == 0 || vocabulary == 0 || vocabulary > (1u << 18) ||
        tokens > chm::kVerifyTokens || uint64_t{sequences} * tokens > 0xFFFFFull)
        return 0;
    return chm::verify_bytes(sequences, tokens, vocabulary);
}

charlotte_hip_matmul_status charlotte_hip_matmul_verify(charlotte_hip_matmul_context* ctx,
                                                        const charlotte_hip_matmul_verify_desc* desc,
                                                        uint32_t sequences, uint32_t tokens, void* stream) {
    return guarded(ctx, "verify", [&] {
        if (!desc) refuse("no descriptor");
        const charlotte_hip_matmul_verify_desc& d = *desc;
        if (sequences == 0 || tokens == 0) refuse("a step of no nodes");
        if (d.vocabulary == 0 || d.vocabulary > (1u << 18)) refuse("vocabulary " + std::to_string(d.vocabulary));
        const uint64_t bytes = charlotte_hip_matmul_verify_workspace_bytes(sequences, tokens, d.vocabulary);
        if (bytes == 0) refuse("too many nodes a step");
        if (d.draft && d.parents) refuse("a draft's probabilities go with a chain, not a tree", CHARLOTTE_HIP_MATMUL_UNSUPPORTED);
        need(d.node_tokens, "node_tokens", 4);
        need(d.target, "target", 4);
        need(d.uniforms, "uniforms", 4);
        need(d.path, "path", 4);
        need(d.emitted, "emitted", 4);
        need(d.count, "count", 4);
        if (d.draft) need(d.accepts, "accepts", 4);
        if (!aligned(d.draft, 4) || !aligned(d.parents, 4) || !aligned(d.lengths, 4)) refuse("a pointer not 4-byte aligned");
        need(d.workspace, "workspace", 16);
        if (d.workspace_bytes < bytes) refuse("needs a workspace of " + std::to_string(bytes) + " bytes");
        chm::Verify a{};
        a.node_tokens = d.node_tokens, a.target = d.target, a.draft = d.draft;
        a.uniforms = d.uniforms, a.accepts = d.accepts, a.parents = d.parents, a.lengths = d.lengths;
        a.path = d.path, a.emitted = d.emitted, a.count = d.count;
        a.target_stride = stride_of(d.target_stride, d.vocabulary, 1, "target stride");
        a.draft_stride = stride_of(d.draft_stride, d.vocabulary, 1, "draft stride");
        a.vocabulary = d.vocabulary, a.sequences = sequences, a.tokens = tokens;
        a.sums = static_cast<uint64_t*>(d.workspace);
        a.drawn = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(d.workspace) + bytes - uint64_t{sequences} * 4);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_verify(a, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
