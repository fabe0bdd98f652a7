// The C ABI's operators of a step over several requests
// (include/charlotte_hip_matmul.h): their checks, on the host and before any
// kernel launches, and their launches. Lengths and tables are device memory, and
// what they hold is checked by the kernels.
#include <algorithm>
#include <cmath>
#include <utility>

#include "checks.hpp"
#include "formats.hpp"
#include "requests.hpp"

struct charlotte_hip_matmul_page_pool {
    const charlotte_hip_matmul_context* ctx = nullptr;  // compared, never followed: it may be gone before the pool
    int device = 0;
    chm::CacheShape shape{};
    uint32_t* counters = nullptr;  // kPieces words a compute unit, 0 between launches
    bool owned = false;
};

namespace {

using chm::aligned;
using chm::guarded;
using chm::need;
using chm::need_grid;
using chm::refuse;
using chm::stride_of;

constexpr uint32_t kRequests = 65536;
constexpr uint32_t kRows = 1u << 20;  // of paged attention

bool pool_type(uint32_t type) {
    return type == CHARLOTTE_HIP_MATMUL_F16 || type == CHARLOTTE_HIP_MATMUL_Q4_0 || type == CHARLOTTE_HIP_MATMUL_Q8_0;
}

bool pool_sizes(uint32_t pages, uint32_t page_tokens, uint32_t kv_heads, uint32_t head_dim) {
    return pages > 0 && page_tokens > 0 && page_tokens % 32 == 0 && page_tokens <= 2048 &&
           uint64_t{pages} * page_tokens < (1ull << 31) && kv_heads > 0 && kv_heads <= 65535 && head_dim >= 32 &&
           head_dim <= 256 && head_dim % 32 == 0;
}

void check_pool(uint32_t type, uint32_t pages, uint32_t page_tokens, uint32_t kv_heads, uint32_t head_dim) {
    if (!pool_type(type)) refuse("GGUF type " + std::to_string(type), CHARLOTTE_HIP_MATMUL_UNSUPPORTED_TYPE);
    if (!pool_sizes(pages, page_tokens, kv_heads, head_dim))
        refuse(std::to_string(pages) + " pages of " + std::to_string(page_tokens) + " tokens, key heads " +
               std::to_string(kv_heads) + ", head " + std::to_string(head_dim));
}

// A pool over `device`, or over memory of its own.
hipError_t make_pool(charlotte_hip_matmul_context* ctx, uint32_t type, uint32_t pages, uint32_t page_tokens,
                     uint32_t kv_heads, uint32_t head_dim, void* device, charlotte_hip_matmul_page_pool** out) {
    const uint64_t bytes = chm::cache_bytes(type, pages, kv_heads, head_dim, page_tokens);
    const uint64_t counted = uint64_t{ctx->compute_units} * chm::kPieces * sizeof(uint32_t);
    if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
    const bool owned = device == nullptr;
    void* counters = nullptr;
    hipError_t e = hipMalloc(&counters, counted);
    if (e == hipSuccess && owned) e = hipMalloc(&device, bytes);
    if (e == hipSuccess) e = hipMemset(counters, 0, counted);
    if (e == hipSuccess && owned) e = hipMemset(device, 0, bytes);
    if (e == hipSuccess) e = hipDeviceSynchronize();
    auto* p = e == hipSuccess ? new (std::nothrow) charlotte_hip_matmul_page_pool : nullptr;
    if (!p) {
        if (counters) (void)hipFree(counters);
        if (owned && device) (void)hipFree(device);
        if (e != hipSuccess) return e;
        refuse("no host memory", CHARLOTTE_HIP_MATMUL_OUT_OF_MEMORY);
    }
    chm::CacheShape s{};
    s.base = static_cast<uint8_t*>(device);
    s.tiles = page_tokens / 32;
    s.format = type;
    s.sequences = pages, s.kv_heads = kv_heads, s.head_dim = head_dim, s.capacity = page_tokens;
    *p = {ctx, ctx->device, s, static_cast<uint32_t*>(counters), owned};
    *out = p;
    return hipSuccess;
}

void own_pool(const charlotte_hip_matmul_context* ctx, const charlotte_hip_matmul_page_pool* pool) {
    if (!pool) refuse("no pool");
    if (pool->ctx != ctx) refuse("a pool of another context");
}

chm::CacheRows rows_of(const charlotte_hip_matmul_context* ctx, const charlotte_hip_matmul_page_pool* pool,
                       const float* keys, const float* values, uint64_t key_stride, uint64_t value_stride,
                       const uint32_t* slots, uint32_t rows) {
    own_pool(ctx, pool);
    if (rows == 0) refuse("a step of no rows");
    need(keys, "keys", 16);
    need(values, "values", 16);
    need(slots, "slots", 4);
    const chm::CacheShape& c = pool->shape;
    const uint64_t width = uint64_t{c.kv_heads} * c.head_dim;
    chm::CacheRows a{};
    a.cache = c;
    a.keys = keys, a.values = values;
    a.key_stride = stride_of(key_stride, width, 4, "key stride");
    a.value_stride = stride_of(value_stride, width, 4, "value stride");
    a.first = slots;
    a.tokens = rows;
    need_grid((uint64_t{rows} * (width / 32) * 8 + 255) / 256);
    return a;
}

// Requests and the pages of each, as page_plan and paged_attention take them.
void check_table(uint32_t requests, uint32_t table_stride, uint32_t page_tokens) {
    if (requests == 0 || requests > kRequests) refuse(std::to_string(requests) + " requests");
    if (table_stride == 0 || uint64_t{table_stride} * page_tokens >= (1ull << 31))
        refuse("table stride " + std::to_string(table_stride));
}

// How a step of attention runs: requests of up to 16 rows of a key head by units of
// 16, of more by units of 32, of many_from and more, where they are load enough, by
// units of `many`; each in launches of its own, of which one that finds no request of
// its kind takes 4 - 5 us. One request, which is of one kind, and groups past 16 have no
// launch of units of 16.
struct PagedPlan {
    bool ones, twos;
    uint32_t many, many_load;  // 0: none
};
PagedPlan paged_plan(const chm::CacheShape& c, uint32_t group, uint32_t most, uint32_t requests, uint64_t most_load) {
    const uint64_t rows = uint64_t{group} * std::max(most, 1u);
    if (rows <= 16) return {true, false, 0, 0};
    PagedPlan plan{requests > 1 && group <= 16, true, 0, 0};
    // the loads at which attention takes its form of many rows (attention_plan.cpp)
    const uint32_t load = c.head_dim <= 64 ? 112 : c.head_dim <= 128 ? 44 : 11;
    if (rows >= chm::many_from(c.head_dim) && chm::many_rows_of(c.format, c.head_dim) && most_load >= load)
        plan.many = c.head_dim <= 128 ? 256 : 128, plan.many_load = load;
    return plan;
}

// Pieces' places, outputs and then offsets and sums, of units of `rows` rows.
uint64_t piece_rows(const charlotte_hip_matmul_context* ctx, uint32_t rows) {
    return uint64_t{ctx->compute_units} * chm::kPieces * rows;
}
uint64_t piece_bytes(const charlotte_hip_matmul_context* ctx, const chm::CacheShape& c, const PagedPlan& plan) {
    return piece_rows(ctx, std::max(plan.twos ? 32u : 16u, plan.many)) * (uint64_t{c.head_dim} * 4 + 8) +
           (plan.many ? ctx->compute_units * sizeof(chm::PagedJoin) : 0);
}

// An output that is an input's memory has its stride.
void in_place(const float* output, uint64_t stride, const float* input, uint64_t input_stride) {
    if (output && output == input && stride != input_stride) refuse("in place with two strides");
}

}  // namespace

extern "C" {

uint64_t charlotte_hip_matmul_page_pool_bytes(uint32_t gguf_type, uint32_t pages, uint32_t page_tokens,
                                              uint32_t kv_heads, uint32_t head_dim) {
    if (!pool_type(gguf_type) || !pool_sizes(pages, page_tokens, kv_heads, head_dim)) return 0;
    return chm::cache_bytes(gguf_type, pages, kv_heads, head_dim, page_tokens);
}

charlotte_hip_matmul_status charlotte_hip_matmul_page_pool_create(charlotte_hip_matmul_context* ctx, uint32_t gguf_type,
                                                                  uint32_t pages, uint32_t page_tokens,
                                                                  uint32_t kv_heads, uint32_t head_dim,
                                                                  charlotte_hip_matmul_page_pool** out) {
    if (out) *out = nullptr;
    return guarded(ctx, "page pool create", [&] {
        if (!out) refuse("nowhere to put the pool");
        check_pool(gguf_type, pages, page_tokens, kv_heads, head_dim);
        return make_pool(ctx, gguf_type, pages, page_tokens, kv_heads, head_dim, nullptr, out);
    });
}

charlotte_hip_matmul_status charlotte_hip_matmul_page_pool_wrap(charlotte_hip_matmul_context* ctx, uint32_t gguf_type,
                                                                uint32_t pages, uint32_t page_tokens,
                                                                uint32_t kv_heads, uint32_t head_dim, void* device,
                                                                uint64_t bytes, charlotte_hip_matmul_page_pool** out) {
    if (out) *out = nullptr;
    return guarded(ctx, "page pool wrap", [&] {
        if (!out) refuse("nowhere to put the pool");
        check_pool(gguf_type, pages, page_tokens, kv_heads, head_dim);
        need(device, "memory", 16);
        if (bytes < chm::cache_bytes(gguf_type, pages, kv_heads, head_dim, page_tokens)) refuse("memory shorter than the pool");
        return make_pool(ctx, gguf_type, pages, page_tokens, kv_heads, head_dim, device, out);
    });
}

charlotte_hip_matmul_status charlotte_hip_matmul_page_pool_free(charlotte_hip_matmul_page_pool* pool) {
    if (!pool) return CHARLOTTE_HIP_MATMUL_OK;
    charlotte_hip_matmul_status s = CHARLOTTE_HIP_MATMUL_OK;
    (void)hipSetDevice(pool->device);
    if (hipFree(pool->counters) != hipSuccess) s = CHARLOTTE_HIP_MATMUL_HIP_ERROR;
    if (pool->owned && hipFree(pool->shape.base) != hipSuccess) s = CHARLOTTE_HIP_MATMUL_HIP_ERROR;
    delete pool;
    return s;
}

charlotte_hip_matmul_status charlotte_hip_matmul_page_plan(charlotte_hip_matmul_context* ctx,
                                                           const charlotte_hip_matmul_page_plan_desc* desc, void* stream) {
    return guarded(ctx, "page plan", [&] {
        if (!desc) refuse("no descriptor");
        const charlotte_hip_matmul_page_plan_desc& d = *desc;
        if (d.pages == 0 || d.page_tokens == 0 || d.page_tokens % 32 != 0 || d.page_tokens > 2048 ||
            uint64_t{d.pages} * d.page_tokens >= (1ull << 31))
            refuse(std::to_string(d.pages) + " pages of " + std::to_string(d.page_tokens) + " tokens");
        check_table(d.requests, d.table_stride, d.page_tokens);
        if (d.rows == 0 || d.rows >= (1u << 31)) refuse(std::to_string(d.rows) + " rows");
        need(d.past, "past", 4);
        need(d.counts, "counts", 4);
        need(d.held, "held", 4);
        need(d.held_after, "held_after", 4);
        need(d.table, "table", 4);
        need(d.free_pages, "free_pages", 4);
        need(d.free_count, "free_count", 4);
        need(d.free_count_after, "free_count_after", 4);
        need(d.starts, "starts", 4);
        need(d.granted, "granted", 4);
        need(d.slots, "slots", 4);
        if (!aligned(d.positions, 4)) refuse("positions not 4-byte aligned");
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_page_plan({d.past, d.counts, d.held, d.held_after, d.table, d.free_pages, d.free_count,
                                      d.free_count_after, d.starts, d.granted, d.slots, d.positions, d.requests, d.rows,
                                      d.table_stride, d.pages, d.page_tokens},
                                     static_cast<hipStream_t>(stream));
    });
}

charlotte_hip_matmul_status charlotte_hip_matmul_page_append(charlotte_hip_matmul_context* ctx,
                                                             charlotte_hip_matmul_page_pool* pool, const float* keys,
                                                             const float* values, uint64_t key_stride,
                                                             uint64_t value_stride, const uint32_t* slots,
                                                             uint32_t rows, void* stream) {
    return guarded(ctx, "page append", [&] {
        const chm::CacheRows a = rows_of(ctx, pool, keys, values, key_stride, value_stride, slots, rows);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_page_append(a, static_cast<hipStream_t>(stream));
    });
}

charlotte_hip_matmul_status charlotte_hip_matmul_page_read(charlotte_hip_matmul_context* ctx,
                                                           const charlotte_hip_matmul_page_pool* pool, float* keys,
                                                           float* values, uint64_t key_stride, uint64_t value_stride,
                                                           const uint32_t* slots, uint32_t rows, void* stream) {
    return guarded(ctx, "page read", [&] {
        const chm::CacheRows a = rows_of(ctx, pool, keys, values, key_stride, value_stride, slots, rows);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_page_read(a, static_cast<hipStream_t>(stream));
    });
}

uint64_t charlotte_hip_matmul_paged_attention_workspace_bytes(const charlotte_hip_matmul_context* ctx,
                                                              const charlotte_hip_matmul_page_pool* pool,
                                                              uint32_t query_heads, uint32_t most) {
    if (!ctx || !pool || query_heads == 0 || query_heads % pool->shape.kv_heads != 0) return 0;
    return piece_bytes(ctx, pool->shape, paged_plan(pool->shape, query_heads / pool->shape.kv_heads, most, 2, UINT64_MAX));
}

charlotte_hip_matmul_status charlotte_hip_matmul_paged_attention(charlotte_hip_matmul_context* ctx,
                                                                 const charlotte_hip_matmul_paged_attention_desc* desc,
                                                                 void* stream) {
    return guarded(ctx, "paged attention", [&] {
        if (!desc) refuse("no descriptor");
        const charlotte_hip_matmul_paged_attention_desc& d = *desc;
        own_pool(ctx, d.pool);
        const chm::CacheShape& c = d.pool->shape;
        check_table(d.requests, d.table_stride, c.capacity);
        if (d.rows == 0 || d.rows > kRows) refuse(std::to_string(d.rows) + " rows");
        if (d.query_heads == 0 || d.query_heads % c.kv_heads != 0)
            refuse("query heads " + std::to_string(d.query_heads) + " over " + std::to_string(c.kv_heads) + " key heads");
        const uint32_t group = d.query_heads / c.kv_heads;
        // 32 rows by a tile, for each compute unit, if every row were to see the longest request
        const uint64_t reach = uint64_t{d.table_stride} * c.capacity, longest = d.longest ? std::min<uint64_t>(d.longest, reach) : reach;
        const uint64_t load = (uint64_t{d.rows} * group + 31) / 32 * c.kv_heads * ((longest + 31) / 32) / ctx->compute_units;
        const PagedPlan plan = paged_plan(c, group, d.most, d.requests, load);
        // all units, each of all the tiles that a table's row holds
        const uint64_t units = (uint64_t{d.rows} * group / (plan.twos ? 32 : 16) + d.requests) * c.kv_heads;
        if (uint64_t{d.rows} * group >= (1ull << 28) || units * (uint64_t{d.table_stride} * (c.capacity / 32) + 16) >= (1ull << 32))
            refuse("too many rows a step for tables so long");
        if (!std::isfinite(d.scale)) refuse("scale not finite");
        need(d.queries, "queries", 16);
        need(d.output, "output", 16);
        need(d.past, "past", 4);
        need(d.counts, "counts", 4);
        need(d.starts, "starts", 4);
        need(d.table, "table", 4);
        const uint64_t width = uint64_t{d.query_heads} * c.head_dim;
        chm::PagedAttention a{};
        a.pool = c;
        a.queries = d.queries, a.output = d.output;
        a.query_stride = stride_of(d.query_stride, width, 4, "query stride");
        a.output_stride = stride_of(d.output_stride, width, 4, "output stride");
        a.past = d.past, a.counts = d.counts, a.starts = d.starts, a.table = d.table;
        a.requests = d.requests, a.rows = d.rows, a.table_stride = d.table_stride;
        a.group = group, a.window = d.window, a.scale = d.scale;
        const uint64_t bytes = piece_bytes(ctx, c, plan);
        need(d.workspace, "workspace", 16);
        if (d.workspace_bytes < bytes) refuse("needs a workspace of " + std::to_string(bytes) + " bytes");
        a.partial = static_cast<float*>(d.workspace);
        a.counters = d.pool->counters;
        a.parts = ctx->compute_units;
        const uint32_t page_tiles = c.capacity / 32;
        a.page_inverse = page_tiles > 1 ? static_cast<uint32_t>(((1ull << 32) + page_tiles - 1) / page_tiles) : 0;
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        auto run = [&](uint32_t rows, uint32_t octets) {
            a.stats = reinterpret_cast<float2*>(a.partial + piece_rows(ctx, rows) * c.head_dim);
            a.joins = reinterpret_cast<chm::PagedJoin*>(a.stats + piece_rows(ctx, rows));
            const auto s = static_cast<hipStream_t>(stream);
            return c.format == chm::kF16    ? chm::launch_paged_f16(a, octets, s)
                   : c.format == chm::kQ4_0 ? chm::launch_paged_q4_0(a, octets, s)
                                            : chm::launch_paged_q8_0(a, octets, s);
        };
        a.many_from = chm::many_from(c.head_dim), a.many_load = plan.many_load;
        a.above = 0, a.upto = 0xFFFFFFFFu;
        if (plan.many)
            if (hipError_t e = run(plan.many, 0); e != hipSuccess) return e;
        if (plan.twos) {
            a.above = plan.ones ? 16 : 0;
            if (hipError_t e = run(32, 2); e != hipSuccess || !plan.ones) return e;
        }
        a.above = 0, a.upto = plan.twos ? 16 : 0xFFFFFFFFu;
        return run(16, 1);
    });
}

charlotte_hip_matmul_status charlotte_hip_matmul_residual_norm(charlotte_hip_matmul_context* ctx,
                                                               const charlotte_hip_matmul_residual_norm_desc* desc,
                                                               uint32_t rows, void* stream) {
    return guarded(ctx, "residual norm", [&] {
        if (!desc) refuse("no descriptor");
        const charlotte_hip_matmul_residual_norm_desc& d = *desc;
        if (rows == 0) refuse("a step of no rows");
        need_grid(uint64_t{rows} * 2);  // workgroups of up to 1,024 threads
        if (d.width == 0 || d.width > 32768) refuse("width " + std::to_string(d.width));
        if (!std::isfinite(d.epsilon) || d.epsilon < 0.0f) refuse("epsilon");
        if (!std::isfinite(d.residual_scale) || !std::isfinite(d.branch_scale)) refuse("a scale not finite");
        if (!d.residual_out && !d.normed) refuse("nowhere to put the result");
        if (!d.branch && (d.branch_weight || d.gate)) refuse("a branch's weight or gate without it");
        need(d.residual, "residual", 4);
        if (d.normed) need(d.weight, "weight", 4);
        if (!aligned(d.branch, 4) || !aligned(d.branch_weight, 4) || !aligned(d.gate, 4) || !aligned(d.residual_out, 4) ||
            !aligned(d.normed, 4))
            refuse("a pointer not 4-byte aligned");
        chm::ResidualNorm a{};
        a.residual = d.residual, a.branch = d.branch, a.branch_weight = d.branch_weight, a.gate = d.gate, a.weight = d.weight;
        a.residual_out = d.residual_out, a.normed = d.normed;
        a.residual_stride = stride_of(d.residual_stride, d.width, 1, "residual stride");
        a.branch_stride = stride_of(d.branch_stride, d.width, 1, "branch stride");
        a.gate_stride = d.gate_stride ? stride_of(d.gate_stride, d.width, 1, "gate stride") : 0;
        a.residual_out_stride = stride_of(d.residual_out_stride, d.width, 1, "residual_out stride");
        a.normed_stride = stride_of(d.normed_stride, d.width, 1, "normed stride");
        if (d.residual_out && d.residual_out == d.normed) refuse("two results in one place");
        for (const float* shared : {d.branch_weight, d.weight})  // other rows read it
            if (shared && (shared == d.residual_out || shared == d.normed)) refuse("a result over a weight");
        // each with a stride of its own, whichever of them are one memory
        for (const auto& [input, stride] : {std::pair{d.residual, a.residual_stride}, std::pair{d.branch, a.branch_stride},
                                            std::pair{d.gate, a.gate_stride}}) {
            in_place(d.residual_out, a.residual_out_stride, input, stride);
            in_place(d.normed, a.normed_stride, input, stride);
        }
        a.width = d.width, a.rows = rows;
        a.epsilon = d.epsilon, a.residual_scale = d.residual_scale, a.branch_scale = d.branch_scale;
        a.fours = d.width % 4 == 0;
        for (uint64_t stride : {a.residual_stride, a.branch_stride, a.gate_stride, a.residual_out_stride, a.normed_stride})
            a.fours = a.fours && stride % 4 == 0;
        for (const float* p : {d.residual, d.branch, d.branch_weight, d.gate, d.weight, static_cast<const float*>(d.residual_out),
                               static_cast<const float*>(d.normed)})
            a.fours = a.fours && aligned(p, 16);
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_residual_norm(a, static_cast<hipStream_t>(stream));
    });
}

uint64_t charlotte_hip_matmul_sample_workspace_bytes(uint32_t rows, uint32_t vocabulary) {
    if (rows == 0 || rows > chm::kGrid || vocabulary == 0 || vocabulary > (1u << 18)) return 0;
    return chm::sample_bytes(rows, vocabulary);
}

charlotte_hip_matmul_status charlotte_hip_matmul_sample(charlotte_hip_matmul_context* ctx,
                                                        const charlotte_hip_matmul_sample_desc* desc, void* stream) {
    return guarded(ctx, "sample", [&] {
        if (!desc) refuse("no descriptor");
        const charlotte_hip_matmul_sample_desc& d = *desc;
        if (d.rows == 0) refuse("no rows");
        if (d.vocabulary == 0 || d.vocabulary > (1u << 18)) refuse("vocabulary " + std::to_string(d.vocabulary));
        need_grid(uint64_t{d.rows} * 2);  // workgroups of 1,024 threads
        if (!d.temperatures && !(d.temperature >= 0.0f)) refuse("temperature " + std::to_string(d.temperature));
        need(d.logits, "logits", 4);
        need(d.uniforms, "uniforms", 4);
        need(d.tokens, "tokens", 4);
        if (!aligned(d.chances, 4) || !aligned(d.temperatures, 4) || !aligned(d.top_ks, 4) || !aligned(d.top_ps, 4) ||
            !aligned(d.min_ps, 4))
            refuse("a pointer not 4-byte aligned");
        need(d.workspace, "workspace", 16);
        const uint64_t bytes = charlotte_hip_matmul_sample_workspace_bytes(d.rows, d.vocabulary);
        if (d.workspace_bytes < bytes) refuse("needs a workspace of " + std::to_string(bytes) + " bytes");
        chm::Sample a{};
        a.logits = d.logits, a.uniforms = d.uniforms, a.tokens = d.tokens, a.chances = d.chances;
        a.temperatures = d.temperatures, a.top_ks = d.top_ks, a.top_ps = d.top_ps, a.min_ps = d.min_ps;
        a.logit_stride = stride_of(d.logit_stride, d.vocabulary, 1, "logit stride");
        a.rows = d.rows, a.vocabulary = d.vocabulary;
        a.temperature = d.temperature, a.top_k = d.top_k, a.top_p = d.top_p, a.min_p = d.min_p;
        a.workspace = d.workspace;
        if (hipError_t e = hipSetDevice(ctx->device); e != hipSuccess) return e;
        return chm::launch_sample(a, static_cast<hipStream_t>(stream));
    });
}

}  // extern "C"
