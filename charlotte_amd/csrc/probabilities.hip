// Softmax of the head's logits at a temperature: p = exp((x - m) / T) / sum. At
// temperature 0 the largest's first index stands in the sum's place.
//
// Rows that a workgroup's registers hold: one launch, a workgroup a row.
//
// Few longer rows: two passes over chunks of the rows, as many as fill the card: each
// chunk's maximum and sum in one read (the sum kept relative to the running
// maximum), then, from all of a row's chunks, its probabilities; the second
// read comes from cache.
//
// Rows past what the caches hold (kWholeBytes), read once: a workgroup keeps
// its chunk in registers, publishes its maximum and sum, waits for those of the
// row's other chunks, and writes its probabilities. The wait is bounded: a
// workgroup that has not seen them all by then reads the row itself and adds it
// in the same order, so that none depends on when another runs. (That needs the logits as they were, so a
// step in place takes the two passes.)
//
// Bound by bytes: 4 read and 4 written a logit. 168 x 262,144: 69.5 us (5.1 TB/s;
// two passes 94), 1,024 x 131,072: 188 us (5.7 TB/s; 324); 6 x 151,936: passes of
// 4.0 and 4.8 us, a launch's latency each.
#include <algorithm>

#include "rows.hpp"
#include "serving.hpp"

namespace chm {

constexpr float kPerOctave = 1.44269504088896340736f;  // log2(e)
constexpr uint32_t kNowhere = 0xFFFFFFFFu;

__device__ __forceinline__ RowStats join_stats(const RowStats& a, const RowStats& b, float rate) {
    RowStats r;
    r.largest = fmaxf(a.largest, b.largest);
    // sums relative to the larger maximum; a side without one has the sum 0, or a NaN
    const float fa = a.largest == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((a.largest - r.largest) * rate);
    const float fb = b.largest == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((b.largest - r.largest) * rate);
    r.sum = a.sum * fa + b.sum * fb;
    r.at = a.largest > b.largest ? a.at : b.largest > a.largest ? b.at : min(a.at, b.at);
    return r;
}

__device__ __forceinline__ RowStats shuffled(const RowStats& s, int o) {
    return {__shfl_xor(s.largest, o), __shfl_xor(s.sum, o), static_cast<uint32_t>(__shfl_xor(static_cast<int>(s.at), o))};
}

// A chunk: `share` entries from the row's boundary (rows.hpp), a multiple of 4.
__device__ __forceinline__ uint32_t share_of(const Probabilities& a) {
    return ((a.vocabulary + 3 + a.chunks - 1) / a.chunks + 3) / 4 * 4;
}

// A thread's part of a row's statistics: fours from `at` to `end`, `step` apart.
__device__ __forceinline__ RowStats running_stats(const float* x, uint32_t lead, uint32_t vocabulary, uint32_t at, uint32_t end,
                                                  uint32_t step, float rate) {
    RowStats s = {-INFINITY, 0.0f, kNowhere};
    for (; at < end; at += step) {
        const float4 q = read4(x, lead, vocabulary, at, -INFINITY);
        const float v[4] = {q.x, q.y, q.z, q.w};
        const float top = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        if (top > s.largest) {
            s.sum *= s.largest == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((s.largest - top) * rate);
            s.largest = top;
            s.at = at - lead + (v[0] == top ? 0 : v[1] == top ? 1 : v[2] == top ? 2 : 3);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            s.sum += v[e] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((v[e] - s.largest) * rate);
    }
    return s;
}

__global__ __launch_bounds__(256) void row_stats(Probabilities a) {
    __shared__ RowStats parts[4];
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const float* x = a.logits + row * a.logit_stride;
    const uint32_t lead = lead_of(x), share = share_of(a);
    const float rate = a.temperature > 0.0f ? kPerOctave / a.temperature : 0.0f;
    RowStats s = running_stats(x, lead, a.vocabulary, chunk * share + 4 * threadIdx.x,
                               min((chunk + 1) * share, lead + a.vocabulary), 1024, rate);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s = join_stats(s, shuffled(s, o), rate);
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        a.stats[blockIdx.x] = join_stats(join_stats(parts[0], parts[1], rate), join_stats(parts[2], parts[3], rate), rate);
}

__global__ __launch_bounds__(256) void row_probabilities(Probabilities a) {
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const float* x = a.logits + row * a.logit_stride;
    float* y = a.output + row * a.output_stride;
    const uint32_t lead = lead_of(x), share = share_of(a);
    const float rate = a.temperature > 0.0f ? kPerOctave / a.temperature : 0.0f;
    // every wave joins the row's chunks, in one order
    RowStats s = {-INFINITY, 0.0f, kNowhere};
    for (uint32_t c = threadIdx.x & 63u; c < a.chunks; c += 64)
        s = join_stats(s, a.stats[static_cast<uint64_t>(row) * a.chunks + c], rate);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s = join_stats(s, shuffled(s, o), rate);
    // nothing but -inf: zeros, where 1 / 0 would make NaNs
    const float inverse = s.sum == 0.0f ? 0.0f : 1.0f / s.sum;
    const float largest = s.largest == -INFINITY ? 0.0f : s.largest;
    const uint32_t end = min((chunk + 1) * share, lead + a.vocabulary);
    for (uint32_t at = chunk * share + 4 * threadIdx.x; at < end; at += 1024) {
        float4 v;
        if (a.temperature > 0.0f) {
            const float4 q = read4(x, lead, a.vocabulary, at, -INFINITY);
            v = {__builtin_amdgcn_exp2f((q.x - largest) * rate) * inverse, __builtin_amdgcn_exp2f((q.y - largest) * rate) * inverse,
                 __builtin_amdgcn_exp2f((q.z - largest) * rate) * inverse, __builtin_amdgcn_exp2f((q.w - largest) * rate) * inverse};
        } else {
            const uint32_t hit = s.at == kNowhere ? kNowhere : s.at + lead - at;
            v = {hit == 0 ? 1.0f : 0.0f, hit == 1 ? 1.0f : 0.0f, hit == 2 ? 1.0f : 0.0f, hit == 3 ? 1.0f : 0.0f};
        }
        write4(y, lead, a.vocabulary, at, v);
    }
}

// ---- whole rows in one read ---------------------------------------------------------

constexpr uint32_t kWholeThreads = 512, kWholeFours = 8, kWholeChunk = 4 * kWholeThreads * kWholeFours;
// Logits past which rows are read once, their second read no longer all from
// cache: of 151,936, 12 rows (7 MB) 10.6 us read once and 10.1 in two passes, 32
// (19 MB) 14.9 and 14.0, 42 (26 MB) 15.7 and 16.9, 64 (39 MB) 18.9 and 23.5, 100 (61
// MB) 27.2 and 33.5; of 262,144, 21 rows (22 MB) 15.4 and 15.6.
constexpr uint64_t kWholeBytes = 22ull << 20;
// Logits past which, with as many probabilities, they leave the caches anyway and
// are read without being kept there: 102 MB 42.4 us either way, 176 MB 69.5 and,
// kept, 75.9, 537 MB 188 and 191 (176 MB with the logits written before and their
// verification after: 171 and 183); of 51 MB, which an earlier launch may have left there, 27.8 and 24.0.
// (Probabilities written past the caches would cost their reader more.)
constexpr uint64_t kOnceBytes = 128ull << 20;
// Rows from which a row of one to two chunks is one workgroup's, in one launch:
// of 32,000, 6 rows 8.0 us so and 7.1 in two passes (one compute unit reads 128
// KB in 4), 48 rows 8.7 and 8.8, 168 rows 11.0 and 14.6, 1,000 rows 39.8 and 46.7.
// Rows of at most a chunk always are: 1 x 4,096 4.8 and 6.6, 6 x 16,000 5.4 and
// 7.0, 168 x 16,000 6.6 and 11.2, 4,000 x 16,000 97.5 and 100.7.
constexpr uint32_t kAloneRows = 48;

// What a chunk publishes, in one word that is never 0: the sum is at least 1
// where the maximum is a number, and 0 only beside -inf; the index is raised by 1.
__device__ __forceinline__ uint64_t published(const RowStats& s, bool at) {
    return static_cast<uint64_t>(__float_as_uint(s.largest)) << 32 | (at ? s.at + 1 : __float_as_uint(s.sum));
}

// The workgroup's statistics from its threads', in every thread.
__device__ __forceinline__ RowStats joined(RowStats s, float rate, RowStats* parts) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s = join_stats(s, shuffled(s, o), rate);
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = s;
    __syncthreads();
    s = parts[threadIdx.x % (kWholeThreads / 64)];
#pragma unroll
    for (int o = kWholeThreads / 128; o > 0; o >>= 1) s = join_stats(s, shuffled(s, o), rate);
    return s;
}

// A chunk's fours from `at0` on, in registers, and the thread's part of its statistics.
template <bool ONCE, uint32_t FOURS>
__device__ __forceinline__ RowStats chunk_stats(const float* x, uint32_t lead, uint32_t vocabulary, uint32_t at0, float rate,
                                                float4 (&q)[FOURS]) {
#pragma unroll
    for (uint32_t i = 0; i < FOURS; ++i) q[i] = read4<ONCE>(x, lead, vocabulary, at0 + 4 * kWholeThreads * i, -INFINITY);
    RowStats s = {-INFINITY, 0.0f, kNowhere};
#pragma unroll
    for (uint32_t i = 0; i < FOURS; ++i) s.largest = fmaxf(s.largest, fmaxf(fmaxf(q[i].x, q[i].y), fmaxf(q[i].z, q[i].w)));
#pragma unroll
    for (uint32_t i = 0; i < FOURS; ++i) {
        const float v[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            s.sum += v[e] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((v[e] - s.largest) * rate);
            if (v[e] == s.largest && v[e] != -INFINITY) s.at = min(s.at, at0 + 4 * kWholeThreads * i + e - lead);
        }
    }
    return s;
}

// The chunk's probabilities, by its row's statistics.
template <uint32_t FOURS>
__device__ __forceinline__ void write_chunk(const Probabilities& a, float* y, uint32_t lead, uint32_t at0, const RowStats& s,
                                            float rate, const float4 (&q)[FOURS]) {
    const float inverse = s.sum == 0.0f ? 0.0f : 1.0f / s.sum;
    const float largest = s.largest == -INFINITY ? 0.0f : s.largest;
#pragma unroll
    for (uint32_t i = 0; i < FOURS; ++i) {
        const uint32_t to = at0 + 4 * kWholeThreads * i;
        if (to >= lead + a.vocabulary) break;
        float4 p;
        if (a.temperature == 0.0f) {
            const uint32_t hit = s.at == kNowhere ? kNowhere : s.at + lead - to;
            p = {hit == 0 ? 1.0f : 0.0f, hit == 1 ? 1.0f : 0.0f, hit == 2 ? 1.0f : 0.0f, hit == 3 ? 1.0f : 0.0f};
        } else {
            p = {__builtin_amdgcn_exp2f((q[i].x - largest) * rate) * inverse, __builtin_amdgcn_exp2f((q[i].y - largest) * rate) * inverse,
                 __builtin_amdgcn_exp2f((q[i].z - largest) * rate) * inverse, __builtin_amdgcn_exp2f((q[i].w - largest) * rate) * inverse};
        }
        write4(y, lead, a.vocabulary, to, p);
    }
}

// A row by one workgroup, in one launch: FOURS fours of logits a thread.
template <uint32_t FOURS>
__global__ __launch_bounds__(kWholeThreads) void row_alone(Probabilities a) {
    __shared__ RowStats parts[kWholeThreads / 64];
    const float* x = a.logits + blockIdx.x * a.logit_stride;
    const uint32_t lead = lead_of(x), at0 = 4 * threadIdx.x;
    const float rate = a.temperature > 0.0f ? kPerOctave / a.temperature : 0.0f;
    float4 q[FOURS];
    // every thread's reads are before the barrier in `joined`: the output may be the logits
    const RowStats s = joined(chunk_stats<false>(x, lead, a.vocabulary, at0, rate, q), rate, parts);
    write_chunk(a, a.output + blockIdx.x * a.output_stride, lead, at0, s, rate, q);
}

__global__ __launch_bounds__(256) void clear_words(uint64_t* words, uint32_t count) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i < count) words[i] = 0;
}

template <bool ONCE>
__global__ __launch_bounds__(kWholeThreads) void row_whole(Probabilities a) {
    __shared__ RowStats parts[kWholeThreads / 64];
    __shared__ RowStats whole;
    __shared__ uint32_t late;
    const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
    const float* x = a.logits + row * a.logit_stride;
    float* y = a.output + row * a.output_stride;
    const uint32_t lead = lead_of(x), at0 = chunk * kWholeChunk + 4 * threadIdx.x;
    const bool at = a.temperature == 0.0f;
    const float rate = at ? 0.0f : kPerOctave / a.temperature;
    uint64_t* words = reinterpret_cast<uint64_t*>(a.stats) + static_cast<uint64_t>(row) * a.chunks;

    float4 q[kWholeFours];
    RowStats s = joined(chunk_stats<ONCE>(x, lead, a.vocabulary, at0, rate, q), rate, parts);
    if (threadIdx.x == 0)
        __hip_atomic_store(words + chunk, published(s, at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // the first wave: the row's statistics from its chunks' words, a lane a chunk
    uint64_t word = 1;
    auto join_words = [&] {
        RowStats r = {-INFINITY, 0.0f, kNowhere};
        if (threadIdx.x < a.chunks) {
            r.largest = __uint_as_float(static_cast<uint32_t>(word >> 32));
            if (at)
                r.at = static_cast<uint32_t>(word) - 1;
            else
                r.sum = __uint_as_float(static_cast<uint32_t>(word));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) r = join_stats(r, shuffled(r, o), rate);
        if (threadIdx.x == 0) whole = r;
    };
    if (threadIdx.x < 64) {
        // it looks until none is 0
        bool all = false;
        for (uint32_t look = 0; look < a.looks && !all; ++look) {
            if (threadIdx.x < a.chunks) word = __hip_atomic_load(words + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            all = __all(word != 0);
            if (!all) __builtin_amdgcn_s_sleep(8);
        }
        join_words();
        if (threadIdx.x == 0) late = !all;
    }
    __syncthreads();
    if (late) {
        // every chunk's word by this workgroup alone, as its own would publish it: the
        // same bits; then its own logits again
#pragma unroll 1
        for (uint32_t c = 0; c < a.chunks; ++c) {
            s = joined(chunk_stats<ONCE>(x, lead, a.vocabulary, c * kWholeChunk + 4 * threadIdx.x, rate, q), rate, parts);
            if (threadIdx.x == c) word = published(s, at);
            __syncthreads();  // `parts` has been read
        }
        if (threadIdx.x < 64) join_words();
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kWholeFours; ++i)
            q[i] = read4<ONCE>(x, lead, a.vocabulary, at0 + 4 * kWholeThreads * i, -INFINITY);
    }
    s = whole;
    write_chunk(a, y, lead, at0, s, rate, q);
}

// Chunks of the two passes: about a thousand workgroups, a chunk of at least 2,048 logits.
static uint32_t pass_chunks(uint32_t rows, uint32_t vocabulary) {
    return std::max(1u, std::min((1024 + rows - 1) / rows, (vocabulary + 2047) / 2048));
}
// Of a row read once (a lane a chunk); 0 where it is not.
static uint32_t whole_chunks(uint32_t rows, uint32_t vocabulary) {
    const uint32_t chunks = (vocabulary + 3 + kWholeChunk - 1) / kWholeChunk;
    return uint64_t{rows} * vocabulary * 4 > kWholeBytes && chunks <= 64 ? chunks : 0;
}

uint64_t probabilities_bytes(uint32_t rows, uint32_t vocabulary) {
    return rows * std::max<uint64_t>(pass_chunks(rows, vocabulary) * sizeof(RowStats), whole_chunks(rows, vocabulary) * 8ull);
}

hipError_t launch_probabilities(Probabilities a, hipStream_t stream) {
    if (a.vocabulary + 3 <= kWholeChunk) {
        hipLaunchKernelGGL(row_alone<kWholeFours>, dim3(a.rows), dim3(kWholeThreads), 0, stream, a);
        return hipGetLastError();
    }
    if (a.vocabulary + 3 <= 2 * kWholeChunk && a.rows >= kAloneRows) {
        hipLaunchKernelGGL(row_alone<2 * kWholeFours>, dim3(a.rows), dim3(kWholeThreads), 0, stream, a);
        return hipGetLastError();
    }
    a.chunks = whole_chunks(a.rows, a.vocabulary);
    if (a.chunks && a.logits != a.output) {
        const uint32_t words = a.rows * a.chunks;
        hipLaunchKernelGGL(clear_words, dim3((words + 255) / 256), dim3(256), 0, stream, reinterpret_cast<uint64_t*>(a.stats), words);
        if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        if (uint64_t{a.rows} * a.vocabulary * 4 > kOnceBytes)
            hipLaunchKernelGGL(row_whole<true>, dim3(words), dim3(kWholeThreads), 0, stream, a);
        else
            hipLaunchKernelGGL(row_whole<false>, dim3(words), dim3(kWholeThreads), 0, stream, a);
        return hipGetLastError();
    }
    a.chunks = pass_chunks(a.rows, a.vocabulary);
    const dim3 grid(a.rows * a.chunks);
    hipLaunchKernelGGL(row_stats, grid, dim3(256), 0, stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    hipLaunchKernelGGL(row_probabilities, grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace chm
