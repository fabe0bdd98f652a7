// A token drawn from each row of logits, by temperature, top-k, top-p, min-p and
// a given uniform number, in whole numbers from the weights on:
//   w = floor(2^40 exp((l - m) / T)), tokens in the order (l falling, index rising).
//
// What is kept is a run of the first tokens whichever way it is cut, so W, its
// weight, is the least of the cuts' running sums, and every cut and the draw
// itself are one question: at which token does the running count or weight pass
// a number? It is answered without sorting, by descent: the weights and counts of
// the logits' leading bits (as keys that rise with them) summed in LDS, the part
// that holds the answer opened by its next bits; tokens of one key have one
// weight, so the place among them is a division, and the token the one of that
// rank among their indices. Sums are of whole numbers, so that atomics may add
// them in any order.
#include "requests.hpp"
#include "rows.hpp"

namespace chm {

constexpr uint32_t kDrawThreads = 1024;
constexpr uint32_t kBins = 2048;
constexpr double kWhole = 1099511627776.0;  // 2^40

// A row's settings, as its kernels use them.
struct Settings {
    double rate;       // 1 / temperature
    uint64_t top_k;    // tokens
    double top_p;      // 1: all
    uint64_t least;    // min_p's weight
    uint64_t draw;     // floor(u 2^31)
    bool greedy;
};

__device__ __forceinline__ Settings settings_of(const Sample& a, uint32_t row) {
    const float t = a.temperatures ? a.temperatures[row] : a.temperature;
    const int32_t k = a.top_ks ? a.top_ks[row] : a.top_k;
    const float p = a.top_ps ? a.top_ps[row] : a.top_p, m = a.min_ps ? a.min_ps[row] : a.min_p;
    const float u = a.uniforms[row];
    Settings s;
    s.greedy = !(t >= 1e-6f) || k == 1;
    s.rate = s.greedy ? 1.0 : 1.0 / static_cast<double>(t);
    s.top_k = k > 0 && static_cast<uint32_t>(k) < a.vocabulary ? static_cast<uint32_t>(k) : a.vocabulary;
    s.top_p = p < 1.0f ? fmax(static_cast<double>(p), 0.0) : 1.0;  // (a NaN: 1)
    s.least = static_cast<uint64_t>(ceil((m > 0.0f ? fmin(static_cast<double>(m), 1.0) : 0.0) * kWhole));
    s.draw = static_cast<uint64_t>((u > 0.0f ? fminf(u, 1.0f - 0x1p-24f) : 0.0f) * 0x1p31f);
    return s;
}

// A logit as a word that rises with it; a NaN as -inf, and one zero.
__device__ __forceinline__ float clean(float l) { return l == l ? l + 0.0f : -INFINITY; }
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t bits = __float_as_uint(l);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

__device__ __forceinline__ uint64_t weight_of(float l, float most, double rate) {
    if (l == most) return 1ull << 40;
    if (l == -INFINITY || most == INFINITY) return 0;
    return static_cast<uint64_t>(exp((static_cast<double>(l) - static_cast<double>(most)) * rate) * kWhole);
}

// The sum over the workgroup's threads before this one, and of all. `parts`: a word a wave.
__device__ __forceinline__ uint64_t sum_before(uint64_t x, uint64_t* parts, uint64_t* total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint64_t sum = x;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint64_t other = __shfl_up(sum, o);
        if (lane >= o) sum += other;
    }
    __syncthreads();  // `parts` of the sum before this one has been read
    if (lane == 63) parts[wave] = sum;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kDrawThreads / 64; ++w) {
        if (w < wave) before += parts[w];
        all += parts[w];
    }
    *total = all;
    return before + sum - x;
}

// A row as its workgroup goes over it.
struct DrawRow {
    const float* x;
    uint32_t lead, vocabulary;
    float most;
    double rate;

    // f(logit, index) for each of the row's tokens.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        for (uint32_t at = 4 * threadIdx.x; at < lead + vocabulary; at += 4 * kDrawThreads) {
            const float4 q = read4(x, lead, vocabulary, at, -INFINITY);
            const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (at + e >= lead && at + e < lead + vocabulary) f(clean(v[e]), at + e - lead);
        }
    }
};

struct Descent {
    uint64_t weights[kBins];
    uint32_t counts[kBins];
    uint64_t parts[kDrawThreads / 64];
    uint32_t found;
    uint64_t before_weight, before_count;
};

// Where the running count (COUNT) or weight of the row passes `target`.
struct Place {
    uint32_t key;
    uint64_t before;  // the weight of the tokens of larger keys
    uint64_t rank;    // among the tokens of its key
    uint64_t weight;  // of each
};

template <bool COUNT>
__device__ Place descend(const DrawRow& row, uint64_t target, Descent& d) {
    uint32_t prefix = 0;  // the key's bits so far
    uint64_t before_weight = 0, before_count = 0;
    const int shifts[3] = {21, 10, 0};
    for (int level = 0; level < 3; ++level) {
        const int shift = shifts[level], above = level == 0 ? 32 : shifts[level - 1];
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < kBins; i += kDrawThreads) d.weights[i] = 0, d.counts[i] = 0;
        __syncthreads();
        row.each([&](float l, uint32_t) {
            const uint32_t key = key_of(l);
            if (level > 0 && key >> above != prefix) return;
            const uint32_t bin = key >> shift & (kBins - 1) & ((1u << (above - shift)) - 1);
            const uint64_t w = weight_of(l, row.most, row.rate);
            if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&d.weights[bin]), static_cast<unsigned long long>(w));
            if (COUNT) atomicAdd(&d.counts[bin], 1u);
        });
        __syncthreads();
        // bins from the largest down, two a thread
        const uint32_t first = kBins - 1 - 2 * threadIdx.x;
        const uint64_t w0 = d.weights[first], w1 = d.weights[first - 1];
        const uint64_t c0 = d.counts[first], c1 = d.counts[first - 1];
        uint64_t all;
        const uint64_t w = before_weight + sum_before(w0 + w1, d.parts, &all);
        const uint64_t c = COUNT ? before_count + sum_before(c0 + c1, d.parts, &all) : 0;
        const uint64_t from = COUNT ? c : w, middle = from + (COUNT ? c0 : w0), to = middle + (COUNT ? c1 : w1);
        if (from <= target && target < to) {  // one thread's
            const bool second = target >= middle;
            d.found = first - (second ? 1 : 0);
            d.before_weight = w + (second ? w0 : 0);
            d.before_count = c + (second ? c0 : 0);
        }
        __syncthreads();
        prefix = level == 0 ? d.found : prefix << (shifts[level - 1] - shift) | d.found;
        before_weight = d.before_weight, before_count = d.before_count;
    }
    Place p;
    p.key = prefix;
    p.before = before_weight;
    p.weight = weight_of(logit_of(prefix), row.most, row.rate);
    p.rank = COUNT ? target - before_count : (target - before_weight) / p.weight;
    return p;
}

// The index of the token of rank `rank` among those of a key.
__device__ uint32_t index_of(const DrawRow& row, uint32_t key, uint64_t rank, Descent& d) {
    const uint32_t share = (row.vocabulary + kDrawThreads - 1) / kDrawThreads;
    __syncthreads();
    d.counts[threadIdx.x] = 0;
    __syncthreads();
    row.each([&](float l, uint32_t i) {
        if (key_of(l) == key) atomicAdd(&d.counts[i / share], 1u);
    });
    __syncthreads();
    uint64_t all;
    const uint64_t mine = d.counts[threadIdx.x], before = sum_before(mine, d.parts, &all);
    if (before <= rank && rank < before + mine) {
        uint64_t left = rank - before;
        for (uint32_t i = threadIdx.x * share;; ++i)
            if (key_of(clean(row.x[i])) == key && left-- == 0) {
                d.found = i;
                break;
            }
    }
    __syncthreads();
    return d.found;
}

__global__ __launch_bounds__(kDrawThreads) void draw_rows(Sample a) {
    __shared__ Descent d;
    __shared__ uint32_t wave_key[kDrawThreads / 64], wave_at[kDrawThreads / 64];
    const uint32_t r = blockIdx.x, lane = threadIdx.x & 63u;
    const Settings s = settings_of(a, r);
    DrawRow row{a.logits + r * a.logit_stride, 0, a.vocabulary, 0.0f, s.rate};
    row.lead = lead_of(row.x);

    // The largest and the first of it.
    uint32_t key = 0, at = 0xFFFFFFFFu;
    row.each([&](float l, uint32_t i) {
        const uint32_t k = key_of(l);
        if (k > key) key = k, at = i;
    });
    auto join = [&](uint32_t k, uint32_t i) {
        if (k > key || (k == key && i < at)) key = k, at = i;
    };
#pragma unroll
    for (uint32_t o = 32; o > 0; o >>= 1) join(__shfl_xor(key, o), __shfl_xor(at, o));
    if (lane == 0) wave_key[threadIdx.x >> 6] = key, wave_at[threadIdx.x >> 6] = at;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kDrawThreads / 64; ++w) join(wave_key[w], wave_at[w]);
    row.most = logit_of(key);

    int32_t token = static_cast<int32_t>(at);
    float chance = 1.0f;
    if (row.most == -INFINITY) {
        token = -1, chance = 0.0f;
    } else if (!s.greedy) {
        // All weights, and those that min_p leaves.
        uint64_t all = 0, some = 0;
        row.each([&](float l, uint32_t) {
            const uint64_t w = weight_of(l, row.most, row.rate);
            all += w;
            if (w >= s.least) some += w;
        });
        uint64_t kept, likely;
        sum_before(all, d.parts, &kept);
        sum_before(some, d.parts, &likely);
        if (s.top_k < a.vocabulary) {
            const Place p = descend<true>(row, s.top_k - 1, d);
            kept = p.before + (p.rank + 1) * p.weight;
        }
        if (s.top_p < 1.0) {
            const uint64_t least = static_cast<uint64_t>(ceil(s.top_p * static_cast<double>(kept)));
            const Place p = descend<false>(row, least > 0 ? min(least, kept) - 1 : 0, d);
            kept = p.before + (p.rank + 1) * p.weight;
        }
        kept = min(kept, max(likely, 1ull << 40));
        // floor(kept draw / 2^31): kept is below 2^59
        const uint64_t target = (kept >> 31) * s.draw + ((kept & 0x7FFFFFFFull) * s.draw >> 31);
        const Place p = descend<false>(row, target, d);
        token = static_cast<int32_t>(index_of(row, p.key, p.rank, d));
        chance = static_cast<float>(static_cast<double>(p.weight) / static_cast<double>(kept));
    }
    if (threadIdx.x == 0) {
        a.tokens[r] = token;
        if (a.chances) a.chances[r] = chance;
    }
}

uint64_t sample_bytes(uint32_t rows, uint32_t) { return uint64_t{rows} * 16; }

hipError_t launch_sample(const Sample& a, hipStream_t stream) {
    hipLaunchKernelGGL(draw_rows, dim3(a.rows), dim3(kDrawThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace chm
