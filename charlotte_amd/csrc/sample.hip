// A token drawn from each row of logits, by temperature, top-k, top-p, min-p and
// a given uniform number, in whole numbers from the weights on:
//   w = floor(2^40 exp((l - m) / T)), tokens in the order (l falling, index rising).
//
// What is kept is a run of the first tokens whichever way it is cut, so W, its
// weight, is the least of the cuts' running sums, and every cut and the draw
// itself are one question: at which token does the running count or weight pass
// a number? It is answered without sorting the row, in three launches over chunks
// of the rows:
//   row_largest   each chunk's largest logit, and its smallest;
//   row_bins      counts and weights of kBins equal steps of m - l, down to where a
//                 weight is 0 or the logits end. The workgroup that ends a row last finds
//                 the bins that the cuts and the draw may fall into: a cut's bins bound
//                 what is kept, that the next one's;
//   row_draw      the tokens in those bins, some hundreds, gathered. The last workgroup
//                 of a row sorts them by finer bins, and answers.
// Where those bins hold more than kList tokens (many equal logits) or the logits'
// distances pass f32, one workgroup answers by descent:
// weights and counts of the logits' leading bits (as keys that rise with them)
// summed in LDS, the part that holds the answer opened by its next bits; tokens of
// one key have one weight, so the place among them is a division.
// Sums are of whole numbers, so that atomics may add them in any order.
//
// What a row's workgroups leave for the last of them goes past the caches that
// they do not share, by atomics and by loads and stores of the device's scope:
// each workgroup waits for its own to arrive, then counts itself; no cache is
// written back or cleared for it.
//
// Bound by the weights' f64 and by what ends a row: 1 x 151,936 logits 22 - 24 us (3.4 + 9.8
// + 9.3); 64 x 128,256, settings a row, 50 (8.2, read at 4.0 TB/s, + 26.0 + 17.7); 24 x
// 262,144 by temperature alone 51. Of row_bins' 26.0 the logits and their bins are 8.0, the
// weights 9.1 (21 of 50 instructions a logit are f64's: 4.4 at its full rate), adds to LDS 0.8,
// to memory 3.0, the search by a row's last workgroup 5.0; of the one row's 9.8 they are 4.0,
// 0.5, 0.1, 1.6 and 3.4. Weights of f32's exponential in the bins, with bounds, and whole
// ones summed in row_draw took as long where few tokens lay within the bounds, and 200 -
// 600 us where a draw near the end of a flat row had thousands. A flat row whose range a mask
// of large finite values makes useless has hundreds of tokens a bin: past kList in those that
// matter it is one workgroup's, as where many logits are equal.
#include <algorithm>
#include <cstddef>

#include "requests.hpp"
#include "rows.hpp"

namespace chm {

constexpr uint32_t kDrawThreads = 512;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kList = 2048;  // tokens gathered of a row
// (m - l) / T from which a weight is 0, and more than rounding's worth past it: 40 ln 2 is 27.73.
constexpr float kReach = 27.8f;
constexpr double kWhole = 1099511627776.0;  // 2^40

// log2(e) / temperature, in two parts.
struct Octaves {
    double high, low;
};
// A row's settings, as its kernels use them.
struct Settings {
    double rate;       // 1 / temperature
    Octaves octaves;
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
    const double heat = s.greedy ? 1.0 : static_cast<double>(t);
    s.rate = 1.0 / heat;
    constexpr double kLog2E = 1.44269504088896340736, kLog2ELow = 2.0355273740931033e-17;
    s.octaves.high = s.rate * kLog2E;
    s.octaves.low = s.rate > 0.0 ? (__builtin_fma(-s.octaves.high, heat, kLog2E) + kLog2ELow) * s.rate : 0.0;
    s.top_k = k > 0 && static_cast<uint32_t>(k) < a.vocabulary ? static_cast<uint32_t>(k) : a.vocabulary;
    s.top_p = p < 1.0f ? fmax(static_cast<double>(p), 0.0) : 1.0;  // (a NaN: 1)
    s.least = static_cast<uint64_t>(ceil((m > 0.0f ? fmin(static_cast<double>(m), 1.0) : 0.0) * kWhole));
    s.draw = static_cast<uint64_t>((u > 0.0f ? fminf(u, 1.0f - 0x1p-24f) : 0.0f) * 0x1p31f);
    return s;
}

// A logit that is a NaN counts as -inf.
__device__ __forceinline__ float clean(float l) { return fmaxf(l, -INFINITY); }
// A logit as a word that rises with it; both zeros as one.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t bits = __float_as_uint(l + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// floor(2^40 exp((l - m) / T)), l not so far below a finite m that the power has no
// exponent: (l - m) log2(e) / T in two parts, whose nearest whole number is taken off
// before it is rounded, and 2^z of what is left by the polynomial of degree 11 whose
// largest relative error there is least (Remez's exchange; 2^-54.7 with its terms in f64).
// In all within 1.25 units of f64's last place; a whole number that f64 holds.
__device__ __forceinline__ double whole_weight(float l, double most, const Octaves& octaves) {
    const double d = static_cast<double>(l) - most, whole = rint(d * octaves.high);
    const double z = __builtin_fma(d, octaves.low, __builtin_fma(d, octaves.high, -whole));
    double p = 4.4352819196017726e-10;
    p = __builtin_fma(p, z, 7.074105632845698e-09);
    p = __builtin_fma(p, z, 1.0178198028606432e-07);
    p = __builtin_fma(p, z, 1.3215433089687149e-06);
    p = __builtin_fma(p, z, 1.525273348996672e-05);
    p = __builtin_fma(p, z, 0.0001540353046251404);
    p = __builtin_fma(p, z, 0.001333355814678995);
    p = __builtin_fma(p, z, 0.009618129107588335);
    p = __builtin_fma(p, z, 0.055504108664819925);
    p = __builtin_fma(p, z, 0.24022650695910155);
    p = __builtin_fma(p, z, 0.6931471805599453);
    p = __builtin_fma(p, z, 1.0);
    return floor(ldexp(p, static_cast<int>(whole) + 40));
}

__device__ __forceinline__ uint64_t weight_of(float l, float most, const Octaves& octaves) {
    if (l == most) return 1ull << 40;
    if (l == -INFINITY || most == INFINITY) return 0;
    if ((static_cast<double>(l) - most) * octaves.high < -64.0) return 0;
    return static_cast<uint64_t>(whole_weight(l, most, octaves));
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
    Octaves octaves;

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
            const uint64_t w = weight_of(l, row.most, row.octaves);
            if (w) atomicAdd(reinterpret_cast<unsigned long long*>(&d.weights[bin]), static_cast<unsigned long long>(w));
            if (COUNT) atomicAdd(&d.counts[bin], 1u);
        });
        __syncthreads();
        // bins from the largest down, some a thread
        constexpr uint32_t kMine = kBins / kDrawThreads;
        const uint32_t first = kBins - 1 - kMine * threadIdx.x;
        uint64_t weight = 0, count = 0, all;
        for (uint32_t i = 0; i < kMine; ++i) weight += d.weights[first - i], count += d.counts[first - i];
        weight = before_weight + sum_before(weight, d.parts, &all);
        count = COUNT ? before_count + sum_before(count, d.parts, &all) : 0;
        for (uint32_t i = 0; i < kMine; ++i) {
            const uint64_t w = d.weights[first - i], c = d.counts[first - i], from = COUNT ? count : weight;
            if (from <= target && target < from + (COUNT ? c : w)) {  // one thread's
                d.found = first - i;
                d.before_weight = weight, d.before_count = count;
            }
            weight += w, count += c;
        }
        __syncthreads();
        prefix = level == 0 ? d.found : prefix << (shifts[level - 1] - shift) | d.found;
        before_weight = d.before_weight, before_count = d.before_count;
    }
    Place p;
    p.key = prefix;
    p.before = before_weight;
    p.weight = weight_of(logit_of(prefix), row.most, row.octaves);
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

// What the running weight passes with the last token that top_p keeps of `kept`.
__device__ __forceinline__ uint64_t passed_by(const Settings& s, uint64_t kept) {
    const uint64_t least = static_cast<uint64_t>(ceil(s.top_p * static_cast<double>(kept)));
    return least > 0 ? min(least, kept) - 1 : 0;
}
// What it passes with the token drawn: floor(kept draw / 2^31), kept below 2^59.
__device__ __forceinline__ uint64_t drawn_at(const Settings& s, uint64_t kept) {
    return (kept >> 31) * s.draw + ((kept & 0x7FFFFFFFull) * s.draw >> 31);
}

__device__ __forceinline__ void write_draw(const Sample& a, uint32_t row, uint32_t token, uint64_t weight, uint64_t kept) {
    a.tokens[row] = static_cast<int32_t>(token);
    if (a.chances) a.chances[row] = static_cast<float>(static_cast<double>(weight) / static_cast<double>(kept));
}

// A row by one workgroup, by descent.
__device__ void draw_alone(const Sample& a, uint32_t r, const Settings& s, float most, Descent& d) {
    DrawRow row{a.logits + r * a.logit_stride, 0, a.vocabulary, most, s.octaves};
    row.lead = lead_of(row.x);
    // All weights, and those that min_p leaves.
    uint64_t all = 0, some = 0;
    row.each([&](float l, uint32_t) {
        const uint64_t w = weight_of(l, row.most, row.octaves);
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
        const Place p = descend<false>(row, passed_by(s, kept), d);
        kept = p.before + (p.rank + 1) * p.weight;
    }
    kept = min(kept, max(likely, 1ull << 40));
    const Place p = descend<false>(row, drawn_at(s, kept), d);
    const uint32_t token = index_of(row, p.key, p.rank, d);
    if (threadIdx.x == 0) write_draw(a, r, token, p.weight, kept);
}

// ---- by bins -----------------------------------------------------------------

// What a row's workgroups share, at the device's scope.
template <typename T>
__device__ __forceinline__ T get(const T& x) {
    return __hip_atomic_load(&x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ void put(T& x, T value) {
    __hip_atomic_store(&x, value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ T add(T& x, T value) {
    return __hip_atomic_fetch_add(&x, value, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Bins whose tokens are gathered: `first` .. `last`, of `count` tokens, those before
// them `before` and their weight `ahead`; the first token's place in the list.
struct Run {
    uint32_t first, last, count, before, start, reserved;
    uint64_t ahead;
};
constexpr uint32_t kRuns = 3;
// A row's part of the workspace.
struct DrawRoom {
    uint64_t weights[kBins];     // the bins' weights
    uint64_t counts[kBins / 2];  // and tokens, two bins' in a word
    uint64_t likely;             // weight that min_p leaves of the bins of its end
    uint32_t binned, gathered;   // workgroups of row_bins, of row_draw, that have ended
    uint32_t listed;             // tokens gathered
    uint32_t runs, alone;        // runs; or by descent
    uint32_t cut;                // top_k's last token is in a run
    uint32_t end_first, end_past;  // the bins that min_p's end may be in
    uint64_t all, end_ahead;     // weight of all tokens; of those before these bins
    Run run[kRuns];
    uint64_t list[kList];        // key, and the index's complement: the first token is the largest
};
constexpr uint32_t kCleared = offsetof(DrawRoom, list) / 8;
static_assert(offsetof(DrawRoom, list) % 8 == 0, "words of 8 bytes");
struct DrawChunks {
    DrawRoom* rooms;
    uint64_t* largest;  // [rows][chunks]: key, and the index's complement
    float* smallest;    // [rows][chunks], of what is finite
    uint32_t chunks, share;
};

// f(logit, index) for each token of a workgroup's chunk; in the fours at the row's
// ends also for what is no token, at -inf.
template <typename F>
__device__ __forceinline__ void each_of_chunk(const Sample& a, const DrawChunks& c, uint32_t row, uint32_t chunk, F f) {
    const float* x = a.logits + row * a.logit_stride;
    const uint32_t lead = lead_of(x), end = min((chunk + 1) * c.share, lead + a.vocabulary);
#pragma unroll 2
    for (uint32_t at = chunk * c.share + 4 * threadIdx.x; at < end; at += 4 * kDrawThreads) {
        const float4 q = read4(x, lead, a.vocabulary, at, -INFINITY);
        f(clean(q.x), at - lead), f(clean(q.y), at + 1 - lead), f(clean(q.z), at + 2 - lead), f(clean(q.w), at + 3 - lead);
    }
}

__device__ __forceinline__ uint64_t most_of_wave(uint64_t x) {
#pragma unroll
    for (uint32_t o = 32; o > 0; o >>= 1) x = max(x, static_cast<uint64_t>(__shfl_xor(x, o)));
    return x;
}
__device__ __forceinline__ float least_of_wave(float x) {
#pragma unroll
    for (uint32_t o = 32; o > 0; o >>= 1) x = fminf(x, __shfl_xor(x, o));
    return x;
}

__global__ __launch_bounds__(kDrawThreads) void row_largest(Sample a, DrawChunks c) {
    __shared__ uint64_t parts[kDrawThreads / 64];
    __shared__ float least_parts[kDrawThreads / 64];
    const uint32_t row = blockIdx.x / c.chunks, chunk = blockIdx.x % c.chunks;
    uint64_t* room = reinterpret_cast<uint64_t*>(c.rooms + row);
    for (uint32_t i = chunk * kDrawThreads + threadIdx.x; i < kCleared; i += c.chunks * kDrawThreads) room[i] = 0;
    uint64_t most = 0;
    float least = INFINITY;
    each_of_chunk(a, c, row, chunk, [&](float l, uint32_t i) {
        most = max(most, uint64_t{key_of(l)} << 32 | ~i);
        least = fminf(least, l == -INFINITY ? INFINITY : l);
    });
    most = most_of_wave(most), least = least_of_wave(least);
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = most, least_parts[threadIdx.x >> 6] = least;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kDrawThreads / 64; ++w) most = max(most, parts[w]), least = fminf(least, least_parts[w]);
        c.largest[blockIdx.x] = most, c.smallest[blockIdx.x] = least;
    }
}

// The row's largest, its key and its index's complement, and its smallest that is finite; in every thread.
struct Ends {
    uint64_t largest;
    float smallest;
};
__device__ __forceinline__ Ends ends_of(const DrawChunks& c, uint32_t row) {
    Ends e{0, INFINITY};
    for (uint32_t i = threadIdx.x & 63u; i < c.chunks; i += 64) {
        e.largest = max(e.largest, c.largest[uint64_t{row} * c.chunks + i]);
        e.smallest = fminf(e.smallest, c.smallest[uint64_t{row} * c.chunks + i]);
    }
    return {most_of_wave(e.largest), least_of_wave(e.smallest)};
}

// An infinite logit, or two whose distance f32 does not hold: the row has no bins. (Of +inf
// and -inf alone the smallest is +inf too, and the distance a NaN.)
__device__ __forceinline__ bool too_far(float most, float smallest) { return !(most - smallest < INFINITY); }

// A logit's place among the bins: it does not fall as the logit does.
__device__ __forceinline__ float place_of(float l, float most, float steps) {
    return fminf((most - l) * steps, static_cast<float>(kBins - 1));
}
// Bins a unit of a logit: over what weighs anything, or over the row's logits where
// they reach less far, so that no bin has much more of them than another (one that
// has more than kList is answered by descent); all that weigh before the last bin.
__device__ __forceinline__ float steps_of(const Settings& s, float most, float smallest) {
    const double range = static_cast<double>(most) - static_cast<double>(smallest);
    return static_cast<float>(fmin(fmax(s.rate * (static_cast<double>(kBins - 1) / kReach), (kBins - 3) / range), 1e30));
}

// Whether this is the last of a row's workgroups to come here.
__device__ __forceinline__ bool last_of(uint32_t& counter, uint32_t workgroups, uint32_t* flag) {
    __asm__ __volatile__("s_waitcnt vmcnt(0)" ::: "memory");  // what each wave wrote has arrived
    __syncthreads();
    if (threadIdx.x == 0) *flag = add(counter, 1u) == workgroups - 1;
    __syncthreads();
    return *flag != 0;
}

struct Planning {
    uint64_t sums[kBins + 1];    // weights before a bin
    uint32_t counts[kBins + 1];
    uint64_t parts[kDrawThreads / 64];
};

// The bins that the row's cuts and its draw may fall into, by the last of its workgroups.
__device__ void plan_row(const Sample& a, const Settings& s, float steps, DrawRoom& room, Planning& d) {
    constexpr uint32_t kMine = kBins / kDrawThreads;
    static_assert(kMine % 2 == 0, "whole words of counts");
    uint64_t weight[kMine], pair[kMine / 2], sum = 0, tokens = 0, all, all_tokens;
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) weight[i] = get(room.weights[kMine * threadIdx.x + i]), sum += weight[i];
#pragma unroll
    for (uint32_t i = 0; i < kMine / 2; ++i) {
        pair[i] = get(room.counts[kMine / 2 * threadIdx.x + i]);
        tokens += (pair[i] & 0xFFFFFFFFull) + (pair[i] >> 32);
    }
    uint64_t before = sum_before(sum, d.parts, &all);
    uint32_t before_tokens = static_cast<uint32_t>(sum_before(tokens, d.parts, &all_tokens));
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
        const uint32_t bin = kMine * threadIdx.x + i;
        d.sums[bin] = before, d.counts[bin] = before_tokens;
        before += weight[i], before_tokens += static_cast<uint32_t>(pair[i / 2] >> (i % 2 * 32));
    }
    if (threadIdx.x == 0) d.sums[kBins] = all, d.counts[kBins] = static_cast<uint32_t>(all_tokens);
    __syncthreads();
    if (threadIdx.x >= 64) return;
    // By one wave: the first bin (of kBins) of which `passed` is true, as it is of all after it.
    const uint32_t lane = threadIdx.x;
    auto first_bin = [&](auto passed) {
        const uint32_t block = __popcll(__ballot(!passed(kBins / 64 * lane + kBins / 64 - 1)));
        if (block == 64) return kBins - 1;
        const uint32_t in = __popcll(__ballot(lane < kBins / 64 && !passed(kBins / 64 * block + lane % (kBins / 64))));
        return kBins / 64 * block + in;
    };
    // a question's bins, its target between `low` and `high`
    auto run_of = [&](uint64_t low, uint64_t high) {
        Run r{};
        r.first = first_bin([&](uint32_t bin) { return d.sums[bin + 1] > low; });
        r.last = first_bin([&](uint32_t bin) { return d.sums[bin + 1] > high; });
        r.last = min(r.last, kBins - 2);  // the last bin's tokens weigh nothing
        return r;
    };
    Run none{kBins, kBins, 0, 0, 0, 0, 0}, top_k = none, top_p = none;
    uint64_t low = d.sums[kBins], high = low;  // of what is kept
    if (s.top_k < a.vocabulary) {
        const uint32_t bin = first_bin([&](uint32_t b) { return d.counts[b + 1] >= s.top_k; });
        if (bin < kBins - 1) {
            top_k.first = top_k.last = bin;
            low = max(d.sums[bin], 1ull << 40), high = d.sums[bin + 1];  // the first token is always kept
        }
    }
    if (s.top_p < 1.0) {
        top_p = run_of(passed_by(s, low), passed_by(s, high));
        low = max(d.sums[top_p.first], 1ull << 40), high = min(high, d.sums[top_p.last + 1]);
    }
    if (s.least > 0) {
        // min_p's last token is in the bin of its distance or, by rounding, one beside it; of a
        // temperature so far above the logits that f64's exponentials are alike over several
        // bins, one of those (of an infinite one, where both are NaNs or infinite: of all)
        const double bins = static_cast<double>(steps) / s.rate;
        const double at = -log(static_cast<double>(s.least) / kWhole) * bins, off = 1.0 + 0x1p-50 * bins;
        const uint32_t from = static_cast<uint32_t>(fmin(fmax(at - off, 0.0), static_cast<double>(kBins - 2)));
        const uint32_t to = static_cast<uint32_t>(fmin(at + off, static_cast<double>(kBins - 1))) + 1;
        low = min(low, max(d.sums[from], 1ull << 40)), high = min(high, d.sums[to]);
        if (lane == 0) room.end_first = from, room.end_past = to, room.end_ahead = d.sums[from];
    }
    const Run draw = run_of(drawn_at(s, low), drawn_at(s, high));
    if (lane != 0) return;
    // in order, and those that meet as one
    Run x = draw, y = top_k, z = top_p;
    auto order = [](Run& u, Run& v) {
        if (v.first < u.first) {
            const Run t = u;
            u = v, v = t;
        }
    };
    order(x, y), order(y, z), order(x, y);
    uint32_t runs = 0, listed = 0;
    auto keep = [&](Run r) {
        r.before = d.counts[r.first], r.count = d.counts[r.last + 1] - r.before, r.start = listed;
        r.ahead = d.sums[r.first];
        listed += r.count;
        room.run[runs++] = r;
    };
    auto meet = [](const Run& u, const Run& v) { return v.first < kBins && v.first <= u.last + 1; };
    if (meet(y, z)) y.last = max(y.last, z.last), z = none;
    if (meet(x, y)) {
        x.last = max(x.last, y.last), y = z, z = none;
        if (meet(x, y)) x.last = max(x.last, y.last), y = none;
    }
    keep(x);
    if (y.first < kBins) keep(y);
    if (z.first < kBins) keep(z);
    room.runs = runs, room.cut = top_k.first < kBins, room.alone = listed > kList;
    room.all = d.sums[kBins];
}

__global__ __launch_bounds__(kDrawThreads) void row_bins(Sample a, DrawChunks c) {
    __shared__ union {
        struct {
            uint64_t weights[kBins];
            uint32_t counts[kBins];
        } bins;
        Planning planning;
    } space;
    __shared__ uint32_t last;
    const uint32_t row = blockIdx.x / c.chunks, chunk = blockIdx.x % c.chunks;
    for (uint32_t i = threadIdx.x; i < kBins; i += kDrawThreads) space.bins.weights[i] = 0, space.bins.counts[i] = 0;
    const Settings s = settings_of(a, row);
    const Ends ends = ends_of(c, row);
    const float most = logit_of(static_cast<uint32_t>(ends.largest >> 32));
    if (s.greedy || most == -INFINITY || too_far(most, ends.smallest)) return;
    DrawRoom& room = c.rooms[row];
    const float steps = steps_of(s, most, ends.smallest);
    __syncthreads();
    uint32_t rest = 0;
    each_of_chunk(a, c, row, chunk, [&](float l, uint32_t) {
        const uint32_t bin = static_cast<uint32_t>(place_of(l, most, steps));
        if (bin == kBins - 1) {
            ++rest;
            return;
        }
        // a whole number below 2^52 in its bits
        const double w = whole_weight(l, most, s.octaves) + 0x1p52;
        atomicAdd(reinterpret_cast<unsigned long long*>(&space.bins.weights[bin]), __builtin_bit_cast(unsigned long long, w) & ((1ull << 52) - 1));
        atomicAdd(&space.bins.counts[bin], 1u);
    });
#pragma unroll
    for (uint32_t o = 32; o > 0; o >>= 1) rest += __shfl_xor(rest, o);
    if ((threadIdx.x & 63u) == 0 && rest > 0) atomicAdd(&space.bins.counts[kBins - 1], rest);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kBins; i += kDrawThreads)
        if (space.bins.weights[i] != 0) add(room.weights[i], space.bins.weights[i]);
    for (uint32_t i = threadIdx.x; i < kBins / 2; i += kDrawThreads)
        if (const uint64_t pair = space.bins.counts[2 * i] | uint64_t{space.bins.counts[2 * i + 1]} << 32) add(room.counts[i], pair);
    if (last_of(room.binned, c.chunks, &last)) plan_row(a, s, steps, room, space.planning);
}

// The row's list sorted, and its questions answered, by the last of its workgroups.
struct Sorting {
    union {
        uint64_t list[kList];
        uint64_t before[kList];    // the list's weight before a token, once it is sorted
    };
    uint64_t sorted[kList];
    uint32_t buckets[kList + 1];   // tokens, then those before
    uint64_t parts[kDrawThreads / 64];
    uint64_t passed, own;
    uint32_t token;
};

__device__ void answer_row(const Sample& a, uint32_t row, const Settings& s, float most, float steps, const DrawRoom& room,
                           Sorting& t) {
    constexpr uint32_t kMine = kList / kDrawThreads;
    Run run[kRuns];
    const uint32_t runs = room.runs;
    uint32_t n = 0, bins = 0;
#pragma unroll
    for (uint32_t q = 0; q < kRuns; ++q) {
        run[q] = q < runs ? room.run[q] : Run{kBins, kBins, 0, 0, kList, 0, 0};
        if (q < runs) n += run[q].count, bins += run[q].last - run[q].first + 1;
    }
    // Buckets: each bin in as many equal parts, which rise as the logits fall.
    const uint32_t each = max(kList / bins, 1u);
    uint64_t token[kMine];
    uint32_t bucket[kMine], slot[kMine];
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) {
        const uint32_t i = kDrawThreads * e + threadIdx.x;
        token[e] = i < n ? get(room.list[i]) : 0;
        t.buckets[i] = 0;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) {
        if (kDrawThreads * e + threadIdx.x >= n) continue;
        const float place = place_of(logit_of(static_cast<uint32_t>(token[e] >> 32)), most, steps);
        uint32_t q = 0, from = 0;
#pragma unroll
        for (uint32_t x = 1; x < kRuns; ++x)
            if (x < runs && place >= static_cast<float>(run[x].first)) q = x;
#pragma unroll
        for (uint32_t x = 0; x + 1 < kRuns; ++x)
            if (x < q) from += run[x].last - run[x].first + 1;
        Run r = run[0];
#pragma unroll
        for (uint32_t x = 1; x < kRuns; ++x)
            if (q == x) r = run[x];
        const uint32_t part = static_cast<uint32_t>((place - static_cast<float>(r.first)) * static_cast<float>(each));
        bucket[e] = min(from * each + min(part, (r.last - r.first + 1) * each - 1), kList - 1);
        slot[e] = atomicAdd(&t.buckets[bucket[e]], 1u);
    }
    __syncthreads();
    uint64_t sum = 0, all;
    uint32_t size[kMine];
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) size[e] = t.buckets[kMine * threadIdx.x + e], sum += size[e];
    sum = sum_before(sum, t.parts, &all);
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) t.buckets[kMine * threadIdx.x + e] = static_cast<uint32_t>(sum), sum += size[e];
    if (threadIdx.x == 0) t.buckets[kList] = n;
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e)
        if (kDrawThreads * e + threadIdx.x < n) t.list[t.buckets[bucket[e]] + slot[e]] = token[e];
    __syncthreads();
    // within a bucket, mostly of one or two, by counting
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) {
        if (kDrawThreads * e + threadIdx.x >= n) continue;
        const uint32_t first = t.buckets[bucket[e]], end = t.buckets[bucket[e] + 1];
        uint32_t rank = 0;
        for (uint32_t j = first; j < end; ++j) rank += t.list[j] > token[e];
        t.sorted[first + rank] = token[e];
    }
    __syncthreads();
    // a thread's tokens: their weights, and the row's weight and count before them
    uint64_t own[kMine], before[kMine];
    uint32_t count[kMine];
    sum = 0;
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) {
        const uint32_t i = kMine * threadIdx.x + e;
        own[e] = i < n ? weight_of(logit_of(static_cast<uint32_t>(t.sorted[i] >> 32)), most, s.octaves) : 0;
        before[e] = sum, sum += own[e];
    }
    sum = sum_before(sum, t.parts, &all);
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) t.before[kMine * threadIdx.x + e] = before[e] += sum;
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) {
        const uint32_t i = kMine * threadIdx.x + e;
        Run r = run[0];
#pragma unroll
        for (uint32_t q = 1; q < kRuns; ++q)
            if (q < runs && run[q].start <= i) r = run[q];
        count[e] = r.before + (i - r.start);
        before[e] = r.ahead + (before[e] - t.before[r.start]);
    }
    // The weight up to the token at which the row's running count or weight passes `target`, its own in t.own.
    auto passed_at = [&](bool by_count, uint64_t target) {
        __syncthreads();
#pragma unroll
        for (uint32_t e = 0; e < kMine; ++e) {
            const uint32_t i = kMine * threadIdx.x + e;
            if (i < n && (by_count ? count[e] == target : before[e] <= target && target < before[e] + own[e]))
                t.passed = before[e] + own[e], t.own = own[e], t.token = ~static_cast<uint32_t>(t.sorted[i]);
        }
        __syncthreads();
        return t.passed;
    };
    uint64_t kept = room.all;
    const uint64_t likely = s.least > 0 ? room.end_ahead + get(room.likely) : kept;
    if (room.cut) kept = passed_at(true, s.top_k - 1);
    if (s.top_p < 1.0) kept = passed_at(false, passed_by(s, kept));
    kept = min(kept, likely);
    passed_at(false, drawn_at(s, kept));
    if (threadIdx.x == 0) write_draw(a, row, t.token, t.own, kept);
}

__global__ __launch_bounds__(kDrawThreads) void row_draw(Sample a, DrawChunks c) {
    __shared__ union {
        Descent descent;
        Sorting sorting;
        uint64_t list[kList];
    } space;
    __shared__ uint64_t likely;
    __shared__ uint32_t last, listed, base;
    const uint32_t row = blockIdx.x / c.chunks, chunk = blockIdx.x % c.chunks;
    const Settings s = settings_of(a, row);
    const Ends ends = ends_of(c, row);
    const float most = logit_of(static_cast<uint32_t>(ends.largest >> 32));
    if (s.greedy || most == -INFINITY) {
        if (chunk == 0 && threadIdx.x == 0) {
            if (most == -INFINITY)
                write_draw(a, row, 0xFFFFFFFFu, 0, 1);
            else
                write_draw(a, row, ~static_cast<uint32_t>(ends.largest), 1, 1);
        }
        return;
    }
    DrawRoom& room = c.rooms[row];
    if (too_far(most, ends.smallest) || room.alone) {
        if (chunk == 0) draw_alone(a, row, s, most, space.descent);
        return;
    }
    if (threadIdx.x == 0) listed = 0, likely = 0;
    __syncthreads();
    const float steps = steps_of(s, most, ends.smallest);
    uint32_t first[kRuns], width[kRuns];  // a run that is not there holds no bin
#pragma unroll
    for (uint32_t q = 0; q < kRuns; ++q) {
        const bool there = q < room.runs;
        first[q] = there ? room.run[q].first : kBins, width[q] = there ? room.run[q].last - first[q] : 0;
    }
    // the bins that min_p's end may be in: none without it
    const uint32_t end_first = s.least > 0 ? room.end_first : kBins, end_bins = s.least > 0 ? room.end_past - end_first : 0;
    uint64_t mine = 0;
    each_of_chunk(a, c, row, chunk, [&](float l, uint32_t i) {
        const uint32_t bin = static_cast<uint32_t>(place_of(l, most, steps));
        if (bin - end_first < end_bins) {
            const uint64_t w = weight_of(l, most, s.octaves);
            mine += w >= s.least ? w : 0;
        }
        bool in = false;
#pragma unroll
        for (uint32_t q = 0; q < kRuns; ++q) in |= bin - first[q] <= width[q];
        if (in && l != -INFINITY) {
            const uint32_t at = atomicAdd(&listed, 1u);
            if (at < kList) space.list[at] = uint64_t{key_of(l)} << 32 | ~i;
        }
    });
    if (s.least > 0) {
#pragma unroll
        for (uint32_t o = 32; o > 0; o >>= 1) mine += __shfl_xor(mine, o);
        if ((threadIdx.x & 63u) == 0 && mine > 0) atomicAdd(reinterpret_cast<unsigned long long*>(&likely), static_cast<unsigned long long>(mine));
    }
    __syncthreads();
    const uint32_t here = min(listed, kList);
    if (threadIdx.x == 0 && likely > 0) add(room.likely, likely);
    if (threadIdx.x == 0 && here > 0) base = add(room.listed, here);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < here; i += kDrawThreads)
        if (base + i < kList) put(room.list[base + i], space.list[i]);
    if (last_of(room.gathered, c.chunks, &last)) answer_row(a, row, s, most, steps, room, space.sorting);
}

// About 512 workgroups, two a CU, a chunk of at least a four a thread; of whole fours.
// 64 x 128,256 logits 52 us; 57 by 256 workgroups, 62 by 1,024 (a row's bins are cleared,
// added up and counted a workgroup); 24 x 262,144 52, 55 and 56.
static uint32_t draw_chunks(uint32_t rows, uint32_t vocabulary) {
    const uint32_t most = (vocabulary + 3 + 4 * kDrawThreads - 1) / (4 * kDrawThreads);
    return std::max(1u, std::min((512 + rows - 1) / rows, most));
}

uint64_t sample_bytes(uint32_t rows, uint32_t vocabulary) {
    return rows * (sizeof(DrawRoom) + uint64_t{draw_chunks(rows, vocabulary)} * 12);
}

hipError_t launch_sample(const Sample& a, hipStream_t stream) {
    DrawChunks c{};
    c.rooms = static_cast<DrawRoom*>(a.workspace);
    c.largest = reinterpret_cast<uint64_t*>(c.rooms + a.rows);
    c.chunks = draw_chunks(a.rows, a.vocabulary);
    c.share = ((a.vocabulary + 3 + c.chunks - 1) / c.chunks + 3) / 4 * 4;
    c.smallest = reinterpret_cast<float*>(c.largest + uint64_t{a.rows} * c.chunks);
    const dim3 grid(a.rows * c.chunks);
    hipLaunchKernelGGL(row_largest, grid, dim3(kDrawThreads), 0, stream, a, c);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    hipLaunchKernelGGL(row_bins, grid, dim3(kDrawThreads), 0, stream, a, c);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    hipLaunchKernelGGL(row_draw, grid, dim3(kDrawThreads), 0, stream, a, c);
    return hipGetLastError();
}

}  // namespace chm
