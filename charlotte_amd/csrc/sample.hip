// A token drawn from each row of logits, by temperature, top-k, top-p, min-p and
// a given uniform number, in whole numbers from the weights on:
//   w = floor(2^40 exp((l - m) / T)), tokens in the order (l falling, index rising).
//
// What is kept is a run of the first tokens whichever way it is cut, so W, its
// weight, is the least of the cuts' running sums, and every cut and the draw
// itself are one question: at which token does the running count or weight pass
// a number? It is answered without sorting the row, in three launches over chunks
// of the rows:
//   row_largest   each chunk's largest logit;
//   row_bins      the weights and counts of kBins equal steps of (m - l) / T, down
//                 to where a weight is 0. The workgroup that ends a row last finds
//                 the bins that the cuts and the draw may fall into: a cut's bin
//                 bounds what is kept, that the bins of the cuts after it;
//   row_draw      the tokens of those bins, few hundreds, gathered. The last
//                 workgroup of a row sorts them, and answers exactly.
// Where those bins hold more than kList tokens (many equal logits, a temperature
// that makes them so) or the largest is +inf, one workgroup answers by descent:
// weights and counts of the logits' leading bits (as keys that rise with them)
// summed in LDS, the part that holds the answer opened by its next bits; tokens of
// one key have one weight, so the place among them is a division.
// Sums are of whole numbers, so that atomics may add them in any order.
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
    DrawRow row{a.logits + r * a.logit_stride, 0, a.vocabulary, most, s.rate};
    row.lead = lead_of(row.x);
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
        const Place p = descend<false>(row, passed_by(s, kept), d);
        kept = p.before + (p.rank + 1) * p.weight;
    }
    kept = min(kept, max(likely, 1ull << 40));
    const Place p = descend<false>(row, drawn_at(s, kept), d);
    const uint32_t token = index_of(row, p.key, p.rank, d);
    if (threadIdx.x == 0) write_draw(a, r, token, p.weight, kept);
}

// ---- by bins -----------------------------------------------------------------

// Runs of bins whose tokens are gathered, in order and apart; what lies before each.
struct Run {
    uint32_t first, last;
    uint64_t weight, count;
    uint32_t start;         // its first token's place in the list
    uint32_t reserved;
};
struct DrawPlan {
    uint64_t likely;            // the weight that min_p leaves
    uint64_t kept;              // without a cut: what top_k leaves
    uint32_t binned, gathered;  // workgroups of row_bins, of row_draw, that have ended
    uint32_t listed;            // tokens gathered
    uint32_t runs, alone;       // runs; or by descent
    uint32_t cut;               // top_k's last token is in a run
    Run run[3];
};

// A row's part of the workspace.
struct DrawRoom {
    uint64_t weights[kBins];
    uint32_t counts[kBins];
    DrawPlan plan;          // (cleared with the bins by row_largest)
    uint64_t list[kList];   // key, and the index's complement: the first token is the largest
};
constexpr uint32_t kCleared = (offsetof(DrawRoom, list) + 3) / 4;

struct DrawChunks {
    DrawRoom* rooms;
    uint64_t* largest;  // [rows][chunks]: key, and the index's complement
    uint32_t chunks, share;
};

// f(logit, index) for each token of a workgroup's chunk.
template <typename F>
__device__ __forceinline__ void each_of_chunk(const Sample& a, const DrawChunks& c, uint32_t row, uint32_t chunk, F f) {
    const float* x = a.logits + row * a.logit_stride;
    const uint32_t lead = lead_of(x), end = min((chunk + 1) * c.share, lead + a.vocabulary);
#pragma unroll 2
    for (uint32_t at = chunk * c.share + 4 * threadIdx.x; at < end; at += 4 * kDrawThreads) {
        const float4 q = read4(x, lead, a.vocabulary, at, -INFINITY);
        const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            if (at + e >= lead && at + e < lead + a.vocabulary) f(clean(v[e]), at + e - lead);
    }
}

__device__ __forceinline__ uint64_t most_of_wave(uint64_t x) {
#pragma unroll
    for (uint32_t o = 32; o > 0; o >>= 1) x = max(x, static_cast<uint64_t>(__shfl_xor(x, o)));
    return x;
}

__global__ __launch_bounds__(kDrawThreads) void row_largest(Sample a, DrawChunks c) {
    __shared__ uint64_t parts[kDrawThreads / 64];
    const uint32_t row = blockIdx.x / c.chunks, chunk = blockIdx.x % c.chunks;
    uint32_t* room = reinterpret_cast<uint32_t*>(c.rooms + row);
    for (uint32_t i = chunk * kDrawThreads + threadIdx.x; i < kCleared; i += c.chunks * kDrawThreads) room[i] = 0;
    uint64_t most = 0;
    each_of_chunk(a, c, row, chunk, [&](float l, uint32_t i) { most = max(most, uint64_t{key_of(l)} << 32 | ~i); });
    most = most_of_wave(most);
    if ((threadIdx.x & 63u) == 0) parts[threadIdx.x >> 6] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t w = 1; w < kDrawThreads / 64; ++w) most = max(most, parts[w]);
        c.largest[blockIdx.x] = most;
    }
}

// The row's largest: its key, and its index's complement; in every thread.
__device__ __forceinline__ uint64_t largest_of(const DrawChunks& c, uint32_t row) {
    uint64_t most = 0;
    for (uint32_t i = threadIdx.x & 63u; i < c.chunks; i += 64) most = max(most, c.largest[uint64_t{row} * c.chunks + i]);
    return most_of_wave(most);
}

// The bin of a logit: it does not fall as the logit does.
__device__ __forceinline__ uint32_t bin_of(float l, float most, float steps) {
    return static_cast<uint32_t>(fminf((most - l) * steps, static_cast<float>(kBins - 1)));
}
__device__ __forceinline__ float steps_of(const Settings& s) {
    return static_cast<float>(s.rate * (static_cast<double>(kBins - 1) / kReach));
}

// Whether this is the last of a row's workgroups to come here; then it sees what they wrote.
__device__ __forceinline__ bool last_of(uint32_t* counter, uint32_t workgroups, uint32_t* flag) {
    __builtin_amdgcn_s_waitcnt(0);  // each wave's writes are out
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        *flag = atomicAdd(counter, 1u) == workgroups - 1;
        __threadfence();
    }
    __syncthreads();
    return *flag != 0;
}

// The bins that the row's cuts and its draw may fall into, by the last of its workgroups.
__device__ void plan_row(const Sample& a, const Settings& s, DrawRoom& room, Descent& d) {
    constexpr uint32_t kMine = kBins / kDrawThreads;
    uint64_t w[kMine], c[kMine], weight = 0, count = 0, total, tokens;
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
        const uint32_t bin = kMine * threadIdx.x + i;
        w[i] = room.weights[bin], c[i] = room.counts[bin];
        weight += w[i], count += c[i];
    }
    weight = sum_before(weight, d.parts, &total);
    count = sum_before(count, d.parts, &tokens);
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
        const uint32_t bin = kMine * threadIdx.x + i;
        d.weights[bin] = weight, d.counts[bin] = static_cast<uint32_t>(count);  // before the bin
        weight += w[i], count += c[i];
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    auto after = [&](uint32_t bin) { return bin + 1 < kBins ? d.weights[bin + 1] : total; };
    auto counted = [&](uint32_t bin) { return bin + 1 < kBins ? uint64_t{d.counts[bin + 1]} : tokens; };
    // the bin whose running weight passes `target`
    auto bin_at = [&](uint64_t target) {
        uint32_t low = 0, high = kBins;
        while (high - low > 1) {
            const uint32_t middle = (low + high) / 2;
            (d.weights[middle] <= target ? low : high) = middle;
        }
        return low;
    };
    __shared__ Run run[3];  // (indexed by thread 0 alone)
    uint32_t runs = 0;
    uint64_t low = total, high = total;  // what is kept weighs no less and no more
    if (s.top_k < a.vocabulary) {
        uint32_t from = 0, to = kBins;
        while (to - from > 1) {
            const uint32_t middle = (from + to) / 2;
            (d.counts[middle] < s.top_k ? from : to) = middle;
        }
        low = d.weights[from], high = after(from);
        if (counted(from) == s.top_k) low = high;
        if (low != high) run[runs++] = {from, from, 0, 0, 0, 0};
    }
    room.plan.cut = low != high, room.plan.kept = low;
    if (s.top_p < 1.0) {
        const uint32_t from = bin_at(passed_by(s, low)), to = bin_at(passed_by(s, high));
        run[runs++] = {from, to, 0, 0, 0, 0};
        low = d.weights[from], high = after(to);
    }
    const uint64_t likely = max(room.plan.likely, 1ull << 40);
    low = max(min(low, likely), 1ull), high = min(high, likely);
    run[runs++] = {bin_at(drawn_at(s, low)), bin_at(drawn_at(s, high)), 0, 0, 0, 0};
    // in order, and those that meet as one
    for (uint32_t i = 1; i < runs; ++i)
        for (uint32_t j = i; j > 0 && run[j].first < run[j - 1].first; --j) {
            const Run t = run[j];
            run[j] = run[j - 1], run[j - 1] = t;
        }
    uint32_t merged = 0;
    for (uint32_t i = 1; i < runs; ++i)
        if (run[i].first <= run[merged].last + 1)
            run[merged].last = max(run[merged].last, run[i].last);
        else
            run[++merged] = run[i];
    uint64_t listed = 0;
    for (uint32_t i = 0; i <= merged; ++i) {
        run[i].weight = d.weights[run[i].first], run[i].count = d.counts[run[i].first];
        run[i].start = static_cast<uint32_t>(listed);
        listed += counted(run[i].last) - run[i].count;
        room.plan.run[i] = run[i];
    }
    room.plan.runs = merged + 1;
    room.plan.alone = listed > kList;
}

__global__ __launch_bounds__(kDrawThreads) void row_bins(Sample a, DrawChunks c) {
    __shared__ Descent d;
    __shared__ uint32_t last;
    const uint32_t row = blockIdx.x / c.chunks, chunk = blockIdx.x % c.chunks;
    const Settings s = settings_of(a, row);
    const float most = logit_of(static_cast<uint32_t>(largest_of(c, row) >> 32));
    if (s.greedy || fabsf(most) == INFINITY) return;
    DrawRoom& room = c.rooms[row];
    const float steps = steps_of(s);
    for (uint32_t i = threadIdx.x; i < kBins; i += kDrawThreads) d.weights[i] = 0, d.counts[i] = 0;
    __syncthreads();
    uint64_t likely = 0;
    uint32_t rest = 0;
    each_of_chunk(a, c, row, chunk, [&](float l, uint32_t) {
        const uint32_t bin = bin_of(l, most, steps);
        if (bin == kBins - 1) {
            ++rest;
            return;
        }
        const uint64_t w = weight_of(l, most, s.rate);
        if (w >= s.least) likely += w;
        atomicAdd(reinterpret_cast<unsigned long long*>(&d.weights[bin]), static_cast<unsigned long long>(w));
        atomicAdd(&d.counts[bin], 1u);
    });
#pragma unroll
    for (uint32_t o = 32; o > 0; o >>= 1) likely += __shfl_xor(likely, o), rest += __shfl_xor(rest, o);
    if ((threadIdx.x & 63u) == 0) {
        if (rest) atomicAdd(&d.counts[kBins - 1], rest);
        if (likely) atomicAdd(reinterpret_cast<unsigned long long*>(&room.plan.likely), static_cast<unsigned long long>(likely));
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kBins; i += kDrawThreads) {
        if (d.counts[i] == 0) continue;
        atomicAdd(reinterpret_cast<unsigned long long*>(&room.weights[i]), static_cast<unsigned long long>(d.weights[i]));
        atomicAdd(&room.counts[i], d.counts[i]);
    }
    if (last_of(&room.plan.binned, c.chunks, &last)) plan_row(a, s, room, d);
}

// The row's list sorted, and its questions answered, by the last of its workgroups.
struct Sorting {
    uint64_t list[kList];
    uint64_t before[kList];  // the list's weight before a token
    uint64_t parts[kDrawThreads / 64];
    uint64_t passed, own;
    uint32_t token;
};

__device__ void answer_row(const Sample& a, uint32_t row, const Settings& s, float most, const DrawRoom& room, Sorting& t) {
    const uint32_t n = min(room.plan.listed, kList);
    uint32_t size = 64;
    while (size < n) size *= 2;
    for (uint32_t i = threadIdx.x; i < size; i += kDrawThreads) t.list[i] = i < n ? room.list[i] : 0;
    // bitonic, falling; the places past the list, zeros, come last
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < size / 2; i += kDrawThreads) {
                const uint32_t x = 2 * i - (i & (j - 1)), y = x + j;
                const uint64_t u = t.list[x], v = t.list[y];
                if ((u < v) == ((x & k) == 0)) t.list[x] = v, t.list[y] = u;
            }
        }
    __syncthreads();
    // a thread's tokens: their weights, and the row's weight and count before them
    constexpr uint32_t kMine = kList / kDrawThreads;
    uint64_t own[kMine], before[kMine], count[kMine], sum = 0, all;
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) {
        const uint32_t i = kMine * threadIdx.x + e;
        own[e] = i < n ? weight_of(logit_of(static_cast<uint32_t>(t.list[i] >> 32)), most, s.rate) : 0;
        before[e] = sum, sum += own[e];
    }
    sum = sum_before(sum, t.parts, &all);
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) t.before[kMine * threadIdx.x + e] = before[e] += sum;
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) {
        const uint32_t i = kMine * threadIdx.x + e;
        Run run = room.plan.run[0];
        for (uint32_t q = 1; q < room.plan.runs; ++q)
            if (room.plan.run[q].start <= i) run = room.plan.run[q];
        count[e] = run.count + (i - run.start);
        before[e] = run.weight + (before[e] - t.before[run.start]);
    }
    // The weight up to the token at which the row's running count or weight passes `target`, its own in t.own.
    auto passed_at = [&](bool by_count, uint64_t target) {
        __syncthreads();
#pragma unroll
        for (uint32_t e = 0; e < kMine; ++e) {
            const uint32_t i = kMine * threadIdx.x + e;
            if (i < n && (by_count ? count[e] == target : before[e] <= target && target < before[e] + own[e]))
                t.passed = before[e] + own[e], t.own = own[e], t.token = ~static_cast<uint32_t>(t.list[i]);
        }
        __syncthreads();
        return t.passed;
    };
    uint64_t kept = room.plan.kept;
    if (room.plan.cut) kept = passed_at(true, s.top_k - 1);
    if (s.top_p < 1.0) kept = passed_at(false, passed_by(s, kept));
    kept = min(kept, max(room.plan.likely, 1ull << 40));
    passed_at(false, drawn_at(s, kept));
    if (threadIdx.x == 0) write_draw(a, row, t.token, t.own, kept);
}

__global__ __launch_bounds__(kDrawThreads) void row_draw(Sample a, DrawChunks c) {
    __shared__ union {
        Descent descent;
        Sorting sorting;
    } space;
    __shared__ uint32_t last, listed, base;
    const uint32_t row = blockIdx.x / c.chunks, chunk = blockIdx.x % c.chunks;
    const Settings s = settings_of(a, row);
    const uint64_t largest = largest_of(c, row);
    const float most = logit_of(static_cast<uint32_t>(largest >> 32));
    if (s.greedy || most == -INFINITY) {
        if (chunk == 0 && threadIdx.x == 0) {
            if (most == -INFINITY)
                write_draw(a, row, 0xFFFFFFFFu, 0, 1);
            else
                write_draw(a, row, ~static_cast<uint32_t>(largest), 1, 1);
        }
        return;
    }
    DrawRoom& room = c.rooms[row];
    if (most == INFINITY || room.plan.alone) {
        if (chunk == 0) draw_alone(a, row, s, most, space.descent);
        return;
    }
    if (threadIdx.x == 0) listed = 0;
    __syncthreads();
    const float steps = steps_of(s);
    uint32_t first[3], width[3];  // a run that is not there holds no bin
#pragma unroll
    for (uint32_t q = 0; q < 3; ++q) {
        const bool there = q < room.plan.runs;
        first[q] = there ? room.plan.run[q].first : kBins, width[q] = there ? room.plan.run[q].last - first[q] : 0;
    }
    each_of_chunk(a, c, row, chunk, [&](float l, uint32_t i) {
        const uint32_t bin = bin_of(l, most, steps);
        if (bin - first[0] > width[0] && bin - first[1] > width[1] && bin - first[2] > width[2]) return;
        const uint32_t at = atomicAdd(&listed, 1u);
        if (at < kList) space.sorting.list[at] = uint64_t{key_of(l)} << 32 | ~i;
    });
    __syncthreads();
    const uint32_t mine = min(listed, kList);
    if (threadIdx.x == 0 && mine > 0) base = atomicAdd(&room.plan.listed, mine);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < mine; i += kDrawThreads)
        if (base + i < kList) room.list[base + i] = space.sorting.list[i];
    if (last_of(&room.plan.gathered, c.chunks, &last)) answer_row(a, row, s, most, room, space.sorting);
}

// About a thousand workgroups, a chunk of at least two fours a thread; of whole fours.
static uint32_t draw_chunks(uint32_t rows, uint32_t vocabulary) {
    const uint32_t most = (vocabulary + 3 + 8 * kDrawThreads - 1) / (8 * kDrawThreads);
    return std::max(1u, std::min((1024 + rows - 1) / rows, most));
}

uint64_t sample_bytes(uint32_t rows, uint32_t vocabulary) {
    return rows * (sizeof(DrawRoom) + uint64_t{draw_chunks(rows, vocabulary)} * 8);
}

hipError_t launch_sample(const Sample& a, hipStream_t stream) {
    DrawChunks c{};
    c.rooms = static_cast<DrawRoom*>(a.workspace);
    c.largest = reinterpret_cast<uint64_t*>(c.rooms + a.rows);
    c.chunks = draw_chunks(a.rows, a.vocabulary);
    c.share = ((a.vocabulary + 3 + c.chunks - 1) / c.chunks + 3) / 4 * 4;
    const dim3 grid(a.rows * c.chunks);
    hipLaunchKernelGGL(row_largest, grid, dim3(kDrawThreads), 0, stream, a, c);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    hipLaunchKernelGGL(row_bins, grid, dim3(kDrawThreads), 0, stream, a, c);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    hipLaunchKernelGGL(row_draw, grid, dim3(kDrawThreads), 0, stream, a, c);
    return hipGetLastError();
}

}  // namespace chm
