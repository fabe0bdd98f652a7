// Block tables and slot maps from the requests' lengths: pages given back go
// onto the stack of free pages, pages that are needed come off its top, in the
// requests' order; then each row's position and slot.
//
// Where each of these lands is a running sum over the requests - of their rows,
// of the pages they give, of the pages they take - found by one workgroup, a
// request a thread. The entries themselves are shared among its threads whatever
// the requests' sizes: entry i is that of the last request whose running sum is not
// above i, by binary search in LDS.
//
// Up to 1,024 requests (page_plan_few) nothing is read that the step writes: a page
// taken that another request gives back is read from that one's row, and a slot in
// a page that is taken now from where the page comes; so all of it is on its way
// at once. More (page_plan) go in two passes over 1,024 at a time.
//
// Bound by latency, chains of dependent reads and barriers: 24 requests 5.1 us by 256
// threads (11.2 in two passes), 512 6.5 by 1,024, 1,100 19.5.
#include "requests.hpp"

namespace chm {

constexpr uint32_t kPlanThreads = 1024;
// Rows past which their slots are a launch of their own, of many workgroups: 4,163
// rows of 64 requests 5.1 and 4.1 us so, 12.0 in one.
constexpr uint32_t kPlanRows = 2048;
constexpr uint32_t kNoSlot = 0xFFFFFFFFu;

// What a request asks for.
struct Wish {
    uint64_t need;           // pages
    uint32_t past, count, held;
    bool fits;               // its rows are the step's, its pages the table row's
    __device__ __forceinline__ uint32_t gives() const { return fits && held > need ? held - static_cast<uint32_t>(need) : 0u; }
    __device__ __forceinline__ uint32_t takes() const { return fits && need > held ? static_cast<uint32_t>(need) - held : 0u; }
};

__device__ __forceinline__ Wish wish_of(const PagePlan& a, uint32_t request) {
    Wish w{0, 0, 0, 0, false};
    if (request < a.requests) {
        w.past = a.past[request], w.count = a.counts[request];
        w.held = min(a.held[request], a.table_stride);
        w.need = (uint64_t{w.past} + w.count + a.page_tokens - 1) / a.page_tokens;
    }
    return w;
}

// The sum of x over the threads before this one; the workgroup's in `total`.
// `parts`: a word a wave.
__device__ __forceinline__ uint64_t sum_before(uint64_t x, uint64_t* parts, uint64_t* total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, waves = blockDim.x / 64;
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
    for (uint32_t w = 0; w < waves; ++w) {
        if (w < wave) before += parts[w];
        all += parts[w];
    }
    *total = all;
    return before + sum - x;
}

__device__ __forceinline__ uint32_t saturated(uint64_t x) { return x < 0xFFFFFFFFull ? static_cast<uint32_t>(x) : 0xFFFFFFFFu; }

// The last of the chunk's requests whose running sum is not above i.
__device__ __forceinline__ uint32_t owner_of(const uint32_t* before, uint32_t requests, uint32_t i) {
    uint32_t low = 0, high = requests;  // before[low] <= i < before[high]
    while (high - low > 1) {
        const uint32_t middle = (low + high) / 2;
        if (before[middle] <= i)
            low = middle;
        else
            high = middle;
    }
    return low;
}

// Two of them at once.
template <uint32_t WAVES>
__device__ __forceinline__ void sums_before(uint64_t& x, uint64_t& y, uint64_t (*parts)[2], uint64_t* all_x, uint64_t* all_y) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint64_t u = x, v = y;
#pragma unroll
    for (uint32_t o = 1; o < 64; o <<= 1) {
        const uint64_t p = __shfl_up(u, o), q = __shfl_up(v, o);
        if (lane >= o) u += p, v += q;
    }
    if (lane == 63) parts[wave][0] = u, parts[wave][1] = v;
    __syncthreads();
    x = u - x, y = v - y, u = 0, v = 0;
#pragma unroll
    for (uint32_t w = 0; w < WAVES; ++w) {
        if (w < wave) x += parts[w][0], y += parts[w][1];
        u += parts[w][0], v += parts[w][1];
    }
    *all_x = u, *all_y = v;
}

// At most as many requests as threads.
template <uint32_t THREADS>
__global__ __launch_bounds__(THREADS) void page_plan_few(PagePlan a) {
    constexpr uint32_t kWaves = THREADS / 64;
    __shared__ uint64_t row_parts[kWaves][2], page_parts[kWaves][2];
    __shared__ uint32_t gives_before[THREADS], takes_before[THREADS], start[THREADS];
    __shared__ uint32_t need[THREADS], held[THREADS], past[THREADS];
    __shared__ uint8_t served_[THREADS];
    __shared__ uint32_t taken_all;
    const uint32_t request = threadIdx.x, n = a.requests;
    if (threadIdx.x == 0) taken_all = 0;
    const uint32_t free_count = *a.free_count;
    Wish w = wish_of(a, request);
    const uint32_t held_there = request < n ? a.held[request] : 0u;

    uint64_t first = w.count, nothing = 0, rows, unused;
    sums_before<kWaves>(first, nothing, row_parts, &rows, &unused);
    w.fits = (w.count == 0 || first + w.count <= a.rows) && w.need <= a.table_stride;
    uint64_t gives_at = w.gives(), takes_at = w.takes(), gives, takes;
    sums_before<kWaves>(gives_at, takes_at, page_parts, &gives, &takes);
    // the stack before, and with what is given: it holds `pages` words, whatever the tables say
    const uint32_t below = min(free_count, a.pages);
    const uint32_t given = static_cast<uint32_t>(min(gives, uint64_t{a.pages - below})), left = below + given;
    const bool served = w.fits && (w.takes() == 0 || takes_at + w.takes() <= left);
    gives_before[request] = saturated(gives_at), takes_before[request] = saturated(takes_at), start[request] = saturated(first);
    need[request] = static_cast<uint32_t>(w.need), held[request] = w.held, past[request] = w.past, served_[request] = served;
    if (request < n) {
        a.held_after[request] = served ? static_cast<uint32_t>(w.need) : held_there;
        a.granted[request] = served ? w.count : 0u;
        a.starts[request] = saturated(first);
        if (served && w.takes() > 0) atomicMax(&taken_all, static_cast<uint32_t>(takes_at + w.takes()));
    }
    __syncthreads();
    // the entry that stands at place i of what is given
    auto given_page = [&](uint32_t i) {
        const uint32_t r = owner_of(gives_before, n, i);
        return a.table[uint64_t{r} * a.table_stride + need[r] + (i - gives_before[r])];
    };
    auto taken_page = [&](uint32_t k) {
        const uint32_t at = left - 1 - k;
        return at < below ? a.free_pages[at] : given_page(at - below);
    };
    if (threadIdx.x == 0) {
        *a.free_count_after = left - taken_all;
        a.starts[n] = saturated(rows);
    }
    for (uint32_t i = threadIdx.x; i < given; i += THREADS) a.free_pages[below + i] = given_page(i);
    // those served are the first of those that take
    for (uint32_t k = threadIdx.x; k < taken_all; k += THREADS) {
        const uint32_t r = owner_of(takes_before, n, k);
        a.table[uint64_t{r} * a.table_stride + held[r] + (k - takes_before[r])] = taken_page(k);
    }
    if (a.rows > kPlanRows) return;
    for (uint32_t i = threadIdx.x; i < a.rows; i += THREADS) {
        uint32_t slot = kNoSlot, position = 0;
        if (i < rows) {
            const uint32_t r = owner_of(start, n, i);
            position = past[r] + (i - start[r]);
            if (served_[r]) {
                const uint32_t entry = position / a.page_tokens;
                const uint32_t page = entry < held[r] ? a.table[uint64_t{r} * a.table_stride + entry]
                                                      : taken_page(takes_before[r] + (entry - held[r]));
                if (page < a.pages) slot = page * a.page_tokens + position % a.page_tokens;
            }
        }
        a.slots[i] = slot;
        if (a.positions) a.positions[i] = position;
    }
}

__global__ __launch_bounds__(kPlanThreads) void page_plan(PagePlan a) {
    __shared__ uint64_t parts[kPlanThreads / 64];
    __shared__ uint32_t before[kPlanThreads], held[kPlanThreads], past[kPlanThreads], start[kPlanThreads];
    __shared__ uint8_t served_[kPlanThreads];
    __shared__ uint32_t taken_all;
    const uint32_t chunk = blockDim.x;
    uint32_t left = min(*a.free_count, a.pages);
    if (threadIdx.x == 0) taken_all = 0;

    // Pages given back.
    uint64_t rows_before = 0, gives_before = 0;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += chunk) {
        const uint32_t here = min(chunk, a.requests - r0);
        Wish w = wish_of(a, r0 + threadIdx.x);
        uint64_t rows, gives;
        const uint64_t end = rows_before + sum_before(w.count, parts, &rows) + w.count;
        w.fits = (w.count == 0 || end <= a.rows) && w.need <= a.table_stride;
        const uint64_t at = sum_before(w.gives(), parts, &gives);
        before[threadIdx.x] = saturated(at);
        held[threadIdx.x] = static_cast<uint32_t>(w.need);  // the first entry given: below table_stride where one is
        __syncthreads();
        // a stack of `pages` words holds no more, whatever the tables say
        const uint64_t room = gives_before < a.pages - left ? a.pages - left - gives_before : 0;
        for (uint64_t i = threadIdx.x; i < (gives < room ? gives : room); i += chunk) {
            const uint32_t r = owner_of(before, here, static_cast<uint32_t>(i));
            const uint64_t entry = held[r] + (i - before[r]);
            a.free_pages[left + gives_before + i] = a.table[uint64_t{r0 + r} * a.table_stride + entry];
        }
        rows_before += rows, gives_before += gives;
        __syncthreads();
    }
    left = static_cast<uint32_t>(min(uint64_t{left} + gives_before, uint64_t{a.pages}));

    // Pages taken, and the rows' slots.
    uint64_t takes_before = 0;
    rows_before = 0;
    for (uint32_t r0 = 0; r0 < a.requests; r0 += chunk) {
        const uint32_t here = min(chunk, a.requests - r0), request = r0 + threadIdx.x;
        Wish w = wish_of(a, request);
        uint64_t rows, takes;
        const uint64_t first = rows_before + sum_before(w.count, parts, &rows);
        w.fits = (w.count == 0 || first + w.count <= a.rows) && w.need <= a.table_stride;
        const uint64_t at = takes_before + sum_before(w.takes(), parts, &takes);
        const bool served = w.fits && (w.takes() == 0 || at + w.takes() <= left);
        before[threadIdx.x] = saturated(at), held[threadIdx.x] = w.held;
        past[threadIdx.x] = w.past, start[threadIdx.x] = saturated(first);
        served_[threadIdx.x] = served;
        if (request < a.requests) {
            a.held_after[request] = served ? static_cast<uint32_t>(w.need) : a.held[request];
            a.granted[request] = served ? w.count : 0u;
            a.starts[request] = saturated(first);
            if (served && w.takes() > 0) atomicMax(&taken_all, static_cast<uint32_t>(at + w.takes()));
        }
        __syncthreads();
        // those served are the first of those that take: their entries are one run
        for (uint64_t i = takes_before + threadIdx.x; i < taken_all; i += chunk) {
            const uint32_t r = owner_of(before, here, static_cast<uint32_t>(i));
            a.table[uint64_t{r0 + r} * a.table_stride + held[r] + (static_cast<uint32_t>(i) - before[r])] =
                a.free_pages[left - 1 - static_cast<uint32_t>(i)];
        }
        if (a.rows <= kPlanRows)
            for (uint64_t i = rows_before + threadIdx.x; i < min(rows_before + rows, uint64_t{a.rows}); i += chunk) {
                const uint32_t r = owner_of(start, here, static_cast<uint32_t>(i));
                const uint32_t position = past[r] + (static_cast<uint32_t>(i) - start[r]), entry = position / a.page_tokens;
                uint32_t slot = kNoSlot;
                if (served_[r]) {
                    const uint32_t page = entry < held[r] ? a.table[uint64_t{r0 + r} * a.table_stride + entry]
                                                          : a.free_pages[left - 1 - (before[r] + (entry - held[r]))];
                    if (page < a.pages) slot = page * a.page_tokens + position % a.page_tokens;
                }
                a.slots[i] = slot;
                if (a.positions) a.positions[i] = position;
            }
        rows_before += rows, takes_before += takes;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        *a.free_count_after = left - taken_all;
        a.starts[a.requests] = saturated(rows_before);
    }
    if (a.rows <= kPlanRows)
        for (uint64_t i = rows_before + threadIdx.x; i < a.rows; i += chunk) {
            a.slots[i] = kNoSlot;
            if (a.positions) a.positions[i] = 0;
        }
}

// The slots of many rows, from the table as page_plan left it.
__global__ __launch_bounds__(256) void page_slots(PagePlan a) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= a.rows) return;
    uint32_t slot = kNoSlot, position = 0;
    if (i < a.starts[a.requests]) {
        const uint32_t r = owner_of(a.starts, a.requests, i);
        position = a.past[r] + (i - a.starts[r]);
        if (a.granted[r] > 0) {
            const uint32_t page = a.table[uint64_t{r} * a.table_stride + position / a.page_tokens];
            if (page < a.pages) slot = page * a.page_tokens + position % a.page_tokens;
        }
    }
    a.slots[i] = slot;
    if (a.positions) a.positions[i] = position;
}

hipError_t launch_page_plan(const PagePlan& a, hipStream_t stream) {
    if (a.requests <= 256 && (a.rows <= 1024 || a.rows > kPlanRows))
        hipLaunchKernelGGL(page_plan_few<256>, dim3(1), dim3(256), 0, stream, a);
    else if (a.requests <= 1024)
        hipLaunchKernelGGL(page_plan_few<1024>, dim3(1), dim3(1024), 0, stream, a);
    else
        hipLaunchKernelGGL(page_plan, dim3(1), dim3(kPlanThreads), 0, stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (a.rows > kPlanRows) hipLaunchKernelGGL(page_slots, dim3((a.rows + 255) / 256), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace chm
