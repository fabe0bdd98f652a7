// Block tables and slot maps from the requests' lengths: pages given back go
// onto the stack of free pages, pages that are needed come off its top, in the
// requests' order; then each row's position and slot.
//
// Where each of these lands is a running sum over the requests - of their rows,
// of the pages they give, of the pages they take - found by one workgroup, a
// request a thread, 1,024 at a time. The entries themselves are shared among its
// threads whatever the requests' sizes: entry i is that of the last request whose
// running sum is not above i, by binary search in LDS. A slot needs no entry that
// the step writes: of a page that is taken now it reads the stack itself.
#include "requests.hpp"

namespace chm {

constexpr uint32_t kPlanThreads = 1024;
// Rows past which their slots are a launch of their own.
constexpr uint32_t kPlanRows = 8192;
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
    hipLaunchKernelGGL(page_plan, dim3(1), dim3(kPlanThreads), 0, stream, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (a.rows > kPlanRows) hipLaunchKernelGGL(page_slots, dim3((a.rows + 255) / 256), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace chm
