// Page tables, slots and positions of a step's tokens from the requests'
// lengths (the bookkeeping of KVCache's blocks, kv_cache.zig:24-141, 279-362,
// and of BatchScheduler, batch_queue.zig:75-232) on gfx950.
//
// Three running sums over the requests decide everything: tokens asked for,
// pages asked for, tokens granted. One workgroup takes them; small calls write
// the step's tokens in the same launch, larger ones in a second one over the
// whole chip. All counts are integers: nothing depends on timing.
//
// Bound: latency. One workgroup's chain is a trip to memory for the lengths, three
// sums (a barrier each), a trip for the pages that come back and one for the
// tables, about a microsecond each: 4 requests 3.8 us, 64 4.8 to 6.1, 500 with 2400
// tokens 8.7. 512 requests with 64 prompts (110 thousand tokens) take three
// dependent launches: 4.5, 2.4 and 4.3, together 11.1.
#include "device_common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"

namespace mmhip {

namespace {

// Threads of the launch over requests; where there are few requests and tokens fewer
// of them, whose barriers are shorter (4 requests 3.8 against 5.2 us, 64 with 93 tokens
// 4.8 and 6.1, with 64 both 6.1; beyond, 250 requests 7.5 and 6.9).
constexpr uint32_t kPlanThreads = 1024, kPlanFew = 256;
// Tokens that the same launch writes: 500 requests with 2387 tokens 8.7 us, in three
// launches 10.1 to 11.5; 900 with 6092 (beyond) 13.2 and 11.4.
constexpr uint32_t kPlanSmall = 4096;
constexpr uint32_t kPlanFill = 256;
constexpr uint32_t kPlanStarts = 2048;                   // of the requests' first tokens, in LDS

__device__ __forceinline__ uint32_t pages_of(const PlanArgs& a, uint64_t positions) {
    return (uint32_t)((positions + ((1u << a.page_shift) - 1)) >> a.page_shift);
}

// Token t of request r at position pos: its outputs, and a new page's table entry.
__device__ __forceinline__ void place(const PlanArgs& a, uint32_t t, uint32_t r, uint32_t pos, uint32_t held, const PlanRow& row,
                                      uint32_t top) {
    const uint32_t page = pos >> a.page_shift, at = pos & ((1u << a.page_shift) - 1);
    int32_t* entry = a.tables + (uint64_t)r * a.table_stride + page;
    int32_t id;
    if (page < held) {
        id = *entry;
    } else {
        id = a.free[top - 1 - (row.pages + (page - held))];
        if (at == 0) *entry = id;
    }
    const bool ok = id >= 0 && (uint32_t)id < a.n_pages;
    if (!ok) report(a.status, kBadPlanPage);
    a.positions[t] = pos;
    a.slots[t] = ok ? (int32_t)(((uint32_t)id << a.page_shift) | at) : -1;
    a.table_of[t] = r;
    a.seen[t] = pos + 1;
}
__device__ __forceinline__ void pad(const PlanArgs& a, uint32_t t) {
    a.positions[t] = 0;
    a.slots[t] = -1;
    a.table_of[t] = 0;
    a.seen[t] = 0;
}

// The last of n ascending starts that is not behind t; starts[0] is not.
__device__ __forceinline__ uint32_t last_start(const uint32_t* starts, uint32_t n, uint32_t t) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Gives request r's pages back: free[row.back_at ..).
__device__ __forceinline__ void give_page(const PlanArgs& a, uint32_t r, const PlanRow& row, uint32_t i) {
    a.free[row.back_at + i] = a.tables[(uint64_t)r * a.table_stride + row.back_from + i];
}
__device__ __forceinline__ void give_back(const PlanArgs& a, uint32_t r, uint32_t i0, uint32_t step) {
    const PlanRow row = a.work[r];
    for (uint32_t i = i0; i < row.back; i += step) give_page(a, r, row, i);
}

// What one workgroup keeps of its requests where it does the whole call.
template <uint32_t N>
struct PlanHeld {
    PlanRow rows[N];
    uint32_t starts[N], backs[N];  // the tokens granted and the pages given back before each
};
struct PlanTotals {
    uint32_t top, tokens, backs;  // free pages before any is taken
};

// The requests' running sums: firsts, granted, last, next_lens, the rows and the
// new count of free pages. With `held` there are at most THREADS requests, and the
// rows stay there.
template <uint32_t THREADS>
__device__ __forceinline__ PlanTotals plan_requests(const PlanArgs& a, PlanHeld<THREADS>* held) {
    __shared__ uint64_t memory[2][2][THREADS / 64];
    Together<THREADS / 64> together{memory};
    const uint64_t capacity = (uint64_t)a.table_pages << a.page_shift;
    const bool once = held != nullptr;
    uint32_t count = *a.free_count;
    PlanRow row{};
    uint32_t add = 0;
    // Pages that come back, tokens asked for.
    uint64_t back_all = 0, asked_all = 0;
    uint32_t fits = 0;  // the last row's
    for (uint32_t r0 = 0; r0 < a.n_requests; r0 += THREADS) {
        const uint32_t r = r0 + threadIdx.x;
        uint64_t len = 0;
        row = PlanRow{};
        add = 0;
        if (r < a.n_requests) {
            len = a.lens[r];
            add = a.added[r];
            const uint32_t release = a.release ? a.release[r] : 0, shared = a.shared ? a.shared[r] : 0;
            if (len > capacity) report(a.status, kBadPlanLength);
            if (release) {
                const uint32_t pages = min(pages_of(a, len), a.table_pages);
                row.back_from = min(shared, pages);
                row.back = pages - row.back_from;
                len = 0;
            }
            if (add > 0 && len + add > capacity) {
                report(a.status, kBadPlanLength);
                add = 0;
            }
        }
        row.start = (uint32_t)len;
        uint64_t back = row.back, asked = add, all_back, all_asked;
        together.scan2(back, asked, all_back, all_asked);
        if (add && asked_all + asked > a.max_tokens) {
            add = 0;
            report(a.status, kBadPlanTokens);
        }
        fits = add;
        // No more than the stack holds (a length may name more pages than the pool has).
        const uint64_t backs = back_all + back - row.back, before = (uint64_t)min(count, a.n_pages) + backs;
        row.back_at = (uint32_t)min(before, (uint64_t)a.n_pages);
        row.back = min(row.back, a.n_pages - row.back_at);
        row.pages = fits;  // until the second sweep
        if (!once && r < a.n_requests) a.work[r] = row;
        if (once) held->backs[threadIdx.x] = (uint32_t)min(backs, (uint64_t)0xFFFFFFFFu);
        back_all += all_back;
        asked_all += all_asked;
    }
    if (count > a.n_pages) {
        if (threadIdx.x == 0) report(a.status, kBadPlanFree);
        count = a.n_pages;
    }
    uint64_t top64 = count + back_all;
    if (top64 > a.n_pages) {
        if (threadIdx.x == 0) report(a.status, kBadPlanFree);
        top64 = a.n_pages;
    }
    const uint32_t top = (uint32_t)top64;
    // Pages asked for, tokens granted and pages taken.
    uint64_t need_all = 0, given_all = 0, taken = 0;
    for (uint32_t r0 = 0; r0 < a.n_requests; r0 += THREADS) {
        const uint32_t r = r0 + threadIdx.x;
        if (!once) {
            row = r < a.n_requests ? a.work[r] : PlanRow{};
            fits = row.pages;
        }
        const uint64_t len = row.start;
        const uint32_t need = fits ? pages_of(a, len + fits) - pages_of(a, len) : 0;
        uint64_t pages = need, all;
        uint64_t none = 0;
        pages = together.scan(pages, all, none);
        if (need && need_all + pages > top) fits = 0;
        const uint64_t before = need_all + pages - need;
        need_all += all;
        uint64_t given = fits, all_given, took = fits ? need : 0;
        given = together.scan(given, all_given, took);
        if (r < a.n_requests) {
            const uint32_t first = (uint32_t)(given_all + given - fits);
            a.firsts[r] = first;
            a.granted[r] = fits != 0;
            if (a.last) a.last[r] = fits ? first + fits - 1 : kNoToken;
            row.pages = (uint32_t)min(before, (uint64_t)a.n_pages);
            if (once) {
                held->starts[r] = first;
                held->rows[r] = row;
            } else {
                a.work[r] = row;
            }
            a.next_lens[r] = (uint32_t)(len + fits);
        }
        given_all += all_given;
        taken += took;
    }
    if (threadIdx.x == 0) {
        a.firsts[a.n_requests] = (uint32_t)given_all;
        *a.next_free_count = top - (uint32_t)taken;
        if (!once) *a.top = top;
    }
    return {top, (uint32_t)given_all, top - count};
}

template <uint32_t THREADS>
__global__ __launch_bounds__(THREADS) void plan_small_kernel(PlanArgs a) {
    __shared__ PlanHeld<THREADS> held;
    const PlanTotals all = plan_requests<THREADS>(a, &held);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < all.backs; i += THREADS) {
        const uint32_t r = last_start(held.backs, a.n_requests, i);
        give_page(a, r, held.rows[r], i - held.backs[r]);
    }
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < a.max_tokens; t += THREADS) {
        if (t >= all.tokens) {
            pad(a, t);
            continue;
        }
        const uint32_t r = last_start(held.starts, a.n_requests, t);
        const PlanRow row = held.rows[r];
        place(a, t, r, row.start + (t - held.starts[r]), pages_of(a, row.start), row, all.top);
    }
}

__global__ __launch_bounds__(kPlanThreads) void plan_requests_kernel(PlanArgs a) { (void)plan_requests<kPlanThreads>(a, nullptr); }
__global__ __launch_bounds__(256) void plan_back_kernel(PlanArgs a) { give_back(a, blockIdx.x, threadIdx.x, 256); }
// starts: of requests 0, 1 << shift, ...
__global__ __launch_bounds__(kPlanFill) void plan_fill_kernel(PlanArgs a, uint32_t shift) {
    __shared__ uint32_t starts[kPlanStarts];
    const uint32_t total = a.firsts[a.n_requests], top = *a.top;
    uint32_t n = 0;
    if (a.n_requests) n = ((a.n_requests - 1) >> shift) + 1;
    for (uint32_t i = threadIdx.x; i < n; i += kPlanFill) starts[i] = a.firsts[i << shift];
    __syncthreads();
    const uint32_t t = blockIdx.x * kPlanFill + threadIdx.x;
    if (t >= a.max_tokens) return;
    if (t >= total) return pad(a, t);
    uint32_t r = last_start(starts, n, t), first = starts[r];
    if (shift) {
        r <<= shift;
        r += last_start(a.firsts + r, min(1u << shift, a.n_requests - r), t);
        first = a.firsts[r];
    }
    const PlanRow row = a.work[r];
    place(a, t, r, row.start + (t - first), pages_of(a, row.start), row, top);
}

}  // namespace

uint64_t plan_workspace_bytes(uint32_t n_requests) { return 16 + (uint64_t)n_requests * sizeof(PlanRow); }

hipError_t launch_kv_plan(const PlanArgs& a_in, void* work, hipStream_t s) {
    PlanArgs a = a_in;
    a.top = static_cast<uint32_t*>(work);
    a.work = reinterpret_cast<PlanRow*>(static_cast<uint8_t*>(work) + 16);
    if (a.n_requests <= kPlanFew / 2 && a.max_tokens <= kPlanFew) {
        plan_small_kernel<kPlanFew><<<1, kPlanFew, 0, s>>>(a);
        return hipGetLastError();
    }
    if (a.n_requests <= kPlanThreads && a.max_tokens <= kPlanSmall) {
        plan_small_kernel<kPlanThreads><<<1, kPlanThreads, 0, s>>>(a);
        return hipGetLastError();
    }
    plan_requests_kernel<<<1, kPlanThreads, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.release && a.n_requests) {
        plan_back_kernel<<<a.n_requests, 256, 0, s>>>(a);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a.max_tokens) {
        uint32_t shift = 0;
        while ((((uint64_t)a.n_requests + (1u << shift) - 1) >> shift) > kPlanStarts) ++shift;
        plan_fill_kernel<<<(unsigned)(((uint64_t)a.max_tokens + kPlanFill - 1) / kPlanFill), kPlanFill, 0, s>>>(a, shift);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace mmhip
