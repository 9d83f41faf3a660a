// Page tables, slots and positions of a step's tokens from the requests'
// lengths (the bookkeeping of KVCache's blocks, kv_cache.zig:24-141, 279-362,
// and of BatchScheduler, batch_queue.zig:75-232) on gfx950.
//
// Three running sums over the requests decide everything: tokens asked for,
// pages asked for, tokens granted. One workgroup takes them; small calls write
// the step's tokens in the same launch, larger ones in a second one over the
// whole chip. All counts are integers: nothing depends on timing.
#include "device_common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"

namespace mmhip {

namespace {

constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

// The sum over threads 0 .. this one, and over all. Two barriers.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* red, uint64_t& all) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t in = wave_scan(v);
    if (lane == 63) red[wave] = in;
    __syncthreads();
    uint64_t before = 0;
    all = 0;
    for (uint32_t w = 0; w < kPlanWaves; ++w) {
        if (w < wave) before += red[w];
        all += red[w];
    }
    __syncthreads();
    return before + in;
}

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

// Token t < the total: the request it belongs to, the last one whose first
// token is not behind t.
__device__ __forceinline__ uint32_t request_of(const uint32_t* firsts, uint32_t n, uint32_t t) {
    uint32_t lo = 0, hi = n;  // firsts[lo] <= t < firsts[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (firsts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ void fill_token(const PlanArgs& a, uint32_t t, uint32_t top) {
    const uint32_t total = a.firsts[a.n_requests];
    if (t >= total) return pad(a, t);
    const uint32_t r = request_of(a.firsts, a.n_requests, t);
    const PlanRow row = a.work[r];
    const uint32_t pos = row.start + (t - a.firsts[r]);
    place(a, t, r, pos, pages_of(a, row.start), row, top);
}

// Gives request r's pages back: free[row.back_at ..).
__device__ __forceinline__ void give_back(const PlanArgs& a, uint32_t r, uint32_t i0, uint32_t step) {
    const PlanRow row = a.work[r];
    for (uint32_t i = i0; i < row.back; i += step) {
        const uint64_t at = (uint64_t)row.back_at + i;
        if (at < a.n_pages) a.free[at] = a.tables[(uint64_t)r * a.table_stride + row.back_from + i];
    }
}

// The requests' running sums: firsts, granted, last, next_lens, the workspace's
// rows and the new count of free pages. *top: free pages before any is taken.
__device__ __forceinline__ uint32_t plan_requests(const PlanArgs& a) {
    __shared__ uint64_t red[kPlanWaves];
    const uint64_t capacity = (uint64_t)a.table_pages << a.page_shift;
    uint32_t count = *a.free_count;
    if (count > a.n_pages) {
        if (threadIdx.x == 0) report(a.status, kBadPlanFree);
        count = a.n_pages;
    }
    // Pages that come back.
    uint64_t back_all = 0;
    for (uint32_t r0 = 0; r0 < a.n_requests; r0 += kPlanThreads) {
        const uint32_t r = r0 + threadIdx.x;
        uint32_t back = 0, from = 0;
        uint64_t len = 0;
        if (r < a.n_requests) {
            len = a.lens[r];
            if (len > capacity) {
                report(a.status, kBadPlanLength);
            }
            if (a.release && a.release[r]) {
                const uint32_t held = min(pages_of(a, len), a.table_pages);
                from = a.shared ? min(a.shared[r], held) : 0;
                back = held - from;
                len = 0;
            }
        }
        uint64_t all;
        const uint64_t in = block_scan(back, red, all);
        if (r < a.n_requests) {
            PlanRow row;
            row.start = (uint32_t)len;
            row.pages = 0;
            row.back = back;
            row.back_from = from;
            row.back_at = (uint32_t)min<uint64_t>(count + back_all + in - back, a.n_pages);
            a.work[r] = row;
        }
        back_all += all;
    }
    uint64_t top64 = count + back_all;
    if (top64 > a.n_pages) {
        if (threadIdx.x == 0) report(a.status, kBadPlanFree);
        top64 = a.n_pages;
    }
    const uint32_t top = (uint32_t)top64;
    // Tokens and pages asked for, tokens granted.
    uint64_t asked_all = 0, need_all = 0, given_all = 0, taken = 0;
    for (uint32_t r0 = 0; r0 < a.n_requests; r0 += kPlanThreads) {
        const uint32_t r = r0 + threadIdx.x;
        uint64_t len = 0, add = 0;
        bool ok = false;
        if (r < a.n_requests) {
            len = a.work[r].start;
            add = a.added[r];
            ok = add > 0 && len + add <= capacity;
            if (add > 0 && !ok) report(a.status, kBadPlanLength);
        }
        uint64_t all;
        uint64_t in = block_scan(ok ? add : 0, red, all);
        if (ok && asked_all + in > a.max_tokens) {
            ok = false;
            report(a.status, kBadPlanTokens);
        }
        asked_all += all;
        const uint32_t need = ok ? pages_of(a, len + add) - pages_of(a, len) : 0;
        in = block_scan(need, red, all);
        if (need && need_all + in > top) ok = false;
        const uint64_t pages = need_all + in - need;
        need_all += all;
        const uint64_t mine = (ok && need ? (uint64_t)need << 32 : 0) | (ok ? add : 0);
        in = block_scan(mine, red, all);
        if (r < a.n_requests) {
            const uint32_t first = (uint32_t)(given_all + (uint32_t)(in - mine));
            a.firsts[r] = first;
            a.granted[r] = ok;
            if (a.last) a.last[r] = ok ? first + (uint32_t)add - 1 : kNoToken;
            a.work[r].pages = (uint32_t)min<uint64_t>(pages, a.n_pages);
            a.next_lens[r] = (uint32_t)(len + (ok ? add : 0));
        }
        given_all += (uint32_t)all;
        taken += all >> 32;
    }
    if (threadIdx.x == 0) {
        a.firsts[a.n_requests] = (uint32_t)given_all;
        *a.next_free_count = top - (uint32_t)taken;
        *a.top = top;
    }
    return top;
}

__global__ __launch_bounds__(kPlanThreads) void plan_small_kernel(PlanArgs a) {
    const uint32_t top = plan_requests(a);
    __syncthreads();
    if (a.release) {
        for (uint32_t r = threadIdx.x >> 6; r < a.n_requests; r += kPlanWaves) give_back(a, r, threadIdx.x & 63, 64);
        __syncthreads();
    }
    for (uint32_t t = threadIdx.x; t < a.max_tokens; t += kPlanThreads) fill_token(a, t, top);
}

__global__ __launch_bounds__(kPlanThreads) void plan_requests_kernel(PlanArgs a) { (void)plan_requests(a); }
__global__ __launch_bounds__(256) void plan_back_kernel(PlanArgs a) { give_back(a, blockIdx.x, threadIdx.x, 256); }
__global__ __launch_bounds__(256) void plan_fill_kernel(PlanArgs a) {
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    if (t < a.max_tokens) fill_token(a, t, *a.top);
}

}  // namespace

uint64_t plan_workspace_bytes(uint32_t n_requests) { return 16 + (uint64_t)n_requests * sizeof(PlanRow); }

hipError_t launch_kv_plan(const PlanArgs& a_in, void* work, hipStream_t s) {
    PlanArgs a = a_in;
    a.top = static_cast<uint32_t*>(work);
    a.work = reinterpret_cast<PlanRow*>(static_cast<uint8_t*>(work) + 16);
    if (a.n_requests <= kPlanThreads && a.max_tokens <= 4096) {
        plan_small_kernel<<<1, kPlanThreads, 0, s>>>(a);
        return hipGetLastError();
    }
    plan_requests_kernel<<<1, kPlanThreads, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.release && a.n_requests) {
        plan_back_kernel<<<a.n_requests, 256, 0, s>>>(a);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a.max_tokens) {
        plan_fill_kernel<<<(unsigned)(((uint64_t)a.max_tokens + 255) / 256), 256, 0, s>>>(a);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace mmhip
