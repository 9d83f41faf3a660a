// Log probabilities of the next token over the vocabulary (computeLogits'
// output, inference.zig:1013-1033) on gfx950: per row the log probabilities of
// given tokens, the entropy and the `top` largest logits, in one pass over the
// row. With m the row's maximum, s = sum exp(x - m) and t = sum exp(x - m) (x - m), a token's
// log probability is (x - m) - ln s and the entropy ln s - t / s.
//
// Bound: HBM, 4 bytes per logit; for few rows the latency of two launches. A
// row is cut into pieces, so that few rows reach the whole chip: the first
// launch leaves every piece's (m, s, t) and its `top` largest logits in the
// workspace, the second joins a row's pieces. Sums are taken in a fixed order:
// nothing but the row and the number of rows decides an output. One row of
// 154880, top 20: 7.4 us and 5.3; 64 rows, top 5: 16.5 and 4.6 (a call 21, without
// the largest 12.5).
//
// The largest logits are keys of 64 bits (rank_key) that no two logits share,
// so their order is total and the order in which candidates are found does not
// matter. A wave keeps only logits that can be among the `top` largest: those
// above the piece's `top`-th so far, and not below the `top`-th largest of its
// lanes' own maxima (as many logits reach that one). What is left, two or three
// times `top` in a first chunk and few later, is ranked by counting.
#include <algorithm>

#include "device_common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"

namespace mmhip {

namespace {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr uint32_t kLpPerThread = 16, kLpChunk = kLpThreads * kLpPerThread;
constexpr uint32_t kLpMostTop = 32;
constexpr uint32_t kLpMostPieces = kLpThreads;  // a thread of the join per piece
// Pieces of a call that are enough: four workgroups per CU of the full chip (64
// rows: 21.9 us; with half as many 23.2, with twice 26.9).
constexpr uint32_t kLpPieces = 1024;

struct LpSum {
    float m, s, t;
    float unused;
};
struct LpPlan {
    uint32_t pieces, chunks;
    LpSum* sums;     // [rows][pieces]
    uint64_t* keys;  // [rows][pieces][top], largest first, 0 behind the last
};

// A logit's place in the order of the largest: larger is earlier, equal ones
// by the lower id, NaN after every number. 0: none.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t id) {
    uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as 0
    b = x != x ? 0u : (b & 0x80000000u ? ~b : b | 0x80000000u);
    return ((uint64_t)b << 32) | (0xFFFFFFFFu - id);
}
__device__ __forceinline__ uint32_t key_id(uint64_t k) { return 0xFFFFFFFFu - (uint32_t)k; }
__device__ __forceinline__ float key_logit(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return b == 0 ? __builtin_nanf("") : __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}

// The number right above a key's logit (NaN above +infinity).
__device__ __forceinline__ float above_of(uint64_t k) { return key_logit(k + (1ull << 32)); }

// Sums are taken in base 2: s = sum 2^y and t = sum 2^y y, y = (x - m) log2 e.
// The product's rounding moves a term by |y| 2^-24 ln 2 of its size at most, up
// or down: a part in 10^6 where y = -24, and what lies further down weighs
// nothing. log2 e enters in two parts: rounded to f32 it is 1.3e-8 too small,
// which would move all terms to one side.
constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596300e-8f;
__device__ __forceinline__ float in_base2(float d) { return fmaf(d, kLog2e, d * kLog2eRest); }
// What a part's weight 2^y, y = (m - M) log2 e, makes of its sums at the larger
// maximum M. Without weight it adds nothing to t, but a NaN in s stays one.
__device__ __forceinline__ void rebase(LpSum& a, float m) {
    if (a.m == m) return;
    const float y = in_base2(a.m - m), f = __builtin_amdgcn_exp2f(y);
    a.t = f == 0.0f ? 0.0f : f * (a.t + a.s * y);
    a.s *= f;
    a.m = m;
}
// Over the workgroup, in a fixed order. For every thread.
__device__ __forceinline__ LpSum join_all(LpSum v, LpSum* red) {
    rebase(v, group_max<64>(v.m));
    v.s = group_sum<64>(v.s);
    v.t = group_sum<64>(v.t);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    LpSum all{-INFINITY, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) all.m = fmaxf(all.m, red[w].m);
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) {
        LpSum o = red[w];
        rebase(o, all.m);
        all.s += o.s;
        all.t += o.t;
    }
    return all;
}

// The `top`-th largest of the lanes' keys (0: none); at least `top` of them
// are not 0. Two that are not 0 differ, so exactly one lane has that rank.
__device__ __forceinline__ uint64_t wave_kth(uint64_t key, uint32_t top) {
    uint32_t above = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) {
        const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)key, i), hi = __builtin_amdgcn_readlane((uint32_t)(key >> 32), i);
        above += (((uint64_t)hi << 32) | lo) > key;
    }
    const int at = __ffsll((unsigned long long)__ballot(above == top - 1 && key != 0)) - 1;
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(key >> 32), at) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((uint32_t)key, at);
}

// Of the lanes' numbers, the `top`-th largest: false where equal ones, NaN or
// infinite ones leave it undecided which `top` lanes reach it.
__device__ __forceinline__ bool wave_kth(float m, uint32_t top, float& kth) {
    uint32_t above = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) above += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m), i)) > m;
    const uint64_t at = __ballot(above == top - 1 && m > -INFINITY);
    if (__popcll(at) != 1) return false;
    kth = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m), __ffsll((unsigned long long)at) - 1));
    return true;
}

// The `top` largest of list[0, n), largest first, into out, 0 behind the last.
// list has room for kRankStep - 1 keys more. Begins with a barrier.
constexpr uint32_t kRankStep = 16;
__device__ __forceinline__ void rank_list(uint64_t* list, uint32_t n, uint64_t* out, uint32_t top) {
    if (threadIdx.x < kRankStep - 1) list[n + threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < max(n, top); i += kLpThreads) {
        if (i >= n) {
            out[i] = 0;
            continue;
        }
        const uint64_t mine = list[i];
        uint32_t above = 0;
        for (uint32_t j = 0; j < n; j += kRankStep)
#pragma unroll
            for (uint32_t e = 0; e < kRankStep; ++e) above += list[j + e] > mine;
        if (above < top) out[above] = mine;
    }
}

// Appends the lanes' keys key(i), i < N, of which want(i) holds to the list.
template <int N, class Want, class Key>
__device__ __forceinline__ void keep(Want want, Key key, uint64_t* list, uint32_t* kept) {
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += (uint32_t)__popcll(__ballot(want(i)));
    if (n == 0) return;
    uint32_t at = 0;
    if ((threadIdx.x & 63) == 0) at = atomicAdd(kept, n);
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint64_t mask = __ballot(want(i));
        if (mask == 0) continue;
        if (want(i)) list[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = key(i);
        at += (uint32_t)__popcll(mask);
    }
}

// The most a chunk keeps: of each wave fewer than `top` lanes that pass the
// piece's `top`-th, or exactly `top` lanes that reach the wave's; and the
// piece's own `top`.
constexpr uint32_t kLpMostKept = kLpWaves * kLpMostTop * kLpPerThread + kLpMostTop + kRankStep;

// One workgroup per piece.
__global__ __launch_bounds__(kLpThreads) void logprobs_split_kernel(LogprobsArgs a, LpPlan p) {
    __shared__ LpSum red[kLpWaves];
    __shared__ uint64_t list[kLpMostKept];
    __shared__ uint64_t best[kLpMostTop];
    __shared__ uint32_t kept[2];
    const uint64_t row = blockIdx.x / p.pieces;
    const uint32_t piece = blockIdx.x - (uint32_t)row * p.pieces;
    const uint32_t c0 = (uint32_t)((uint64_t)piece * p.chunks / p.pieces);
    const uint32_t c1 = (uint32_t)((uint64_t)(piece + 1) * p.chunks / p.pieces);
    const float* x = a.logits + row * a.stride;
    const uint32_t top = a.top, tid = threadIdx.x;
    if (tid < kLpMostTop) best[tid] = 0;
    if (tid < 2) kept[tid] = 0;
    LpSum sum{-INFINITY, 0.0f, 0.0f, 0.0f};
    uint64_t floor_key = 0;  // the piece's `top`-th so far
    __syncthreads();
    // Thread t has logits t + 256 i of a chunk, the next one's on their way
    // while it works on one (nothing is read where there is none).
    uint32_t pre[kLpPerThread];
    const auto read = [&](uint32_t c) {
        const uint32_t first = c * kLpChunk;
        const BufRsrc r = make_rsrc(x + first, c < c1 ? min(a.vocab - first, kLpChunk) * 4 : 0);
#pragma unroll
        for (uint32_t i = 0; i < kLpPerThread; ++i) pre[i] = buf_load_b32<kCacheStream>(r, tid * 4, i * (kLpThreads * 4));
    };
    read(c0);
    for (uint32_t c = c0; c < c1; ++c) {
        const uint32_t first = c * kLpChunk, n = min(a.vocab - first, kLpChunk);
        float v[kLpPerThread];
#pragma unroll
        for (uint32_t i = 0; i < kLpPerThread; ++i) v[i] = tid + i * kLpThreads < n ? __uint_as_float(pre[i]) : -INFINITY;
        read(c + 1);
        float m = v[0];
#pragma unroll
        for (uint32_t i = 1; i < kLpPerThread; ++i) m = fmaxf(m, v[i]);  // leaves NaN out
        {
            const float old = sum.m;
            LpSum here{fmaxf(old, m), 0.0f, 0.0f, 0.0f};
            const float base = here.m == -INFINITY ? 0.0f : here.m;
#pragma unroll
            for (uint32_t i = 0; i < kLpPerThread; ++i) {
                // (below y = -256 e is 0; a NaN stays one in e)
                const float y = in_base2(v[i] - base), e = __builtin_amdgcn_exp2f(y);
                here.s += e;
                here.t = fmaf(e, fmaxf(y, -256.0f), here.t);
            }
            rebase(sum, here.m);
            sum.s += here.s;
            sum.t += here.t;
        }
        if (top == 0) continue;
        // Lanes with a number above the floor's (which may be a NaN's, or none
        // yet: NaN, which bars nothing). An equal one comes later in the order.
        const float floor_x = key_logit(floor_key);
        const uint32_t pass = (uint32_t)__popcll(__ballot(m == m && !(m <= floor_x)));
        float least_x = above_of(floor_key);
        bool plain = floor_x == floor_x;
        if (pass >= top) plain = wave_kth(m, top, least_x);
        if (plain) {
            // Compared as numbers. None of the absent: least_x is above -infinity.
            if (pass)
                keep<kLpPerThread>([&](int i) { return v[i] >= least_x; },
                                   [&](int i) { return rank_key(v[i], first + tid + i * kLpThreads); }, list, &kept[c & 1]);
        } else {
            // Equal maxima, or NaN among the largest: as keys.
            uint64_t k[kLpPerThread], key = 0;
#pragma unroll
            for (uint32_t i = 0; i < kLpPerThread; ++i) {
                const uint32_t at = tid + i * kLpThreads;
                k[i] = at < n ? rank_key(v[i], first + at) : 0;
                key = max(key, k[i]);
            }
            if (key <= floor_key) key = 0;
            uint64_t least = floor_key + 1;
            if ((uint32_t)__popcll(__ballot(key != 0)) >= top) least = wave_kth(key, top);
            keep<kLpPerThread>([&](int i) { return k[i] >= least; }, [&](int i) { return k[i]; }, list, &kept[c & 1]);
        }
        __syncthreads();
        uint32_t found = kept[c & 1];
        if (tid == 0) kept[(c + 1) & 1] = 0;
        if (found) {
            // The piece's own behind them.
            if (tid < top && best[tid]) list[found + tid] = best[tid];
            found += (uint32_t)__popcll(__ballot((tid & 63) < top && best[tid & 63]));
            rank_list(list, found, best, top);
        }
        __syncthreads();
        floor_key = best[top - 1];
    }
    sum = join_all(sum, red);
    if (tid == 0) p.sums[row * p.pieces + piece] = sum;
    if (tid < top) p.keys[(row * p.pieces + piece) * top + tid] = best[tid];
}

// One workgroup per row.
__global__ __launch_bounds__(kLpThreads) void logprobs_join_kernel(LogprobsArgs a, LpPlan p) {
    __shared__ LpSum red[kLpWaves];
    __shared__ uint64_t list[kLpMostPieces / 64 * kLpMostTop * kLpMostTop + kRankStep];
    __shared__ uint64_t best[kLpMostTop];
    __shared__ uint32_t kept;
    const uint64_t row = blockIdx.x;
    const float* x = a.logits + row * a.stride;
    const uint32_t top = a.top, tid = threadIdx.x, lane = tid & 63;
    if (tid == 0) kept = 0;
    LpSum sum{-INFINITY, 0.0f, 0.0f, 0.0f};
    if (tid < p.pieces) sum = p.sums[row * p.pieces + tid];
    sum = join_all(sum, red);
    // The logarithm and what follows in 64 bits, rounded once: logf is up to two
    // units too small and hardly ever too large (half a unit on average).
    const double log_s = log((double)sum.s);
    const auto log_prob = [&](float x) { return (float)(((double)x - (double)sum.m) - log_s); };
    if (a.entropy && tid == 0) a.entropy[row] = (float)(log_s - M_LN2 * ((double)sum.t / (double)sum.s));
    for (uint64_t i = tid; i < a.n_given; i += kLpThreads) {
        const uint32_t id = a.tokens[row * a.n_given + i];
        if (id >= a.vocab) report(a.status, kBadToken);
        a.token_logprobs[row * a.n_given + i] = id < a.vocab ? log_prob(x[id]) : __builtin_nanf("");
    }
    if (top == 0) return;
    // 64 keys, the largest of each piece (of every 64th piece) and where there
    // are fewer pieces their next ones: the `top`-th largest of these is a
    // floor. Every wave finds it for itself.
    const uint64_t* keys = p.keys + row * p.pieces * top;
    uint64_t largest = 0;
    if (p.pieces >= 64) {
        for (uint32_t i = lane; i < p.pieces; i += 64) largest = max(largest, keys[(uint64_t)i * top]);
    } else if (lane / p.pieces < top) {
        largest = keys[lane % p.pieces * top + lane / p.pieces];
    }
    uint64_t least = 1;
    if ((uint32_t)__popcll(__ballot(largest != 0)) >= top) least = wave_kth(largest, top);
    for (uint32_t i = tid; i < (p.pieces * top + 63) / 64 * 64; i += kLpThreads) {
        const uint64_t k = i < p.pieces * top ? keys[i] : 0;
        keep<1>([&](int) { return k >= least; }, [&](int) { return k; }, list, &kept);
    }
    __syncthreads();
    rank_list(list, kept, best, top);
    __syncthreads();
    if (tid < top) {
        a.top_ids[row * top + tid] = key_id(best[tid]);
        if (a.top_logprobs) a.top_logprobs[row * top + tid] = log_prob(key_logit(best[tid]));
    }
}

LpPlan lp_plan(uint64_t n_rows, uint64_t vocab) {
    LpPlan p{};
    p.chunks = (uint32_t)((vocab + kLpChunk - 1) / kLpChunk);
    const uint64_t want = (kLpPieces + n_rows - 1) / n_rows;
    p.pieces = (uint32_t)std::min<uint64_t>(std::min<uint64_t>(want, kLpMostPieces), p.chunks);
    return p;
}
uint64_t up16(uint64_t v) { return (v + 15) / 16 * 16; }

}  // namespace

uint64_t logprobs_workspace_bytes(uint64_t n_rows, uint64_t vocab, uint32_t top) {
    if (n_rows == 0 || vocab == 0) return 0;
    const LpPlan p = lp_plan(n_rows, vocab);
    return n_rows * p.pieces * sizeof(LpSum) + up16(n_rows * p.pieces * top * 8);
}

hipError_t launch_logprobs(const LogprobsArgs& a, uint64_t n_rows, hipStream_t s) {
    if (n_rows == 0) return hipSuccess;
    LpPlan p = lp_plan(n_rows, a.vocab);
    p.sums = static_cast<LpSum*>(a.work);
    p.keys = reinterpret_cast<uint64_t*>(p.sums + n_rows * p.pieces);
    logprobs_split_kernel<<<(unsigned)(n_rows * p.pieces), kLpThreads, 0, s>>>(a, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    logprobs_join_kernel<<<(unsigned)n_rows, kLpThreads, 0, s>>>(a, p);
    return hipGetLastError();
}

}  // namespace mmhip
