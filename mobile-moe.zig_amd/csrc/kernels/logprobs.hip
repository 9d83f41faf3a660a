// Log probabilities of the next token over the vocabulary (computeLogits'
// output, inference.zig:1013-1033) on gfx950: per row the log probabilities of
// given tokens, the entropy and the `top` largest logits, in one pass over the
// row. With m the row's maximum, s = sum exp(x - m) and t = sum exp(x - m) (x - m),
// a token's log probability is (x - m) - ln s and the entropy ln s - t / s.
//
// Bound: HBM, 4 bytes per logit; for few rows the latency of two launches. A
// row is cut into pieces, so that few rows reach the whole chip: the first
// launch leaves every piece's (m, s, t) and its `top` largest logits in the
// workspace, the second joins a row's pieces. Sums are taken in a fixed order:
// nothing but the row and the number of rows decides an output.
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

namespace mmhip {

namespace {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr uint32_t kLpPerThread = 16, kLpChunk = kLpThreads * kLpPerThread;
constexpr uint32_t kLpMostTop = 32;
constexpr uint32_t kLpMostPieces = kLpThreads;  // a thread of the join per piece
// Pieces of a call that are enough: four workgroups per CU of the full chip.
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

// Adds a part (m, s, t) to another. A part without weight at the new maximum
// adds nothing to t, but a NaN in its sum stays one.
__device__ __forceinline__ void join(LpSum& a, const LpSum& b) {
    const float m = fmaxf(a.m, b.m), da = a.m - m, db = b.m - m;
    const float fa = a.m == m ? 1.0f : expf(da), fb = b.m == m ? 1.0f : expf(db);
    const float ta = fa == 0.0f ? 0.0f : (a.m == m ? a.t : fa * (a.t + a.s * da));
    const float tb = fb == 0.0f ? 0.0f : (b.m == m ? b.t : fb * (b.t + b.s * db));
    a.m = m;
    a.s = a.s * fa + b.s * fb;
    a.t = ta + tb;
}
// Over the workgroup: a wave's lanes, then the waves, in a fixed order (lane
// 0's). For every thread.
__device__ __forceinline__ LpSum join_all(LpSum v, LpSum* red) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        LpSum o;
        o.m = __shfl_xor(v.m, off, 64);
        o.s = __shfl_xor(v.s, off, 64);
        o.t = __shfl_xor(v.t, off, 64);
        join(v, o);
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < kLpWaves; ++w) join(v, red[w]);
    return v;
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

// The `top` largest of list[0, n), largest first, into out, 0 behind the last.
// Between two barriers of the caller's.
__device__ __forceinline__ void rank_list(const uint64_t* list, uint32_t n, uint64_t* out, uint32_t top) {
    for (uint32_t i = threadIdx.x; i < max(n, top); i += kLpThreads) {
        if (i >= n) {
            out[i] = 0;
            continue;
        }
        const uint64_t mine = list[i];
        uint32_t above = 0;
        for (uint32_t j = 0; j < n; ++j) above += list[j] > mine;
        if (above < top) out[above] = mine;
    }
}

// The most a chunk keeps: of each wave fewer than `top` lanes that pass the
// piece's `top`-th, or exactly `top` lanes that reach the wave's; and the
// piece's own `top`.
constexpr uint32_t kLpMostKept = kLpWaves * kLpMostTop * kLpPerThread + kLpMostTop;

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
    for (uint32_t c = c0; c < c1; ++c) {
        // Thread t has logits 4 t .. 4 t + 3 of each quarter of the chunk.
        const uint32_t first = c * kLpChunk, n = min(a.vocab - first, kLpChunk);
        const BufRsrc r = make_rsrc(x + first, n * 4);
        float v[kLpPerThread];
        if (n == kLpChunk) {
#pragma unroll
            for (uint32_t j = 0; j < kLpPerThread / 4; ++j) {
                const uint4 q = buf_load_b128<kCacheStream>(r, tid * 16, j * kLpThreads * 16);
                v[4 * j] = __uint_as_float(q.x);
                v[4 * j + 1] = __uint_as_float(q.y);
                v[4 * j + 2] = __uint_as_float(q.z);
                v[4 * j + 3] = __uint_as_float(q.w);
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kLpPerThread; ++i) {
                const uint32_t at = tid * 4 + (i >> 2) * (kLpThreads * 4) + (i & 3);
                const uint32_t q = buf_load_b32<kCacheStream>(r, at * 4, 0);
                v[i] = at < n ? __uint_as_float(q) : -INFINITY;
            }
        }
        float m = v[0];
#pragma unroll
        for (uint32_t i = 1; i < kLpPerThread; ++i) m = fmaxf(m, v[i]);  // leaves NaN out
        {
            LpSum here{m, 0.0f, 0.0f, 0.0f};
            const float base = m == -INFINITY || m != m ? 0.0f : m;
#pragma unroll
            for (uint32_t i = 0; i < kLpPerThread; ++i) {
                const float d = v[i] - base, e = expf(d);
                here.s += e;
                here.t += e == 0.0f ? 0.0f : e * d;
            }
            join(sum, here);
        }
        if (top == 0) continue;
        // Nothing to do where every lane's largest number is below the floor's
        // (no number: a NaN's, or no floor yet), NaN being below every number.
        if (__any(!(m < key_logit(floor_key)))) {
            uint64_t key = 0;
#pragma unroll
            for (uint32_t i = 0; i < kLpPerThread; ++i) {
                const uint32_t at = tid * 4 + (i >> 2) * (kLpThreads * 4) + (i & 3);
                if (at < n) key = max(key, rank_key(v[i], first + at));
            }
            if (key <= floor_key) key = 0;
            uint64_t least = floor_key + 1;
            if ((uint32_t)__popcll(__ballot(key != 0)) >= top) least = wave_kth(key, top);
            if (key >= least) {
#pragma unroll
                for (uint32_t i = 0; i < kLpPerThread; ++i) {
                    const uint32_t at = tid * 4 + (i >> 2) * (kLpThreads * 4) + (i & 3);
                    const uint64_t k = rank_key(v[i], first + at);
                    if (at < n && k >= least) list[atomicAdd(&kept[c & 1], 1u)] = k;
                }
            }
        }
        __syncthreads();
        uint32_t found = kept[c & 1];
        if (tid == 0) kept[(c + 1) & 1] = 0;
        if (found) {
            // The piece's own behind them.
            if (tid < top && best[tid]) list[found + tid] = best[tid];
            found += (uint32_t)__popcll(__ballot((tid & 63) < top && best[tid & 63]));
            __syncthreads();
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
    __shared__ uint64_t list[kLpMostPieces / 64 * kLpMostTop * kLpMostTop];
    __shared__ uint64_t best[kLpMostTop];
    __shared__ uint32_t kept;
    const uint64_t row = blockIdx.x;
    const float* x = a.logits + row * a.stride;
    const uint32_t top = a.top, tid = threadIdx.x, lane = tid & 63;
    if (tid == 0) kept = 0;
    LpSum sum{-INFINITY, 0.0f, 0.0f, 0.0f};
    if (tid < p.pieces) sum = p.sums[row * p.pieces + tid];
    sum = join_all(sum, red);
    const float log_s = logf(sum.s);
    if (a.entropy && tid == 0) a.entropy[row] = log_s - sum.t / sum.s;
    for (uint64_t i = tid; i < a.n_given; i += kLpThreads) {
        const uint32_t id = a.tokens[row * a.n_given + i];
        if (id >= a.vocab) report(a.status, kBadToken);
        a.token_logprobs[row * a.n_given + i] = id < a.vocab ? (x[id] - sum.m) - log_s : __builtin_nanf("");
    }
    if (top == 0) return;
    // A lane stands for the pieces lane + 64 i: the `top`-th largest of the
    // lanes' largest is a floor, where there are as many lanes. Every wave
    // finds it for itself.
    const uint64_t* keys = p.keys + row * p.pieces * top;
    uint64_t largest = 0;
    for (uint32_t i = lane; i < p.pieces; i += 64) largest = max(largest, keys[(uint64_t)i * top]);
    uint64_t least = 1;
    if ((uint32_t)__popcll(__ballot(largest != 0)) >= top) least = wave_kth(largest, top);
    for (uint32_t i = tid; i < p.pieces * top; i += kLpThreads) {
        const uint64_t k = keys[i];
        if (k >= least) list[atomicAdd(&kept, 1u)] = k;
    }
    __syncthreads();
    rank_list(list, kept, best, top);
    __syncthreads();
    if (tid < top) {
        a.top_ids[row * top + tid] = key_id(best[tid]);
        if (a.top_logprobs) a.top_logprobs[row * top + tid] = (key_logit(best[tid]) - sum.m) - log_s;
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
