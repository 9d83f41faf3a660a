// Log probabilities of the next token over the vocabulary on gfx950.
#include "device_common.hpp"
#include "kernels.hpp"

namespace mmhip {

namespace {

constexpr int kLpThreads = 256;

// A logit's place in the order of the largest: larger is earlier, equal ones
// by the lower id, NaN after every number. 0: none.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t id) {
    uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as 0
    b = x != x ? 0u : (b & 0x80000000u ? ~b : b | 0x80000000u);
    return ((uint64_t)b << 32) | (0xFFFFFFFFu - id);
}

__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* red) {
    for (int off = 32; off > 0; off >>= 1) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, off, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return max(max(red[0], red[1]), max(red[2], red[3]));
}
__device__ __forceinline__ float block_sum(float v, float* red) {
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// One workgroup per row.
__global__ __launch_bounds__(kLpThreads) void logprobs_simple_kernel(LogprobsArgs a) {
    __shared__ uint64_t r64[kLpThreads / 64];
    __shared__ float r32[kLpThreads / 64];
    const uint64_t row = blockIdx.x;
    const float* x = a.logits + row * a.stride;
    uint64_t key = 0;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kLpThreads) key = max(key, rank_key(x[i], i));
    key = block_max(key, r64);
    const float m = x[0xFFFFFFFFu - (uint32_t)key];
    float s = 0.0f, t = 0.0f;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kLpThreads) {
        const float d = x[i] - m, e = expf(d);
        s += e;
        t += e == 0.0f ? 0.0f : e * d;
    }
    s = block_sum(s, r32);
    t = block_sum(t, r32);
    const float log_s = logf(s);
    if (a.entropy && threadIdx.x == 0) a.entropy[row] = log_s - t / s;
    for (uint64_t i = threadIdx.x; i < a.n_given; i += kLpThreads) {
        const uint32_t id = a.tokens[row * a.n_given + i];
        if (id >= a.vocab) report(a.status, kBadToken);
        a.token_logprobs[row * a.n_given + i] = id < a.vocab ? (x[id] - m) - log_s : __builtin_nanf("");
    }
    uint64_t below = ~0ull;
    for (uint32_t j = 0; j < a.top; ++j) {
        key = 0;
        for (uint32_t i = threadIdx.x; i < a.vocab; i += kLpThreads) {
            const uint64_t k = rank_key(x[i], i);
            if (k < below) key = max(key, k);
        }
        below = block_max(key, r64);
        if (threadIdx.x == 0) {
            const uint32_t id = 0xFFFFFFFFu - (uint32_t)below;
            a.top_ids[row * a.top + j] = id;
            if (a.top_logprobs) a.top_logprobs[row * a.top + j] = (x[id] - m) - log_s;
        }
    }
}

}  // namespace

uint64_t logprobs_workspace_bytes(uint64_t, uint64_t, uint32_t) { return 0; }

hipError_t launch_logprobs(const LogprobsArgs& a, uint64_t n_rows, hipStream_t s) {
    if (n_rows == 0) return hipSuccess;
    logprobs_simple_kernel<<<(unsigned)n_rows, kLpThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace mmhip
