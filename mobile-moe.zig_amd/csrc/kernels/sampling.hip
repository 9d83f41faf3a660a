// Tokens drawn from logits with temperature, top-k, top-p and min-p and given
// random numbers, on gfx950.
//
// With m the row's largest logit and T the temperature a token's weight is
// w = exp((x - m) / T). All three filters keep the front of one order (larger
// logits first, equal ones by the lower id), so what is kept is every token
// with a key (rank_key) at or above one cut. The token drawn is the first kept id
// at which the running sum of the kept weights, by id, exceeds u times their
// sum.
//
// A comparison of sums must not depend on how they were taken, so weights are
// computed in 64 bits (weight()) and summed as whole multiples of 2^-shift
// (44 for up to 2^18 tokens): integer sums have no order.
#include "device_common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"

namespace mmhip {

namespace {

constexpr uint32_t kSmThreads = 1024, kSmWaves = kSmThreads / 64;
constexpr uint32_t kSmDigit = 11, kSmBins = 1u << kSmDigit;

// A logit's place in the order: larger is earlier, equal ones by the lower id.
// NaN and -infinity, which are never drawn, are below kLeastKey.
__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);  // -0 counts as 0
    return x != x ? 0u : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(float x, uint32_t id) { return (uint64_t)order_bits(x) << 32 | (0xFFFFFFFFu - id); }
constexpr uint64_t kLeastKey = 0x00800000ull << 32;
__device__ __forceinline__ float key_value(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}

// (x - m) / T; 0 for the largest itself, an infinite one too.
__device__ __forceinline__ double scaled(float x, float m, double inv_t) {
    return x == m ? 0.0 : ((double)x - (double)m) * inv_t;
}
// exp(z) * 2^shift for z <= 0: 2^n 2^f with |f| <= 1/2, 2^f by its series to the
// eleventh power (the next term is below 7e-15). From z = -70 on 0 for every shift.
__device__ __forceinline__ double weight(double z, int shift) {
    const double t = fmax(z * 1.4426950408889634, -101.0);
    const double n = rint(t), f = (t - n) * 0.6931471805599453;
    double p = 1.0 / 39916800.0;
    p = fma(p, f, 1.0 / 3628800.0);
    p = fma(p, f, 1.0 / 362880.0);
    p = fma(p, f, 1.0 / 40320.0);
    p = fma(p, f, 1.0 / 5040.0);
    p = fma(p, f, 1.0 / 720.0);
    p = fma(p, f, 1.0 / 120.0);
    p = fma(p, f, 1.0 / 24.0);
    p = fma(p, f, 1.0 / 6.0);
    p = fma(p, f, 0.5);
    p = fma(p, f, 1.0);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)n + shift);
}
// The same as a whole number: at most 2^44, so adding 2^52 rounds it to the
// lower bits of the sum.
__device__ __forceinline__ uint64_t whole_weight(double z, int shift) {
    return __double_as_longlong(weight(z, shift) + 0x1p52) & 0xFFFFFFFFFFFFFull;
}

__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* red) {
    __syncthreads();
    v = wave_scan(v);
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t all = 0;
    for (uint32_t w = 0; w < kSmWaves; ++w) all += red[w];
    return all;
}
__device__ __forceinline__ uint64_t block_max(uint64_t v, uint64_t* red) {
    __syncthreads();
#pragma unroll
    for (int off = 32; off; off >>= 1) v = max(v, (uint64_t)__shfl_xor((unsigned long long)v, off, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t all = 0;
    for (uint32_t w = 0; w < kSmWaves; ++w) all = max(all, red[w]);
    return all;
}

struct RowSettings {
    float m;
    double inv_t, least_z;
    int shift;
};

struct Bins {
    unsigned long long mass[kSmBins];
    uint32_t count[kSmBins];
    uint32_t found;
    uint64_t above;
};

// The key at which the running total of keys >= floor in descending order first
// reaches `target`: of tokens (MASS false) or of weights. 64-bit keys in six digits
// of 11 bits, each by a histogram of the row's keys with the digits before it.
template <bool MASS>
__device__ uint64_t find_cut(const float* x, uint32_t vocab, const RowSettings& s, uint64_t floor, uint64_t target, Bins& b) {
    uint64_t prefix = 0, before = 0;
    for (int level = 0; level < 6; ++level) {
        const int low = level == 5 ? 0 : 53 - 11 * level, bits = level == 5 ? 9 : 11;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < kSmBins; i += kSmThreads) b.mass[i] = 0, b.count[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < vocab; i += kSmThreads) {
            const float v = x[i];
            const uint64_t k = order_key(v, i);
            if (k < floor || (level && (k >> (low + bits)) != prefix)) continue;
            const uint32_t at = (uint32_t)(k >> low) & ((1u << bits) - 1);
            atomicAdd(&b.count[at], 1u);
            if (MASS) atomicAdd(&b.mass[at], (unsigned long long)whole_weight(scaled(v, s.m, s.inv_t), s.shift));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            // The last digit there is where all of them fall short.
            uint32_t last = 0;
            uint64_t sum = before, above = before;
            for (uint32_t at = 1u << bits; at-- > 0;) {
                if (b.count[at] == 0) continue;
                last = at;
                above = sum;
                sum += MASS ? b.mass[at] : b.count[at];
                if (sum >= target) break;
            }
            b.found = last;
            b.above = above;
        }
        __syncthreads();
        prefix = prefix << bits | b.found;
        before = b.above;
    }
    return prefix;
}

__global__ __launch_bounds__(kSmThreads) void sample_row_kernel(SampleArgs a) {
    __shared__ uint64_t red[kSmWaves];
    __shared__ Bins bins;
    const uint32_t out = blockIdx.x, tid = threadIdx.x;
    uint32_t row = out;
    if (a.rows) {
        row = a.rows[out];
        if (row == kNoToken) return;
        if (row >= a.n_logits) {
            if (tid == 0) {
                report(a.status, kBadSampleRow);
                a.tokens[out] = kNoToken;
                if (a.probs) a.probs[out] = __builtin_nanf("");
                if (a.kept) a.kept[out] = 0;
            }
            return;
        }
    }
    const float* x = a.logits + row * a.stride;
    const float t = a.temperature ? a.temperature[out] : 1.0f, p = a.top_p ? a.top_p[out] : 1.0f;
    const float min_p = a.min_p ? a.min_p[out] : 0.0f, u = a.uniform[out];
    uint32_t k = a.top_k ? a.top_k[out] : 0;
    const bool ok = t >= 0.0f && t <= 3.4028235e38f && p >= 0.0f && min_p >= 0.0f && min_p <= 1.0f && u >= 0.0f && u < 1.0f;
    uint64_t best = 0;
    for (uint32_t i = tid; i < a.vocab; i += kSmThreads) best = max(best, order_key(x[i], i));
    best = block_max(best, red);
    if (!ok || best < kLeastKey) {
        if (tid == 0) {
            report(a.status, ok ? kNoSampleToken : kBadSampleSetting);
            a.tokens[out] = kNoToken;
            if (a.probs) a.probs[out] = __builtin_nanf("");
            if (a.kept) a.kept[out] = 0;
        }
        return;
    }
    if (t == 0.0f || k == 1) {
        if (tid == 0) {
            a.tokens[out] = 0xFFFFFFFFu - (uint32_t)best;
            if (a.probs) a.probs[out] = 1.0f;
            if (a.kept) a.kept[out] = 1;
        }
        return;
    }
    const RowSettings s{key_value(best), 1.0 / (double)t, log((double)min_p), a.shift};
    uint64_t cut = kLeastKey;
    if (k != 0 && k < a.vocab) cut = max(cut, find_cut<false>(x, a.vocab, s, cut, k, bins));
    if (p < 1.0f) {
        uint64_t sum = 0;
        for (uint32_t i = tid; i < a.vocab; i += kSmThreads) {
            const float v = x[i];
            if (order_key(v, i) >= cut) sum += whole_weight(scaled(v, s.m, s.inv_t), s.shift);
        }
        sum = block_sum(sum, red);
        cut = max(cut, find_cut<true>(x, a.vocab, s, cut, (uint64_t)ceil((double)p * (double)sum), bins));
    }
    const auto weight_of = [&](uint32_t i, uint64_t& kept) -> uint64_t {
        const float v = x[i];
        if (order_key(v, i) < cut) return 0;
        const double z = scaled(v, s.m, s.inv_t);
        if (!(z >= s.least_z)) return 0;
        ++kept;
        return whole_weight(z, s.shift);
    };
    uint64_t sum = 0, kept = 0;
    for (uint32_t i = tid; i < a.vocab; i += kSmThreads) sum += weight_of(i, kept);
    sum = block_sum(sum, red);
    kept = block_sum(kept, red);
    // The first id whose running sum is above u times all of it.
    const uint64_t target = (uint64_t)((double)u * (double)sum);
    uint64_t before = 0, none = 0;
    for (uint32_t i0 = 0; i0 < a.vocab; i0 += kSmThreads) {
        const uint32_t i = i0 + tid;
        const uint64_t w = i < a.vocab ? weight_of(i, none) : 0;
        const uint64_t all = block_sum(w, red);
        if (before + all > target) {
            const uint64_t in = wave_scan(w);
            uint64_t here = before + in;
            for (uint32_t v = 0; v < tid >> 6; ++v) here += red[v];
            if (w && here > target && here - w <= target) {
                a.tokens[out] = i;
                if (a.probs) a.probs[out] = (float)(weight(scaled(x[i], s.m, s.inv_t), s.shift) / (double)sum);
                if (a.kept) a.kept[out] = (uint32_t)kept;
            }
            return;
        }
        before += all;
    }
}

}  // namespace

uint64_t sample_workspace_bytes(uint64_t n_rows, uint64_t vocab) {
    (void)n_rows;
    (void)vocab;
    return 0;
}

hipError_t launch_sample(const SampleArgs& a_in, uint64_t n_rows, hipStream_t s) {
    if (n_rows == 0) return hipSuccess;
    SampleArgs a = a_in;
    uint32_t bits = 0;
    while ((1ull << bits) < a.vocab) ++bits;
    a.shift = bits <= 18 ? 44 : 62 - bits;
    sample_row_kernel<<<(unsigned)n_rows, kSmThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace mmhip
