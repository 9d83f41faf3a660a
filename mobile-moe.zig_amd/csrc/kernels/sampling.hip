// Tokens drawn from logits with temperature, top-k, top-p and min-p and given
// random numbers, on gfx950.
//
// With m the row's largest logit and T the temperature a token's weight is
// w = exp((x - m) / T). All three filters keep the front of one order (larger
// logits first, equal ones by the lower id), so what is kept is every token
// with a key (order_key) at or above one cut. The token drawn is the first kept id
// at which the running sum of the kept weights, by id, exceeds u times their
// sum.
//
// A comparison of sums must not depend on how they were taken, so weights are
// computed in 64 bits (weight()) and summed as whole multiples of 2^-shift
// (44 for up to 2^18 tokens): integer sums have no order.
//
// Four launches: the largest logit (pieces of rows); a histogram of tokens and
// weights over bins of (m - x) / T; the tokens of the bins that hold the cuts, in a
// list, and what each chunk of logits keeps for certain; the cuts in the list, the
// chunk and the token that u falls on (a workgroup per row). Bound: with few rows
// the latency of four launches, each two or three dependent trips to memory and a
// few barriers; with many by vector instructions, about 30 for each logit and
// weight. Measured with 154880 tokens, us (largest, histogram, list, draw): one
// row with top-p 3.7, 5.1, 6.0, 7.1, together 22.6; 16 rows with top-k 5.6, 6.0, 7.8,
// 6.0, together 24.1; 64 rows with settings of their own 10.1, 14.2, 14.6, 11.6, together
// 49.9 (their logits are 39.7 MB, 8.3 us of copying). One workgroup per row for all
// of it took 586, 542 and 1036.
#include <algorithm>
#include <type_traits>

#include "device_common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"

namespace mmhip {

namespace {

constexpr uint32_t kSmThreads = 1024, kSmWaves = kSmThreads / 64;  // of the launch over rows
// Logits of a piece's turn, and the waves that share them. Eight waves with half as
// many each, up to a piece per workgroup of the limit below, are 2 us faster for few
// rows (1 row 23.7 against 25.9 us, 8 rows 29.2 and 31.2, 16 rows 32.3 and 32.8) and 1
// slower for many (64 rows 51.8 and 50.7). (More workgroups instead of wider ones: the
// histogram's sums in memory meet as many more of them, 16 rows took 37 us for 26.)
constexpr uint32_t kSmTurn = 4096, kSmWide = 8, kSmNarrow = 4;
constexpr uint32_t kSmBins = 1024;  // of the row's histogram
// Pieces of a call that are enough: with 64 rows 512, 1024 and 2048 took 57.7, 53.2
// and 55.7 us.
constexpr uint32_t kSmWorkgroups = 1024;
constexpr uint32_t kSmBeside = 4;  // of a lane's logits, worked on beside each other
constexpr uint32_t kSmPerThread = 8;  // tokens beside the cut that a thread of the last launch takes
constexpr uint32_t kSmList = kSmPerThread * kSmThreads;

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

// A weight is 2^(t / 256) with t = (x - m) 256 / (T ln 2), rounded to n + f:
// 2^(n / 256) is a table's entry and an exponent, 2^(f / 256) a series of four
// powers (the next is below 4e-17). Half the instructions of a series of eleven.
constexpr int kSmParts = 256;
struct Parts {
    double of[kSmParts];
};
constexpr Parts make_parts() {
    Parts t{};
    for (int i = 0; i < kSmParts; ++i) {
        const double f = (i < kSmParts / 2 ? i : i - kSmParts) * (0.6931471805599453 / kSmParts);
        double p = 1.0;
        for (int n = 14; n > 0; --n) p = 1.0 + p * f / n;
        t.of[i] = i < kSmParts / 2 ? p : 2.0 * p;
    }
    return t;
}
__constant__ const Parts kParts = make_parts();
__device__ __forceinline__ void fill_parts(double* parts) {  // by the first 256 threads; a barrier follows
    if (threadIdx.x < kSmParts) parts[threadIdx.x] = kParts.of[threadIdx.x];
}
// (The compiler copies a constant addend to a vector register before each step.)
__device__ __forceinline__ double fma_to(double a, double b, double addend) {
    double d;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(addend));
    return d;
}
// The weight times 2^shift, for t <= 0. From 2^-64 on down as 2^-64, which is 0 for every shift.
__device__ __forceinline__ double weight(double t, int shift, const double* parts) {
    constexpr double kLn2 = 0.6931471805599453 / kSmParts;
    const double whole = 0x1.8p52 + kSmParts * shift;
    t = fmax(t, -64.0 * kSmParts);
    const double r = t + whole;  // n and the shift in its lowest bits
    const uint32_t n = (uint32_t)__double_as_longlong(r);
    const double f = t - (r - whole);
    double p = kLn2 * kLn2 * kLn2 * kLn2 / 24;
    p = fma_to(f, p, kLn2 * kLn2 * kLn2 / 6);
    p = fma_to(p, f, kLn2 * kLn2 / 2);
    p = fma_to(p, f, kLn2);
    const double part = parts[n & (uint32_t)(kSmParts - 1)];
    const double w = fma(part, p * f, part);
    return __hiloint2double(__double2hiint(w) + ((int)n >> 8 << 20), __double2loint(w));
}
// The same as a whole number: at most 2^44, so adding 2^52 rounds it to the
// lower bits of the sum.
__device__ __forceinline__ uint64_t whole_weight(double t, int shift, const double* parts) {
    return __double_as_longlong(weight(t, shift, parts) + 0x1p52) & 0xFFFFFFFFFFFFFull;
}

// What a row asks for.
enum SmMode : uint32_t { kSmAbsent, kSmNoRow, kSmBadSetting, kSmEmpty, kSmFirst, kSmAll, kSmCut };
struct RowSettings {
    SmMode mode;
    const float* x;
    uint64_t best;  // the first token's key
    bool far;                // is the largest logit infinite
    float bin_c, bin_m;
    double m, per_t, least;  // t per logit, and t of min_p
    float p, u;
    uint32_t k;     // 0: no cut by number
    bool by_mass;   // a cut by probability
    int shift;
};

struct SmRow {
    uint32_t listed;           // tokens in bins beside a cut (at most kSmList are in the list)
    uint32_t k_bin, k_rank;    // the cut by number: the bin, and which of its tokens is the last
    uint32_t p_lo, p_hi;       // the cut by probability: the bins that it may be in
    uint64_t k_mass, p_mass;   // of the tokens in bins before k_bin, before p_lo
    uint64_t mass;             // of all
};
struct SmPlan {
    uint32_t chunks, pieces, list;
    uint32_t chunk, per;       // logits of a chunk, chunks of a piece
    uint32_t waves;            // of a piece
    uint64_t* best;            // [rows][pieces]
    float* lowest;             // [rows][pieces]
    unsigned long long* mass;  // [rows][kSmBins]
    uint32_t* count;           // [rows][kSmBins]
    uint64_t* chunk_mass;      // [rows][chunks]: kept for certain
    uint32_t* chunk_count;     // [rows][chunks]
    uint64_t* keys;            // [rows][list]
    SmRow* rows;
    RowSettings *asked, *settings;
};
constexpr uint32_t kNoBin = 0xFFFFFFFFu;

// What a row asks for, as far as that does not depend on its logits.
__device__ __forceinline__ RowSettings row_asked(const SampleArgs& a, uint32_t out) {
    RowSettings s{};
    uint32_t row = out;
    if (a.rows) row = a.rows[out];
    const float t = a.temperature ? a.temperature[out] : 1.0f, least = a.min_p ? a.min_p[out] : 0.0f;
    s.p = a.top_p ? a.top_p[out] : 1.0f;
    s.u = a.uniform[out];
    s.k = a.top_k ? a.top_k[out] : 0;
    if (a.rows && row == kNoToken) s.mode = kSmAbsent;
    else if (a.rows && row >= a.n_logits) s.mode = kSmNoRow;
    else if (!(t >= 0.0f && t <= 3.4028235e38f && s.p >= 0.0f && least >= 0.0f && least <= 1.0f && s.u >= 0.0f && s.u < 1.0f))
        s.mode = kSmBadSetting;
    else if (t == 0.0f || s.k == 1) s.mode = kSmFirst;
    else {
        if (s.k >= a.vocab) s.k = 0;
        s.by_mass = s.p < 1.0f;
        s.mode = s.k || s.by_mass ? kSmCut : kSmAll;
    }
    if (s.mode < kSmFirst) return s;
    s.x = a.logits + row * a.stride;
    s.per_t = 369.3299304675746 / (double)t;  // 256 / ln 2
    s.least = 369.3299304675746 * log((double)least);
    s.shift = a.shift;
    s.bin_c = 0.25f / t;
    return s;
}
// With the row's largest token's key and its lowest logit.
__device__ __forceinline__ void row_settings(RowSettings& s, const RowSettings& asked, uint64_t best, float low) {
    const float m = key_value(best);
    const bool far = m > 3.4028235e38f;
    s.mode = asked.mode >= kSmFirst && best < kLeastKey ? kSmEmpty : asked.mode;
    s.x = asked.x;
    s.best = best;
    s.far = far;
    // Bins of 1/32 of the temperature next to the largest logit, twice as wide
    // from four temperatures below it on, and so on; narrower ones where the
    // row's logits are closer together than that.
    s.bin_c = fminf(fmaxf(asked.bin_c, 7.0f * __builtin_amdgcn_rcpf(m - low)), 1e30f);
    s.m = far ? 0.0 : (double)m;
    s.per_t = far ? 369.3299304675746 : asked.per_t;
    s.bin_m = fmaf((float)s.m, s.bin_c, 1.0f);
    s.least = asked.least;
    s.p = asked.p;
    s.u = asked.u;
    s.k = asked.k;
    s.by_mass = asked.by_mass;
    s.shift = asked.shift;
}
// A logit as the weights and bins see it: beside an infinite one no other one
// weighs anything, so in such a row that is 0 and all others are far below.
__device__ __forceinline__ float seen(float x, const RowSettings& s) {
    return !s.far || !(x > -INFINITY) ? x : x > 3.4028235e38f ? 0.0f : -3.4028235e38f;
}
// t of a logit.
__device__ __forceinline__ double scaled(float x, const RowSettings& s) { return ((double)x - s.m) * s.per_t; }
// The bin of a logit above -infinity: never smaller for a smaller logit.
__device__ __forceinline__ uint32_t bin_bits(float x, const RowSettings& s) {
    return __float_as_uint(__builtin_amdgcn_fmed3f(fmaf(-x, s.bin_c, s.bin_m), 1.0f, 255.9f));
}
__device__ __forceinline__ uint32_t bin_of(float x, const RowSettings& s) { return (bin_bits(x, s) - 0x3F800000u) >> 16; }
// The least bits of a bin; more than any where there is none.
__device__ __forceinline__ uint32_t bin_start(uint32_t bin) { return bin < kSmBins ? 0x3F800000u + (bin << 16) : 0x80000000u; }
__device__ __forceinline__ uint64_t mass_target(float p, uint64_t sum) {
    return max((uint64_t)ceil((double)p * (double)sum), (uint64_t)1);
}

// A wave's chunk: a lane's i-th logit stands at place_of(i), NaN where there is none.
__device__ __forceinline__ uint32_t place_of(uint32_t i) { return (i >> 2) * 256 + (threadIdx.x & 63) * 4 + (i & 3); }
template <uint32_t EACH>
__device__ __forceinline__ void load_chunk(const float* x, uint32_t vocab, uint32_t chunk, float (&v)[EACH]) {
    const uint32_t first = chunk * (EACH * 64), n = min(vocab - first, EACH * 64), lane = threadIdx.x & 63;
    const BufRsrc r = make_rsrc(x + first, n * 4);
    if (n == EACH * 64) {
#pragma unroll
        for (uint32_t j = 0; j < EACH / 4; ++j) {
            const uint4 q = buf_load_b128(r, lane * 16, j * 1024);
            v[4 * j] = __uint_as_float(q.x);
            v[4 * j + 1] = __uint_as_float(q.y);
            v[4 * j + 2] = __uint_as_float(q.z);
            v[4 * j + 3] = __uint_as_float(q.w);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) v[i] = __uint_as_float(buf_load_b32(r, lane * 16, (i >> 2) * 1024 + (i & 3) * 4));
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i)
            if (place_of(i) >= n) v[i] = __builtin_nanf("");
    }
}

// The row of logits that the row's number names, or null.
__device__ __forceinline__ const float* row_logits(const SampleArgs& a, uint32_t out) {
    uint32_t row = out;
    if (a.rows) row = a.rows[out];
    return !a.rows || row < a.n_logits ? a.logits + row * a.stride : nullptr;
}

// The largest and lowest logits of a piece, and the row's memory cleared.
template <uint32_t WAVES, uint32_t EACH>
__global__ __launch_bounds__(WAVES * 64) void sample_best_kernel(SampleArgs a, SmPlan p) {
    __shared__ uint64_t memory[2][2][WAVES];
    const uint32_t out = blockIdx.x / p.pieces, piece = blockIdx.x - out * p.pieces;
    const uint32_t c0 = piece * p.per, c1 = min(c0 + p.per, p.chunks);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (uint32_t i = piece * WAVES * 64 + threadIdx.x; i < kSmBins; i += p.pieces * WAVES * 64) {
        p.mass[(uint64_t)out * kSmBins + i] = 0;
        p.count[(uint64_t)out * kSmBins + i] = 0;
    }
    if (piece == 0 && threadIdx.x == 0) p.rows[out].listed = 0;
    const float* x = row_logits(a, out);
    float top = -INFINITY;
    uint32_t id = 0, under = 0, over = 0xFFFFFFFFu;
    float v[EACH];
    if (x && c0 + wave < c1) load_chunk(x, a.vocab, c0 + wave, v);
    if (piece == 0 && threadIdx.x == 0) p.asked[out] = row_asked(a, out);
    if (x)
        for (uint32_t c = c0 + wave; c < c1; c += WAVES) {
            if (c != c0 + wave) load_chunk(x, a.vocab, c, v);
            float here = -INFINITY;
#pragma unroll
            for (uint32_t i = 0; i < EACH; i += 2) {
                const float v0 = v[i] > -INFINITY ? v[i] : -INFINITY, v1 = v[i + 1] > -INFINITY ? v[i + 1] : -INFINITY;
                here = __builtin_amdgcn_fmed3f(__builtin_amdgcn_fmed3f(here, v0, INFINITY), v1, INFINITY);
                const uint32_t b0 = __float_as_uint(v0), b1 = __float_as_uint(v1);
                under = max(under, max(b0 + 0x00800000u, b1 + 0x00800000u));
                over = min(over, min(b0, b1));
            }
            // The wave's largest, at its lowest id.
            here = key_value(lane_value(wave_max_scan((uint64_t)order_bits(here)), 63) << 32);
            if (!(here > top)) continue;
            top = here;
#pragma unroll
            for (uint32_t j = EACH / 4; j-- > 0;) {
                uint32_t lowest_place = 256;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const uint64_t at = __ballot(v[4 * j + e] == here);
                    if (at) lowest_place = min(lowest_place, (uint32_t)__builtin_ctzll(at) * 4 + e);
                }
                if (lowest_place < 256) id = c * (EACH * 64) + j * 256 + lowest_place;
            }
        }
    // Of finite numbers and +infinity the lowest: a negative one's bits, more for a
    // lower number, go past those of -infinity with 2^23 added; if there is none, the
    // least bits are the lowest number's.
    float low = under >= 0x80800000u ? __uint_as_float(under - 0x00800000u) : over < 0x7F800001u ? __uint_as_float(over) : INFINITY;
    uint64_t best = order_key(top, id), lowest = order_bits(-low);
    Together<WAVES> all{memory};
    all.largest(best, lowest);
    if (threadIdx.x == 0) {
        p.best[blockIdx.x] = best;
        p.lowest[blockIdx.x] = -key_value(lowest << 32);
    }
}

// How many tokens, and how much of the weights, each bin of the row holds. Rows
// without a cut: what each chunk keeps. The row's settings for the launches behind.
template <uint32_t WAVES, uint32_t EACH>
__global__ __launch_bounds__(WAVES * 64) void sample_bins_kernel(SampleArgs a, SmPlan p) {
    __shared__ uint64_t memory[2][2][WAVES];
    __shared__ double parts[kSmParts];
    __shared__ unsigned long long mass[kSmBins];
    __shared__ uint32_t count[kSmBins];
    const uint32_t out = blockIdx.x / p.pieces, piece = blockIdx.x - out * p.pieces;
    const uint32_t c0 = piece * p.per, c1 = min(c0 + p.per, p.chunks);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float* x = row_logits(a, out);
    float v[EACH];
    if (x && c0 + wave < c1) load_chunk(x, a.vocab, c0 + wave, v);  // its latency beside the settings'
    const RowSettings& asked = p.asked[out];
    uint64_t best = 0, lowest = 0;
    for (uint32_t i = threadIdx.x; i < p.pieces; i += WAVES * 64) {
        best = max(best, p.best[(uint64_t)out * p.pieces + i]);
        lowest = max(lowest, (uint64_t)order_bits(-p.lowest[(uint64_t)out * p.pieces + i]));
    }
    fill_parts(parts);
    for (uint32_t i = threadIdx.x; i < kSmBins; i += WAVES * 64) mass[i] = 0, count[i] = 0;
    Together<WAVES> all{memory};
    all.largest(best, lowest);
    RowSettings s;
    row_settings(s, asked, best, -key_value(lowest << 32));
    if (piece == 0 && threadIdx.x == 0) p.settings[out] = s;
    if (s.mode < kSmAll) return;
    const auto next = [&](uint32_t c) {
        if (c != c0 + wave) load_chunk(x, a.vocab, c, v);
        if (s.far) {
#pragma unroll
            for (uint32_t i = 0; i < EACH; ++i) v[i] = seen(v[i], s);
        }
    };
    if (s.mode == kSmAll) {
        for (uint32_t c = c0 + wave; c < c1; c += WAVES) {
            next(c);
            uint64_t sum = 0;
            uint32_t n = 0;
#pragma unroll
            for (uint32_t i = 0; i < EACH; ++i) {
                const double t = scaled(v[i], s);
                const uint64_t w = whole_weight(t, s.shift, parts);
                const bool keep = v[i] > -INFINITY && t >= s.least;
                sum += keep ? w : 0;
                n += keep;
            }
            sum = wave_scan(sum);
            n = (uint32_t)wave_scan(n);
            if (lane == 63) {
                p.chunk_mass[(uint64_t)out * p.chunks + c] = sum;
                p.chunk_count[(uint64_t)out * p.chunks + c] = n;
            }
        }
        return;
    }
    const auto fill = [&](auto by_number, auto by_mass) {
        for (uint32_t c = c0 + wave; c < c1; c += WAVES) {
            next(c);
#pragma unroll
            for (uint32_t i0 = 0; i0 < EACH; i0 += kSmBeside) {
                uint32_t b[kSmBeside];
                uint64_t w[kSmBeside];
#pragma unroll
                for (uint32_t i = 0; i < kSmBeside; ++i) {
                    b[i] = bin_of(v[i0 + i], s);
                    if (by_mass()) w[i] = whole_weight(scaled(v[i0 + i], s), s.shift, parts);
                }
#pragma unroll
                for (uint32_t i = 0; i < kSmBeside; ++i) {
                    if (!(v[i0 + i] > -INFINITY)) continue;
                    if (by_number()) atomicAdd(&count[b[i]], 1u);
                    if (by_mass()) atomicAdd(&mass[b[i]], (unsigned long long)w[i]);
                }
            }
        }
    };
    if (!s.by_mass) fill(std::true_type(), std::false_type());
    else if (!s.k) fill(std::false_type(), std::true_type());
    else fill(std::true_type(), std::true_type());
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kSmBins; i += WAVES * 64) {
        if (count[i]) atomicAdd(&p.count[(uint64_t)out * kSmBins + i], count[i]);
        if (mass[i]) atomicAdd(&p.mass[(uint64_t)out * kSmBins + i], mass[i]);
    }
}

// The bins that the cuts are in: their tokens go into the row's list, and what
// each chunk has in the bins before all of them is kept for certain.
template <uint32_t WAVES, uint32_t EACH>
__global__ __launch_bounds__(WAVES * 64) void sample_list_kernel(SampleArgs a, SmPlan p) {
    constexpr uint32_t kPer = kSmBins / (WAVES * 64);
    __shared__ uint64_t memory[2][2][WAVES];
    __shared__ uint64_t most;
    __shared__ uint32_t listed, listed_at;
    __shared__ float queue[WAVES][EACH * 64];
    __shared__ uint16_t place[WAVES][EACH * 64];
    __shared__ double parts[kSmParts];
    __shared__ SmRow row;
    const uint32_t out = blockIdx.x / p.pieces, piece = blockIdx.x - out * p.pieces;
    const uint32_t c0 = piece * p.per, c1 = min(c0 + p.per, p.chunks);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tid = threadIdx.x;
    const RowSettings s = p.settings[out];
    const float* x = row_logits(a, out);
    float v[EACH];
    if (x && c0 + wave < c1) load_chunk(x, a.vocab, c0 + wave, v);
    uint64_t m[kPer], mass_to = 0, all_mass, num_to = 0, all_num;
    uint32_t n[kPer];
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        m[i] = p.mass[(uint64_t)out * kSmBins + tid * kPer + i];
        n[i] = p.count[(uint64_t)out * kSmBins + tid * kPer + i];
    }
    if (s.mode != kSmCut) return;
    if (tid == 0) {
        row = SmRow{0, kNoBin, 0, kNoBin, kNoBin, 0, 0, 0};
        most = 0;
        listed = 0;
    }
    fill_parts(parts);
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) mass_to += m[i], num_to += n[i];
    const uint64_t mass_here = mass_to, num_here = num_to;
    Together<WAVES> all{memory};
    all.scan2(mass_to, num_to, all_mass, all_num);
    mass_to -= mass_here;
    num_to -= num_here;
    const bool by_k = s.k && s.k < all_num;
    if (by_k) {
        uint64_t at = num_to, w = mass_to;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) {
            if (at < s.k && s.k <= at + n[i]) {
                row.k_bin = tid * kPer + i;
                row.k_rank = (uint32_t)(s.k - at);
                row.k_mass = w;
                most = w + m[i];
            }
            at += n[i];
            w += m[i];
        }
        __syncthreads();
    }
    if (s.by_mass) {
        // The sum that the cut is a part of, at least and at most.
        const uint64_t lo = mass_target(s.p, by_k ? row.k_mass : all_mass), hi = mass_target(s.p, by_k ? most : all_mass);
        uint64_t w = mass_to;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) {
            if (w < lo && lo <= w + m[i]) {
                row.p_lo = tid * kPer + i;
                row.p_mass = w;
            }
            if (w < hi && hi <= w + m[i]) row.p_hi = tid * kPer + i;
            w += m[i];
        }
        __syncthreads();
    }
    const SmRow r = row;
    if (piece == 0 && tid == 0) {
        SmRow* to = &p.rows[out];
        to->k_bin = r.k_bin;
        to->k_rank = r.k_rank;
        to->p_lo = r.p_lo;
        to->p_hi = r.p_hi;
        to->k_mass = r.k_mass;
        to->p_mass = r.p_mass;
        to->mass = all_mass;
    }
    // Bits of the bins before all cuts, from the cuts' bins on and how many.
    const uint32_t sure = bin_start(min(r.k_bin, r.p_lo)), k_from = bin_start(r.k_bin), k_bits = r.k_bin < kSmBins ? 0x10000u : 0u;
    const uint32_t p_from = bin_start(r.p_lo), p_bits = r.p_lo < kSmBins ? (r.p_hi - r.p_lo + 1) << 16 : 0u;
    // Every wave takes as many turns: they ask for their tokens' places together.
    for (uint32_t c = c0 + wave; c < c0 + p.per; c += WAVES) {
        float next[EACH];
        if (c + WAVES < c1) load_chunk(x, a.vocab, c + WAVES, next);
        if (c >= c1) {
#pragma unroll
            for (uint32_t i = 0; i < EACH; ++i) v[i] = __builtin_nanf("");
        }
        if (s.far) {
#pragma unroll
            for (uint32_t i = 0; i < EACH; ++i) v[i] = seen(v[i], s);
        }
        uint64_t mine = 0;
        uint32_t kept = 0, n_sure = 0, n_list = 0;
        // Both go to the wave's queue first, what is kept for certain from its front
        // and what is listed from its end: few lanes have some.
        const auto before = [](uint64_t which) {
            return __builtin_amdgcn_mbcnt_hi((uint32_t)(which >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)which, 0));
        };
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) {
            const uint32_t bits = bin_bits(v[i], s);
            const bool there = v[i] > -INFINITY, is_sure = there && bits < sure;
            const bool in_list = there && (bits - k_from < k_bits || bits - p_from < p_bits);
            const uint64_t sures = __ballot(is_sure), lists = __ballot(in_list);
            if (sures) {
                if (is_sure) queue[wave][n_sure + before(sures)] = v[i];
                n_sure += (uint32_t)__popcll(sures);
            }
            if (lists) {
                const uint32_t to = EACH * 64 - 1 - (n_list + before(lists));
                if (in_list) queue[wave][to] = v[i], place[wave][to] = (uint16_t)place_of(i);
                n_list += (uint32_t)__popcll(lists);
            }
        }
        __builtin_amdgcn_wave_barrier();
        for (uint32_t i = lane; i < n_sure; i += 64) {
            const double t = scaled(queue[wave][i], s);
            if (t >= s.least) {
                mine += whole_weight(t, s.shift, parts);
                kept += 1;
            }
        }
        mine = wave_scan(mine);
        kept = (uint32_t)wave_scan(kept);
        if (lane == 63 && c < c1) {
            p.chunk_mass[(uint64_t)out * p.chunks + c] = mine;
            p.chunk_count[(uint64_t)out * p.chunks + c] = kept;
        }
        uint32_t at = 0;
        if (lane == 0 && n_list) at = atomicAdd(&listed, n_list);
        __syncthreads();
        if (tid == 0 && listed) listed_at = atomicAdd(&p.rows[out].listed, listed);
        __syncthreads();
        at = listed_at + (uint32_t)__builtin_amdgcn_readfirstlane(at);
        for (uint32_t i = lane; i < n_list; i += 64) {
            if (at + i >= p.list) break;
            const uint32_t from = EACH * 64 - 1 - i, id = c * (EACH * 64) + place[wave][from];
            p.keys[(uint64_t)out * p.list + at + i] = order_key(s.far ? x[id] : queue[wave][from], id);
        }
        if (c + WAVES < c0 + p.per) {
            __syncthreads();
            if (tid == 0) listed = 0;
            __syncthreads();
        }
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) v[i] = next[i];
    }
}

// The key at which the running total of keys >= floor of the row, largest first,
// reaches `target`: of tokens (MASS false) or of weights. 64-bit keys in digits of
// ten bits, each by a histogram of the row's keys with the digits before it: for
// rows with more tokens in one bin than the list holds.
struct Bins {
    unsigned long long mass[kSmBins];
    uint32_t count[kSmBins];
    uint32_t found, found_n;
    uint64_t above, cut;
    // The keys of a bin that one wave looks through.
    uint64_t few_key[64], few_weight[64];
    uint32_t few;
};
template <bool MASS>
__device__ uint64_t find_cut(const RowSettings& s, const double* parts, uint32_t vocab, uint64_t floor, uint64_t target, Bins& b,
                             Together<kSmWaves>& all) {
    const uint32_t tid = threadIdx.x;
    uint64_t prefix = 0, before = 0;
    for (int low = 54, bits = 10;; bits = low < 10 ? 4 : 10, low -= bits) {
        __syncthreads();
        b.mass[tid] = 0;
        b.count[tid] = 0;
        __syncthreads();
        const auto add = [&](float v, uint32_t i) {
            const uint64_t k = order_key(v, i);
            if (k < floor || (low < 54 && (k >> (low + bits)) != prefix)) return;
            const uint32_t at = (1u << bits) - 1 - ((uint32_t)(k >> low) & ((1u << bits) - 1));  // larger ones first
            atomicAdd(&b.count[at], 1u);
            if (MASS) atomicAdd(&b.mass[at], (unsigned long long)whole_weight(scaled(seen(v, s), s), s.shift, parts));
        };
        uint32_t i = tid;
        for (; i + 7 * kSmThreads < vocab; i += 8 * kSmThreads) {
            float v[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) v[e] = s.x[i + e * kSmThreads];
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) add(v[e], i + e * kSmThreads);
        }
        for (; i < vocab; i += kSmThreads) add(s.x[i], i);
        __syncthreads();
        const uint64_t here = MASS ? b.mass[tid] : b.count[tid];
        uint64_t sum, none = 0;
        const uint64_t to = before + all.scan(here, sum, none);
        target = min(target, before + sum);  // where all of them fall short the last one is it
        if (to - here < target && target <= to) {
            b.found = (1u << bits) - 1 - tid;
            b.above = to - here;
        }
        __syncthreads();
        prefix = prefix << bits | b.found;
        before = b.above;
        if (low == 0) return prefix;
    }
}

// The same among one wave's keys (0: none), each against each.
template <bool MASS>
__device__ __forceinline__ uint64_t find_few(uint64_t key, uint64_t w, uint64_t target) {
    uint64_t to = 0;
    for (uint64_t left = __ballot(key != 0); left; left &= left - 1) {
        const uint32_t j = (uint32_t)__builtin_ctzll(left);
        const uint64_t other = MASS ? lane_value(w, j) : 1;
        if (lane_value(key, j) >= key) to += other;
    }
    const uint64_t at = __ballot(key != 0 && to >= target && to - (MASS ? w : 1) < target);
    return at ? lane_value(key, (uint32_t)__builtin_ctzll(at)) : 0;
}

// The same among the keys that a workgroup's threads hold (those of `in`), by
// their distance from the largest of them: 1024 bins over the distances, then over
// those of the bin that the key is in, until that holds no more than a wave's.
// clear: the bins are.
template <bool MASS>
__device__ uint64_t find_listed(const uint64_t (&key)[kSmPerThread], const uint64_t (&w)[kSmPerThread], uint32_t in, uint64_t target,
                                Bins& b, bool& clear, Together<kSmWaves>& all) {
    const uint32_t tid = threadIdx.x;
    uint64_t top = 0, under = 0;  // under: the complement of the smallest
#pragma unroll
    for (uint32_t i = 0; i < kSmPerThread; ++i)
        if (in >> i & 1u) top = max(top, key[i]), under = max(under, ~key[i]);
    all.largest(top, under);
    uint64_t low = ~under, above = 0;
    // Each turn leaves at most a 1024th of the span: seven for 64 bits.
    for (int turn = 0; turn < 7; ++turn) {
        const uint64_t span = top - low;
        const uint32_t sh = span < kSmBins ? 0 : 54 - (uint32_t)__clzll((long long)span);
        if (!clear) {
            b.mass[tid] = 0;
            b.count[tid] = 0;
            if (tid == 0) b.few = 0;
            __syncthreads();
        }
        clear = false;
#pragma unroll
        for (uint32_t i = 0; i < kSmPerThread; ++i)
            if (in >> i & 1u) {
                const uint32_t at = (uint32_t)((top - key[i]) >> sh);
                atomicAdd(&b.count[at], 1u);
                if (MASS) atomicAdd(&b.mass[at], (unsigned long long)w[i]);
            }
        __syncthreads();
        const uint32_t num = b.count[tid];
        const uint64_t here = MASS ? b.mass[tid] : num;
        uint64_t sum, none = 0;
        const uint64_t to = above + all.scan(here, sum, none);
        if (to - here < target && target <= to) {
            b.found = tid;
            b.found_n = num;
            b.above = to - here;
        }
        __syncthreads();
        const uint32_t at = b.found, n = b.found_n;
        above = b.above;
        if (sh == 0) return top - at;
#pragma unroll
        for (uint32_t i = 0; i < kSmPerThread; ++i) {
            if (!(in >> i & 1u)) continue;
            if ((uint32_t)((top - key[i]) >> sh) != at) {
                in &= ~(1u << i);
            } else if (n <= 64) {
                const uint32_t to_few = atomicAdd(&b.few, 1u);
                b.few_key[to_few] = key[i];
                b.few_weight[to_few] = w[i];
            }
        }
        if (n <= 64) {
            __syncthreads();
            if (tid < 64) {
                const uint64_t cut = find_few<MASS>(tid < n ? b.few_key[tid] : 0, tid < n ? b.few_weight[tid] : 0, target - above);
                if (tid == 0) b.cut = cut;
            }
            __syncthreads();
            return b.cut;
        }
        const uint64_t end = top - ((uint64_t)at << sh), last = end - (((uint64_t)1 << sh) - 1);
        low = max(low, last);  // (of two different integer types max would go through doubles)
        top = end;
    }
    return top;
}

// One workgroup per row: the cut among the listed tokens, the chunk in which the
// running sum passes u times all, and the token in it. What does not depend on
// another load is loaded first.
__global__ __launch_bounds__(kSmThreads) void sample_draw_kernel(SampleArgs a, SmPlan p) {
    __shared__ uint64_t memory[2][2][kSmWaves];
    __shared__ double parts[kSmParts];
    __shared__ Bins bins;
    __shared__ unsigned long long in_chunks[kSmThreads];  // the list's kept weights, by group of chunks
    __shared__ uint32_t found;
    __shared__ uint64_t found_before;
    const uint32_t out = blockIdx.x, tid = threadIdx.x;
    const RowSettings s = p.settings[out];
    const SmRow r = p.rows[out];
    // Kept weights by group of chunks, a thread for each group.
    const uint32_t per = (p.chunks + kSmThreads - 1) / kSmThreads;
    uint64_t mine = 0, kept = 0;
    const auto add_chunks = [&] {
        for (uint32_t c = tid * per; c < min((tid + 1) * per, p.chunks); ++c) {
            mine += p.chunk_mass[(uint64_t)out * p.chunks + c];
            kept += p.chunk_count[(uint64_t)out * p.chunks + c];
        }
    };
    if (s.mode >= kSmAll) add_chunks();
    uint64_t key[kSmPerThread], w[kSmPerThread];
    key[0] = tid < p.list ? p.keys[(uint64_t)out * p.list + tid] : 0;
    fill_parts(parts);
    if (s.mode == kSmAbsent) return;
    if (s.mode < kSmAll) {
        if (tid == 0) {
            const bool first = s.mode == kSmFirst;
            if (!first) report(a.status, s.mode == kSmNoRow ? kBadSampleRow : s.mode == kSmBadSetting ? kBadSampleSetting : kNoSampleToken);
            a.tokens[out] = first ? 0xFFFFFFFFu - (uint32_t)s.best : kNoToken;
            if (a.probs) a.probs[out] = first ? 1.0f : __builtin_nanf("");
            if (a.kept) a.kept[out] = first;
        }
        return;
    }
    Together<kSmWaves> all{memory};
    bins.mass[tid] = 0;
    bins.count[tid] = 0;
    in_chunks[tid] = 0;
    if (tid == 0) bins.few = 0;
    __syncthreads();
    uint64_t cut = kLeastKey;
    uint32_t in = 0, in_k = 0, in_p = 0;
    bool clear = true;  // the bins are
    if (s.mode == kSmCut) {
        if (r.listed <= p.list) {
#pragma unroll
            for (uint32_t i = 0; i < kSmPerThread; ++i) {
                const uint32_t at = i * kSmThreads + tid;
                w[i] = 0;
                if (at >= r.listed) {
                    key[i] = 0;
                    continue;
                }
                if (i) key[i] = p.keys[(uint64_t)out * p.list + at];
                const float v = seen(key_value(key[i]), s);
                const uint32_t b = bin_of(v, s);
                w[i] = whole_weight(scaled(v, s), s.shift, parts);
                in |= 1u << i;
                in_k |= (uint32_t)(b == r.k_bin) << i;
                in_p |= (uint32_t)(b >= r.p_lo && b <= r.p_hi) << i;
            }
            // Up to 64 are the first wave's.
            const bool few = r.listed <= 64;
            const auto find = [&](auto mass, uint32_t among, uint64_t target) -> uint64_t {
                constexpr bool kMass = decltype(mass)::value;
                if (!few) return find_listed<kMass>(key, w, among, target, bins, clear, all);
                if (tid < 64) {
                    const uint64_t c = find_few<kMass>(among & 1u ? key[0] : 0, w[0], target);
                    if (tid == 0) bins.cut = c;
                }
                __syncthreads();
                return bins.cut;
            };
            uint64_t sum = 0;
            if (r.k_bin != kNoBin) {
                cut = find(std::false_type(), in_k, r.k_rank);
                if (s.by_mass) {
#pragma unroll
                    for (uint32_t i = 0; i < kSmPerThread; ++i)
                        if ((in_k >> i & 1u) && key[i] >= cut) sum += w[i];
                    sum = r.k_mass + all.sum(sum);  // (its barrier: all have read bins.cut)
                }
            } else {
                sum = r.mass;
            }
            if (s.by_mass) {
#pragma unroll
                for (uint32_t i = 0; i < kSmPerThread; ++i)
                    if ((in_p >> i & 1u) && key[i] < cut) in_p &= ~(1u << i);
                cut = max(cut, find(std::true_type(), in_p, mass_target(s.p, sum) - r.p_mass));
            }
        } else {
            // More than the list holds: over all logits again.
            if (s.k) cut = max(cut, find_cut<false>(s, parts, a.vocab, cut, s.k, bins, all));
            if (s.by_mass) {
                uint64_t sum = 0;
                for (uint32_t i = tid; i < a.vocab; i += kSmThreads) {
                    const float v = s.x[i];
                    if (order_key(v, i) >= cut) sum += whole_weight(scaled(seen(v, s), s), s.shift, parts);
                }
                sum = all.sum(sum);
                cut = max(cut, find_cut<true>(s, parts, a.vocab, cut, mass_target(s.p, sum), bins, all));
            }
            // (as the launches over pieces leave them where the list suffices)
            for (uint32_t c = tid >> 6; c < p.chunks; c += kSmWaves) {
                uint64_t sum = 0;
                uint32_t n = 0;
                for (uint32_t i = c * p.chunk + (tid & 63); i < min((c + 1) * p.chunk, a.vocab); i += 64) {
                    const float v = s.x[i];
                    const double t = scaled(seen(v, s), s);
                    if (order_key(v, i) >= cut && t >= s.least) sum += whole_weight(t, s.shift, parts), ++n;
                }
                sum = wave_scan(sum);
                n = (uint32_t)wave_scan(n);
                if ((tid & 63) == 63) {
                    p.chunk_mass[(uint64_t)out * p.chunks + c] = sum;
                    p.chunk_count[(uint64_t)out * p.chunks + c] = n;
                }
            }
            __syncthreads();
            mine = kept = 0;
            add_chunks();
        }
        // What the list keeps, to its groups.
#pragma unroll
        for (uint32_t i = 0; i < kSmPerThread; ++i) {
            if (!(in >> i & 1u)) continue;
            if (key[i] < cut || !(scaled(seen(key_value(key[i]), s), s) >= s.least)) {
                in &= ~(1u << i);
                continue;
            }
            ++kept;
            atomicAdd(&in_chunks[(0xFFFFFFFFu - (uint32_t)key[i]) / p.chunk / per], (unsigned long long)w[i]);
        }
        __syncthreads();
        mine += in_chunks[tid];
    }
    uint64_t sum;
    const uint64_t to = all.scan(mine, sum, kept);
    const uint64_t target = (uint64_t)((double)s.u * (double)sum);
    if (mine && to > target && to - mine <= target) found = tid, found_before = to - mine;
    __syncthreads();
    // The chunk of the group.
    const uint32_t group = found;
    uint64_t before = found_before;
    uint32_t chunk = group * per;
    if (per > 1) {
        bins.mass[tid] = tid < per && chunk + tid < p.chunks ? p.chunk_mass[(uint64_t)out * p.chunks + chunk + tid] : 0;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kSmPerThread; ++i) {
            const uint32_t c = (0xFFFFFFFFu - (uint32_t)key[i]) / p.chunk;
            if ((in >> i & 1u) && c / per == group) atomicAdd(&bins.mass[c - chunk], (unsigned long long)w[i]);
        }
        __syncthreads();
        for (uint32_t c = 0; c + 1 < per && before + bins.mass[c] <= target; ++c) {
            before += bins.mass[c];
            ++chunk;
        }
    }
    const uint32_t id = chunk * p.chunk + tid;
    uint64_t here = 0;
    double t = 0.0;
    if (tid < p.chunk && id < a.vocab) {
        const float v = s.x[id];
        t = scaled(seen(v, s), s);
        if (order_key(v, id) >= cut && t >= s.least) here = whole_weight(t, s.shift, parts);
    }
    uint64_t in_chunk, none = 0;
    const uint64_t now = before + all.scan(here, in_chunk, none);
    if (here && now > target && now - here <= target) {
        a.tokens[out] = id;
        if (a.probs) a.probs[out] = (float)(weight(t, s.shift, parts) / (double)sum);
        if (a.kept) a.kept[out] = (uint32_t)kept;
    }
}

SmPlan sm_plan(uint64_t n_rows, uint64_t vocab) {
    SmPlan p{};
    // Whole chunks for each of a piece's waves, in as few turns as leave enough pieces.
    const uint64_t most = (vocab + kSmTurn - 1) / kSmTurn;
    const uint64_t turns = std::max<uint64_t>(n_rows * most / kSmWorkgroups, 1);
    p.waves = n_rows * most <= kSmWorkgroups ? kSmWide : kSmNarrow;
    p.chunk = kSmTurn / p.waves;
    p.chunks = (uint32_t)((vocab + p.chunk - 1) / p.chunk);
    p.per = (uint32_t)std::min(turns, most) * p.waves;
    p.pieces = (p.chunks + p.per - 1) / p.per;
    p.list = (uint32_t)std::min<uint64_t>(kSmList, vocab);
    return p;
}
uint64_t sm_layout(SmPlan& p, uint64_t n_rows, uint8_t* base) {
    uint64_t at = 0;
    const auto take = [&](uint64_t bytes) {
        uint8_t* here = base + at;
        at += (bytes + 15) / 16 * 16;
        return here;
    };
    p.best = reinterpret_cast<uint64_t*>(take(n_rows * p.pieces * 8));
    p.lowest = reinterpret_cast<float*>(take(n_rows * p.pieces * 4));
    p.mass = reinterpret_cast<unsigned long long*>(take(n_rows * kSmBins * 8));
    p.count = reinterpret_cast<uint32_t*>(take(n_rows * kSmBins * 4));
    p.chunk_mass = reinterpret_cast<uint64_t*>(take(n_rows * p.chunks * 8));
    p.chunk_count = reinterpret_cast<uint32_t*>(take(n_rows * p.chunks * 4));
    p.keys = reinterpret_cast<uint64_t*>(take(n_rows * p.list * 8));
    p.rows = reinterpret_cast<SmRow*>(take(n_rows * sizeof(SmRow)));
    p.asked = reinterpret_cast<RowSettings*>(take(n_rows * sizeof(RowSettings)));
    p.settings = reinterpret_cast<RowSettings*>(take(n_rows * sizeof(RowSettings)));
    return at;
}

}  // namespace

uint64_t sample_workspace_bytes(uint64_t n_rows, uint64_t vocab) {
    if (n_rows == 0 || vocab == 0) return 0;
    SmPlan p = sm_plan(n_rows, vocab);
    return sm_layout(p, n_rows, nullptr);
}

hipError_t launch_sample(const SampleArgs& a_in, uint64_t n_rows, hipStream_t s) {
    if (n_rows == 0) return hipSuccess;
    SampleArgs a = a_in;
    uint32_t bits = 0;
    while ((1ull << bits) < a.vocab) ++bits;
    a.shift = bits <= 18 ? 44 : 62 - bits;
    SmPlan p = sm_plan(n_rows, a.vocab);
    sm_layout(p, n_rows, static_cast<uint8_t*>(a.work));
    const unsigned grid = (unsigned)(n_rows * p.pieces);
    const bool wide = p.waves == kSmWide;
    const unsigned threads = p.waves * 64;
    (wide ? sample_best_kernel<kSmWide, kSmTurn / kSmWide / 64> : sample_best_kernel<kSmNarrow, kSmTurn / kSmNarrow / 64>)
        <<<grid, threads, 0, s>>>(a, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    (wide ? sample_bins_kernel<kSmWide, kSmTurn / kSmWide / 64> : sample_bins_kernel<kSmNarrow, kSmTurn / kSmNarrow / 64>)
        <<<grid, threads, 0, s>>>(a, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    (wide ? sample_list_kernel<kSmWide, kSmTurn / kSmWide / 64> : sample_list_kernel<kSmNarrow, kSmTurn / kSmNarrow / 64>)
        <<<grid, threads, 0, s>>>(a, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    sample_draw_kernel<<<(unsigned)n_rows, kSmThreads, 0, s>>>(a, p);
    return hipGetLastError();
}

}  // namespace mmhip
