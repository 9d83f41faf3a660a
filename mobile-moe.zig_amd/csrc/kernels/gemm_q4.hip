// 4-bit weights (q4_ops.hpp) times many f32 vectors on gfx950's f16 matrix
// cores: prompts.
//
// The integer weights are exact in f16. A vector's value, times a power of two, is
// the sum of two f16 numbers: the nearest one, and the nearest to what that leaves.
// That is off by 2^-23 of the value at most, or by half of f16's smallest step, 2^-25,
// where that is more. So the power of two goes with the vector's values: the largest
// of every 128 columns lies in [2^6, 2^15) (the last step is at most 2^-31 of it), and
// where the power changes the sums so far change with it. It stays within 2^64 of its
// smallest, which keeps the sums in range: beside a value 2^64 and more times as large
// a value may be off by 2^-95 of that. A 32-column block of 16 weight rows times 16
// vectors is two v_mfma_f32_16x16x32_f16 (the smaller parts first) and one
// multiply-add per output with the block's scale.
//
// Bound: vector instructions (per value of x two conversions, per eight weights
// 9 or 21 operations, per output and block one multiply-add), matrix cores and LDS
// together: of a large prompt's time they take 46, 34 and 47 hundredths. A workgroup's waves share the x tile in LDS: each converts its part of
// the next 64 columns while the matrix cores work on the last ones, and a wave
// unpacks weights of its own rows straight from their records. Waves may also
// split the columns (KS groups), their sums added at the end.
//
// Measured: [10240 x 2048] times 256 vectors 33.0 us (325 Tflop/s of products; the
// two matrix instructions per product alone would take 17 us), [3840 x 768] times
// 77 vectors 7.5 us; with bf16 parts (three instructions per product, four
// conversions) 74 and 10.9 us.
#include <type_traits>

#include "device_common.hpp"
#include "gemm_tile_ops.hpp"
#include "kernels.hpp"
#include "q4_ops.hpp"

namespace mmhip {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct GemmQ4Args {
    const uint4* recs;
    const uint16_t* dvals;
    const float* x;
    float* y;
    uint64_t x_stride, y_slot, y_row;  // y[slot * y_slot + row * y_row]
    uint32_t batch, cols, tiles, units, rows, d_row;
    uint32_t rec_bytes, d_bytes;
    uint32_t groups, items;  // tile groups, groups of vectors
    uint32_t wg_tiles;       // weight tiles of a workgroup: at most NJ for each of its RS waves
};

// Eight weights as f16, in the order of columns 0 2, 4 6, 1 3, 5 7: 0x6400 | u is
// 1024 + u, 0x5400 | u << 4 is 64 + u.
__device__ __forceinline__ uint32_t f16_less(uint32_t h, float by) {
    const f16x2 b = {(_Float16)by, (_Float16)by};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, h) - b);
}
template <int FMT>
__device__ __forceinline__ f16x8 q4_bop_f16(uint32_t d) {
    uint32_t h[4];
    if constexpr (FMT == kFmtQ4) {
        // (the stored codes have their top bit flipped)
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const uint32_t e = d >> (4 * k);
            h[k] = f16_less((e & 0x000F000Fu) ^ 0x64086408u, 1032.0f);
            h[k + 1] = f16_less((e & 0x00F000F0u) ^ 0x54805480u, 72.0f);
        }
    } else {
        uint32_t w[2];
        q4_words<FMT>(d, w[0], w[1]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            h[k] = f16_less(__builtin_amdgcn_perm(0x64646464u, w[k & 1] ^ 0x80808080u, k < 2 ? 0x04020400u : 0x04030401u), 1152.0f);
    }
    return __builtin_bit_cast(f16x8, make_uint4(h[0], h[1], h[2], h[3]));
}

// A half step's x tile in LDS: 64 columns of MT * 16 vectors, per 16 vectors and
// part eight runs (block, column group), each the 16 vectors' eight columns in
// the weights' order. Vectors' places are changed four by four, in an order of
// its own for each column group: a wave's 16-byte reads meet no bank twice, its
// 4-byte writes (eight runs, four vectors) none more than twice.
constexpr uint32_t kQ4Run = 256, kQ4Part = 8 * kQ4Run;
__device__ __forceinline__ uint32_t run_place(uint32_t vec, uint32_t group) {
    return (vec & 15) ^ ((0x2130u >> (4 * group) & 3u) << 2);  // 0 3 1 2 fours for groups 0 1 2 3
}

// The power of two that takes a largest |x| into [2^12, 2^13), or as near to that as
// f32 has one: room for values four times as large, and for a 64th.
__device__ __forceinline__ int fit(float most) { return 139 - (int)min(max(__float_as_uint(most) >> 23, 12u), 254u); }
__device__ __forceinline__ float power_of_two(int k) { return __uint_as_float((uint32_t)(127 + k) << 23); }
constexpr float kQ4Fits = 32768.0f, kQ4Low = 64.0f;
constexpr int kQ4Up = 64;
__device__ __forceinline__ float row_max(float m) {  // over 16 lanes
    m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0xB1, 0xF, 0xF, false)));
    m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0x4E, 0xF, 0xF, false)));
    m = fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0x141, 0xF, 0xF, false)));
    return fmaxf(m, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(m), 0x140, 0xF, 0xF, false)));
}
// The largest of eight |x|, NaN left out (fmaxf would quiet each operand first).
__device__ __forceinline__ float max_abs(const uint4& v, const uint4& w) {
    float m;
    asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(m) : "v"(v.x), "v"(v.y), "v"(v.z));
    asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m) : "v"(v.w), "v"(w.x));
    asm("v_max3_f32 %0, %0, |%1|, |%2|" : "+v"(m) : "v"(w.y), "v"(w.z));
    asm("v_max_f32 %0, %0, |%1|" : "+v"(m) : "v"(w.w));
    return m;
}
// Of 64 lanes' truth values, one bit for each 16: is one of them true.
__device__ __forceinline__ uint32_t any_of_rows(uint64_t which) {
    uint64_t b;
    asm("s_quadmask_b64 %0, %1\n\ts_quadmask_b64 %0, %0" : "=&s"(b) : "s"(which) : "scc");
    return (uint32_t)b;
}

// MT: 16 vectors each; NJ: 16 weight rows each of a wave; RS waves share an x
// tile, KS groups of them the columns. WAVES of a SIMD fit its registers.
//
// The wave that stages a unit's values looks at their largest before. Where one has
// left the range of its vector's power of two, the wave takes another one and says so
// in LDS, and the waves that read the values change their sums before that unit;
// otherwise nothing of this is in the loop but seven vector instructions for eight
// columns and two branches a unit. (For values of a normal distribution the power
// stays as the first unit sets it. A branch each 64 columns instead of 128 costs
// [10240 x 2048] times 256 2 us.)
template <int FMT, int MT, int NJ, int RS, int KS, int WAVES>
__global__ __launch_bounds__(RS * KS * 64, WAVES) void gemm_q4_kernel(GemmQ4Args a) {
    constexpr int kQuads = MT * 4 / RS;                              // of x, a thread and half step
    static_assert(kQuads >= 1 && MT * 4 % RS == 0, "a wave stages whole rows of four vectors");
    constexpr uint32_t kBuf = MT * 2 * kQ4Part;
    constexpr uint32_t kSlot = MT * NJ * 4 * 64;                     // floats of a wave's sums
    constexpr uint32_t kRed = KS > 1 ? RS * KS * kSlot * 4 : 0, kMain = KS * 2 * kBuf;
    constexpr int kAhead = 2;
    __shared__ __align__(16) uint8_t lds[kRed > kMain ? kRed : kMain];
    // For two turns: how much the vectors' powers of two have grown, and the turn for which
    // each staging wave (any of them) has said so. In the end, the powers undone.
    __shared__ __align__(16) int grown[KS][2][MT * 16];
    __shared__ uint32_t grown_at[KS][2][RS], any_at[KS][2];
    // Tile group tg runs on XCD tg % 8, its groups of vectors one after the other:
    // each XCD's L2 holds an eighth of the matrix, read once.
    const uint32_t r8 = blockIdx.x >> 3, item = r8 % a.items, tg = r8 / a.items * 8 + (blockIdx.x & 7);
    if (tg >= a.groups) return;  // whole workgroup
    const uint32_t first = item * (MT * 16), count = min(a.batch - first, MT * 16u);
    const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t rw = wave % RS, kg = wave / RS;
    const BufRsrc rec_r = make_rsrc(a.recs, a.rec_bytes), d_r = make_rsrc(a.dvals, a.d_bytes);
    const BufRsrc x_r = make_rsrc(a.x + first * a.x_stride, (uint32_t)(((count - 1) * a.x_stride + a.cols) * 4));
    uint8_t* const xs = lds + kg * 2 * kBuf;
    // Its tiles, as evenly over the waves as they go.
    const uint32_t each = a.wg_tiles / RS, more = a.wg_tiles % RS;
    const uint32_t tile0 = tg * a.wg_tiles + rw * each + min(rw, more), n_tiles = each + (rw < more);
    if (lane < 2) grown_at[kg][lane][rw] = any_at[kg][lane] = 0;

    // Units of this group; all groups take as many turns.
    const uint32_t u0 = a.units * kg / KS, u1 = a.units * (kg + 1) / KS, turns = (a.units + KS - 1) / KS;
    // This lane stages four columns of vectors r0 + 4 RS i.
    const uint32_t r0 = 4 * rw + g;
    uint32_t x_voff[kQuads];
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
        const uint32_t r = r0 + 4 * RS * i;
        x_voff[i] = r < count ? (uint32_t)(r * a.x_stride + 4 * n) * 4 : kBufOob;
    }
    const uint32_t upper = n >= 8 ? kBufOob : 0;  // of a half step: out of range where columns end in its middle
    uint8_t* const dst = xs + (n >> 1) * kQ4Run + (n & 1) * 4 + (r0 >> 4) * (2 * kQ4Part);
    uint32_t place[4];  // of vectors r0 + 4 RS i: the same for all where RS is 4 or 8
#pragma unroll
    for (int i = 0; i < 4; ++i) place[i] = run_place(r0 + 4 * RS * i, (n >> 1) & 3) * 16;

    f32x4 acc[MT][NJ];
    int power[kQuads], least[kQuads];  // a vector's power of two, and the smallest it has had
    float absent[kQuads];              // in range where there is no vector, otherwise 0
#pragma unroll
    for (int i = 0; i < kQuads; ++i) absent[i] = r0 + 4 * RS * i < count ? 0.0f : kQ4Low;
    // Loads in flight: of x one unit's first half and two units' second ones (a unit's
    // largest is looked at before its first half goes to LDS), of the weights kAhead units.
    uint4 x0[kQuads], x1[2][kQuads], wv[kAhead][NJ];
    uint32_t dv[kAhead][NJ];
    const auto load_x = [&](uint32_t u, int h, uint4 (&to)[kQuads]) {
        const uint32_t col = u * kQ4UnitCols + 64 * h;
        const uint32_t part = u < u1 && col + 32 == a.cols ? upper : 0;
        const uint32_t soff = u < u1 && col < a.cols ? col * 4 : kBufOob;
#pragma unroll
        for (int i = 0; i < kQuads; ++i) to[i] = buf_load_b128(x_r, x_voff[i] | part, soff);
    };
    const auto load_w = [&](auto nj, uint32_t u, uint4 (&wq)[NJ], uint32_t (&dq)[NJ]) {
#pragma unroll
        for (int j = 0; j < nj(); ++j) {
            const uint32_t t = tile0 + j;
            const bool ok = u < u1 && t < a.tiles && j < (int)n_tiles;
            wq[j] = buf_load_b128(rec_r, lane * 16, ok ? (t * a.units + u) * 1024 : kBufOob);
            dq[j] = buf_load_b16(d_r, lane * 8, ok ? t * a.d_row * 32 + (u >> 2) * kQ4StepScaleBytes + (u & 3) * 2 : kBufOob);
        }
    };
    // Are the largest of a unit, as loaded, out of range of the last one's power of two?
    // (Yes also where a lane has not one of all its vectors in range: adapt() tells.)
    const auto out_of_range = [&](uint32_t u, int q) {
        float low = kQ4Low, most = kQ4Low;
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            const float at = fmaf(max_abs(x0[i], x1[q][i]), power_of_two(power[i]), absent[i]);
            low = i ? fminf(low, at) : at;
            most = i ? fmaxf(most, at) : at;
        }
        const bool out = (__ballot(most >= kQ4Fits) != 0) | (any_of_rows(__ballot(low >= kQ4Low)) != 15);
        return out && u < u1;
    };
    // The powers of two for it, the turn-th.
    const auto adapt = [&](uint32_t turn, int q) {
        bool changed = false;
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            const float m = row_max(max_abs(x0[i], x1[q][i])), at = m * power_of_two(power[i]);
            int by = 0;
            if (at >= kQ4Fits || (m > 0.0f && at < kQ4Low)) by = min(fit(m), least[i] + kQ4Up) - power[i];
            power[i] += by;
            least[i] = min(least[i], power[i]);
            changed |= by != 0;
            if (n == 0) grown[kg][turn & 1][r0 + 4 * RS * i] = by;
        }
        if (__any(changed) && lane == 0) grown_at[kg][turn & 1][rw] = any_at[kg][turn & 1] = turn;
    };
    // The sums so far, as the turn-th unit wants them.
    const auto follow = [&](uint32_t turn) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int4 by = *reinterpret_cast<const int4*>(&grown[kg][turn & 1][m * 16 + 4 * g]);
            const bool said = grown_at[kg][turn & 1][(4 * m + g) % RS] == turn;
            const int b[4] = {said ? by.x : 0, said ? by.y : 0, said ? by.z : 0, said ? by.w : 0};
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[m][j][e] = ldexpf(acc[m][j][e], b[e]);
        }
    };
    // Half h's loaded values into its buffer.
    const auto stage = [&](int h, const uint4 (&from)[kQuads]) {
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            const float s = power_of_two(power[i]);
            const float v[4] = {__uint_as_float(from[i].x), __uint_as_float(from[i].y), __uint_as_float(from[i].z),
                                __uint_as_float(from[i].w)};
            _Float16 hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi[e] = (_Float16)(v[e] * s);
                lo[e] = (_Float16)fmaf(v[e], s, -(float)hi[e]);
            }
            uint8_t* p = dst + place[RS >= 4 ? 0 : i & 3] + h * kBuf + (4 * RS * i >> 4) * (2 * kQ4Part);
            *reinterpret_cast<f16x2*>(p) = f16x2{hi[0], hi[2]};
            *reinterpret_cast<f16x2*>(p + 8) = f16x2{hi[1], hi[3]};
            *reinterpret_cast<f16x2*>(p + kQ4Part) = f16x2{lo[0], lo[2]};
            *reinterpret_cast<f16x2*>(p + kQ4Part + 8) = f16x2{lo[1], lo[3]};
        }
    };
    const auto products = [&](auto nj, int h, const uint4 (&w)[NJ], const float (&c)[NJ][4]) {
        const uint8_t* src = xs + h * kBuf + g * kQ4Run + run_place(n, g) * 16;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            f16x8 hi[MT], lo[MT];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const uint8_t* p = src + m * (2 * kQ4Part) + b * 4 * kQ4Run;
                hi[m] = __builtin_bit_cast(f16x8, *reinterpret_cast<const uint4*>(p));
                lo[m] = __builtin_bit_cast(f16x8, *reinterpret_cast<const uint4*>(p + kQ4Part));
            }
#pragma unroll
            for (int j = 0; j < nj(); ++j) {
                const f16x8 wb = q4_bop_f16<FMT>(h == 0 ? (b == 0 ? w[j].x : w[j].y) : (b == 0 ? w[j].z : w[j].w));
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
                    p = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo[m], wb, p, 0, 0, 0);
                    p = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi[m], wb, p, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[m][j][e] = fmaf(p[e], c[j][2 * h + b], acc[m][j][e]);
                }
            }
        }
    };

    // A wave that shares its tile with no other needs only the order of its own accesses
    // ([768 x 8192] times 64 15.9 us, with barriers 19.0).
    const auto staged = [] {
        if constexpr (RS == 1) wave_lds_order();
        else lds_barrier();
    };
    // Sums that the compiler does not put off beyond a branch, where a wave's products
    // would not fit the registers otherwise: [10240 x 2048] times 256 33.0 us, without them
    // 34.3; times 512 with four waves a SIMD 61.8 and 107.
    constexpr int kSettleFirst = MT >= 4 ? 1 : MT * NJ == 4 && WAVES == 4 ? 2 : 0, kSettleSecond = MT >= 4 ? 1 : 0;
    const auto settle = [&](auto nj, auto count) {
#pragma unroll
        for (int m = 0; m < count(); ++m)
#pragma unroll
            for (int j = 0; j < nj(); ++j) {
                f32x4& sums = acc[m][j];
                asm volatile("" : "+v"(sums));
            }
    };
    // All columns, for a wave with so many tiles. As many barriers whatever it has.
    const auto sweep = [&](auto nj) {
        load_x(u0, 0, x0);
        load_x(u0, 1, x1[0]);
#pragma unroll
        for (int q = 0; q < kAhead; ++q) load_w(nj, u0 + q, wv[q], dv[q]);
        load_x(u0 + 1, 1, x1[1]);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[m][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kQuads; ++i) power[i] = least[i] = fit(row_max(max_abs(x0[i], x1[0][i])));
        stage(0, x0);
        load_x(u0 + 1, 0, x0);
        staged();
        bool said = false;
        for (uint32_t k = 0; k < turns; k += kAhead) {
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
                if (k + q >= turns) break;  // for the whole workgroup
                const uint32_t u = u0 + k + q;
                if (said) follow(k + q);
                float c[NJ][4];
#pragma unroll
                for (int j = 0; j < nj(); ++j) broadcast_rows4(f16_scale((uint16_t)dv[q][j]), c[j]);
                stage(1, x1[q]);
                load_x(u + 2, 1, x1[q]);
                products(nj, 0, wv[q], c);
                settle(nj, std::integral_constant<int, kSettleFirst>());
                if (out_of_range(u + 1, q ^ 1)) adapt(k + q + 1, q ^ 1);
                staged();
                const uint32_t any = any_at[kg][q ^ 1];
                stage(0, x0);
                load_x(u + 2, 0, x0);
                products(nj, 1, wv[q], c);
                load_w(nj, u + kAhead, wv[q], dv[q]);
                settle(nj, std::integral_constant<int, kSettleSecond>());
                said = (uint32_t)__builtin_amdgcn_readfirstlane(any) == k + q + 1;
                staged();
            }
        }
    };
    if (NJ > 1 && n_tiles < NJ) sweep(std::integral_constant<int, (NJ > 1 ? NJ - 1 : 1)>());
    else sweep(std::integral_constant<int, NJ>());

    // The vectors' powers of two, undone.
#pragma unroll
    for (int i = 0; i < kQuads; ++i)
        if (n == 0) grown[kg][0][r0 + 4 * RS * i] = -power[i];
    lds_barrier();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int4 by = *reinterpret_cast<const int4*>(&grown[kg][0][m * 16 + 4 * g]);
        const int b[4] = {by.x, by.y, by.z, by.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[m][j][e] = ldexpf(acc[m][j][e], b[e]);
    }
    float odd = 0.0f;  // NaN once a result is infinite or NaN
    const auto place_in_y = [&](uint32_t m, uint32_t j, uint32_t e) -> float* {
        const uint32_t t = m * 16 + 4 * g + e, row = (tile0 + j) * 16 + n;
        return j < n_tiles && t < count && row < a.rows ? a.y + ((uint64_t)(first + t) * a.y_slot + (uint64_t)row * a.y_row) : nullptr;
    };
    const auto put = [&](uint32_t m, uint32_t j, uint32_t e, float v) {
        const uint32_t t = m * 16 + 4 * g + e, row = (tile0 + j) * 16 + n;
        if (j < n_tiles && t < count && row < a.rows) a.y[(uint64_t)(first + t) * a.y_slot + (uint64_t)row * a.y_row] = v;
        odd = fmaf(v, 0.0f, odd);
    };
    if constexpr (KS == 1) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) put(m, j, e, acc[m][j][e]);
    } else {
        float* const red = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) red[wave * kSlot + ((m * NJ + j) * 4 + e) * 64 + lane] = acc[m][j][e];
        lds_barrier();
        for (uint32_t q = kg; q < MT * NJ; q += KS) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; ++k) v += red[(k * RS + rw) * kSlot + (q * 4 + e) * 64 + lane];
                put(q / NJ, q % NJ, e, v);
            }
        }
    }
    if (odd == odd) return;
#pragma unroll 1
    for (uint32_t q = KS > 1 ? kg : 0; q < MT * NJ; q += KS)
#pragma unroll 1
        for (uint32_t e = 0; e < 4; ++e) {
            float* const y = place_in_y(q / NJ, q % NJ, e);
            if (y && !(fabsf(*y) < INFINITY))
                *y = q4_defined<FMT>(a.recs, a.dvals, a.units, a.d_row, a.cols, (tile0 + q % NJ) * 16 + n,
                                     a.x + (uint64_t)(first + q / NJ * 16 + 4 * g + e) * a.x_stride);
        }
}

// A launch's tile: 16 mt vectors by `tiles` weight tiles (at most nj for each of
// rs waves), ks groups of columns; waves a SIMD.
struct Shape {
    int mt, nj, rs, ks;
    uint32_t tiles;
    int waves = 2;
};
template <int FMT>
const void* fn_of(const Shape& t) {
    if (t.mt == 4) return reinterpret_cast<const void*>(&gemm_q4_kernel<FMT, 4, 2, 8, 1, 2>);
    if (t.mt == 2 && t.ks == 2) return reinterpret_cast<const void*>(&gemm_q4_kernel<FMT, 2, 1, 8, 2, 4>);
    if (t.mt == 2 && t.waves == 2) return reinterpret_cast<const void*>(&gemm_q4_kernel<FMT, 2, 2, 8, 1, 2>);
    if (t.mt == 2) return reinterpret_cast<const void*>(&gemm_q4_kernel<FMT, 2, 2, 8, 1, 4>);
    if (t.ks == 8) return reinterpret_cast<const void*>(&gemm_q4_kernel<FMT, 1, 1, 1, 8, 2>);
    if (t.ks == 4 && t.rs == 2) return reinterpret_cast<const void*>(&gemm_q4_kernel<FMT, 1, 1, 2, 4, 2>);
    if (t.ks == 4 && t.nj == 2) return reinterpret_cast<const void*>(&gemm_q4_kernel<FMT, 1, 2, 4, 4, 4>);
    if (t.ks == 4) return reinterpret_cast<const void*>(&gemm_q4_kernel<FMT, 1, 1, 4, 4, 4>);
    if (t.ks == 2) return reinterpret_cast<const void*>(&gemm_q4_kernel<FMT, 1, 2, 4, 2, 2>);
    return reinterpret_cast<const void*>(&gemm_q4_kernel<FMT, 1, 2, 4, 1, 2>);
}

// By the number of 16 x 16 tiles of the result. Few: up to a workgroup per CU with
// four groups of columns and two or four tiles (or eight groups, where rows are long
// and one tile makes enough workgroups). {1,1,1,8} / {1,1,2,4} / {1,1,4,4}, us:
// [768 x 8192] times 64 (192 tiles) 15.2 / 20.6 / 23.1, [2048 x 2560] times 20 (256) 8.3 /
// 8.6 / 9.9, times 64 (512) 14.8 / 8.7 / 9.9, times 100 (896) 27.2 / 12.7 / 10.0,
// [3840 x 768] times 32 (480) 9.0 / 5.4 / 6.3.
//
// Then larger tiles and fewer groups. {1,1,4,4} / {1,2,4,2} / {2,1,8,2} / {2,2,8,1} /
// {4,2,8,1}: [2048 x 2560] times 128 (1024 tiles) 10.5 / 14.9 / 19.7 / 30.0 / 34.6, times
// 256 (2048) 18.7 / 15.1 / 19.9 / 30.2 / 34.9; [3840 x 768] times 256 (3840) 20.5 / 10.0 /
// 9.3 / 12.0 / 13.9; [10240 x 2048] times 64 (2560) 23.0 / 18.3 / 16.8 / 25.0 / 29.1, times
// 256 (10240) 72 / 42.7 / 46.9 / 40.2 / 33.3.
// Between four and eight tiles per CU {1,2,4,4} is ahead of {1,2,4,2} where rows are
// long: [3840 x 2048] times 77 11.7 / 12.5, [1536 x 4096] times 256 19.7 / 21.7, but [5120
// x 1664] times 64 11.6 / 11.4.
//
// Many: the two largest tiles by what they cost, rounds of one workgroup per CU
// times a round's time, in hundredths of a microsecond a unit (fitted to the above
// and, {2,2,8,1} before {4,2,8,1}: times 128 25.4 / 29.5, times 512 61.9 / 63.6; [3840 x
// 768] times 512 12.7 / 14.7). The largest takes as many weight tiles as cost
// least: a SIMD's two waves have a quarter of them. Up to 32 vectors leave it no
// choice, and up to 16 the smallest tile is ahead: [154880 x 2048] times 16 {1,2,4,1}
// 50, {1,2,4,2} 54, {2,2,8,1} 67; times 32 84, 91, 72.
Shape shape_of(uint32_t tiles, uint32_t units, uint32_t batch, uint32_t cus) {
    const uint64_t results = (uint64_t)tiles * ((batch + 15) / 16);
    if (results <= cus && units >= 32) return Shape{1, 1, 1, 8, 1};
    if (results <= 2ull * cus) return Shape{1, 1, 2, 4, 2};
    if (results <= 4ull * cus) return Shape{1, 1, 4, 4, 4};
    if (results <= 8ull * cus && units >= 16) return Shape{1, 2, 4, 4, 8};
    if (results <= 16ull * cus) return results > 8ull * cus && batch > 16 ? Shape{2, 1, 8, 2, 8} : Shape{1, 2, 4, 2, 8};
    if (batch <= 16) return Shape{1, 2, 4, 1, 8};
    const auto rounds = [&](uint32_t t, uint32_t vecs) {
        return ((uint64_t)((tiles + t - 1) / t) * ((batch + vecs - 1) / vecs) + cus - 1) / cus;
    };
    // (In a second round a CU has room for two workgroups: [10240 x 2048] times 512 61.8
    // us, with one 72.8; times 128, one round, 26.8 and 25.4.)
    Shape best{2, 2, 8, 1, 16, rounds(16, 32) > 1 ? 4 : 2};
    uint64_t least = 30 + 110 * rounds(16, 32);
    for (uint32_t t = 16; t >= 8 && batch > 32; --t) {
        const uint64_t cost = rounds(t, 64) * (70 + 42 * ((t + 3) / 4));
        if (cost < least) {
            least = cost;
            best = Shape{4, 2, 8, 1, t};
        }
    }
    return best;
}

}  // namespace

// Vectors of one launch: fewer than 2^32 threads.
uint64_t gemm_q4_most(const TileGeom& g) {
    const uint64_t items = ((1ull << 21) - 1) / (g.tiles + 8);
    return items ? items * 16 : 16;
}

hipError_t launch_gemm_q4(const uint4* recs, const uint16_t* dvals, const TileGeom& g, uint64_t mat, const float* x,
                          uint64_t x_stride, uint32_t batch, float* y, uint64_t y_slot, uint64_t y_row, int num_cu,
                          hipStream_t s) {
    if (batch == 0) return hipSuccess;
    if (x_stride >= kQ4MostCols || batch > gemm_q4_most(g)) return hipErrorInvalidValue;
    GemmQ4Args a{};
    a.recs = recs + mat * g.rec_stride;
    a.dvals = dvals + mat * g.d_stride;
    a.rec_bytes = (uint32_t)(g.rec_stride * 16);
    a.d_bytes = (uint32_t)(g.d_stride * 2);
    a.x = x;
    a.y = y;
    a.x_stride = x_stride;
    a.y_slot = y_slot;
    a.y_row = y_row;
    a.batch = batch;
    a.cols = (uint32_t)g.cols;
    a.tiles = (uint32_t)g.tiles;
    a.units = (uint32_t)g.units;
    a.rows = (uint32_t)g.rows;
    a.d_row = (uint32_t)g.d_row;
    const Shape t = shape_of(a.tiles, a.units, batch, num_cu > 0 ? num_cu : 256);
    a.wg_tiles = t.tiles;
    a.groups = (a.tiles + t.tiles - 1) / t.tiles;
    a.items = (batch + t.mt * 16 - 1) / (t.mt * 16);
    const void* fn = g.fmt == kFmtQ4 ? fn_of<kFmtQ4>(t) : fn_of<kFmtIq4>(t);
    void* args[] = {&a};
    return hipLaunchKernel(fn, dim3((a.groups + 7) / 8 * 8 * a.items), dim3(t.rs * t.ks * 64), args, 0, s);
}

}  // namespace mmhip
