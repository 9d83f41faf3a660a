// Sums and maxima over a wave's lanes. Inside rows of 16 lanes by the vector
// unit's lane permutes (a shuffle through LDS takes about 0.05 us), over whole
// waves by two shuffles more. Every lane gets the result, in a fixed order of
// additions; NaN does not enter a maximum.
#pragma once

#include "device_common.hpp"

namespace mmhip {

constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140, kRotate8 = 0x128;
template <int CTRL>
__device__ __forceinline__ float permuted(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ double permuted(double v) {
    const uint64_t b = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)b, CTRL, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(b >> 32), CTRL, 0xF, 0xF, true);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
// Over 8, 16 or all 64 lanes.
template <int LANES>
__device__ __forceinline__ float group_max(float v) {
    v = fmaxf(v, permuted<kXor1>(v));
    v = fmaxf(v, permuted<kXor2>(v));
    v = fmaxf(v, permuted<kHalfMirror>(v));
    if constexpr (LANES >= 16) v = fmaxf(v, permuted<kMirror>(v));
    if constexpr (LANES == 64) {
        v = fmaxf(v, __shfl_xor(v, 16, 64));
        v = fmaxf(v, __shfl_xor(v, 32, 64));
    }
    return v;
}
template <int LANES, class T>
__device__ __forceinline__ T group_sum(T v) {
    v += permuted<kXor1>(v);
    v += permuted<kXor2>(v);
    v += permuted<kHalfMirror>(v);
    if constexpr (LANES >= 16) v += permuted<kMirror>(v);
    if constexpr (LANES == 64) {
        v += __shfl_xor(v, 16, 64);
        v += __shfl_xor(v, 32, 64);
    }
    return v;
}

// The sum over lanes 0 .. this one, of all 64 lanes.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {  // 0 where no lane moves to
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)v, CTRL, ROWS, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(v >> 32), CTRL, ROWS, 0xF, true);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
    v += moved<0x111, 0xF>(v);  // within rows of 16: from 1, 2, 4, 8 lanes below
    v += moved<0x112, 0xF>(v);
    v += moved<0x114, 0xF>(v);
    v += moved<0x118, 0xF>(v);
    v += moved<0x142, 0xA>(v);  // a row's last lane to the row above: rows 1 and 3
    v += moved<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
    return v;
}
// A lane's value, the same for all.
__device__ __forceinline__ uint64_t lane_value(uint64_t v, uint32_t lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, lane);
}

// The maximum over lanes 0 .. this one.
__device__ __forceinline__ uint64_t wave_max_scan(uint64_t v) {
    v = max(v, moved<0x111, 0xF>(v));
    v = max(v, moved<0x112, 0xF>(v));
    v = max(v, moved<0x114, 0xF>(v));
    v = max(v, moved<0x118, 0xF>(v));
    v = max(v, moved<0x142, 0xA>(v));
    v = max(v, moved<0x143, 0xC>(v));
    return v;
}
// Sums and maxima of two numbers at once over a workgroup, one barrier each: the
// memory of one is written again two calls later, when the next one's barrier has
// shown that all have read it.
template <uint32_t WAVES>
struct Together {
    uint64_t (*memory)[2][WAVES];  // [2]
    uint32_t turn = 0;
    __device__ __forceinline__ void exchange(uint64_t& a, uint64_t& b) {  // lane 63's, to lanes 0 .. WAVES - 1
        uint64_t(&red)[2][WAVES] = memory[turn & 1];
        turn += 1;
        const uint32_t lane = threadIdx.x & 63;
        if (lane == 63) red[0][threadIdx.x >> 6] = a, red[1][threadIdx.x >> 6] = b;
        __syncthreads();
        a = lane < WAVES ? red[0][lane] : 0;
        b = lane < WAVES ? red[1][lane] : 0;
    }
    // a: over threads 0 .. this one, and of all; b: of all.
    __device__ __forceinline__ uint64_t scan(uint64_t a, uint64_t& all, uint64_t& b) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint64_t mine = wave_scan(a);
        a = mine;
        b = wave_scan(b);
        exchange(a, b);
        a = wave_scan(a);
        b = lane_value(wave_scan(b), 63);
        all = lane_value(a, 63);
        return mine + (wave ? lane_value(a, wave - 1) : 0);
    }
    // Both over threads 0 .. this one.
    __device__ __forceinline__ void scan2(uint64_t& a, uint64_t& b, uint64_t& all_a, uint64_t& all_b) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint64_t mine_a = wave_scan(a), mine_b = wave_scan(b);
        a = mine_a;
        b = mine_b;
        exchange(a, b);
        a = wave_scan(a);
        b = wave_scan(b);
        all_a = lane_value(a, 63);
        all_b = lane_value(b, 63);
        a = mine_a + (wave ? lane_value(a, wave - 1) : 0);
        b = mine_b + (wave ? lane_value(b, wave - 1) : 0);
    }
    __device__ __forceinline__ uint64_t sum(uint64_t a) {
        uint64_t all, none = 0;
        scan(a, all, none);
        return all;
    }
    __device__ __forceinline__ void largest(uint64_t& a, uint64_t& b) {
        a = wave_max_scan(a);
        b = wave_max_scan(b);
        exchange(a, b);
        a = lane_value(wave_max_scan(a), 63);
        b = lane_value(wave_max_scan(b), 63);
    }
};

}  // namespace mmhip
