// 4-bit weights in groups of 32 with an f16 scale (Q4_0: code - 8 times the
// scale; IQ4_NL: an entry of a table of 16 int8 values times the scale) in the
// tile layout of the other formats:
//
//   unit (four 32-column blocks of 16 rows, 1152 B = 64 x 18 B)
//     recs: lane l = 16 g + n holds 4 dwords, dword b the codes of columns
//           8 g .. 8 g + 7 of block b, row n: byte i has column i in its lower
//           four bits and column 4 + i in its upper four. Q4_0 codes are stored
//           with their top bit flipped, so that a nibble is code - 8 as a signed
//           number.
//     d:    per four units (a step) 64 lanes x 4 f16: lane l holds the scale of
//           block g, row n of each of the four units, so that a step's scales
//           are one 8-byte load per lane. Absent units have zeros.
#pragma once

#include "device_common.hpp"
#include "kernels.hpp"

namespace mmhip {

constexpr uint32_t kQ4UnitCols = 128;

// What a weight's int8 form (q4_words) is times its value: a nibble that is
// moved to the upper half of its byte is a signed byte of 16 times the value.
template <int FMT>
constexpr float q4_unscale() { return FMT == kFmtQ4 ? 0.0625f : 1.0f; }

// The eight weights of a record dword as int8: columns 0..3 and 4..7.
//
// IQ4_NL looks four codes up at a time with v_perm_b32, which picks bytes out
// of eight: both halves of the table by the lower three bits, then the half by
// the fourth (selector 8 gives the sign of a constant's byte 1, 0xFF, selector 0
// its byte 0, 0x00). 13 operations a dword; Q4_0 takes 3.
template <int FMT>
__device__ __forceinline__ void q4_words(uint32_t d, uint32_t& w0, uint32_t& w1) {
    if constexpr (FMT == kFmtQ4) {
        w0 = (d << 4) & 0xF0F0F0F0u;
        w1 = d & 0xF0F0F0F0u;
    } else {
        const auto look = [](uint32_t c) {
            const uint32_t low = __builtin_amdgcn_perm(0xF6EADDCFu, 0xBFAD9881u, c & 0x07070707u);   // -127 .. -10
            const uint32_t high = __builtin_amdgcn_perm(0x71594535u, 0x26190D01u, c & 0x07070707u);  // 1 .. 113
            const uint32_t upper = __builtin_amdgcn_perm(0u, 0x00008000u, c & 0x08080808u);
            return (upper & high) | (~upper & low);
        };
        w0 = look(d);
        w1 = look(d >> 4);
    }
}
template <int FMT>
__device__ __forceinline__ long q4_bop(uint32_t d) {
    uint32_t w0, w1;
    q4_words<FMT>(d, w0, w1);
    return (long)(((uint64_t)w1 << 32) | w0);
}

// The value of one code, before its scale.
template <bool NL>
__device__ __forceinline__ int q4_code(uint32_t c) {
    return NL ? (int)(int8_t)((c & 8u ? 0x7159453526190D01ull : 0xF6EADDCFBFAD9881ull) >> (8 * (c & 7u))) : (int)c - 8;
}

// A row's product with a vector by its definition, in 64 bits, one column after the
// other: for results that the fast forms left infinite or NaN, which an infinity or NaN
// spreads over (digits and parts of one are NaN), or sums beyond f32 on the way.
template <int FMT>
__device__ __forceinline__ float q4_defined(const uint4* recs, const uint16_t* dvals, uint32_t units, uint32_t d_row, uint32_t cols,
                                            uint32_t row, const float* x) {
    const uint32_t n = row & 15;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(recs + (uint64_t)(row >> 4) * units * 64 + n);
    const uint16_t* d = dvals + (uint64_t)(row >> 4) * 16 * d_row + n * 4;
    double sum = 0.0;
#pragma unroll 1
    for (uint32_t c = 0; c < cols; c += 8) {
        const uint32_t u = c >> 7, b = (c >> 5) & 3, g = (c >> 3) & 3;
        const double scale = f16_bits_to_f32(d[(u >> 2) * 256 + b * 64 + (u & 3)]);
        uint32_t codes = w[(uint64_t)u * 256 + g * 64 + b];
        if (FMT == kFmtQ4) codes ^= 0x88888888u;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            sum += scale * q4_code<FMT == kFmtIq4>((codes >> (8 * (i & 3) + 4 * (i >> 2))) & 15u) * (double)x[c + i];
        if (sum != sum) break;
    }
    return (float)sum;
}

// Where a step's scales of a tile begin, in bytes (steps: of a tile).
constexpr uint32_t kQ4StepScaleBytes = 64 * 4 * 2;

}  // namespace mmhip
