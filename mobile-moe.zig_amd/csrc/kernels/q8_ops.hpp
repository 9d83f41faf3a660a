// Q8_0 block quantisation (quantizeQ8_0, dequant.zig:98-130): the scale of a
// block of 32 values and their codes, 8 consecutive lanes per block with four
// values each. Shared by the codec, the norm and the cache writer, so that all
// of them give the same codes for the same values.
#pragma once

#include "device_common.hpp"

namespace mmhip {

// f32ToF16 (dequant.zig:50-95) as the quantiser stores a block scale: round
// to nearest even on the normal range, 0 for f32 subnormals and below 2^-25,
// Inf / NaN kept. On the f16 subnormal range, [2^-25, 2^-14), the reference
// shifts the significand by 1 - e16, which spills out of the 10-bit field: a
// trap in safe builds for [2^-21, 2^-14), a corrupted code for [2^-25, 2^-21)
// (2^-22 -> 0x8000). This takes the branch's evident intent on the whole
// range, a shift by 14 - e16: the subnormal value truncated toward zero.
__device__ __forceinline__ uint32_t f32_to_f16_scale(float v) {
    const uint32_t bits = __float_as_uint(v);
    const uint32_t er = (bits >> 23) & 0xFFu, mant = bits & 0x7FFFFFu;
    uint32_t e = 0, m = 0;
    if (er == 0xFFu) {
        e = 0x1Fu;
        m = mant >> 13;
        if (mant != 0 && m == 0) m = 1;
    } else if (er != 0) {
        const int e16 = (int)er - 112;
        if (e16 >= 31) {
            e = 0x1Fu;
        } else if (e16 <= 0) {
            if (e16 >= -10) m = (mant | 0x800000u) >> (uint32_t)(14 - e16);
        } else {
            e = (uint32_t)e16;
            m = mant >> 13;
            const uint32_t rb = mant & 0x1FFFu;
            if (rb > 0x1000u || (rb == 0x1000u && (m & 1u))) {
                ++m;
                if (m == 0x400u) {
                    m = 0;
                    ++e;
                }
            }
        }
    }
    return ((bits >> 31) << 15) | (e << 10) | m;
}

// The codes (one per byte) of a lane's four values, n_live of them present
// (absent ones, NaN included, count as 0), and the block's scale d before its
// rounding to f16. All 8 lanes of a block call it together.
__device__ __forceinline__ uint32_t q8_quad(const float (&v)[4], uint32_t n_live, float& d) {
    // The block's largest |x| (a NaN never compares greater).
    float m = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float av = fabsf(v[e]);
        m = ((uint32_t)e < n_live && av > m) ? av : m;
    }
    m = max8_lanes(m);
    d = m > 0.0f ? m / 127.0f : 0.0f;
    // x / d rounded half away from zero (@round of the f32 quotient).
    // z = x * rcp(d) is within |x/d| * (2^-23 + 2^-24) <= 2.3e-5 of
    // the exact quotient (rcp: 1 ulp; |x/d| <= 127.00002), and the
    // correctly rounded quotient is within 2^-17 of it; where z is
    // more than 1e-4 from every half-integer both round to the same
    // integer. Lanes with a value closer, with |z| > 127.25 (a
    // subnormal d can push the quotient past 127.5, which the exact
    // path clamps) or with a non-finite z (d = 0, Inf or NaN inputs)
    // redo their block with the IEEE division.
    const float rd = __builtin_amdgcn_rcpf(d);
    uint32_t q4 = 0;
    bool near = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        // y = |z| + 0.5 (rounding error <= 2^-18 for |z| < 128): |z| is
        // near a half-integer where y is near an integer.
        const float z = v[e] * rd, az = fabsf(z), y = az + 0.5f, r = truncf(y);
        near |= !(az <= 127.25f) || !(fabsf((y - r) - 0.5f) < 0.5f - 1.0e-4f);
        // Not near: |z| <= 127.25 and away from half-integers, so the
        // rounded value is in [-127, 127]; absent values are 0.
        q4 |= ((uint32_t)(int)copysignf(r, z) & 0xFFu) << (8 * e);
    }
    if (__any(near) && near) {
        q4 = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float r = roundf(v[e] / d);
            const float re = (r == r && d > 0.0f && (uint32_t)e < n_live) ? r : 0.0f;  // NaN input (@intFromFloat traps)
            const int q = (int)fminf(fmaxf(re, -127.0f), 127.0f);
            q4 |= (uint32_t)(q & 0xFF) << (8 * e);
        }
    }
    return q4;
}

}  // namespace mmhip
