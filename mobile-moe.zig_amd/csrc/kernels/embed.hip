// Rows of an embedding table (embedToken, inference.zig:388-404) on gfx950:
// y[t] = scale * row tokens[t], the table in the raw blocks of its file.
//
// Bound: HBM (a row's blocks in, 4 bytes per value out); one token: the launch
// and two dependent reads. A lane makes two times four consecutive values, both
// read before the first is written, and the output passes the caches by: 4096
// rows of 2048 values in 4 bits take 8.0 us (37.6 MB; only writing their 33.5 MB
// takes 6.4 to 7), with ordinary stores 10.1; with one or four times four values 9.2
// and 8.3. One row: 3.8 us, of which a launch that does nothing is 3.4.
#include "device_common.hpp"
#include "kernels.hpp"
#include "q4_ops.hpp"

namespace mmhip {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kEmbedThreads = 256;
constexpr uint32_t kEmbedEach = 2;

__device__ __forceinline__ uint32_t half_at(const uint8_t* p) { return *reinterpret_cast<const uint16_t*>(p); }
__device__ __forceinline__ uint32_t word_at(const uint8_t* p) {  // at any even address
    uint32_t v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, 2), 4);
    return v;
}

enum EmbedType { kEmbF32, kEmbF16, kEmbQ8, kEmbIq2, kEmbQ4, kEmbIq4 };

// Values 4 q .. 4 q + 3 of a row (n of them there).
template <int T>
__device__ __forceinline__ void quad(const uint8_t* row, uint32_t q, uint32_t n, float (&v)[4]) {
    if constexpr (T == kEmbF32 || T == kEmbF16) {
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            v[e] = 0.0f;
            if (e < n) v[e] = T == kEmbF32 ? reinterpret_cast<const float*>(row)[4 * q + e]
                                           : f16_bits_to_f32(reinterpret_cast<const uint16_t*>(row)[4 * q + e]);
        }
    } else if constexpr (T == kEmbQ8) {
        const uint8_t* b = row + (q >> 3) * 34;
        const float d = f16_bits_to_f32(half_at(b));
        const uint32_t c = word_at(b + 2 + 4 * (q & 7));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = d * (float)(int8_t)(c >> (8 * e));
    } else if constexpr (T == kEmbIq2) {
        const uint8_t* b = row + (q >> 6) * 66;
        const float d = f16_bits_to_f32(half_at(b));
        const uint8_t* s = b + 2 + 8 * ((q >> 3) & 7);
        const uint32_t l = (q >> 1) & 3, half = q & 1, word = word_at(s + 4);
        const uint32_t code = (word >> (7 * l)) & 0x7Fu, sign = code | ((uint32_t)(__popc(code) & 1) << 7);
        const uint32_t mag = (uint32_t)(c_iq2_grid[s[l]] >> (32 * half));
        const float db = d * (0.5f + (float)(word >> 28)) * 0.25f;
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            const float m = (float)((mag >> (8 * e)) & 0xFFu);
            v[e] = db * ((sign >> (4 * half + e)) & 1u ? -m : m);
        }
    } else {
        const uint8_t* b = row + (q >> 3) * 18;
        const float d = f16_bits_to_f32(half_at(b));
        const uint32_t c = word_at(b + 2 + 4 * (q & 3)) >> ((q & 4) ? 4 : 0);  // columns 16 .. 31: the upper four bits
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = d * (float)q4_code<T == kEmbIq4>((c >> (8 * e)) & 15u);
    }
}

// A wave takes 64 kEmbedEach quads of a row, a lane every 64th.
template <int T>
__global__ __launch_bounds__(kEmbedThreads) void embed_kernel(EmbedArgs a, uint64_t n_tokens, uint32_t parts) {
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t unit = (uint64_t)blockIdx.x * (kEmbedThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t t = unit / parts;
    if (t >= n_tokens) return;
    const uint32_t part = (uint32_t)(unit - t * parts);
    const uint32_t token = a.tokens[t];
    if (token == kNoToken) return;
    const bool bad = token >= a.rows;
    if (bad && part == 0 && lane == 0) report(a.status, kBadEmbedToken);
    const uint8_t* row = a.table + (bad ? 0 : token) * a.row_bytes;
    float* y = a.y + t * a.y_stride;
    float v[kEmbedEach][4];
#pragma unroll
    for (uint32_t i = 0; i < kEmbedEach; ++i) {
        const uint32_t q = (part * kEmbedEach + i) * 64 + lane;
        if (4 * q < a.cols) quad<T>(row, q, min(a.cols - 4 * q, 4u), v[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kEmbedEach; ++i) {
        const uint32_t q = (part * kEmbedEach + i) * 64 + lane;
        if (4 * q >= a.cols) return;
        const uint32_t n = min(a.cols - 4 * q, 4u);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = bad ? __builtin_nanf("") : v[i][e] * a.scale;
        if (a.vec && n == 4) {
            __builtin_nontemporal_store(f32x4{v[i][0], v[i][1], v[i][2], v[i][3]}, reinterpret_cast<f32x4*>(y + 4 * q));
        } else {
            for (uint32_t e = 0; e < n; ++e) y[4 * q + e] = v[i][e];
        }
    }
}

}  // namespace

hipError_t launch_embed(const EmbedArgs& a_in, uint32_t type, uint64_t n_tokens, hipStream_t s) {
    EmbedArgs a = a_in;
    a.vec = (reinterpret_cast<uintptr_t>(a.y) & 15u) == 0 && a.y_stride % 4 == 0;
    constexpr uint32_t kWaves = kEmbedThreads / 64;
    const uint32_t parts = (a.cols + 256 * kEmbedEach - 1) / (256 * kEmbedEach);
    const unsigned grid = (unsigned)((n_tokens * parts + kWaves - 1) / kWaves);
    switch (type) {
        case 0: embed_kernel<kEmbF32><<<grid, kEmbedThreads, 0, s>>>(a, n_tokens, parts); break;
        case 1: embed_kernel<kEmbF16><<<grid, kEmbedThreads, 0, s>>>(a, n_tokens, parts); break;
        case 2: embed_kernel<kEmbQ4><<<grid, kEmbedThreads, 0, s>>>(a, n_tokens, parts); break;
        case 8: embed_kernel<kEmbQ8><<<grid, kEmbedThreads, 0, s>>>(a, n_tokens, parts); break;
        case 16: embed_kernel<kEmbIq2><<<grid, kEmbedThreads, 0, s>>>(a, n_tokens, parts); break;
        case 20: embed_kernel<kEmbIq4><<<grid, kEmbedThreads, 0, s>>>(a, n_tokens, parts); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace mmhip
