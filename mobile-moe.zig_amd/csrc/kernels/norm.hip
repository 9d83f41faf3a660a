// Root-mean-square norm, rotary positions and the paged cache's writer
// (math.rmsNorm, math.zig:7-35; RoPECache, 197-240; KVCache.put,
// kv_cache.zig:279-362) on gfx950. All three are bound by HBM for many rows and
// by one launch's latency for few.
//
// Norm: a row's sum of squares and the inverse root are in f64 and the root is
// rounded to f32 once; every other operation is one f32 operation per value,
// never contracted. The sum's order depends on the width alone, and the cache
// writer keeps it (both give thread t columns 4t .. 4t + 3, and rows end within
// the first two waves), so it stores the bits that norm and codec would give one
// after the other. The f64 sum costs a conversion and an FMA
// per value, hidden behind the row's loads. 4099 rows of 2048 with a residual,
// its sum and Q8_0 out: 18.5 us, 5.9 TB/s; one row 1.8 us.
//
// Rotary positions: 4096 tokens of 20 heads of 192 values, 64 of them turned:
// 19.2 us, 6.6 TB/s; one token 2.3 us. The angles' 64-bit arithmetic is a
// wave's work per token and runs while the other values are copied.
//
// Cache writer: 4096 positions to Q8_0 7.2 us a call, 1.7 TB/s: a workgroup's
// chain of slot, row, angles, sum and root is longer than its bytes; 64 positions
// 3 us.
#include "device_common.hpp"
#include "kernels.hpp"
#include "lanes.hpp"
#include "q8_ops.hpp"

namespace mmhip {

namespace {

constexpr int kNormThreads = 256;
enum NormOut : uint32_t { kOutF32 = 0, kOutF16 = 1, kOutQ8 = 2 };

// Four values from p + c, those at or past `cols` absent (0).
__device__ __forceinline__ void load4(float (&v)[4], const float* p, uint32_t c, uint32_t cols, bool vec) {
    if (vec && c + 4 <= cols) {
        const float4 q = *reinterpret_cast<const float4*>(p + c);
        v[0] = q.x;
        v[1] = q.y;
        v[2] = q.z;
        v[3] = q.w;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = c + e < cols ? p[c + e] : 0.0f;
    }
}
// Stores past the caches: lines left in L2 are written back at the launch's end
// (norm of 4099 rows 21.9 -> 18.5 us, rotary positions of 4096 tokens 27.1 ->
// 19.2 us, whole calls; loads past them as well: 21.7 and 23.7). A reader right
// behind takes back what it saves: norm to f32 and the product of its rows with
// 1344 Q8_0 columns, ordinary stores against these, 256 rows 15.8 / 16.1 us, 2048
// rows 77.5 / 76.6, 4099 rows 142.9 / 143.3; rotation and a norm of the whole
// rows, 4096 tokens, 48.1 / 48.9. A wave's stores fill whole lines.
__device__ __forceinline__ void stream4(float* p, float a, float b, float c, float d) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store((f4){a, b, c, d}, reinterpret_cast<f4*>(p));
}
template <bool STREAM>
__device__ __forceinline__ void store4(float* p, const float (&v)[4], uint32_t c, uint32_t cols, bool vec) {
    if (vec && c + 4 <= cols) {
        if constexpr (STREAM) stream4(p + c, v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<float4*>(p + c) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < cols) p[c + e] = v[e];
    }
}

__device__ __forceinline__ uint32_t half_bits(float v) { return __half_as_ushort(__float2half_rn(v)); }

// 1 / sqrt(mean + eps) to a few units of the 53rd bit, rounded to f32. (A
// division and a square root instead took every wave about 0.3 us.)
__device__ __forceinline__ float inverse_root(double sum, double inv_cols, float eps) {
    return (float)rsqrt(fma(sum, inv_cols, (double)eps));
}

// Values c .. c + 3 of a row's output.
template <uint32_t OUT>
__device__ __forceinline__ void store_normed(const NormArgs& a, uint64_t row, uint32_t c, const float (&v)[4]) {
    if constexpr (OUT == kOutF32) {
        store4<true>(static_cast<float*>(a.y) + row * a.y_stride, v, c, a.cols, a.vec);
    } else if constexpr (OUT == kOutF16) {
        uint16_t* y = static_cast<uint16_t*>(a.y) + row * a.y_stride + c;
        if (c + 4 <= a.cols) {
            const uint2 q = make_uint2(half_bits(v[0]) | half_bits(v[1]) << 16, half_bits(v[2]) | half_bits(v[3]) << 16);
            __builtin_memcpy(y, &q, 8);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (c + e < a.cols) y[e] = (uint16_t)half_bits(v[e]);
        }
    } else {
        // A block's 8 lanes are together.
        float d;
        const uint32_t q4 = q8_quad(v, c < a.cols ? min(a.cols - c, 4u) : 0u, d);
        const uint32_t blocks = (a.cols + 31) / 32, j = (c / 4) & 7;
        if (c / 32 < blocks) {
            uint16_t* y = static_cast<uint16_t*>(a.y) + (row * blocks + c / 32) * 17;
            __builtin_memcpy(y + 1 + 2 * j, &q4, 4);  // 2-byte aligned
            if (j == 0) y[0] = (uint16_t)f32_to_f16_scale(d);
        }
    }
}

// The workgroup's sum.
__device__ __forceinline__ double block_sum(double acc, double* part) {
    acc = group_sum<64>(acc);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
    __syncthreads();
    acc = 0.0;
#pragma unroll
    for (int i = 0; i < kNormThreads / 64; ++i) acc += part[i];
    return acc;
}

// One workgroup per row, which stays in registers: thread t has columns
// 4 (t + 256 i) .. + 3, i < NV, and reads all of them, the residual and the
// weight before it uses any.
template <uint32_t OUT, int NV>
__global__ __launch_bounds__(kNormThreads) void rms_norm_kernel(NormArgs a) {
    __shared__ double part[kNormThreads / 64];
    const uint64_t row = blockIdx.x;
    // Columns past the row's end, and a residual that is not there, read 0.
    const BufRsrc x = make_rsrc(a.x + row * a.x_stride, a.cols * 4);
    const BufRsrc res = make_rsrc(a.residual + row * a.residual_stride, a.residual ? a.cols * 4 : 0);
    const BufRsrc weight = make_rsrc(a.weight, a.cols * 4);
    float v[NV][4], r[NV][4], w[NV][4];
    const auto read = [&](float (&to)[NV][4], BufRsrc from) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (a.vec) {
                const uint4 q = buf_load_b128(from, threadIdx.x * 16, i * (kNormThreads * 16));
                to[i][0] = __uint_as_float(q.x);
                to[i][1] = __uint_as_float(q.y);
                to[i][2] = __uint_as_float(q.z);
                to[i][3] = __uint_as_float(q.w);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    to[i][e] = __uint_as_float(buf_load_b32(from, threadIdx.x * 16 + 4 * e + i * (kNormThreads * 16), 0));
            }
        }
    };
    read(v, x);
    read(r, res);
    read(w, weight);
    double acc = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (a.residual) v[i][e] = __fadd_rn(v[i][e], r[i][e]);
            acc = fma((double)v[i][e], (double)v[i][e], acc);
        }
        if (a.sum) store4<true>(a.sum + row * a.sum_stride, v[i], (threadIdx.x + i * kNormThreads) * 4, a.cols, a.vec);
    }
    const float root = inverse_root(block_sum(acc, part), a.inv_cols, a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][e] = __fmul_rn(__fmul_rn(v[i][e], root), w[i][e]);
        store_normed<OUT>(a, row, (threadIdx.x + i * kNormThreads) * 4, v[i]);
    }
}

// Longer rows are read twice.
template <uint32_t OUT>
__global__ __launch_bounds__(kNormThreads) void rms_norm_long_kernel(NormArgs a) {
    __shared__ double part[kNormThreads / 64];
    const uint64_t row = blockIdx.x;
    const float* x = a.x + row * a.x_stride;
    const float* res = a.residual ? a.residual + row * a.residual_stride : nullptr;
    float* sum = a.sum ? a.sum + row * a.sum_stride : nullptr;
    double acc = 0.0;
    for (uint32_t c = threadIdx.x * 4; c < a.cols; c += kNormThreads * 4) {
        float v[4], w[4];
        load4(v, x, c, a.cols, a.vec);
        if (res) {
            load4(w, res, c, a.cols, a.vec);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __fadd_rn(v[e], w[e]);
        }
        if (sum) store4<false>(sum, v, c, a.cols, a.vec);  // read again below
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = fma((double)v[e], (double)v[e], acc);
    }
    const float root = inverse_root(block_sum(acc, part), a.inv_cols, a.eps);
    // Every thread takes every step, so that a Q8_0 block's 8 lanes are together.
    const uint32_t steps = (a.cols + kNormThreads * 4 - 1) / (kNormThreads * 4);
    for (uint32_t i = 0; i < steps; ++i) {
        const uint32_t c = (threadIdx.x + i * kNormThreads) * 4;
        float v[4], w[4];
        // A sum that replaced its input is read back, by the thread that wrote it.
        load4(v, sum ? sum : x, c, a.cols, a.vec);
        if (res && !sum) {
            load4(w, res, c, a.cols, a.vec);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __fadd_rn(v[e], w[e]);
        }
        load4(w, a.weight, c, a.cols, a.vec);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __fmul_rn(__fmul_rn(v[e], root), w[e]);
        store_normed<OUT>(a, row, c, v);
    }
}

// The fewest registers that hold a row. With residual, sum and Q8_0 out, by
// this rule / re-reading every row: 8192 x 512 17.9 / 21.7 us, 8192 x 1024
// 22.0 / 26.4, 4096 x 2048 23.0 / 27.9, 2048 x 4096 25.4 / 32.5; one run more
// than a row has costs up to half as much again (8192 x 512 with two: 25.7).
template <uint32_t OUT>
void launch_norm(const NormArgs& a, unsigned grid, hipStream_t s) {
    if (a.cols <= 1024) rms_norm_kernel<OUT, 1><<<grid, kNormThreads, 0, s>>>(a);
    else if (a.cols <= 2048) rms_norm_kernel<OUT, 2><<<grid, kNormThreads, 0, s>>>(a);
    else if (a.cols <= 4096) rms_norm_kernel<OUT, 4><<<grid, kNormThreads, 0, s>>>(a);
    else rms_norm_long_kernel<OUT><<<grid, kNormThreads, 0, s>>>(a);
}

// Cosine and sine of position * frequency, times the magnitude, from the
// angle in turns: its whole turns are dropped in f64, so far positions keep
// their angle.
__device__ __forceinline__ float2 turn(double turns_per_position, double magnitude, uint32_t position) {
    double t = (double)position * turns_per_position;
    t -= rint(t);
    double s, c;
    sincospi(2.0 * t, &s, &c);
    return make_float2((float)(c * magnitude), (float)(s * magnitude));
}

// One rotated value: dim `i` of the rotated dims, `v` its value, `o` its
// partner's. The products and the sum are rounded one by one.
__device__ __forceinline__ float rotate(float v, float o, float2 cs, bool second) {
#pragma clang fp contract(off)
    return second ? o * cs.y + v * cs.x : v * cs.x - o * cs.y;
}

constexpr int kRopeThreads = 256;

// A thread's n-th unit of a token's heads x per_head units, 256 apart, by steps
// without a division.
struct RopeUnit {
    uint32_t h, j;
    uint32_t step_h, step_j, per_head;
    __device__ RopeUnit(uint32_t first, uint32_t per)
        : h(first / per), j(first % per), step_h(kRopeThreads / per), step_j(kRopeThreads % per), per_head(per) {}
    __device__ void next() {
        h += step_h;
        j += step_j;
        if (j >= per_head) {
            j -= per_head;
            ++h;
        }
    }
};

// One workgroup per token. A thread's units are W pairs (both values of each),
// read before the token's cosines are known; the other dims are copied W at a
// time in the meantime. W = 4: 16-byte accesses.
template <int W>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
    __shared__ float2 cs[kRopeMaxPairs];
    const uint64_t t = blockIdx.x;
    const uint32_t pairs = a.dims / 2;
    const float* x = a.x + t * a.x_token_stride;
    float* y = a.y + t * a.y_token_stride;
    // Where pair j's values are in a head. Of W = 4 pairs: two runs of 4.
    const auto place = [&](uint32_t j, uint32_t& ia, uint32_t& ib) {
        ia = a.first + (a.half ? j : 2 * j);
        ib = a.half ? ia + pairs : ia + W;
    };
    const auto read = [&](float (&v)[W], const float* p) {
        if constexpr (W == 4) {
            const float4 q = *reinterpret_cast<const float4*>(p);
            v[0] = q.x;
            v[1] = q.y;
            v[2] = q.z;
            v[3] = q.w;
        } else {
            v[0] = *p;
        }
    };
    const auto write = [&](float* p, const float (&v)[W]) {
        if constexpr (W == 4) stream4(p, v[0], v[1], v[2], v[3]);
        else *p = v[0];
    };
    RopeUnit u(threadIdx.x, pairs / W);
    float va[W], vb[W];
    uint32_t ia, ib;
    place(u.j * W, ia, ib);
    if (u.h < a.n_heads) {
        read(va, x + u.h * a.x_head_stride + ia);
        read(vb, x + u.h * a.x_head_stride + ib);
    }
    if (threadIdx.x < pairs) cs[threadIdx.x] = turn(a.turns[threadIdx.x], a.magnitude, a.positions[t]);
    const uint32_t rest = a.copy ? (a.head_dim - a.dims) / W : 0;
    if (rest) {
        for (RopeUnit c(threadIdx.x, rest); c.h < a.n_heads; c.next()) {
            const uint32_t k = c.j * W, i = k < a.first ? k : k + a.dims;
            float v[W];
            read(v, x + c.h * a.x_head_stride + i);
            write(y + c.h * a.y_head_stride + i, v);
        }
    }
    __syncthreads();
    while (u.h < a.n_heads) {
        const float2* p = cs + u.j * W;
        float* to = y + u.h * a.y_head_stride;
        float ra[W], rb[W];
        if (W == 1 || a.half) {
#pragma unroll
            for (int e = 0; e < W; ++e) {
                ra[e] = rotate(va[e], vb[e], p[e], false);
                rb[e] = rotate(vb[e], va[e], p[e], true);
            }
        } else {
#pragma unroll
            for (int e = 0; e + 1 < W; e += 2) {
                ra[e] = rotate(va[e], va[e + 1], p[e / 2], false);
                ra[e + 1] = rotate(va[e + 1], va[e], p[e / 2], true);
                rb[e] = rotate(vb[e], vb[e + 1], p[(W + e) / 2], false);
                rb[e + 1] = rotate(vb[e + 1], vb[e], p[(W + e) / 2], true);
            }
        }
        write(to + ia, ra);
        write(to + ib, rb);
        u.next();
        if (u.h >= a.n_heads) break;
        place(u.j * W, ia, ib);
        read(va, x + u.h * a.x_head_stride + ia);
        read(vb, x + u.h * a.x_head_stride + ib);
    }
}

// One workgroup per position: thread t has values 4t.. of the row.
constexpr int kStoreThreads = 192;
static_assert(kStoreThreads * 4 >= kKvMaxRank + kKvMaxRope, "a row fits one pass");
__global__ __launch_bounds__(kStoreThreads) void kv_store_kernel(StoreArgs a) {
    __shared__ double part[kStoreThreads / 64];
    __shared__ float2 cs[kKvMaxRope / 2];
    const uint64_t t = blockIdx.x;
    const PagedGeom g = a.geom;
    const float* x = a.kv + t * a.kv_stride;
    const uint32_t c = threadIdx.x * 4, pe = g.width - g.rank;
    const bool live = c < g.width, latent = c < g.rank;
    // The row, its weight, its slot and its position are read at once.
    float v[4], w[4];
    load4(v, x, live ? c : 0, live ? g.width : 0, a.vec);
    if (a.weight) load4(w, a.weight, latent ? c : 0, latent ? g.rank : 0, a.vec);
    const int32_t slot = a.slots[t];
    const uint32_t position = a.turns ? a.positions[t] : 0;
    uint32_t page, at;
    if (!paged_slot(g, slot, page, at)) {
        if (slot >= 0 && threadIdx.x == 0) report(a.status, kBadSlot);
        return;
    }
    if (a.turns && threadIdx.x < pe / 2) cs[threadIdx.x] = turn(a.turns[threadIdx.x], a.magnitude, position);
    double acc = 0.0;
    if (latent && a.weight) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc = fma((double)v[e], (double)v[e], acc);
    }
    acc = group_sum<64>(acc);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (latent && a.weight) {
        acc = 0.0;
#pragma unroll
        for (int i = 0; i < kStoreThreads / 64; ++i) acc += part[i];
        const float r = inverse_root(acc, a.inv_rank, a.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __fmul_rn(__fmul_rn(v[e], r), w[e]);
    } else if (live && !latent && a.turns) {
        const uint32_t k = c - g.rank, half = pe / 2;
        if (a.half) {
            float o[4];
            const bool second = k >= half;
            load4(o, x, second ? c - half : c + half, g.width, a.vec);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = rotate(v[e], o[e], cs[(second ? k - half : k) + e], second);
        } else {
            const float2 c0 = cs[k / 2], c1 = cs[k / 2 + 1];
            const float u[4] = {rotate(v[0], v[1], c0, false), rotate(v[1], v[0], c0, true),
                                rotate(v[2], v[3], c1, false), rotate(v[3], v[2], c1, true)};
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = u[e];
        }
    }
    if (g.q8) {
        // (A block without values would send its wave through the exact
        // divisions: lanes past the row have ones.)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = live ? v[e] : 1.0f;
        float d;
        const uint32_t q4 = q8_quad(v, 4u, d);
        if (live) {
            *reinterpret_cast<uint32_t*>(a.pool + paged_row(g, page, at) + c) = q4;
            if ((threadIdx.x & 7) == 0)
                *reinterpret_cast<uint16_t*>(a.pool + paged_scales(g, page, at) + c / 32 * 2) = (uint16_t)f32_to_f16_scale(d);
        }
    } else if (live) {
        *reinterpret_cast<uint2*>(a.pool + paged_row(g, page, at) + 2 * c) =
            make_uint2(half_bits(v[0]) | half_bits(v[1]) << 16, half_bits(v[2]) | half_bits(v[3]) << 16);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

hipError_t launch_rms_norm(const NormArgs& in, uint32_t out, uint64_t n_rows, hipStream_t s) {
    if (n_rows == 0) return hipSuccess;
    NormArgs a = in;
    a.inv_cols = 1.0 / a.cols;
    a.vec = a.cols % 4 == 0 && aligned16(a.x) && a.x_stride % 4 == 0 && aligned16(a.weight) &&
            (!a.residual || (aligned16(a.residual) && a.residual_stride % 4 == 0)) &&
            (!a.sum || (aligned16(a.sum) && a.sum_stride % 4 == 0)) &&
            (out != kOutF32 || (aligned16(a.y) && a.y_stride % 4 == 0));
    const unsigned grid = (unsigned)n_rows;
    if (out == kOutF32) launch_norm<kOutF32>(a, grid, s);
    else if (out == kOutF16) launch_norm<kOutF16>(a, grid, s);
    else launch_norm<kOutQ8>(a, grid, s);
    return hipGetLastError();
}

hipError_t launch_rope(const RopeArgs& a, uint64_t n_tokens, hipStream_t s) {
    if (n_tokens == 0 || a.n_heads == 0) return hipSuccess;
    const bool vec = a.dims % 8 == 0 && a.first % 4 == 0 && a.head_dim % 4 == 0 && aligned16(a.x) && aligned16(a.y) &&
                     a.x_token_stride % 4 == 0 && a.x_head_stride % 4 == 0 && a.y_token_stride % 4 == 0 &&
                     a.y_head_stride % 4 == 0;
    // (The kernel alone, 4096 tokens of 20 heads of 192, with ordinary stores:
    // 21.4 us; pair by pair 30.5.)
    if (vec) rope_kernel<4><<<(unsigned)n_tokens, kRopeThreads, 0, s>>>(a);
    else rope_kernel<1><<<(unsigned)n_tokens, kRopeThreads, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv_store(const StoreArgs& in, uint64_t n_tokens, hipStream_t s) {
    if (n_tokens == 0) return hipSuccess;
    StoreArgs a = in;
    a.inv_rank = 1.0 / a.geom.rank;
    a.vec = aligned16(a.kv) && a.kv_stride % 4 == 0 && aligned16(a.weight);
    kv_store_kernel<<<(unsigned)n_tokens, kStoreThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace mmhip
