// 4-bit weights (q4_ops.hpp) times many f32 vectors on gfx950's bf16 matrix
// cores: prompts.
//
// The integer weights are exact in bf16 and an f32 value is the sum of three
// bf16 numbers, so a 32-column block of 16 weight rows times 16 vectors is
// three v_mfma_f32_16x16x32_bf16 (the smallest parts first) and one multiply-add
// per output with the block's scale: the sums of f32 products, no coarser.
#include "device_common.hpp"
#include "gemm_tile_ops.hpp"
#include "kernels.hpp"
#include "q4_ops.hpp"

namespace mmhip {

namespace {

struct GemmQ4Args {
    const uint4* recs;
    const uint16_t* dvals;
    const float* x;
    float* y;
    uint64_t x_stride, y_slot, y_row;  // y[slot * y_slot + row * y_row]
    uint32_t batch, cols, tiles, units, rows, d_row;
    uint32_t rec_bytes, d_bytes;
    uint32_t groups, items;  // tile groups, groups of vectors
};

// Four f32 values as three times four bf16: what each rounding leaves goes into
// the next part, 24 bits of significand together. Times 2^-12 (kActScale), so
// that a block's products stay finite for every finite x.
__device__ __forceinline__ void split3(const uint4& q, uint2 (&part)[3]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    uint32_t out[3][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f32x2 v = {__uint_as_float(w[2 * i]) * kActScale, __uint_as_float(w[2 * i + 1]) * kActScale};
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const uint32_t h = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
            out[p][i] = h;
            v = f32x2{v[0] - __uint_as_float(h << 16), v[1] - __uint_as_float(h & 0xFFFF0000u)};
        }
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) part[p] = make_uint2(out[p][0], out[p][1]);
}

template <int FMT>
__device__ __forceinline__ bf16x8 q4_bop_bf16(uint32_t d) {
    uint32_t w0, w1;
    q4_words<FMT>(d, w0, w1);
    return q8_bop(w0, w1);
}

// Waves of a workgroup split the columns: wave v takes the v-th share of the
// units and the shares are added at the end. MT: 16 vectors each, NJ: 16 weight
// rows each.
template <int FMT, int MT, int NJ, int KS>
__global__ __launch_bounds__(KS * 64, 2) void gemm_q4_kernel(GemmQ4Args a) {
    constexpr uint32_t kSlot = MT * NJ * 4 * 64;                  // floats of a wave's sums
    constexpr uint32_t kX = MT * 3 * kPlaneBytes;                 // a wave's 64 columns of x
    constexpr uint32_t kRed = KS * kSlot * 4, kMain = KS * kX;
    __shared__ __align__(16) uint8_t lds[kRed > kMain ? kRed : kMain];
    const uint32_t item = blockIdx.x % a.items, tg = blockIdx.x / a.items;
    const uint32_t first = item * (MT * 16), count = min(a.batch - first, MT * 16u);
    const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const BufRsrc rec_r = make_rsrc(a.recs, a.rec_bytes), d_r = make_rsrc(a.dvals, a.d_bytes);
    const BufRsrc x_r = make_rsrc(a.x + first * a.x_stride, (uint32_t)(((count - 1) * a.x_stride + a.cols) * 4));
    uint8_t* const xs = lds + wave * kX;

    f32x4 acc[MT][NJ];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[m][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    const uint32_t u0 = a.units * wave / KS, u1 = a.units * (wave + 1) / KS;
    uint4 xv[2][MT * 4], wv[NJ];
    uint32_t dv[NJ];
    const auto load_x = [&](uint32_t u, int h) {
        const uint32_t col = u * kQ4UnitCols + 64 * h + 4 * n;
#pragma unroll
        for (int i = 0; i < MT * 4; ++i) {
            const uint32_t r = 4 * i + g;
            xv[h][i] = buf_load_b128(x_r, u < u1 && r < count && col < a.cols ? (uint32_t)(r * a.x_stride + col) * 4 : kBufOob, 0);
        }
    };
    const auto load_w = [&](uint32_t u) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const uint32_t t = tg * NJ + j;
            const bool ok = u < u1 && t < a.tiles;
            wv[j] = buf_load_b128(rec_r, lane * 16, ok ? (t * a.units + u) * 1024 : kBufOob);
            dv[j] = buf_load_b16(d_r, lane * 8, ok ? t * a.d_row * 32 + (u >> 2) * kQ4StepScaleBytes + (u & 3) * 2 : kBufOob);
        }
    };
    load_w(u0);
    load_x(u0, 0);
    load_x(u0, 1);
    for (uint32_t u = u0; u < u1; ++u) {
        uint4 w[NJ];
        float c[NJ][4];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            w[j] = wv[j];
            broadcast_rows4(f16_scale((uint16_t)dv[j]) * (q4_unscale<FMT>() * kActUnscale), c[j]);
        }
        load_w(u + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            {
                uint8_t* dst = xs + (n >> 1) * kRunBytes + g * 16 + (n & 1) * 8;
#pragma unroll
                for (int i = 0; i < MT * 4; ++i) {
                    uint2 part[3];
                    split3(xv[h][i], part);
#pragma unroll
                    for (int p = 0; p < 3; ++p)
                        *reinterpret_cast<uint2*>(dst + (i >> 2) * (3 * kPlaneBytes) + p * kPlaneBytes + (i & 3) * 64) = part[p];
                }
            }
            load_x(u + 1, h);
            wave_lds_order();
            const uint8_t* src = xs + g * kRunBytes + n * 16;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                bf16x8 part[MT][3];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int p = 0; p < 3; ++p)
                        part[m][p] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(
                            src + (m * 3 + p) * kPlaneBytes + b * 4 * kRunBytes));
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const uint32_t d = h == 0 ? (b == 0 ? w[j].x : w[j].y) : (b == 0 ? w[j].z : w[j].w);
                    const bf16x8 wb = q4_bop_bf16<FMT>(d);
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
                        p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(part[m][2], wb, p, 0, 0, 0);
                        p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(part[m][1], wb, p, 0, 0, 0);
                        p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(part[m][0], wb, p, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[m][j][e] = fmaf(p[e], c[j][2 * h + b], acc[m][j][e]);
                    }
                }
            }
            wave_lds_order();
        }
    }

    lds_barrier();  // the sums take the memory over
    float* const red = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) red[wave * kSlot + ((m * NJ + j) * 4 + r) * 64 + lane] = acc[m][j][r];
    lds_barrier();
    for (uint32_t e = wave; e < MT * NJ; e += KS) {
        const uint32_t m = e / NJ, j = e % NJ, row = (tg * NJ + j) * 16 + n;
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; ++k) v += red[k * kSlot + (e * 4 + r) * 64 + lane];
            const uint32_t t = m * 16 + 4 * g + r;
            if (t < count && row < a.rows) a.y[(uint64_t)(first + t) * a.y_slot + (uint64_t)row * a.y_row] = v;
        }
    }
}

}  // namespace

// Vectors of one launch: x is read through 32-bit offsets from a group's first
// row, and a launch has fewer than 2^32 threads.
uint64_t gemm_q4_most(const TileGeom& g) {
    const uint64_t groups = (g.tiles + 3) / 4;
    const uint64_t items = ((1ull << 23) - 1) / groups;
    return items ? items * 16 : 16;
}

hipError_t launch_gemm_q4(const uint4* recs, const uint16_t* dvals, const TileGeom& g, uint64_t mat, const float* x,
                          uint64_t x_stride, uint32_t batch, float* y, uint64_t y_slot, uint64_t y_row, int num_cu,
                          hipStream_t s) {
    (void)num_cu;
    if (batch == 0) return hipSuccess;
    if (x_stride >= 1ull << 25 || batch > gemm_q4_most(g)) return hipErrorInvalidValue;
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
    a.groups = (a.tiles + 3) / 4;
    a.items = (batch + 15) / 16;
    const unsigned blocks = a.groups * a.items;
    if (g.fmt == kFmtQ4) gemm_q4_kernel<kFmtQ4, 1, 4, 8><<<blocks, 512, 0, s>>>(a);
    else gemm_q4_kernel<kFmtIq4, 1, 4, 8><<<blocks, 512, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace mmhip
