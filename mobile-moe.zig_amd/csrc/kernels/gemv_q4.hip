// 4-bit weights (q4_ops.hpp) times one to four vectors, or a few fours, on gfx950:
// decode.
//
// y[t][r] = sum_b d[r][b] sum_{i < 32} v[r][32 b + i] x[t][32 b + i]. A vector's
// block of 32 becomes integers of up to 2^30 with the block's own power of two
// (exact down to 2^-6 of the block's largest value, below that off by at most
// 2^-30 of it), cut into four int8 digits. The digits are rows of the A
// operand of v_mfma_i32_16x16x32_i8, which has sixteen: one product per block
// and 16 weight rows gives the exact integer sums of all four digits of up to
// four vectors, so the weights are read and unpacked once for all of them and
// the sums are those of f32 values, not of rounded ones.
//
// Bound: HBM, 0.5625 bytes per weight. A workgroup owns a run of 16-row tiles;
// its waves share the run's steps (four units of 128 columns) evenly, each a
// contiguous part, with the next steps' loads in flight. Tiles that two waves
// share are joined in wave order, so the result does not depend on timing.
// Measured: 64 IQ4_NL matrices of [1536 x 2048], one vector each, 21.0 us (5.4
// TB/s); [154880 x 2048] times four vectors 32.1 us (5.6 TB/s), in IQ4_NL, whose
// lookups take more instructions than Q4_0's unpacking, 38.1 (4.8); times one 29.2 and
// 31.7; [768 x 2048] times one 4.1 us, a launch's time.
#include "device_common.hpp"
#include "gemm_tile_ops.hpp"
#include "kernels.hpp"
#include "q4_ops.hpp"
#include "tile_ops.hpp"

namespace mmhip {

namespace {

constexpr uint32_t kQ4Ups = 4;        // units per step

// Columns whose digits are in LDS at once, in units.
template <int TOK>
constexpr uint32_t q4_chunk() { return TOK == 1 ? 64 : 24; }
// Tiles per workgroup (LDS row sums; all of its LDS stays below 64 KiB).
template <int TOK>
constexpr uint32_t q4_tiles() { return TOK == 1 ? 64 : 40; }
// LDS digits of a unit, by the lane (row m of A, column group g) that reads them.
// One vector: A has the four digits of block b in rows 4 b .. 4 b + 3, so a lane
// reads 8 bytes of the one block it has a row of. Four vectors: rows 4 t .. 4 t + 3
// are vector t's digits, 8 bytes of every block (two halves of two blocks).
template <int TOK>
constexpr uint32_t q4_unit_bytes() { return TOK == 1 ? 64 * 8 : 64 * 32; }

// The four digits of four columns' integers (digit 0 the highest), a word per
// digit, column e in byte e.
__device__ __forceinline__ void digits4(const float (&v)[4], int up, uint32_t (&out)[4]) {
    uint32_t q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = ((uint32_t)(int)rintf(ldexpf(v[e], up)) + 0x00808080u) ^ 0x00808080u;
    const uint32_t a = __builtin_amdgcn_perm(q[1], q[0], 0x05010400u);  // bytes 0 0 1 1 of q0, q1
    const uint32_t b = __builtin_amdgcn_perm(q[3], q[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(q[1], q[0], 0x07030602u);  // bytes 2 2 3 3
    const uint32_t d = __builtin_amdgcn_perm(q[3], q[2], 0x07030602u);
    out[3] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    out[2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    out[1] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    out[0] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// A block's scale, a power of two, and the power that undoes it, from the bits of its
// largest |x|: integers of at most 2^30, and no steps below f32's own, 2^-149. A
// block with an infinity or NaN gets a NaN scale (and its results q4_defined()).
__device__ __forceinline__ float block_scale(uint32_t m_bits, int& up) {
    up = 156 - (int)max(m_bits >> 23, 7u);
    return m_bits >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : ldexpf(1.0f, -up);
}

// A quarter block of a vector, four columns per lane, into the LDS digits.
template <int TOK>
__device__ __forceinline__ void store_digits(const float (&v)[4], uint32_t tok, uint32_t blk, uint32_t jq, uint8_t* aq,
                                             float* xs) {
    uint32_t m = quad_abs_max_bits(v);
    m = umax_dpp<0xB1>(m);
    m = umax_dpp<0x4E>(m);
    m = umax_dpp<0x141>(m);
    int up;
    const float s = block_scale(m, up);
    uint32_t d[4];
    digits4(v, up, d);
    const uint32_t g = jq >> 1, half = jq & 1;
    uint8_t* const unit = aq + (blk >> 2) * q4_unit_bytes<TOK>();
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        uint8_t* at = TOK == 1 ? unit + (g * 16 + (blk & 3) * 4 + e) * 8
                               : unit + ((blk >> 1) & 1) * 1024 + (g * 16 + tok * 4 + e) * 16 + (blk & 1) * 8;
        *reinterpret_cast<uint32_t*>(at + half * 4) = d[e];
    }
    if (jq == 0) xs[TOK == 1 ? blk : (blk >> 2) * 16 + tok * 4 + (blk & 3)] = s;
}

// Four digits' sums as one number: the upper two's and the lower two's (below 2^28)
// are rounded to f32 where they have more than 24 bits, and their sum once more.
// Times the weights' scale first (at most 2^60) and the vector's last: no product of
// scales that could leave f32's normal numbers.
__device__ __forceinline__ float digits_value(int t1, int t2) { return fmaf((float)t1, 65536.0f, (float)t2); }

struct Q4Args {
    GemvArgs a;
    uint32_t n_vec;  // vectors of one problem (TOK 4): x_stride, y_stride are between these
};
template <int N>
struct Q4Set {
    Q4Args seg[N];
};

// TOK 1: grid row y is a problem, a matrix and a vector of its own. TOK 4: grid
// row y is a group of up to four vectors, all with the first matrix.
template <int FMT, int TOK, int WG, int DEPTH, int NSEG>
__global__ __launch_bounds__(WG, WG == 256 ? 2 : 4) void gemv_q4_kernel(Q4Set<NSEG> set) {
    constexpr uint32_t kWaves = WG / 64, kRing = DEPTH + 1;
    constexpr uint32_t kChunk = q4_chunk<TOK>(), kOut = TOK == 1 ? 16 : 64;
    const GemvArgs& a = set.seg[NSEG > 1 ? blockIdx.z : 0].a;
    pin_gemv_args(a);
    const uint32_t n_vec = TOK == 1 ? 1 : min(set.seg[0].n_vec - blockIdx.y * TOK, (uint32_t)TOK);
    const uint32_t t_begin = blockIdx.x * a.tiles_per_wg;
    if (t_begin >= a.tiles || (TOK == 1 && blockIdx.y >= a.n_probs)) return;  // whole workgroup
    __shared__ float row_sum[q4_tiles<TOK>() * kOut];
    __shared__ float edge[2][kWaves * kOut];
    extern __shared__ __align__(16) uint8_t smem[];
    const uint32_t chunk = min(a.units, kChunk);
    uint8_t* const aq = smem;
    float* const xs = reinterpret_cast<float*>(smem + chunk * q4_unit_bytes<TOK>());

    const uint32_t lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t mat = a.first_mat + (TOK == 1 ? blockIdx.y : 0);
    const float* x = a.x + (uint64_t)blockIdx.y * (TOK == 1 ? 1 : TOK) * a.x_stride;
    const uint32_t n_tiles = min(a.tiles - t_begin, a.tiles_per_wg);
    const BufRsrc rec_r = make_rsrc(a.recs + mat * a.rec_stride, (uint32_t)(a.rec_stride * 16));
    const BufRsrc d_r = make_rsrc(a.dvals + mat * a.d_stride, (uint32_t)(a.d_stride * 2));
    const uint32_t rec_voff = lane * 16, d_voff = lane * 8;
    const uint32_t rec_tile = keep_sgpr(a.units * 1024u), d_tile = keep_sgpr(a.d_row * 32u);
    const uint32_t a_lane = lane * (TOK == 1 ? 8 : 16);
    uint32_t mine[4];  // all ones for the block that this lane has a row of
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) mine[b] = TOK != 1 || n >> 2 == b ? 0xFFFFFFFFu : 0u;

    // The chunk's steps [0, L) of the run, S per tile; this wave's [j0, j1).
    uint32_t u_begin = 0, n_units = 0, S = 1, L = 0, j0 = 0, j1 = 0, tf = 0;
    uint32_t cur_t = 0, cur_s = 0, nxt_t = 0, nxt_s = 0;
    uint4 rb[kRing][kQ4Ups];
    uint2 db[kRing];
    const auto load = [&](bool ok, uint32_t t, uint32_t s, uint4 (&r)[kQ4Ups], uint2& d) {
        const uint32_t u = u_begin + s * kQ4Ups;
#pragma unroll
        for (uint32_t i = 0; i < kQ4Ups; ++i)
            r[i] = buf_load_b128<kCacheStream>(rec_r, rec_voff + i * 1024,
                                               ok && u + i < a.units ? (t_begin + t) * rec_tile + u * 1024 : kBufOob);
        d = buf_load_b64<kCacheStream>(d_r, d_voff, ok ? (t_begin + t) * d_tile + (u >> 2) * kQ4StepScaleBytes : kBufOob);
    };
    const auto start = [&](uint32_t units) {
        n_units = units;
        S = (units + kQ4Ups - 1) / kQ4Ups;
        L = n_tiles * S;
        j0 = wave * L / kWaves;
        j1 = (wave + 1) * L / kWaves;
        tf = j0 / S;
        cur_t = nxt_t = tf;
        cur_s = nxt_s = j0 - tf * S;
#pragma unroll
        for (uint32_t q = 0; q < DEPTH; ++q) {
            load(j0 + q < j1, nxt_t, nxt_s, rb[q], db[q]);
            if (++nxt_s == S) nxt_s = 0, ++nxt_t;
        }
    };
    // The vectors' digits: 8 lanes a block, four columns each (columns past the
    // end are zeros), a pass of the workgroup over WG / 8 blocks. Vectors that are
    // not there leave rows of A that only results that are not there come from.
    const auto x_load = [&](uint32_t u0, uint32_t i, uint32_t tok) {
        const BufRsrc r = make_rsrc(x + (tok < n_vec ? tok * a.x_stride : 0), tok < n_vec ? a.cols * 4 : 0);
        return buf_load_b128(r, (u0 * kQ4UnitCols + i * 4) * 4, 0);
    };
    const auto x_store = [&](const uint4& q, uint32_t i, uint32_t units, uint32_t tok) {
        if (i >= units * 32 || tok >= n_vec) return;
        const float v[4] = {__uint_as_float(q.x), __uint_as_float(q.y), __uint_as_float(q.z), __uint_as_float(q.w)};
        store_digits<TOK>(v, tok, i >> 3, i & 7, aq, xs);
    };
    const auto fill = [&](uint32_t u0, uint32_t units, uint32_t i0) {
        for (uint32_t i = i0 + threadIdx.x; i < units * 32; i += WG) {
            uint4 q[TOK];
#pragma unroll
            for (uint32_t tok = 0; tok < TOK; ++tok) q[tok] = x_load(u0, i, tok);
#pragma unroll
            for (uint32_t tok = 0; tok < TOK; ++tok) x_store(q[tok], i, units, tok);
        }
    };

    {
        // The first passes' vectors are asked for before any weight: a CU returns
        // loads in the order of their issue, and the barrier orders the waves'.
        constexpr uint32_t kPre = TOK == 1 ? 1024 / WG : 1;
        uint4 pre[kPre][TOK];
#pragma unroll
        for (uint32_t q = 0; q < kPre; ++q)
#pragma unroll
            for (uint32_t tok = 0; tok < TOK; ++tok) pre[q][tok] = x_load(0, q * WG + threadIdx.x, tok);
        __builtin_amdgcn_s_barrier();
        start(chunk);
        for (uint32_t i = threadIdx.x; i < n_tiles * kOut; i += WG) row_sum[i] = 0.0f;
#pragma unroll
        for (uint32_t q = 0; q < kPre; ++q)
#pragma unroll
            for (uint32_t tok = 0; tok < TOK; ++tok) x_store(pre[q][tok], q * WG + threadIdx.x, chunk, tok);
        fill(0, chunk, kPre * WG);
    }
    float acc = 0.0f;
    bool whole = cur_s == 0;  // the current tile's part began at its first step
    const auto compute = [&](uint32_t j, const uint4 (&r)[kQ4Ups], const uint2& d) {
        const uint32_t scale4[2] = {d.x, d.y};
#pragma unroll
        for (uint32_t i = 0; i < kQ4Ups; ++i) {
            const uint32_t u = cur_s * kQ4Ups + i;  // of the chunk
            const uint32_t ul = min(u, n_units - 1);  // (a step's absent units have scales of 0)
            const uint8_t* p = aq + ul * q4_unit_bytes<TOK>() + a_lane;
            const uint32_t w[4] = {r[i].x, r[i].y, r[i].z, r[i].w};
            const float dw = f16_scale((uint16_t)(scale4[i >> 1] >> (16 * (i & 1)))) * q4_unscale<FMT>();
            if constexpr (TOK == 1) {
                // Block b's digits are in rows 4 b ..: four products into one
                // accumulator leave block g's four sums in lane group g.
                const uint2 h = *reinterpret_cast<const uint2*>(p);
                v4i dv = {0, 0, 0, 0};
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const long av = (long)(((uint64_t)(h.y & mine[b]) << 32) | (h.x & mine[b]));
                    dv = __builtin_amdgcn_mfma_i32_16x16x32_i8(av, q4_bop<FMT>(w[b]), dv, 0, 0, 0);
                }
                acc = fmaf(digits_value(dv[0] * 256 + dv[1], dv[2] * 256 + dv[3]) * dw, xs[ul * 4 + g], acc);
            } else {
                const uint4 h0 = *reinterpret_cast<const uint4*>(p), h1 = *reinterpret_cast<const uint4*>(p + 1024);
                const long av[4] = {(long)(((uint64_t)h0.y << 32) | h0.x), (long)(((uint64_t)h0.w << 32) | h0.z),
                                    (long)(((uint64_t)h1.y << 32) | h1.x), (long)(((uint64_t)h1.w << 32) | h1.z)};
                // Lane group g holds vector g's sums of all four blocks, and the
                // scale of block g, which the others need too.
                const float4 xv = *reinterpret_cast<const float4*>(xs + ul * 16 + g * 4);
                const float xb[4] = {xv.x, xv.y, xv.z, xv.w};
                float db4[4];
                broadcast_rows4(dw, db4);
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const v4i dv = mfma_i8(av[b], q4_bop<FMT>(w[b]));
                    acc = fmaf(digits_value(dv[0] * 256 + dv[1], dv[2] * 256 + dv[3]) * db4[b], xb[b], acc);
                }
            }
        }
        const bool tile_end = cur_s + 1 == S;
        if (tile_end || j + 1 == j1) {
            const float tot = TOK == 1 ? reduce_groups(acc) : acc;
            acc = 0.0f;
            if (lane < kOut) {
                if (whole && tile_end)
                    row_sum[cur_t * kOut + lane] += tot;
                else
                    edge[cur_t == tf ? 0 : 1][wave * kOut + lane] = tot;
            }
            whole = true;
        }
        if (++cur_s == S) cur_s = 0, ++cur_t;
    };

    // Results that are infinite or NaN, once more. (Asked for behind the loop it costs a
    // single small matrix 0.05 us more, before its end four vectors 0.15.)
    bool odd = false;
    const auto defined = [&] {
        for (uint32_t i = threadIdx.x; i < n_tiles * kOut; i += WG) {
            const uint32_t row = (t_begin + i / kOut) * 16 + (i & 15), tok = i % kOut >> 4;
            if (row >= a.rows || tok >= n_vec) continue;
            float* const y = a.y + ((uint64_t)blockIdx.y * (TOK == 1 ? 1 : TOK) + tok) * a.y_stride + row;
            if (!(fabsf(*y) < INFINITY))
                *y = q4_defined<FMT>(a.recs + mat * a.rec_stride, a.dvals + mat * a.d_stride, a.units, a.d_row, a.cols, row,
                                     x + (uint64_t)tok * a.x_stride);
        }
    };
    for (uint32_t kb = 0;;) {
        lds_barrier();  // the digits are there
        for (uint32_t j = j0; j < j1; j += kRing) {
#pragma unroll
            for (uint32_t q = 0; q < kRing; ++q) {
                if (j + q < j1) {
                    load(j + q + DEPTH < j1, nxt_t, nxt_s, rb[(q + DEPTH) % kRing], db[(q + DEPTH) % kRing]);
                    if (++nxt_s == S) nxt_s = 0, ++nxt_t;
                    compute(j + q, rb[q], db[q]);
                }
            }
        }
        lds_barrier();  // the chunk's sums are there
        const bool last = kb + chunk >= a.units;
        for (uint32_t i = threadIdx.x; i < n_tiles * kOut; i += WG) {
            const uint32_t t = i / kOut, at = i % kOut;
            const uint32_t w_first = ((t * S + 1) * kWaves - 1) / L, w_last = ((t * S + S) * kWaves - 1) / L;
            float v = row_sum[i];
            if (w_first != w_last) {
                float sum = 0.0f;
                for (uint32_t w = w_first; w <= w_last; ++w) {
                    const uint32_t b0 = w * L / kWaves, b1 = (w + 1) * L / kWaves;
                    if (b0 == b1) continue;
                    sum += edge[b0 / S == t ? 0 : 1][w * kOut + at];
                }
                v += sum;
                if (!last) row_sum[i] = v;
            }
            if (last) {
                const uint32_t row = (t_begin + t) * 16 + (at & 15), tok = at >> 4;
                if (row < a.rows && tok < n_vec) {
                    if (!(fabsf(v) < INFINITY)) odd = true;
                    a.y[((uint64_t)blockIdx.y * (TOK == 1 ? 1 : TOK) + tok) * a.y_stride + row] = v;
                }
            }
        }
        if (TOK == 1 && __builtin_expect(odd, 0)) defined();
        if (last) break;
        kb += chunk;
        lds_barrier();  // digits and edge slots are free again
        u_begin = kb;
        const uint32_t units = min(chunk, a.units - kb);
        start(units);
        whole = cur_s == 0;
        fill(kb, units, 0);
    }
    if (TOK == 4 && __builtin_expect(odd, 0)) defined();
}

template <int TOK>
size_t q4_lds(uint32_t units) {
    const uint32_t chunk = units < q4_chunk<TOK>() ? units : q4_chunk<TOK>();
    return (size_t)chunk * (q4_unit_bytes<TOK>() + 16 * TOK);
}

template <int TOK, int WG, int DEPTH, int N>
hipError_t launch_set(const Q4Args* segs, uint32_t n, uint32_t fmt, uint32_t grid_x, uint32_t grid_y, size_t lds, hipStream_t s) {
    Q4Set<N> set{};
    for (uint32_t i = 0; i < (uint32_t)N; ++i) set.seg[i] = segs[i < n ? i : 0];
    const void* fn = fmt == kFmtQ4 ? reinterpret_cast<const void*>(&gemv_q4_kernel<kFmtQ4, TOK, WG, DEPTH, N>)
                                   : reinterpret_cast<const void*>(&gemv_q4_kernel<kFmtIq4, TOK, WG, DEPTH, N>);
    void* args[] = {&set};
    return hipLaunchKernel(fn, dim3(grid_x, grid_y, n), dim3(WG), args, lds, s);
}

}  // namespace

hipError_t launch_gemv_q4(const GemvArgs* segs_in, uint32_t n_segs, uint32_t fmt, int num_cu, hipStream_t s) {
    Q4Args segs[kGemvMaxSegs];
    uint32_t n = 0;
    uint64_t units = 0;
    for (uint32_t i = 0; i < n_segs; ++i) {
        if (!segs_in[i].n_probs || !segs_in[i].tiles) continue;
        if (segs_in[i].probs || segs_in[i].n_active || segs_in[i].silu_mul || segs_in[i].route_decode) return hipErrorInvalidValue;
        units += (uint64_t)segs_in[i].n_probs * segs_in[i].tiles * segs_in[i].units;
        segs[n++] = Q4Args{segs_in[i], 1};
    }
    if (n == 0) return hipSuccess;
    // About the same number of units for every workgroup, one workgroup per CU.
    const uint64_t per_wg = (units + num_cu - 1) / num_cu;
    uint32_t grid_x = 1, grid_y = 1, steps = 0;
    size_t lds = 0;
    for (uint32_t i = 0; i < n; ++i) {
        GemvArgs& a = segs[i].a;
        const uint64_t t = (per_wg + a.units - 1) / a.units;
        a.tiles_per_wg = (uint32_t)(t > q4_tiles<1>() ? q4_tiles<1>() : t);
        if (a.tiles_per_wg > a.tiles) a.tiles_per_wg = a.tiles;
        const uint32_t chunk = a.units < q4_chunk<1>() ? a.units : q4_chunk<1>();
        if (a.tiles_per_wg * ((chunk + kQ4Ups - 1) / kQ4Ups) > steps) steps = a.tiles_per_wg * ((chunk + kQ4Ups - 1) / kQ4Ups);
        const uint32_t gx = (a.tiles + a.tiles_per_wg - 1) / a.tiles_per_wg;
        if (gx > grid_x) grid_x = gx;
        if (a.n_probs > grid_y) grid_y = a.n_probs;
        if (q4_lds<1>(a.units) > lds) lds = q4_lds<1>(a.units);
    }
    if (grid_y > 65535) return hipErrorInvalidValue;
    // Eight waves a workgroup (64 matrices of [1536 x 2048] 21.9 us, four waves 27.4;
    // [154880 x 2048] 29.4 and 30.8), but four where that is a step for each ([768 x
    // 2048] 4.13 us against 4.51, [3840 x 768] 3.85 against 4.19).
    if (n == 1 && steps <= 4) return launch_set<1, 256, 2, 1>(segs, 1, fmt, grid_x, grid_y, lds, s);
    if (n == 1) return launch_set<1, 512, 1, 1>(segs, 1, fmt, grid_x, grid_y, lds, s);
    return launch_set<1, 512, 1, kGemvMaxSegs>(segs, n, fmt, grid_x, grid_y, lds, s);
}

hipError_t launch_gemv_q4_vecs(const GemvArgs& a_in, uint32_t n_vec, uint32_t fmt, int num_cu, hipStream_t s) {
    if (n_vec == 0 || a_in.tiles == 0) return hipSuccess;
    Q4Args seg{a_in, n_vec};
    GemvArgs& a = seg.a;
    const uint64_t t = (a.tiles + num_cu - 1) / num_cu;
    a.tiles_per_wg = (uint32_t)(t > q4_tiles<4>() ? q4_tiles<4>() : t);
    a.n_probs = 1;
    return launch_set<4, 512, 1, 1>(&seg, 1, fmt, (a.tiles + a.tiles_per_wg - 1) / a.tiles_per_wg, (n_vec + 3) / 4, q4_lds<4>(a.units), s);
}

}  // namespace mmhip
