// Attention of single tokens over the paged latent cache (mlaAttention's
// cached part, inference.zig:539-660) on gfx950.
#include "device_common.hpp"
#include "kernels.hpp"

namespace mmhip {

namespace {

constexpr int kMlaThreads = 256;

// One workgroup per token and head; positions in tiles of 256.
__global__ __launch_bounds__(kMlaThreads) void mla_simple_kernel(MlaArgs a) {
    __shared__ float q[kKvMaxRank + kKvMaxRope];
    __shared__ float p[kMlaThreads];
    __shared__ uint64_t at_row[kMlaThreads], at_scale[kMlaThreads];
    __shared__ float red[kMlaThreads / 64];
    const PagedGeom g = a.geom;
    const uint32_t t = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads;
    const uint32_t row = a.table_of ? a.table_of[t] : t;
    uint32_t bad;
    const uint32_t len = paged_seen(g, a.lens[t], row, a.n_tables, a.table_pages, bad);
    if (bad && threadIdx.x == 0) report(a.status, bad == 1 ? kBadTableRow : kBadLength);
    for (uint32_t c = threadIdx.x; c < g.width; c += kMlaThreads)
        q[c] = a.scale * (c < g.rank ? a.q[t * a.q_token_stride + h * a.q_head_stride + c]
                                     : a.q_pe[t * a.q_pe_token_stride + h * a.q_pe_head_stride + c - g.rank]);
    float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
    for (uint32_t p0 = 0; p0 < len; p0 += kMlaThreads) {
        __syncthreads();
        const uint32_t pos = p0 + threadIdx.x;
        float s = -INFINITY;
        uint64_t ro = ~0ull, so = 0;
        if (pos < len) {
            const int32_t id = a.tables[row * a.table_stride + (pos >> g.page_shift)];
            if (paged_has(g, id)) {
                const uint32_t at = pos & ((1u << g.page_shift) - 1);
                ro = paged_row(g, (uint32_t)id, at);
                so = paged_scales(g, (uint32_t)id, at);
                s = 0.0f;
                for (uint32_t c = 0; c < g.width; ++c)
                    s += q[c] * (g.q8 ? (float)(int8_t)a.pool[ro + c] * f16_scale(*reinterpret_cast<const uint16_t*>(a.pool + so + c / 32 * 2))
                                      : f16_scale(*reinterpret_cast<const uint16_t*>(a.pool + ro + 2 * c)));
            } else {
                report(a.status, kBadPage);
            }
        }
        at_row[threadIdx.x] = ro;
        at_scale[threadIdx.x] = so;
        float top = s;
        for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float m2 = fmaxf(m, top), base = m2 == -INFINITY ? 0.0f : m2;
        const float f = expf(m - base);
        p[threadIdx.x] = expf(s - base);
        float sum = p[threadIdx.x];
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
        __syncthreads();
        l = l * f + ((red[0] + red[1]) + (red[2] + red[3]));
        m = m2;
        const uint32_t n = min(len - p0, (uint32_t)kMlaThreads);
        for (int e = 0; e < 2; ++e) {
            const uint32_t c = threadIdx.x + e * kMlaThreads;
            o[e] *= f;
            if (c >= g.rank) continue;
            for (uint32_t i = 0; i < n; ++i) {
                if (at_row[i] == ~0ull) continue;
                o[e] += p[i] * (g.q8 ? (float)(int8_t)a.pool[at_row[i] + c] * f16_scale(*reinterpret_cast<const uint16_t*>(a.pool + at_scale[i] + c / 32 * 2))
                                     : f16_scale(*reinterpret_cast<const uint16_t*>(a.pool + at_row[i] + 2 * c)));
            }
        }
    }
    for (int e = 0; e < 2; ++e) {
        const uint32_t c = threadIdx.x + e * kMlaThreads;
        if (c < g.rank) a.out[t * a.out_token_stride + h * a.out_head_stride + c] = l == 0.0f ? 0.0f : o[e] / l;
    }
    if (a.lse && threadIdx.x == 0) a.lse[(uint64_t)t * a.n_heads + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace

uint64_t mla_workspace_bytes(uint32_t, uint32_t, uint32_t, int) { return 0; }

hipError_t launch_mla(const MlaArgs& a, hipStream_t s) {
    if (a.n_tokens == 0 || a.n_heads == 0) return hipSuccess;
    mla_simple_kernel<<<a.n_tokens * a.n_heads, kMlaThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace mmhip
