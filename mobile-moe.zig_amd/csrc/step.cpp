// extern "C" surface of the operators between a decode step's products: norm,
// rotary positions, the paged latent cache and its attention, log
// probabilities; and of those at a step's two ends: embedding rows, the page
// plan, sampling (declared in include/mmhip.h). Host side: argument checks,
// the rotary plan's frequencies, launches. Arguments are checked before the
// context, so that every refusal can be met without a device.
#include <cmath>
#include <cstring>
#include <mutex>
#include <new>
#include <string>
#include <vector>

#include "../../include/mmhip.h"
#include "backend.hpp"

static_assert(MMHIP_ROPE_MAX_DIMS == 2 * mmhip::kRopeMaxPairs, "rope limit in the header and the library differ");
static_assert(MMHIP_KV_MAX_RANK == mmhip::kKvMaxRank && MMHIP_KV_MAX_ROPE == mmhip::kKvMaxRope,
              "cache limits in the header and the library differ");
static_assert(MMHIP_LOGPROBS_MAX_TOP == mmhip::kLogprobsMaxTop, "top limit in the header and the library differ");

static_assert(MMHIP_NO_TOKEN == mmhip::kNoToken, "the absent token in the header and the library differ");

using namespace mmhip;

struct mmhip_rope {
    mmhip_rope_params params{};
    double magnitude = 1.0;
    double* turns = nullptr;  // device: turns per position of each pair
    int device = 0;
};

namespace {

// One workgroup of at most 256 threads per row or token, and fewer than 2^32
// threads in a launch.
constexpr uint64_t kMostRows = 0xFFFFFF;

int refuse(int code, const char* what, const char* why) {
    set_error(code, std::string(what) + ": " + why);
    return code;
}
int invalid(const char* what, const char* why) { return refuse(MMHIP_ERR_INVALID, what, why); }

// No exception leaves the C entry points.
template <class F>
int guarded(F&& f) noexcept {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return MMHIP_ERR_NOMEM;
    } catch (...) {
        return MMHIP_ERR_HIP;
    }
}

// The context's device for the launches of a call, the caller's after it.
struct OnDevice {
    int before = -1;
    hipError_t e = hipSuccess;
    explicit OnDevice(int device) {
        int now = -1;
        e = hipGetDevice(&now);
        if (e == hipSuccess && now != device) {
            e = hipSetDevice(device);
            if (e == hipSuccess) before = now;
        }
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

template <class Launch>
int launch(mmhip_ctx* ctx, const char* family, Launch&& fn) {
    if (!ctx) return refuse(MMHIP_ERR_INVALID, family, "null context");
    std::lock_guard<std::mutex> lk(ctx->mu);
    OnDevice on(ctx->device);
    if (on.e != hipSuccess) return hip_fail(on.e, family);
    hipError_t e;
    {
        TimedLaunch tl(ctx, family);
        e = fn();
    }
    return e == hipSuccess ? MMHIP_OK : hip_fail(e, family);
}

bool misaligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }

const char* rope_wrong(const mmhip_rope_params& p) {
    if (p.dims < 2 || p.dims % 2 || p.dims > MMHIP_ROPE_MAX_DIMS) return "dims must be even, 2..256";
    if (p.layout > MMHIP_ROPE_HALF) return "unknown layout";
    if (p.scaling > MMHIP_ROPE_YARN) return "unknown scaling";
    if (!(p.base > 1.0f) || !std::isfinite(p.base)) return "base must be finite and above 1";
    if (!std::isfinite(p.magnitude)) return "magnitude must be finite";
    if (p.scaling != MMHIP_ROPE_NONE && (!(p.factor > 0.0f) || !std::isfinite(p.factor))) return "factor must be positive";
    if (p.scaling == MMHIP_ROPE_YARN &&
        (p.original_context == 0 || !(p.beta_fast > 0.0f) || !(p.beta_slow > 0.0f) || !std::isfinite(p.beta_fast) ||
         !std::isfinite(p.beta_slow)))
        return "YaRN needs original_context, beta_fast and beta_slow above 0";
    return nullptr;
}

// Radians per position of each pair, and the magnitude.
void rope_tables(const mmhip_rope_params& p, double* out, double* magnitude) {
    const double dims = p.dims, base = p.base, factor = p.scaling == MMHIP_ROPE_NONE ? 1.0 : (double)p.factor;
    double low = 0.0, high = 0.0;
    if (p.scaling == MMHIP_ROPE_YARN) {
        const auto at = [&](double turns) {
            return dims * std::log((double)p.original_context / (turns * 2.0 * M_PI)) / (2.0 * std::log(base));
        };
        const auto within = [&](double v) { return std::fmin(std::fmax(v, 0.0), dims - 1.0); };
        low = within(std::floor(at(p.beta_fast)));
        high = within(std::ceil(at(p.beta_slow)));
    }
    for (uint32_t i = 0; i < p.dims / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / dims);
        if (p.scaling == MMHIP_ROPE_YARN) {
            // 0.001: a ramp of no width is a step.
            const double r = std::fmin(std::fmax((i - low) / std::fmax(high - low, 0.001), 0.0), 1.0);
            out[i] = f * (1.0 - r) + f / factor * r;
        } else {
            out[i] = f / factor;
        }
    }
    if (p.magnitude != 0.0f) *magnitude = p.magnitude;
    else *magnitude = p.scaling == MMHIP_ROPE_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
}

const char* cache_wrong(const mmhip_kv_cache& c) {
    if (c.rank == 0 || c.rank % 32 || c.rank > MMHIP_KV_MAX_RANK) return "rank must be a multiple of 32 up to 512";
    if (c.rope_dims % 32 || c.rope_dims > MMHIP_KV_MAX_ROPE) return "rope_dims must be 0, 32 or 64";
    if (c.page_tokens < 16 || c.page_tokens > 1024 || (c.page_tokens & (c.page_tokens - 1)))
        return "page_tokens must be a power of two, 16..1024";
    if (c.n_pages == 0 || (uint64_t)c.n_pages * c.page_tokens >= 0x80000000ull)
        return "n_pages * page_tokens must be in [1, 2^31)";
    return nullptr;
}
bool cache_type(uint32_t type) { return type == kF16 || type == kQ8_0; }

PagedGeom paged_geom(const mmhip_kv_cache& c) {
    PagedGeom g{};
    g.width = c.rank + c.rope_dims;
    g.rank = c.rank;
    while ((1u << g.page_shift) < c.page_tokens) ++g.page_shift;
    g.n_pages = c.n_pages;
    g.q8 = c.type == kQ8_0;
    g.page_bytes = paged_page_bytes(g.q8 != 0, g.width, c.page_tokens);
    return g;
}

int check_cache(const char* what, const mmhip_kv_cache* c) {
    if (!c || !c->pool_dev) return invalid(what, "null cache or pool");
    if (!cache_type(c->type)) return refuse(MMHIP_ERR_UNSUPPORTED, what, "the cache holds F16 or Q8_0");
    if (const char* why = cache_wrong(*c)) return invalid(what, why);
    if (misaligned(c->pool_dev, 16)) return invalid(what, "pool_dev must be 16-byte aligned");
    return MMHIP_OK;
}

}  // namespace

extern "C" {

int mmhip_rms_norm_dev(mmhip_ctx* ctx, void* y, uint32_t y_type, uint64_t y_stride, float* sum, uint64_t sum_stride,
                       const float* x, uint64_t x_stride, const float* residual, uint64_t residual_stride,
                       const float* weight, uint64_t n_rows, uint32_t cols, float eps) {
    return guarded([&]() -> int {
        const char* what = "rms_norm";
        if (y_type != kF32 && y_type != kF16 && y_type != kQ8_0)
            return refuse(MMHIP_ERR_UNSUPPORTED, what, "y_type must be F32, F16 or Q8_0");
        if (cols == 0 || cols > 0x7FFFFFFFu) return invalid(what, "cols outside [1, 2^31)");
        if (!(eps >= 0.0f)) return invalid(what, "eps must be at least 0");
        if (n_rows > kMostRows) return invalid(what, "2^24 rows or more");
        if (n_rows == 0) return ctx ? MMHIP_OK : invalid(what, "null context");
        if (!y || !x || !weight) return invalid(what, "null pointer");
        if (x_stride < cols || (residual && residual_stride < cols) || (sum && sum_stride < cols) ||
            (y_type != kQ8_0 && y_stride < cols))
            return invalid(what, "a stride is below cols");
        if (y == sum) return invalid(what, "y_dev and sum_dev are the same buffer");
        if (y == x && (y_type != kF32 || y_stride != x_stride)) return invalid(what, "y_dev on x_dev needs f32 and its stride");
        if (y == residual && (y_type != kF32 || y_stride != residual_stride))
            return invalid(what, "y_dev on residual_dev needs f32 and its stride");
        if (sum && ((sum == x && sum_stride != x_stride) || (sum == residual && sum_stride != residual_stride)))
            return invalid(what, "sum_dev on an input needs its stride");
        if (misaligned(y, y_type == kF32 ? 4 : 2) || misaligned(x, 4) || misaligned(weight, 4) || misaligned(sum, 4) ||
            misaligned(residual, 4))
            return invalid(what, "misaligned pointer");
        NormArgs a{};
        a.y = y;
        a.y_stride = y_stride;
        a.sum = sum;
        a.sum_stride = sum_stride;
        a.x = x;
        a.x_stride = x_stride;
        a.residual = residual;
        a.residual_stride = residual_stride;
        a.weight = weight;
        a.cols = cols;
        a.eps = eps;
        return launch(ctx, what, [&] {
            return launch_rms_norm(a, y_type == kF32 ? 0u : y_type == kF16 ? 1u : 2u, n_rows, ctx->stream);
        });
    });
}

int mmhip_rope_frequencies(const mmhip_rope_params* params, double* out, double* magnitude) {
    return guarded([&]() -> int {
        if (!params || !out || !magnitude) return invalid("rope_frequencies", "null pointer");
        if (const char* why = rope_wrong(*params)) return invalid("rope_frequencies", why);
        rope_tables(*params, out, magnitude);
        return MMHIP_OK;
    });
}

int mmhip_rope_create(mmhip_ctx* ctx, const mmhip_rope_params* params, mmhip_rope** out_rope) {
    return guarded([&]() -> int {
        const char* what = "rope_create";
        if (!params || !out_rope) return invalid(what, "null pointer");
        *out_rope = nullptr;
        if (const char* why = rope_wrong(*params)) return invalid(what, why);
        if (!ctx) return invalid(what, "null context");
        double turns[kRopeMaxPairs], magnitude;
        rope_tables(*params, turns, &magnitude);
        for (uint32_t i = 0; i < params->dims / 2; ++i) turns[i] /= 2.0 * M_PI;
        std::lock_guard<std::mutex> lk(ctx->mu);
        OnDevice on(ctx->device);
        if (on.e != hipSuccess) return hip_fail(on.e, what);
        mmhip_rope* r = new mmhip_rope();
        r->params = *params;
        r->magnitude = magnitude;
        r->device = ctx->device;
        hipError_t e = hipMalloc((void**)&r->turns, params->dims / 2 * sizeof(double));
        if (e == hipSuccess)
            e = hipMemcpyAsync(r->turns, turns, params->dims / 2 * sizeof(double), hipMemcpyHostToDevice, ctx->stream);
        if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
        if (e != hipSuccess) {
            if (r->turns) (void)hipFree(r->turns);
            delete r;
            return hip_fail(e, what);
        }
        *out_rope = r;
        return MMHIP_OK;
    });
}

void mmhip_rope_destroy(mmhip_ctx* ctx, mmhip_rope* rope) {
    if (!rope) return;
    if (ctx) (void)hipStreamSynchronize(ctx->stream);
    if (rope->turns) (void)hipFree(rope->turns);
    delete rope;
}

int mmhip_rope_dev(mmhip_ctx* ctx, const mmhip_rope* rope, float* y, uint64_t y_token_stride, uint64_t y_head_stride,
                   const float* x, uint64_t x_token_stride, uint64_t x_head_stride, const uint32_t* positions,
                   uint64_t n_tokens, uint32_t n_heads, uint32_t head_dim, uint32_t first) {
    return guarded([&]() -> int {
        const char* what = "rope";
        if (!rope) return invalid(what, "null rope");
        if (head_dim < rope->params.dims || first > head_dim - rope->params.dims)
            return invalid(what, "the rotated dims leave the head");
        if (n_tokens > kMostRows) return invalid(what, "2^24 tokens or more");
        if (n_heads > kMostRows) return invalid(what, "2^24 heads or more");
        if (n_tokens == 0 || n_heads == 0) return ctx ? MMHIP_OK : invalid(what, "null context");
        if (!y || !x || !positions) return invalid(what, "null pointer");
        if (n_heads > 1 && (x_head_stride < head_dim || y_head_stride < head_dim))
            return invalid(what, "a head stride is below head_dim");
        const uint64_t heads = n_heads - 1;
        if (n_tokens > 1 && (x_token_stride < heads * x_head_stride + head_dim || y_token_stride < heads * y_head_stride + head_dim))
            return invalid(what, "a token stride is below the heads' extent");
        if (y == x && ((n_tokens > 1 && y_token_stride != x_token_stride) || (n_heads > 1 && y_head_stride != x_head_stride)))
            return invalid(what, "in place needs equal strides");
        if (misaligned(y, 4) || misaligned(x, 4) || misaligned(positions, 4)) return invalid(what, "misaligned pointer");
        if (ctx && ctx->device != rope->device) return invalid(what, "the rope belongs to another device");
        RopeArgs a{};
        a.y = y;
        a.x = x;
        a.y_token_stride = y_token_stride;
        a.y_head_stride = y_head_stride;
        a.x_token_stride = x_token_stride;
        a.x_head_stride = x_head_stride;
        a.positions = positions;
        a.turns = rope->turns;
        a.magnitude = rope->magnitude;
        a.dims = rope->params.dims;
        a.half = rope->params.layout == MMHIP_ROPE_HALF;
        a.n_heads = n_heads;
        a.head_dim = head_dim;
        a.first = first;
        a.copy = y != x;
        return launch(ctx, what, [&] { return launch_rope(a, n_tokens, ctx->stream); });
    });
}

uint64_t mmhip_kv_page_bytes(const mmhip_kv_cache* cache) {
    if (!cache || !cache_type(cache->type) || cache_wrong(*cache)) return 0;
    return paged_page_bytes(cache->type == kQ8_0, cache->rank + cache->rope_dims, cache->page_tokens);
}

int mmhip_kv_store_dev(mmhip_ctx* ctx, const mmhip_kv_cache* cache, const float* kv, uint64_t kv_stride,
                       const float* norm_weight, float eps, const mmhip_rope* rope, const uint32_t* positions,
                       const int32_t* slots, uint64_t n_tokens) {
    return guarded([&]() -> int {
        const char* what = "kv_store";
        if (int rc = check_cache(what, cache)) return rc;
        if (rope && rope->params.dims != cache->rope_dims) return invalid(what, "the rope's dims differ from rope_dims");
        if (norm_weight && !(eps >= 0.0f)) return invalid(what, "eps must be at least 0");
        if (n_tokens > kMostRows) return invalid(what, "2^24 tokens or more");
        if (n_tokens == 0) return ctx ? MMHIP_OK : invalid(what, "null context");
        if (!kv || !slots || (rope && !positions)) return invalid(what, "null pointer");
        if (n_tokens > 1 && kv_stride < cache->rank + cache->rope_dims) return invalid(what, "kv_stride is below a row");
        if (misaligned(kv, 4) || misaligned(slots, 4) || misaligned(norm_weight, 4) || misaligned(positions, 4))
            return invalid(what, "misaligned pointer");
        if (ctx && rope && ctx->device != rope->device) return invalid(what, "the rope belongs to another device");
        StoreArgs a{};
        a.pool = static_cast<uint8_t*>(cache->pool_dev);
        a.geom = paged_geom(*cache);
        a.kv = kv;
        a.kv_stride = kv_stride;
        a.weight = norm_weight;
        a.eps = eps;
        a.turns = rope ? rope->turns : nullptr;
        a.magnitude = rope ? rope->magnitude : 1.0;
        a.half = rope && rope->params.layout == MMHIP_ROPE_HALF;
        a.positions = positions;
        a.slots = slots;
        return launch(ctx, what, [&] {
            a.status = ctx->step_status_dev();
            return launch_kv_store(a, n_tokens, ctx->stream);
        });
    });
}

uint64_t mmhip_mla_attention_workspace(mmhip_ctx* ctx, uint32_t n_tokens, uint32_t n_heads, uint32_t rank) {
    if (!ctx) return 0;
    return mla_workspace_bytes(n_tokens, n_heads, rank, ctx->num_cu);
}

int mmhip_mla_attention_dev(mmhip_ctx* ctx, const mmhip_mla_attention* args) {
    return guarded([&]() -> int {
        const char* what = "attention";
        if (!args) return invalid(what, "null arguments");
        const mmhip_mla_attention& p = *args;
        if (int rc = check_cache(what, &p.cache)) return rc;
        if (!std::isfinite(p.scale)) return invalid(what, "scale must be finite");
        if (p.n_heads == 0) return invalid(what, "n_heads must be above 0");
        if ((uint64_t)p.n_tokens * p.n_heads > 0x7FFFFFFF) return invalid(what, "more than 2^31 - 1 tokens times heads");
        if (p.n_tables == 0 || p.table_pages == 0 || p.table_stride < p.table_pages)
            return invalid(what, "tables need rows, pages and a stride of at least table_pages");
        if (((uint64_t)p.table_pages * p.cache.page_tokens) > 0xFFFFFFFFull)
            return invalid(what, "a table names 2^32 positions or more");
        if (p.n_tokens == 0) return ctx ? MMHIP_OK : invalid(what, "null context");
        const uint32_t pe = p.cache.rope_dims;
        if (!p.q_dev || (pe && !p.q_pe_dev) || !p.out_dev || !p.tables_dev || !p.lens_dev) return invalid(what, "null pointer");
        const uint64_t heads = p.n_heads - 1;
        const bool many = p.n_heads > 1, tokens = p.n_tokens > 1;
        if (many && (p.q_head_stride < p.cache.rank || p.out_head_stride < p.cache.rank || (pe && p.q_pe_head_stride < pe)))
            return invalid(what, "a head stride is below its row");
        if (tokens && (p.q_token_stride < p.cache.rank || (pe && p.q_pe_token_stride < pe)))
            return invalid(what, "a token stride is below its row");
        if (tokens && p.out_token_stride < heads * p.out_head_stride + p.cache.rank)
            return invalid(what, "out_token_stride is below the heads' extent");
        if (misaligned(p.q_dev, 4) || misaligned(p.q_pe_dev, 4) || misaligned(p.out_dev, 4) || misaligned(p.lse_dev, 4) ||
            misaligned(p.tables_dev, 4) || misaligned(p.table_of_dev, 4) || misaligned(p.lens_dev, 4))
            return invalid(what, "misaligned pointer");
        if (!ctx) return invalid(what, "null context");
        const uint64_t need = mla_workspace_bytes(p.n_tokens, p.n_heads, p.cache.rank, ctx->num_cu);
        if (p.workspace_bytes < need || (need && (!p.workspace_dev || misaligned(p.workspace_dev, 16))))
            return invalid(what, "the workspace is too small, null or not 16-byte aligned");
        MlaArgs a{};
        a.pool = static_cast<const uint8_t*>(p.cache.pool_dev);
        a.geom = paged_geom(p.cache);
        a.q = p.q_dev;
        a.q_pe = p.q_pe_dev;
        a.out = p.out_dev;
        a.lse = p.lse_dev;
        a.q_token_stride = p.q_token_stride;
        a.q_head_stride = p.q_head_stride;
        a.q_pe_token_stride = p.q_pe_token_stride;
        a.q_pe_head_stride = p.q_pe_head_stride;
        a.out_token_stride = p.out_token_stride;
        a.out_head_stride = p.out_head_stride;
        a.tables = p.tables_dev;
        a.table_stride = p.table_stride;
        a.n_tables = p.n_tables;
        a.table_pages = p.table_pages;
        a.table_of = p.table_of_dev;
        a.lens = p.lens_dev;
        a.n_tokens = p.n_tokens;
        a.n_heads = p.n_heads;
        a.scale = p.scale;
        a.work = p.workspace_dev;
        a.status = ctx->step_status_dev();
        a.num_cu = ctx->num_cu;
        return launch(ctx, what, [&] { return launch_mla(a, ctx->stream); });
    });
}

uint64_t mmhip_logprobs_workspace(mmhip_ctx* ctx, uint64_t n_rows, uint64_t vocab, uint32_t top) {
    if (!ctx) return 0;
    return logprobs_workspace_bytes(n_rows, vocab, top);
}

int mmhip_logprobs_dev(mmhip_ctx* ctx, const float* logits, uint64_t stride, uint64_t n_rows, uint64_t vocab,
                       const uint32_t* tokens, uint64_t n_given, float* token_logprobs, float* entropy, uint32_t top,
                       uint32_t* top_ids, float* top_logprobs, void* workspace, uint64_t workspace_bytes) {
    return guarded([&]() -> int {
        const char* what = "logprobs";
        if (vocab == 0 || vocab >= 0x80000000ull) return invalid(what, "vocab outside [1, 2^31)");
        if (top > MMHIP_LOGPROBS_MAX_TOP || top > vocab) return invalid(what, "top is above 32 or above vocab");
        if (n_given >= 0x80000000ull) return invalid(what, "2^31 given tokens or more");
        if (n_rows > kMostRows) return invalid(what, "2^24 rows or more");
        if (n_rows == 0) return ctx ? MMHIP_OK : invalid(what, "null context");
        if (!logits || (n_given && (!tokens || !token_logprobs)) || (top && !top_ids)) return invalid(what, "null pointer");
        if (n_rows > 1 && stride < vocab) return invalid(what, "the stride is below vocab");
        if (misaligned(logits, 4) || misaligned(tokens, 4) || misaligned(token_logprobs, 4) || misaligned(entropy, 4) ||
            misaligned(top_ids, 4) || misaligned(top_logprobs, 4))
            return invalid(what, "misaligned pointer");
        if (!ctx) return invalid(what, "null context");
        const uint64_t need = logprobs_workspace_bytes(n_rows, vocab, top);
        if (workspace_bytes < need || (need && (!workspace || misaligned(workspace, 16))))
            return invalid(what, "the workspace is too small, null or not 16-byte aligned");
        LogprobsArgs a{};
        a.logits = logits;
        a.stride = stride;
        a.vocab = (uint32_t)vocab;
        a.tokens = tokens;
        a.n_given = n_given;
        a.token_logprobs = token_logprobs;
        a.entropy = entropy;
        a.top = top;
        a.top_ids = top_ids;
        a.top_logprobs = top_logprobs;
        a.work = workspace;
        a.status = ctx->step_status_dev();
        return launch(ctx, what, [&] { return launch_logprobs(a, n_rows, ctx->stream); });
    });
}

int mmhip_embed_dev(mmhip_ctx* ctx, float* y, uint64_t y_stride, const void* table, uint32_t type, uint64_t rows,
                    uint32_t cols, const uint32_t* tokens, uint64_t n_tokens, float scale) {
    return guarded([&]() -> int {
        const char* what = "embed";
        if (block_size(type) == 0) return refuse(MMHIP_ERR_UNSUPPORTED, what, "the table's type is not on this path");
        if (rows == 0 || rows > 0xFFFFFFFFull) return invalid(what, "rows outside [1, 2^32)");
        if (cols == 0 || cols > 0x7FFFFFFFu) return invalid(what, "cols outside [1, 2^31)");
        if ((type == kIq2Xxs || type_4bit(type)) && cols % block_size(type))
            return invalid(what, "cols must hold whole blocks of the table's type");
        if (n_tokens > kMostRows) return invalid(what, "2^24 tokens or more");
        // A wave per 512 values, and fewer than 2^32 threads.
        if (n_tokens * (((uint64_t)cols + 1023) / 1024) > kMostRows) return invalid(what, "2^24 pieces of 1024 values or more");
        if (n_tokens == 0) return ctx ? MMHIP_OK : invalid(what, "null context");
        if (!y || !table || !tokens) return invalid(what, "null pointer");
        if (n_tokens > 1 && y_stride < cols) return invalid(what, "y_stride is below cols");
        if (misaligned(y, 4) || misaligned(tokens, 4) || misaligned(table, type == kF32 ? 4 : 2))
            return invalid(what, "misaligned pointer");
        EmbedArgs a{};
        a.y = y;
        a.y_stride = y_stride;
        a.table = static_cast<const uint8_t*>(table);
        a.row_bytes = tensor_bytes(type, cols);
        a.rows = rows;
        a.cols = cols;
        a.tokens = tokens;
        a.scale = scale;
        return launch(ctx, what, [&] {
            a.status = ctx->step_status_dev();
            return launch_embed(a, type, n_tokens, ctx->stream);
        });
    });
}

uint64_t mmhip_kv_plan_workspace(mmhip_ctx* ctx, uint32_t n_requests) {
    if (!ctx) return 0;
    return plan_workspace_bytes(n_requests);
}

int mmhip_kv_plan_dev(mmhip_ctx* ctx, const mmhip_kv_plan* args) {
    return guarded([&]() -> int {
        const char* what = "kv_plan";
        if (!args) return invalid(what, "null arguments");
        const mmhip_kv_plan& p = *args;
        if (p.page_tokens < 16 || p.page_tokens > 1024 || (p.page_tokens & (p.page_tokens - 1)))
            return invalid(what, "page_tokens must be a power of two, 16..1024");
        if (p.n_pages == 0 || (uint64_t)p.n_pages * p.page_tokens >= 0x80000000ull)
            return invalid(what, "n_pages * page_tokens must be in [1, 2^31)");
        if (p.n_requests > kMostRows) return invalid(what, "2^24 requests or more");
        if (p.table_pages == 0 || (p.n_requests > 1 && p.table_stride < p.table_pages))
            return invalid(what, "tables need pages and a stride of at least table_pages");
        if ((uint64_t)p.table_pages * p.page_tokens > 0xFFFFFFFFull) return invalid(what, "a table names 2^32 positions or more");
        if (p.max_tokens > 0x7FFFFFFFu) return invalid(what, "2^31 tokens or more");
        if (!p.free_dev || !p.free_count_dev || !p.next_free_count_dev || !p.firsts_dev) return invalid(what, "null pointer");
        if (p.n_requests && (!p.lens_dev || !p.new_dev || !p.next_lens_dev || !p.tables_dev || !p.granted_dev))
            return invalid(what, "null pointer");
        if (p.max_tokens && (!p.positions_dev || !p.slots_dev || !p.table_of_dev || !p.seen_dev)) return invalid(what, "null pointer");
        if (p.shared_dev && !p.release_dev) return invalid(what, "shared_dev without release_dev");
        const void* all[] = {p.lens_dev, p.new_dev, p.release_dev, p.shared_dev, p.next_lens_dev, p.tables_dev, p.free_dev,
                             p.free_count_dev, p.next_free_count_dev, p.positions_dev, p.slots_dev, p.table_of_dev, p.seen_dev,
                             p.firsts_dev, p.granted_dev, p.last_dev};
        for (const void* b : all)
            if (misaligned(b, 4)) return invalid(what, "misaligned pointer");
        if (!ctx) return invalid(what, "null context");
        if (p.workspace_bytes < plan_workspace_bytes(p.n_requests) || !p.workspace_dev || misaligned(p.workspace_dev, 16))
            return invalid(what, "the workspace is too small, null or not 16-byte aligned");
        PlanArgs a{};
        a.n_requests = p.n_requests;
        while ((1u << a.page_shift) < p.page_tokens) ++a.page_shift;
        a.n_pages = p.n_pages;
        a.table_pages = p.table_pages;
        a.max_tokens = p.max_tokens;
        a.lens = p.lens_dev;
        a.added = p.new_dev;
        a.release = p.release_dev;
        a.shared = p.shared_dev;
        a.next_lens = p.next_lens_dev;
        a.tables = p.tables_dev;
        a.table_stride = p.table_stride;
        a.free = p.free_dev;
        a.free_count = p.free_count_dev;
        a.next_free_count = p.next_free_count_dev;
        a.positions = p.positions_dev;
        a.slots = p.slots_dev;
        a.table_of = p.table_of_dev;
        a.seen = p.seen_dev;
        a.firsts = p.firsts_dev;
        a.granted = p.granted_dev;
        a.last = p.last_dev;
        a.status = ctx->step_status_dev();
        return launch(ctx, what, [&] { return launch_kv_plan(a, p.workspace_dev, ctx->stream); });
    });
}

uint64_t mmhip_sample_workspace(mmhip_ctx* ctx, uint64_t n_rows, uint64_t vocab) {
    if (!ctx) return 0;
    return sample_workspace_bytes(n_rows, vocab);
}

int mmhip_sample_dev(mmhip_ctx* ctx, const mmhip_sample* args) {
    return guarded([&]() -> int {
        const char* what = "sample";
        if (!args) return invalid(what, "null arguments");
        const mmhip_sample& p = *args;
        if (p.vocab == 0 || p.vocab > MMHIP_SAMPLE_MAX_VOCAB) return invalid(what, "vocab outside [1, 2^24]");
        if (p.n_rows >= 1u << 22) return invalid(what, "2^22 rows or more");
        if (p.rows_dev && (p.n_logits == 0 || p.n_logits >= MMHIP_NO_TOKEN)) return invalid(what, "n_logits outside [1, 2^32 - 1)");
        if (p.n_rows == 0) return ctx ? MMHIP_OK : invalid(what, "null context");
        if (!p.logits_dev || !p.uniform_dev || !p.tokens_dev) return invalid(what, "null pointer");
        if ((p.rows_dev ? p.n_logits : p.n_rows) > 1 && p.stride < p.vocab) return invalid(what, "the stride is below vocab");
        const void* all[] = {p.logits_dev, p.rows_dev, p.temperature_dev, p.top_k_dev, p.top_p_dev,
                             p.min_p_dev, p.uniform_dev, p.tokens_dev, p.probs_dev, p.kept_dev};
        for (const void* b : all)
            if (misaligned(b, 4)) return invalid(what, "misaligned pointer");
        if (!ctx) return invalid(what, "null context");
        const uint64_t need = sample_workspace_bytes(p.n_rows, p.vocab);
        if (p.workspace_bytes < need || (need && (!p.workspace_dev || misaligned(p.workspace_dev, 16))))
            return invalid(what, "the workspace is too small, null or not 16-byte aligned");
        SampleArgs a{};
        a.logits = p.logits_dev;
        a.stride = p.stride;
        a.n_logits = p.n_logits;
        a.vocab = (uint32_t)p.vocab;
        a.rows = p.rows_dev;
        a.temperature = p.temperature_dev;
        a.top_k = p.top_k_dev;
        a.top_p = p.top_p_dev;
        a.min_p = p.min_p_dev;
        a.uniform = p.uniform_dev;
        a.tokens = p.tokens_dev;
        a.probs = p.probs_dev;
        a.kept = p.kept_dev;
        a.work = p.workspace_dev;
        a.status = ctx->step_status_dev();
        return launch(ctx, what, [&] { return launch_sample(a, p.n_rows, ctx->stream); });
    });
}

}  // extern "C"
