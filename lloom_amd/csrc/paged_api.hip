// paged_api.hip -- the C ABI of the paged cache (include/lloom_hip.h): argument
// checks and launches.
#include <hip/hip_runtime.h>

#include <cmath>
#include <mutex>

#include "api_internal.hpp"
#include "kq_common.hpp"
#include "paged.hpp"
#include "paged_launch.hpp"

using namespace lloom;

namespace {

constexpr int64_t I32 = 0x7fffffff;

// log2 of a page size the kernels take, or -1.
int page_shift(int64_t page) {
    if (page < 16 || page > 4096 || (page & (page - 1))) return -1;
    return __builtin_ctzll((unsigned long long)page);
}

bool misaligned(const void* p, int64_t stride, int act) {
    return (uintptr_t)p % 16 || stride % (act == T_F32 ? 4 : 8);
}

int check_cache(const char* what, int act, int64_t pages, int64_t kv_heads, int64_t dim, int64_t page) {
    if (act != T_F32 && act != T_F16)
        return fail(LLOOM_HIP_EDTYPE, "%s: activation dtype %d must be F32 or F16", what, act);
    if (pages < 1 || pages > I32 || kv_heads < 1 || kv_heads > 65535)
        return fail(LLOOM_HIP_EINVAL, "%s: %lld pages of %lld key heads", what, (long long)pages, (long long)kv_heads);
    if (!paged_dim_fits(dim))
        return fail(LLOOM_HIP_ESHAPE, "%s: head_dim %lld is none of 64, 96, 128, 256", what, (long long)dim);
    if (page_shift(page) < 0)
        return fail(LLOOM_HIP_ESHAPE, "%s: page_size %lld is no power of two from 16 to 4096", what, (long long)page);
    return LLOOM_HIP_OK;
}

}  // namespace

extern "C" {

int lloom_hip_paged_plan(lloom_hip_ctx* ctx, const uint32_t* cached_dev, const uint32_t* new_dev, int64_t requests,
                         int64_t tokens, void* tables_dev, int64_t table_stride, int64_t max_blocks,
                         const uint32_t* free_dev, int64_t free_count, int64_t page_size, void* q_start_dev,
                         void* seq_lens_dev, void* positions_dev, void* slots_dev, void* taken_dev, void* stream) {
    if (!ctx || !cached_dev || !new_dev || !tables_dev || !q_start_dev || !seq_lens_dev || !taken_dev ||
        (tokens && (!positions_dev || !slots_dev)) || (free_count && !free_dev))
        return fail(LLOOM_HIP_EINVAL, "paged_plan: null argument");
    if (requests < 1 || tokens < 0 || max_blocks < 1 || free_count < 0)
        return fail(LLOOM_HIP_EINVAL, "paged_plan: %lld requests, %lld tokens, %lld blocks, %lld free pages",
                    (long long)requests, (long long)tokens, (long long)max_blocks, (long long)free_count);
    if (requests > PAGED_MAX_REQUESTS || tokens > I32 / 2 || max_blocks > I32 || free_count > I32 ||
        table_stride < max_blocks)
        return fail(LLOOM_HIP_ESHAPE, "paged_plan: %lld requests (at most %d), %lld tokens, tables of %lld blocks %lld apart",
                    (long long)requests, PAGED_MAX_REQUESTS, (long long)tokens, (long long)max_blocks,
                    (long long)table_stride);
    const int shift = page_shift(page_size);
    if (shift < 0)
        return fail(LLOOM_HIP_ESHAPE, "paged_plan: page_size %lld is no power of two from 16 to 4096", (long long)page_size);
    HIP_OK(hipSetDevice(ctx->device));
    HIP_OK(launch_paged_plan((const int*)cached_dev, (const int*)new_dev, (int)requests, (int)tokens, (int*)tables_dev,
                             table_stride, (int)max_blocks, (const int*)free_dev, (int)free_count, shift,
                             (int*)q_start_dev, (int*)seq_lens_dev, (int*)positions_dev, (int64_t*)slots_dev,
                             (int*)taken_dev, ctx->flags + 1, (hipStream_t)stream));
    return LLOOM_HIP_OK;
}

int lloom_hip_paged_append(lloom_hip_ctx* ctx, int act_dtype, const void* k_dev, int64_t k_stride, const void* v_dev,
                           int64_t v_stride, const void* slots_dev, int64_t tokens, void* k_cache_dev,
                           void* v_cache_dev, int64_t pages, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                           void* stream) {
    if (!ctx || !k_cache_dev || !v_cache_dev || (tokens && (!k_dev || !v_dev || !slots_dev)))
        return fail(LLOOM_HIP_EINVAL, "paged_append: null argument");
    if (int rc = check_cache("paged_append", act_dtype, pages, kv_heads, head_dim, page_size)) return rc;
    if (tokens < 0 || tokens > I32 / 2) return fail(LLOOM_HIP_EINVAL, "paged_append: %lld tokens", (long long)tokens);
    if (k_stride < kv_heads * head_dim || v_stride < kv_heads * head_dim)
        return fail(LLOOM_HIP_ESHAPE, "paged_append: rows %lld and %lld apart overlap (%lld heads of %lld)",
                    (long long)k_stride, (long long)v_stride, (long long)kv_heads, (long long)head_dim);
    if (misaligned(k_dev, k_stride, act_dtype) || misaligned(v_dev, v_stride, act_dtype) ||
        misaligned(k_cache_dev, 0, T_F16) || misaligned(v_cache_dev, 0, T_F16))
        return fail(LLOOM_HIP_EINVAL, "paged_append: rows and caches must be 16-byte aligned");
    if (tokens == 0) return LLOOM_HIP_OK;
    HIP_OK(hipSetDevice(ctx->device));
    HIP_OK(launch_paged_append(act_dtype, k_dev, k_stride, v_dev, v_stride, (const int64_t*)slots_dev, (int)tokens,
                               k_cache_dev, v_cache_dev, (int)pages, (int)kv_heads, (int)head_dim,
                               page_shift(page_size), ctx->flags + 1, (hipStream_t)stream));
    return LLOOM_HIP_OK;
}

static int check_attention(int64_t tokens, int64_t requests, int64_t kv_heads, int64_t group, int64_t max_new) {
    if (tokens < 0 || requests < 1 || kv_heads < 1 || group < 1 || max_new < 0)
        return fail(LLOOM_HIP_EINVAL, "paged_attention: %lld tokens of %lld requests, %lld key heads of %lld, max_new %lld",
                    (long long)tokens, (long long)requests, (long long)kv_heads, (long long)group, (long long)max_new);
    // rows of a request, and items of a call, are counted in 32 bits
    if (requests > PAGED_MAX_REQUESTS || kv_heads > 1024 || group > 1024 || tokens > I32 / 8 / (group * kv_heads))
        return fail(LLOOM_HIP_ESHAPE, "paged_attention: %lld requests (at most %d), %lld tokens of %lld x %lld heads",
                    (long long)requests, PAGED_MAX_REQUESTS, (long long)tokens, (long long)kv_heads, (long long)group);
    return LLOOM_HIP_OK;
}

int lloom_hip_paged_attention(lloom_hip_ctx* ctx, int act_dtype, const void* q_dev, int64_t q_stride, int64_t tokens,
                              const void* k_cache_dev, const void* v_cache_dev, int64_t pages, int64_t kv_heads,
                              int64_t group, int64_t head_dim, int64_t page_size, const void* tables_dev,
                              int64_t table_stride, int64_t max_blocks, const void* q_start_dev,
                              const void* seq_lens_dev, int64_t requests, float scale, int64_t window, int64_t sinks,
                              int64_t max_new, void* out_dev, void* stream) {
    if (!ctx || !k_cache_dev || !v_cache_dev || !tables_dev || !q_start_dev || !seq_lens_dev ||
        (tokens && (!q_dev || !out_dev)))
        return fail(LLOOM_HIP_EINVAL, "paged_attention: null argument");
    if (int rc = check_cache("paged_attention", act_dtype, pages, kv_heads, head_dim, page_size)) return rc;
    if (int rc = check_attention(tokens, requests, kv_heads, group, max_new)) return rc;
    if (max_blocks < 1 || max_blocks > I32 || table_stride < max_blocks)
        return fail(LLOOM_HIP_ESHAPE, "paged_attention: tables of %lld blocks %lld apart", (long long)max_blocks,
                    (long long)table_stride);
    if (q_stride < kv_heads * group * head_dim)
        return fail(LLOOM_HIP_ESHAPE, "paged_attention: q rows %lld apart overlap (%lld heads of %lld)",
                    (long long)q_stride, (long long)(kv_heads * group), (long long)head_dim);
    if (window < 0 || window > I32 || sinks < 0 || sinks > I32 || !std::isfinite(scale))
        return fail(LLOOM_HIP_EINVAL, "paged_attention: window %lld, sinks %lld, scale %g", (long long)window,
                    (long long)sinks, (double)scale);
    if (misaligned(q_dev, q_stride, act_dtype) || misaligned(out_dev, 0, act_dtype) ||
        misaligned(k_cache_dev, 0, T_F16) || misaligned(v_cache_dev, 0, T_F16))
        return fail(LLOOM_HIP_EINVAL, "paged_attention: q, out and the caches must be 16-byte aligned");
    if (tokens == 0) return LLOOM_HIP_OK;
    HIP_OK(hipSetDevice(ctx->device));
    hipStream_t s = (hipStream_t)stream;
    std::lock_guard<std::mutex> lock(ctx->mu);
    void* ws = nullptr;
    const size_t need =
        paged_attention_workspace_bytes(tokens, requests, (int)kv_heads, (int)group, (int)head_dim, (int)max_new);
    if (need)
        if (int rc = ensure_ws(ctx, need, s, &ws)) return rc;
    if (ctx->joins_left.exchange(false)) {
        hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
        const hipError_t e = launch_paged_clear(ctx->joins, s);
        // recorded into a graph, it has not been done
        if (e != hipSuccess || hipStreamIsCapturing(s, &cap) != hipSuccess || cap != hipStreamCaptureStatusNone)
            ctx->joins_left = true;
        HIP_OK(e);
    }
    PagedCall c{q_dev, (const uint16_t*)k_cache_dev, (const uint16_t*)v_cache_dev, out_dev, (const int*)q_start_dev,
                (const int*)seq_lens_dev, (const int*)tables_dev, ctx->flags + 1, ctx->joins, q_stride, table_stride, (int)tokens,
                (int)requests, (int)kv_heads, (int)group, (int)pages, page_shift(page_size), (int)max_blocks,
                (int)window, (int)sinks, scale * 1.44269504088896340736f,
                group > 1 ? (uint32_t)(((1ull << 32) + group - 1) / group) : 0u};
    HIP_OK(launch_paged_attention(act_dtype, (int)head_dim, c, (int)max_new, ws, s));
    return LLOOM_HIP_OK;
}

int lloom_hip_paged_attention_workspace_bytes(int64_t tokens, int64_t requests, int64_t kv_heads, int64_t group,
                                              int64_t head_dim, int64_t max_new, size_t* bytes) {
    if (!bytes) return fail(LLOOM_HIP_EINVAL, "paged_attention_workspace_bytes: null argument");
    if (int rc = check_attention(tokens, requests, kv_heads, group, max_new)) return rc;
    if (!paged_dim_fits(head_dim))
        return fail(LLOOM_HIP_ESHAPE, "paged_attention: head_dim %lld is none of 64, 96, 128, 256", (long long)head_dim);
    *bytes = paged_attention_workspace_bytes(tokens, requests, (int)kv_heads, (int)group, (int)head_dim, (int)max_new);
    return LLOOM_HIP_OK;
}

}  // extern "C"
