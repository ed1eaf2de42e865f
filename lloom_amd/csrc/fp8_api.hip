// fp8_api.hip -- the C ABI of the 8-bit floating-point products
// (include/lloom_hip.h): argument checks, routes and launches.
#include <hip/hip_runtime.h>

#include <mutex>

#include "api_internal.hpp"
#include "fp8.hpp"

using namespace lloom;

namespace {

constexpr int64_t MAX_ROWS = 1 << 24, MAX_N = 1 << 24, MAX_K = 1 << 22;

bool is_act(int t) { return t == T_F32 || t == T_F16 || t == T_BF16; }
int64_t type_bytes(int t) { return t == T_F32 ? 4 : t == T_E4M3 ? 1 : 2; }

int check_act(const char* what, int type) {
    if (is_act(type)) return LLOOM_HIP_OK;
    return fail(LLOOM_HIP_EDTYPE, "%s: activation dtype %d must be F32, F16 or BF16", what, type);
}

int check_k(const char* what, int64_t k) {
    if (k < 1) return fail(LLOOM_HIP_EINVAL, "%s: k %lld", what, (long long)k);
    if (k % 16 || k > MAX_K)
        return fail(LLOOM_HIP_ESHAPE, "%s: k %lld is no multiple of 16 up to %lld", what, (long long)k, (long long)MAX_K);
    return LLOOM_HIP_OK;
}

// Rows of x: `stride` elements apart, 16-byte aligned.
int check_rows(const char* what, int type, const void* x, int64_t stride, int64_t rows, int64_t k) {
    if (rows < 0 || rows > MAX_ROWS)
        return fail(rows < 0 ? LLOOM_HIP_EINVAL : LLOOM_HIP_ESHAPE, "%s: %lld rows (at most %lld)", what, (long long)rows,
                    (long long)MAX_ROWS);
    if (rows * k > ((int64_t)1 << 36))  // a launch's threads, 8 values each
        return fail(LLOOM_HIP_ESHAPE, "%s: %lld rows of %lld", what, (long long)rows, (long long)k);
    if (stride < k)
        return fail(LLOOM_HIP_ESHAPE, "%s: rows of %lld, %lld apart, overlap", what, (long long)k, (long long)stride);
    if ((uintptr_t)x % 16 || stride * type_bytes(type) % 16)
        return fail(LLOOM_HIP_EINVAL, "%s: rows must be 16-byte aligned", what);
    return LLOOM_HIP_OK;
}

// Bytes that a call reads or writes: rows of `row` bytes, `apart` from each other.
struct Span {
    const void* at;
    int64_t rows, apart, row;
};
// Workgroups read what others have written already where an output shares memory
// with an input or another output.
int check_apart(const char* what, const Span* out, int outs, const Span* in, int ins) {
    auto meet = [](const Span& a, const Span& b) {
        if (!a.at || !b.at || a.rows < 1 || b.rows < 1) return false;
        typedef unsigned __int128 Address;  // rows may be any number of bytes apart
        auto end = [](const Span& s) { return (Address)(uintptr_t)s.at + (Address)(s.rows - 1) * s.apart + s.row; };
        return (uintptr_t)a.at < end(b) && (uintptr_t)b.at < end(a);
    };
    for (int i = 0; i < outs; i++) {
        for (int j = 0; j < ins; j++)
            if (meet(out[i], in[j])) return fail(LLOOM_HIP_EINVAL, "%s: an output overlaps an input", what);
        for (int j = 0; j < i; j++)
            if (meet(out[i], out[j])) return fail(LLOOM_HIP_EINVAL, "%s: outputs overlap", what);
    }
    return LLOOM_HIP_OK;
}
Span rows_span(int type, const void* x, int64_t stride, int64_t rows, int64_t k) {
    return {x, rows, stride * type_bytes(type), k * type_bytes(type)};
}
Span scales_span(const float* s, int64_t rows, int64_t row, int64_t blocks, int64_t block) {
    return {rows > 0 ? s : nullptr, blocks, 4 * block, 4 * ((rows - 1) * row + 1)};
}

int check_product(const char* what, const void* w, const float* ws, int64_t experts, int64_t n, int64_t k, const void* x,
                  int x_type, int64_t x_stride, const float* xs, int64_t xs_row, int64_t xs_block, int64_t x_rows,
                  const void* y, int y_type) {
    if (!w || !ws || (x_rows && !x)) return fail(LLOOM_HIP_EINVAL, "%s: null argument", what);
    if (x_type != T_E4M3)
        if (int rc = check_act(what, x_type)) return rc;
    if (int rc = check_act(what, y_type)) return rc;
    if (int rc = check_k(what, k)) return rc;
    if (n < 1) return fail(LLOOM_HIP_EINVAL, "%s: n %lld", what, (long long)n);
    if (n > MAX_N) return fail(LLOOM_HIP_ESHAPE, "%s: n %lld is over %lld", what, (long long)n, (long long)MAX_N);
    if (experts < 1) return fail(LLOOM_HIP_EINVAL, "%s: %lld experts", what, (long long)experts);
    if (experts > MOE_MAX_EXPERTS)
        return fail(LLOOM_HIP_ESHAPE, "%s: %lld experts, at most %d", what, (long long)experts, MOE_MAX_EXPERTS);
    if (int rc = check_rows(what, x_type, x, x_stride, x_rows, k)) return rc;
    if (x_type == T_E4M3) {
        if (x_rows && !xs) return fail(LLOOM_HIP_EINVAL, "%s: E4M3 rows without scales", what);
        if (xs_row < 0 || xs_block < 0)
            return fail(LLOOM_HIP_EINVAL, "%s: scales %lld and %lld apart", what, (long long)xs_row, (long long)xs_block);
        if ((uintptr_t)xs % 4) return fail(LLOOM_HIP_EINVAL, "%s: scales must be 4-byte aligned", what);
    }
    if ((uintptr_t)w % 16 || (uintptr_t)ws % 4 || (uintptr_t)y % 16)
        return fail(LLOOM_HIP_EINVAL, "%s: the weight and y must be 16-byte, the scales 4-byte aligned", what);
    return LLOOM_HIP_OK;
}

// x in 8 bits, where a call brings it there in a launch before the product's:
// q [rows][k], then the scales, block by block.
struct XCopy {
    bool needed;
    size_t scales_at, bytes;
};
XCopy x_copy(int x_type, int64_t rows, int64_t x_rows, int64_t k, int64_t experts, bool grouped) {
    const size_t q = ((size_t)x_rows * k + 255) & ~(size_t)255;
    return {x_type != T_E4M3 && !fp8_few_fuses(x_type, rows, k, experts, grouped), q,
            q + (size_t)x_rows * ((k + 127) / 128) * sizeof(float)};
}

// The kernels' 32-bit offsets: of a tile's rows of e4m3 x, or of all rows that may
// be gathered, and of their scales.
int check_offsets(const char* what, int x_type, int64_t rows, int64_t x_rows, int64_t stride, int64_t xs_row,
                  int64_t xs_block, int64_t k, int64_t experts, bool grouped, bool gathered) {
    if (x_type != T_E4M3) {
        if (!x_copy(x_type, rows, x_rows, k, experts, grouped).needed) return LLOOM_HIP_OK;
        stride = k, xs_row = 1, xs_block = x_rows;
    }
    const int64_t most = (int64_t)1 << 31, reach = gathered ? x_rows : 256;
    if (stride < most && xs_row < most && xs_block < most && reach * stride + k < most &&
        (reach * xs_row + (k + 127) / 128 * xs_block) * 4 < most)
        return LLOOM_HIP_OK;
    return fail(LLOOM_HIP_ESHAPE, "%s: %lld rows of x, %lld bytes apart, or their scales, are past 2^31 bytes", what,
                (long long)reach, (long long)stride);
}

// A product's launch, in either mode of lloom_hip_ctx_set_fp8_mma.
int check_grid(const char* what, int x_type, int64_t rows, int64_t n, int64_t k, int64_t experts, bool grouped) {
    static const int none = 0;
    Fp8Call c = {};
    c.n = (int)n, c.k = (int)k, c.kb = (int)((k + 127) / 128), c.nb = (int)((n + 127) / 128), c.m = (int)rows;
    c.experts = (int)experts, c.starts = grouped ? &none : nullptr;
    if (x_type != T_E4M3 && !fp8_few_fuses(x_type, rows, k, experts, grouped)) x_type = T_E4M3;
    bool fits = true;
    if (fp8_few_rows(rows, n, experts, grouped)) {
        fits = fp8_few_fits(x_type, c);
    } else {
        for (bool cut : {false, true}) c.cut = cut, c.y_type = cut ? T_F16 : T_F32, fits = fits && fp8_tile_fits(c);
    }
    if (fits) return LLOOM_HIP_OK;
    return fail(LLOOM_HIP_ESHAPE, "%s: %lld rows by n %lld are over the threads of a launch", what, (long long)rows,
                (long long)n);
}

int run_product(lloom_hip_ctx* ctx, int x_type, Fp8Call c, hipStream_t s) {
    const XCopy copy = x_copy(x_type, c.m, c.x_rows, c.k, c.experts, c.starts != nullptr);
    std::unique_lock<std::mutex> lock(ctx->mu, std::defer_lock);
    if (copy.needed && c.x_rows) {
        lock.lock();
        void* ws = nullptr;
        if (int rc = ensure_ws(ctx, copy.bytes, s, &ws)) return rc;
        float* scales = (float*)((uint8_t*)ws + copy.scales_at);
        HIP_OK(launch_fp8_rows(x_type, c.x, c.x_stride, nullptr, 0, c.x_rows, c.k, ws, scales, c.x_rows, s));
        c.x = ws, c.x_stride = c.k, c.xs = scales, c.xs_row = 1, c.xs_block = c.x_rows;
    }
    if (copy.needed) x_type = T_E4M3;
    if (fp8_few_rows(c.m, c.n, c.experts, c.starts != nullptr)) HIP_OK(launch_fp8_few(x_type, c, s));
    else HIP_OK(launch_fp8_tile(c, s));
    return LLOOM_HIP_OK;
}

}  // namespace

extern "C" {

int lloom_hip_fp8_quantize(lloom_hip_ctx* ctx, const void* x_dev, int x_dtype, int64_t x_stride, int64_t rows, int64_t k,
                           void* q_dev, float* scales_dev, int64_t scales_stride, void* stream) {
    if (!ctx || (rows && (!x_dev || !q_dev || !scales_dev))) return fail(LLOOM_HIP_EINVAL, "fp8_quantize: null argument");
    if (int rc = check_act("fp8_quantize", x_dtype)) return rc;
    if (int rc = check_k("fp8_quantize", k)) return rc;
    if (int rc = check_rows("fp8_quantize", x_dtype, x_dev, x_stride, rows, k)) return rc;
    if (scales_stride < rows)
        return fail(LLOOM_HIP_ESHAPE, "fp8_quantize: scales of %lld rows, %lld apart, overlap", (long long)rows,
                    (long long)scales_stride);
    if ((uintptr_t)q_dev % 8 || (uintptr_t)scales_dev % 4)
        return fail(LLOOM_HIP_EINVAL, "fp8_quantize: q must be 8-byte, scales 4-byte aligned");
    const Span out[] = {{q_dev, rows, k, k}, scales_span(scales_dev, rows, 1, (k + 127) / 128, scales_stride)};
    const Span in = rows_span(x_dtype, x_dev, x_stride, rows, k);
    if (int rc = check_apart("fp8_quantize", out, 2, &in, 1)) return rc;
    if (rows == 0) return LLOOM_HIP_OK;
    HIP_OK(hipSetDevice(ctx->device));
    HIP_OK(launch_fp8_rows(x_dtype, x_dev, x_stride, nullptr, 0, rows, k, q_dev, scales_dev, scales_stride,
                           (hipStream_t)stream));
    return LLOOM_HIP_OK;
}

int lloom_hip_fp8_silu_mul(lloom_hip_ctx* ctx, const void* gate_dev, int64_t gate_stride, const void* up_dev,
                           int64_t up_stride, int dtype, int64_t rows, int64_t k, void* q_dev, float* scales_dev,
                           int64_t scales_stride, void* stream) {
    if (!ctx || (rows && (!gate_dev || !up_dev || !q_dev || !scales_dev)))
        return fail(LLOOM_HIP_EINVAL, "fp8_silu_mul: null argument");
    if (int rc = check_act("fp8_silu_mul", dtype)) return rc;
    if (int rc = check_k("fp8_silu_mul", k)) return rc;
    if (int rc = check_rows("fp8_silu_mul", dtype, gate_dev, gate_stride, rows, k)) return rc;
    if (int rc = check_rows("fp8_silu_mul", dtype, up_dev, up_stride, rows, k)) return rc;
    if (scales_stride < rows)
        return fail(LLOOM_HIP_ESHAPE, "fp8_silu_mul: scales of %lld rows, %lld apart, overlap", (long long)rows,
                    (long long)scales_stride);
    if ((uintptr_t)q_dev % 8 || (uintptr_t)scales_dev % 4)
        return fail(LLOOM_HIP_EINVAL, "fp8_silu_mul: q must be 8-byte, scales 4-byte aligned");
    const Span out[] = {{q_dev, rows, k, k}, scales_span(scales_dev, rows, 1, (k + 127) / 128, scales_stride)};
    const Span in[] = {rows_span(dtype, gate_dev, gate_stride, rows, k), rows_span(dtype, up_dev, up_stride, rows, k)};
    if (int rc = check_apart("fp8_silu_mul", out, 2, in, 2)) return rc;
    if (rows == 0) return LLOOM_HIP_OK;
    HIP_OK(hipSetDevice(ctx->device));
    HIP_OK(launch_fp8_rows(dtype, gate_dev, gate_stride, up_dev, up_stride, rows, k, q_dev, scales_dev, scales_stride,
                           (hipStream_t)stream));
    return LLOOM_HIP_OK;
}

int lloom_hip_fp8_quantize_weight(lloom_hip_ctx* ctx, const void* w_dev, int w_dtype, int64_t experts, int64_t n,
                                  int64_t k, void* q_dev, float* scales_dev, void* stream) {
    if (!ctx || !w_dev || !q_dev || !scales_dev) return fail(LLOOM_HIP_EINVAL, "fp8_quantize_weight: null argument");
    if (int rc = check_act("fp8_quantize_weight", w_dtype)) return rc;
    if (int rc = check_k("fp8_quantize_weight", k)) return rc;
    if (experts < 1 || n < 1)
        return fail(LLOOM_HIP_EINVAL, "fp8_quantize_weight: %lld weights of %lld rows", (long long)experts, (long long)n);
    if (n > MAX_N || experts > MOE_MAX_EXPERTS || experts * ((n + 127) / 128) * ((k + 127) / 128) >= (1 << 24))
        return fail(LLOOM_HIP_ESHAPE, "fp8_quantize_weight: %lld weights of [%lld, %lld]", (long long)experts, (long long)n,
                    (long long)k);
    if ((uintptr_t)w_dev % 16 || (uintptr_t)q_dev % 8 || (uintptr_t)scales_dev % 4)
        return fail(LLOOM_HIP_EINVAL, "fp8_quantize_weight: the weight must be 16-byte, q 8-byte, scales 4-byte aligned");
    const int64_t blocks = experts * ((n + 127) / 128) * ((k + 127) / 128);
    const Span out[] = {{q_dev, experts * n, k, k}, {scales_dev, blocks, 4, 4}};
    const Span in = rows_span(w_dtype, w_dev, k, experts * n, k);
    if (int rc = check_apart("fp8_quantize_weight", out, 2, &in, 1)) return rc;
    HIP_OK(hipSetDevice(ctx->device));
    HIP_OK(launch_fp8_weights(w_dtype, w_dev, experts, n, k, q_dev, scales_dev, (hipStream_t)stream));
    return LLOOM_HIP_OK;
}

int lloom_hip_fp8_matmul(lloom_hip_ctx* ctx, const void* w_dev, const float* w_scales_dev, int64_t n, int64_t k,
                         const void* x_dev, int x_dtype, int64_t x_stride, const float* x_scales_dev, int64_t xs_row,
                         int64_t xs_block, int64_t m, void* y_dev, int y_dtype, void* stream) {
    if (!ctx || (m && !y_dev)) return fail(LLOOM_HIP_EINVAL, "fp8_matmul: null argument");
    if (int rc = check_product("fp8_matmul", w_dev, w_scales_dev, 1, n, k, x_dev, x_dtype, x_stride, x_scales_dev, xs_row,
                               xs_block, m, y_dev, y_dtype))
        return rc;
    if (int rc = check_offsets("fp8_matmul", x_dtype, m, m, x_stride, xs_row, xs_block, k, 1, false, false)) return rc;
    if (int rc = check_grid("fp8_matmul", x_dtype, m, n, k, 1, false)) return rc;
    const int64_t kb = (k + 127) / 128;
    const Span out = {y_dev, m, n * type_bytes(y_dtype), n * type_bytes(y_dtype)};
    const Span in[] = {rows_span(x_dtype, x_dev, x_stride, m, k), {w_dev, n, k, k}, {w_scales_dev, (n + 127) / 128, 4 * kb, 4 * kb},
                       scales_span(x_dtype == T_E4M3 ? x_scales_dev : nullptr, m, xs_row, kb, xs_block)};
    if (int rc = check_apart("fp8_matmul", &out, 1, in, 4)) return rc;
    if (m == 0) return LLOOM_HIP_OK;
    HIP_OK(hipSetDevice(ctx->device));
    const Fp8Call c = {(const uint8_t*)w_dev, w_scales_dev, x_dev, x_scales_dev, y_dev, nullptr, nullptr, nullptr,
                       ctx->flags, x_stride, xs_row, xs_block, (int)n, (int)k, (int)((k + 127) / 128),
                       (int)((n + 127) / 128), (int)m, (int)m, (int)m, 1, y_dtype,
                       y_dtype != T_F32 && ctx->fp8_cut};
    return run_product(ctx, x_dtype, c, (hipStream_t)stream);
}

int lloom_hip_fp8_grouped_matmul(lloom_hip_ctx* ctx, const void* w_dev, const float* w_scales_dev, int64_t experts,
                                 int64_t n, int64_t k, const void* x_dev, int x_dtype, int64_t x_stride,
                                 const float* x_scales_dev, int64_t xs_row, int64_t xs_block, int64_t x_rows,
                                 const uint32_t* starts_dev, const uint32_t* gather_dev, const uint32_t* scatter_dev,
                                 int64_t rows, void* y_dev, int y_dtype, int64_t y_rows, void* stream) {
    if (!ctx || !starts_dev || (rows && !y_dev)) return fail(LLOOM_HIP_EINVAL, "fp8_grouped_matmul: null argument");
    if (int rc = check_product("fp8_grouped_matmul", w_dev, w_scales_dev, experts, n, k, x_dev, x_dtype, x_stride,
                               x_scales_dev, xs_row, xs_block, x_rows, y_dev, y_dtype))
        return rc;
    if (rows < 0 || y_rows < 0)
        return fail(LLOOM_HIP_EINVAL, "fp8_grouped_matmul: %lld rows into %lld", (long long)rows, (long long)y_rows);
    if (rows > MAX_ROWS || y_rows > MAX_ROWS || (!gather_dev && x_rows < rows) || (!scatter_dev && y_rows < rows))
        return fail(LLOOM_HIP_ESHAPE, "fp8_grouped_matmul: %lld rows (at most %lld) of %lld into %lld", (long long)rows,
                    (long long)MAX_ROWS, (long long)x_rows, (long long)y_rows);
    if (int rc = check_offsets("fp8_grouped_matmul", x_dtype, rows, x_rows, x_stride, xs_row, xs_block, k, experts, true,
                               gather_dev != nullptr))
        return rc;
    if (int rc = check_grid("fp8_grouped_matmul", x_dtype, rows, n, k, experts, true)) return rc;
    const int64_t kb = (k + 127) / 128;
    const Span out = {y_dev, y_rows, n * type_bytes(y_dtype), n * type_bytes(y_dtype)};
    const Span in[] = {rows_span(x_dtype, x_dev, x_stride, x_rows, k), {w_dev, experts * n, k, k},
                       {w_scales_dev, experts * ((n + 127) / 128), 4 * kb, 4 * kb},
                       scales_span(x_dtype == T_E4M3 ? x_scales_dev : nullptr, x_rows, xs_row, kb, xs_block),
                       {starts_dev, experts + 1, 4, 4}, {gather_dev, rows, 4, 4}, {scatter_dev, rows, 4, 4}};
    if (int rc = check_apart("fp8_grouped_matmul", &out, 1, in, 7)) return rc;
    if (rows == 0) return LLOOM_HIP_OK;
    HIP_OK(hipSetDevice(ctx->device));
    const Fp8Call c = {(const uint8_t*)w_dev, w_scales_dev, x_dev, x_scales_dev, y_dev, (const int*)starts_dev,
                       (const int*)gather_dev, (const int*)scatter_dev, ctx->flags, x_stride, xs_row, xs_block, (int)n,
                       (int)k, (int)((k + 127) / 128), (int)((n + 127) / 128), (int)rows, (int)x_rows, (int)y_rows,
                       (int)experts, y_dtype, y_dtype != T_F32 && ctx->fp8_cut};
    return run_product(ctx, x_dtype, c, (hipStream_t)stream);
}

int lloom_hip_expert_plan(lloom_hip_ctx* ctx, const uint32_t* ids_dev, int64_t tokens, int64_t topk, int64_t experts,
                          void* starts_dev, void* planes_dev, void* tokens_dev, void* stream) {
    if (!ctx || !starts_dev || (tokens && (!ids_dev || !planes_dev || !tokens_dev)))
        return fail(LLOOM_HIP_EINVAL, "expert_plan: null argument");
    if (tokens < 0 || topk < 1 || experts < 1)
        return fail(LLOOM_HIP_EINVAL, "expert_plan: %lld tokens of %lld, %lld experts", (long long)tokens, (long long)topk,
                    (long long)experts);
    if (topk > MOE_MAX_EXPERTS || experts > MOE_MAX_EXPERTS || tokens > MAX_ROWS || tokens * topk >= MAX_ROWS)
        return fail(LLOOM_HIP_ESHAPE, "expert_plan: %lld tokens of %lld (under %lld planes), %lld experts (at most %d)",
                    (long long)tokens, (long long)topk, (long long)MAX_ROWS, (long long)experts, MOE_MAX_EXPERTS);
    const int64_t planes = tokens * topk;
    const Span out[] = {{starts_dev, experts + 1, 4, 4}, {planes_dev, planes, 4, 4}, {tokens_dev, planes, 4, 4}};
    const Span in = {ids_dev, planes, 4, 4};
    if (int rc = check_apart("expert_plan", out, 3, &in, 1)) return rc;
    HIP_OK(hipSetDevice(ctx->device));
    HIP_OK(launch_expert_plan((const int*)ids_dev, tokens * topk, (int)topk, (int)experts, (int*)starts_dev,
                              (int*)planes_dev, (int*)tokens_dev, ctx->flags, (hipStream_t)stream));
    return LLOOM_HIP_OK;
}

int lloom_hip_fp8_workspace_bytes(int x_dtype, int64_t rows, int64_t x_rows, int64_t experts, int64_t k, size_t* bytes) {
    if (!bytes) return fail(LLOOM_HIP_EINVAL, "fp8_workspace_bytes: null argument");
    if (x_dtype != T_E4M3)
        if (int rc = check_act("fp8_workspace_bytes", x_dtype)) return rc;
    if (int rc = check_k("fp8_workspace_bytes", k)) return rc;
    if (rows < 0 || x_rows < 0 || experts < 0)
        return fail(LLOOM_HIP_EINVAL, "fp8_workspace_bytes: %lld rows of %lld, %lld experts", (long long)rows,
                    (long long)x_rows, (long long)experts);
    if (rows > MAX_ROWS || x_rows > MAX_ROWS || experts > MOE_MAX_EXPERTS)
        return fail(LLOOM_HIP_ESHAPE, "fp8_workspace_bytes: %lld rows of %lld (at most %lld), %lld experts (at most %d)",
                    (long long)rows, (long long)x_rows, (long long)MAX_ROWS, (long long)experts, MOE_MAX_EXPERTS);
    const XCopy copy = x_copy(x_dtype, rows, x_rows, k, experts, experts > 0);
    *bytes = copy.needed ? copy.bytes : 0;
    return LLOOM_HIP_OK;
}

}  // extern "C"
