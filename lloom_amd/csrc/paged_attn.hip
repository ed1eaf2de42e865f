// paged_attn.hip -- the paged attention of calls with few rows a request alone
// (paged_rows.hpp).
#include "kernels.hpp"
#include "kq_common.hpp"
#include "paged_rows.hpp"

namespace lloom {

constexpr int ATT_WAVES = 8;

template <int D, bool F32>
__global__ __launch_bounds__(64 * ATT_WAVES) void k_paged_rows(PagedCall c, PagedCut cut, float* parts) {
    __shared__ float acc[ATT_WAVES][ATT_ROWS][D + 4], stat[ATT_WAVES][2][ATT_ROWS];
    paged_rows<D, F32, ATT_WAVES>(c, cut, parts, blockIdx.x, gridDim.x, acc, stat, c.joins);
}

// One workgroup a CU: a second round costs more than the last of the balance
// (512: 26.5 against 20.0 us for 32 requests, 62 MB; 119 against 105 us for 537 MB
// of one request).
constexpr int ATT_TARGET_SHIFT = 8;

template <int D, bool F32>
static hipError_t rows_as(const PagedCall& c, const PagedCut& cut, int64_t grid, float* parts, hipStream_t s) {
    hipLaunchKernelGGL((k_paged_rows<D, F32>), dim3((unsigned)grid), dim3(64 * ATT_WAVES), 0, s, c, cut, parts);
    return hipGetLastError();
}

hipError_t launch_paged_rows(int act, int dim, const PagedCall& c, void* ws, hipStream_t s) {
    const PagedCut cut{4, 8, 1, ATT_TARGET_SHIFT, (ATT_ROWS - 1) / c.group + 1, 0, 0};
    const int64_t grid = paged_items_most(c, cut);
    float* parts = (float*)ws;
    switch (dim) {
        case 64: return act == T_F32 ? rows_as<64, true>(c, cut, grid, parts, s) : rows_as<64, false>(c, cut, grid, parts, s);
        case 96: return act == T_F32 ? rows_as<96, true>(c, cut, grid, parts, s) : rows_as<96, false>(c, cut, grid, parts, s);
        case 128: return act == T_F32 ? rows_as<128, true>(c, cut, grid, parts, s) : rows_as<128, false>(c, cut, grid, parts, s);
        case 256: return act == T_F32 ? rows_as<256, true>(c, cut, grid, parts, s) : rows_as<256, false>(c, cut, grid, parts, s);
    }
    return hipErrorInvalidValue;
}

size_t paged_rows_workspace_bytes(int kv_heads, int dim) {
    return ((size_t)paged_parts(ATT_TARGET_SHIFT) + kv_heads) * ATT_ROWS * (dim + 2) * sizeof(float);
}

}  // namespace lloom
