// paged_attn.hip -- the paged attention of calls with few rows a request alone
// (paged_rows.hpp).
#include "paged_launch.hpp"
#include "kq_common.hpp"
#include "paged_rows.hpp"

namespace lloom {

constexpr int ATT_WAVES = 8;

template <int D, bool F32>
__global__ __launch_bounds__(64 * ATT_WAVES) void k_paged_rows(PagedCall c, PagedCut cut, float* parts) {
    __shared__ float acc[ATT_WAVES][ATT_ROWS][D + 4], stat[ATT_WAVES][2][ATT_ROWS];
    paged_rows<D, F32, ATT_WAVES>(c, cut, parts, blockIdx.x, gridDim.x, acc, stat, c.joins);
}

// The sums over a call's requests that paged_find looks an item up in, a workgroup a
// cut: 4 consecutive requests a thread.  4 us with its launch.  Without it every wave
// read every request: 241 us against 90 + 5 for 1024 single tokens (188 MB), 57 against
// 51 + 4 for 256, 208 against 145 + 5 for 224 requests with 24 chunks of 509 tokens; the
// search by every wave is 2 us faster up to 128 requests, which is left.
constexpr int INDEX_WG = 1024, INDEX_EACH = PAGED_MAX_REQUESTS / INDEX_WG;

__global__ __launch_bounds__(INDEX_WG) void k_paged_index(PagedCall c, PagedCut cut0, PagedCut cut1, int* to) {
    __shared__ float part[INDEX_WG / 64];
    __shared__ int2 parts[INDEX_WG / 64];
    const PagedCut cut = blockIdx.x ? cut1 : cut0;
    to += blockIdx.x * PAGED_INDEX;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cap = paged_key_cap(c), b = threadIdx.x * INDEX_EACH;
    PagedLane at[INDEX_EACH];
    float mine = 0.0f;
    bool order = true;
#pragma unroll
    for (int i = 0; i < INDEX_EACH; i++) {
        at[i] = paged_lane(c, cut, cap, b + i);
        order &= at[i].order;
        mine += (float)at[i].tiles * at[i].units;
    }
    mine = paged_scan(mine);
    if (lane == 63) part[wave] = mine;
    const int refused = __syncthreads_or(!order);
    float total = 0.0f;
    for (int w = 0; w < INDEX_WG / 64; w++) total += part[w];
    const int chunk = paged_chunk(c, cut, total);
    PagedCount n[INDEX_EACH];
    int items = 0, split = 0;
#pragma unroll
    for (int i = 0; i < INDEX_EACH; i++) {
        n[i] = paged_count(at[i], chunk);
        items += n[i].items;
        split += n[i].split;
    }
    int ie = paged_scan(items), se = paged_scan(split);
    if (lane == 63) parts[wave] = make_int2(ie, se);
    __syncthreads();
    ie -= items, se -= split;
    for (int w = 0; w < wave; w++) ie += parts[w].x, se += parts[w].y;
#pragma unroll
    for (int i = 0; i < INDEX_EACH; i++) {
        ie += n[i].items;
        se += n[i].split;
        if (b + i < c.requests) {
            to[16 + b + i] = ie;
            to[16 + PAGED_MAX_REQUESTS + b + i] = se;
        }
    }
    if (threadIdx.x == 0) {
        to[0] = chunk;
        to[1] = refused;
    }
}

__global__ __launch_bounds__(INDEX_WG) void k_paged_clear(int* joins) {
    for (int i = threadIdx.x; i < PAGED_JOINS; i += INDEX_WG) joins[i] = 0;
}

hipError_t launch_paged_clear(int* joins, hipStream_t s) {
    hipLaunchKernelGGL(k_paged_clear, dim3(1), dim3(INDEX_WG), 0, s, joins);
    return hipGetLastError();
}

size_t paged_index_workspace_bytes(int64_t requests) { return requests > 64 ? 2 * PAGED_INDEX * sizeof(int) : 0; }

hipError_t launch_paged_index(PagedCall& c, const PagedCut* cuts, int count, int* to, hipStream_t s) {
    if (c.requests <= 64) return hipSuccess;
    hipLaunchKernelGGL(k_paged_index, dim3(count), dim3(INDEX_WG), 0, s, c, cuts[0], cuts[count - 1], to);
    c.index = to;
    return hipGetLastError();
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

hipError_t launch_paged_rows(int act, int dim, PagedCall c, int* index, void* ws, hipStream_t s) {
    const PagedCut cut{4, 8, 1, ATT_TARGET_SHIFT, (ATT_ROWS - 1) / c.group + 1, 0, 0};
    if (const hipError_t e = launch_paged_index(c, &cut, 1, index, s)) return e;
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
