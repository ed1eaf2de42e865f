// paged_launch.hpp -- launches of the paged cache's kernels, for its entry points
// (paged_api.hip).  Apart from kernels.hpp: the other kernels' sources, and what was
// measured on them, do not change with these.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lloom {

// paged.hip: block tables and slots of a step's tokens; rows into the pages.
hipError_t launch_paged_plan(const int* cached, const int* fresh, int requests, int tokens, int* tables,
                             int64_t table_stride, int max_blocks, const int* free, int free_count, int page_shift,
                             int* q_start, int* seq_lens, int* positions, int64_t* slots, int* taken, int* flags,
                             hipStream_t s);
hipError_t launch_paged_append(int act, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                               const int64_t* slots, int tokens, void* kc, void* vc, int pages, int kv_heads, int dim,
                               int page_shift, int* flags, hipStream_t s);
// paged_attn.hip, paged_tile.hip: head dims that paged_dim_fits names.  A call's
// requests go to the one kernel or the other by their rows (paged.hpp); no request
// has over max_new new tokens where that is not 0 (results do not depend on it).
constexpr bool paged_dim_fits(int64_t d) { return d == 64 || d == 96 || d == 128 || d == 256; }
// With over 64 requests a launch before sums what they are cut into (c.index).
struct PagedCall;
struct PagedCut;
hipError_t launch_paged_clear(int* joins, hipStream_t s);
size_t paged_index_workspace_bytes(int64_t requests);
hipError_t launch_paged_index(PagedCall& c, const PagedCut* cuts, int count, int* to, hipStream_t s);
hipError_t launch_paged_rows(int act, int dim, PagedCall c, int* index, void* ws, hipStream_t s);
size_t paged_rows_workspace_bytes(int kv_heads, int dim);
hipError_t launch_paged_tiles(int act, int dim, const PagedCall& c, int* index, void* tile_ws, void* row_ws, hipStream_t s);
size_t paged_tiles_workspace_bytes(int kv_heads, int dim);
size_t paged_attention_workspace_bytes(int64_t tokens, int64_t requests, int kv_heads, int group, int dim,
                                       int max_new);
hipError_t launch_paged_attention(int act, int dim, const PagedCall& c, int max_new, void* ws, hipStream_t s);

}  // namespace lloom
