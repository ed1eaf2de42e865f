// paged.hpp -- what the paged-cache kernels share: the cache's layout, the
// requests of a call, and how a call's work is cut into items.
//
// The cache is two f16 arrays of pages:
//   k [pages][kv_heads][page][head_dim]
//   v [pages][kv_heads][head_dim][page]
// V is kept with a page's tokens innermost: the second product of attention
// contracts over tokens, and a matrix instruction's operand holds 8
// consecutive contraction elements a lane, so both products load their operands
// as 16-byte pieces of the cache with no transpose on the way.  Every 8 tokens
// that start at a multiple of 8 lie in one page (pages are powers of two from
// 16).
//
// A call has `requests` requests over `tokens` rows of q: request b owns rows
// q_start[b] .. q_start[b + 1), its last row is at position seq_lens[b] - 1, and
// position p is in page tables[b][p / page].  The `group` query heads of a
// key head and the tokens of a request form one axis of rows, (token, head in
// group), so that one pass over a key head's cache serves them all.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lloom {

constexpr int PAGED_MAX_REQUESTS = 4096;

// A call's arguments as the kernels see them.
struct PagedCall {
    const void* q;
    const uint16_t *k, *v;
    void* out;
    const int *q_start, *seq_lens, *tables;
    int* flags;  // sticky page error
    int64_t q_stride, table_stride;
    int tokens, requests, kv_heads, group, pages, page_shift, max_blocks;
    int window, sinks;
    float scale;  // log2(e) * the caller's
};

// How a kernel cuts its requests: `rows` rows of a request and `unit` keys at a
// time, at least `unit_min` units an item, and about `target` items in all.
// route: 0 every request, 1 those of at most `few` rows, 2 the others.
struct PagedCut {
    int rows, unit, unit_min, target, route, few, split;
};

// The keys that rows at positions lo .. hi see: [first, hi] and the first
// `sink` tokens before it, as steps of `step` keys.  Step i of the list is
// step i of the cache while i < sink_steps, then step skip + i.
struct PagedSpan {
    int first, sink_steps, skip, steps;
};
__host__ __device__ inline PagedSpan paged_span(int lo, int hi, int window, int sinks, int step) {
    PagedSpan s;
    s.first = window > 0 && lo >= window ? lo - window + 1 : 0;
    const int sink = sinks < s.first ? sinks : s.first;
    const int fs = s.first / step;
    s.sink_steps = (sink + step - 1) / step;
    if (s.sink_steps > fs) s.sink_steps = fs;
    s.skip = fs - s.sink_steps;
    s.steps = hi < 0 ? 0 : hi / step + 1 - s.skip;
    if (s.steps < s.sink_steps) s.steps = s.sink_steps;  // a window past the last key that there is
    return s;
}

// The most units of keys that a tile of `rows` rows of a request sees.
__host__ __device__ inline int paged_units(int T, int L, const PagedCut& c, int group, int window, int sinks) {
    const int full = L > 0 ? (L + c.unit - 1) / c.unit : 1;
    if (window <= 0) return full;
    const int more = (c.rows - 1) / group + 1;  // a tile's last token is at most this far past its first
    const int64_t keys = (int64_t)window + (T - 1 < more ? T - 1 : more);
    // a list of steps may start and end inside one: counted in units, one more for each end
    const int64_t most = (keys + c.unit - 1) / c.unit + 1 + (sinks + c.unit - 1) / c.unit;
    return most < full ? (int)most : full;
}

#if defined(__HIPCC__)

// One item: rows row0 .. of request b, split `split` of `splits` of its keys.
struct PagedItem {
    int b, T, L, start, tile, split, splits, chunk;  // chunk: units a split
    int group_index;                                 // this (request, tile) among the call's
    bool found;
};

__device__ __forceinline__ void paged_request(const PagedCall& c, int b, int* start, int* T, int* L) {
    int s = c.q_start[b], e = c.q_start[b + 1];
    s = min(max(s, 0), c.tokens);
    e = min(max(e, s), c.tokens);
    *start = s;
    *T = e - s;
    *L = max(c.seq_lens[b], 0);
}
// The last key that a table has a place for.
__device__ __forceinline__ int paged_key_cap(const PagedCall& c) {
    return (int)min(((int64_t)c.max_blocks << c.page_shift) - 1, (int64_t)0x7fffffff);
}

__device__ __forceinline__ int paged_scan(int v) {  // inclusive over the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d, 64);
        if ((int)__lane_id() >= d) v += o;
    }
    return v;
}

// Item `want` (or, by_group, the first item of tile `want`) of the call, found
// by every wave on its own: the lengths are known on the GPU alone, and a wave
// of requests costs two scans.  No LDS, no barrier.
template <bool BY_GROUP>
__device__ __forceinline__ PagedItem paged_find(const PagedCall& c, const PagedCut& cut, int want) {
    const int lane = __lane_id(), cap = paged_key_cap(c);
    PagedItem it;
    it.found = false;
    // chunk: the units a split takes
    int chunk = 0x7fffffff;
    if (cut.split) {
        unsigned long long total = 0;
        for (int b0 = 0; b0 < c.requests; b0 += 64) {
            const int b = b0 + lane;
            if (b < c.requests) {
                int s, T, L;
                paged_request(c, b, &s, &T, &L);
                const int rows = T * c.group;
                if (T > 0 && (cut.route == 0 || (rows <= cut.few) == (cut.route == 1)))
                    total += (unsigned long long)((rows + cut.rows - 1) / cut.rows) *
                             paged_units(T, min(L - 1, cap) + 1, cut, c.group, c.window, c.sinks);
            }
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d, 64);
        const unsigned long long per = (total * c.kv_heads + cut.target - 1) / cut.target;
        chunk = (int)min(per > (unsigned)cut.unit_min ? per : (unsigned long long)cut.unit_min, 0x7fffffffull);
    }
    // every field is the same in all lanes: readfirstlane keeps them scalar
    it.b = it.T = it.L = it.start = it.tile = it.split = it.splits = it.group_index = 0;
    it.chunk = __builtin_amdgcn_readfirstlane(chunk);
    int items_before = 0, tiles_before = 0;
    for (int b0 = 0; b0 < c.requests && !it.found; b0 += 64) {
        const int b = b0 + lane;
        int s = 0, T = 0, L = 0, tiles = 0, splits = 1;
        if (b < c.requests) {
            paged_request(c, b, &s, &T, &L);
            const int rows = T * c.group;
            if (T > 0 && (cut.route == 0 || (rows <= cut.few) == (cut.route == 1))) {
                tiles = (rows + cut.rows - 1) / cut.rows;
                const int u = paged_units(T, min(L - 1, cap) + 1, cut, c.group, c.window, c.sinks);
                splits = u <= chunk ? 1 : (u + chunk - 1) / chunk;
            }
        }
        const int items = tiles * splits;
        const int ie = items_before + paged_scan(items), te = tiles_before + paged_scan(tiles);
        const bool mine = BY_GROUP ? (want < te && want >= te - tiles) : (want < ie && want >= ie - items);
        const unsigned long long hit = __ballot(mine);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            it.found = true;
            it.b = b0 + src;
            it.start = __builtin_amdgcn_readlane(s, src);
            it.T = __builtin_amdgcn_readlane(T, src);
            it.L = __builtin_amdgcn_readlane(L, src);
            it.splits = __builtin_amdgcn_readlane(splits, src);
            const int ib = __builtin_amdgcn_readlane(ie - items, src), tb = __builtin_amdgcn_readlane(te - tiles, src);
            if (BY_GROUP) {
                it.tile = want - tb;
                it.split = ib + it.tile * it.splits;  // its first item's index
                it.group_index = want;
            } else {
                it.tile = (want - ib) / it.splits;
                it.split = (want - ib) - it.tile * it.splits;
                it.group_index = tb + it.tile;
            }
        }
        items_before = __builtin_amdgcn_readlane(ie, 63);
        tiles_before = __builtin_amdgcn_readlane(te, 63);
    }
    return it;
}

// Rows of q that no request owns are zero.
template <bool F32>
__device__ __forceinline__ void paged_zero_tail(const PagedCall& c, int dim, int wg, int wgs) {
    const int end = min(max(c.q_start[c.requests], 0), c.tokens);
    const int per = c.kv_heads * c.group * dim;
    for (int n = end + wg; n < c.tokens; n += wgs)
        for (int i = threadIdx.x; i < per; i += blockDim.x) {
            if (F32) ((float*)c.out)[(int64_t)n * per + i] = 0.0f;
            else ((uint16_t*)c.out)[(int64_t)n * per + i] = 0;
        }
}

#endif

}  // namespace lloom
