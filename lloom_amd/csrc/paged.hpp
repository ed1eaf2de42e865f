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
constexpr int PAGED_JOINS = 2048;

// A call's arguments as the kernels see them.
struct PagedCall {
    const void* q;
    const uint16_t *k, *v;
    void* out;
    const int *q_start, *seq_lens, *tables;
    int* flags;  // sticky page error
    int* joins;  // PAGED_JOINS counters, zero between calls
    int64_t q_stride, table_stride;
    int tokens, requests, kv_heads, group, pages, page_shift, max_blocks;
    int window, sinks;
    float scale;  // log2(e) * the caller's
    uint32_t group_magic;  // 2^32 / group, rounded up (0 for a group of one)
};

// How a kernel cuts its requests: 2^row_shift rows of a request and 2^unit_shift
// keys at a time, at least `unit_min` units an item, and about 2^target_shift
// items in all.  A tile's last token is at most `more` past its first.
// route: 0 every request, 1 those of at most `few` rows, 2 the others.
struct PagedCut {
    int row_shift, unit_shift, unit_min, target_shift, more, route, few, split;
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

// The most units of keys that a tile of a request sees.
__host__ __device__ inline int paged_units(int T, int L, const PagedCut& c, int window, int sinks) {
    const int round = (1 << c.unit_shift) - 1;
    const int full = L > 0 ? (int)(((int64_t)L + round) >> c.unit_shift) : 1;
    if (window <= 0) return full;
    const int64_t keys = (int64_t)window + (T - 1 < c.more ? T - 1 : c.more);
    // a list of steps may start and end inside one: counted in units, one more for each end
    const int64_t most = ((keys + round) >> c.unit_shift) + 1 + (((int64_t)sinks + round) >> c.unit_shift);
    return most < full ? (int)most : full;
}

#if defined(__HIPCC__)

// One item: rows row0 .. of request b, split `split` of `splits` of its keys.
struct PagedItem {
    int b, T, L, start, tile, split, splits, chunk;  // chunk: units a split
    int first;                                       // the item of split 0
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

// n / group for n < 2^32 / group: the magic's error, under group / 2^32, times n
// stays under one.
__device__ __forceinline__ int paged_token(const PagedCall& c, int n) {
    return c.group_magic ? (int)__umulhi((uint32_t)n, c.group_magic) : n;
}

// Bits 0 .. 7: which of the keys key .. key + 7 are in [lo, hi] or under `sinks`
// and at most hi.
__device__ __forceinline__ uint32_t paged_seen8(int key, int lo, int hi, int sinks) {
    const auto under = [key](int end) { return (1u << min(max(end - key, 0), 8)) - 1u; };
    return under(hi + 1) & (~under(lo) | under(sinks));
}

__device__ __forceinline__ int paged_scan(int v) {  // inclusive over the wave
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d, 64);
        if ((int)__lane_id() >= d) v += o;
    }
    return v;
}

// A lane's request: its rows' tiles, and the units of keys of one.
struct PagedLane {
    int start, T, L, tiles, units;
};
__device__ __forceinline__ PagedLane paged_lane(const PagedCall& c, const PagedCut& cut, int cap, int b) {
    PagedLane r{0, 0, 0, 0, 0};
    if (b >= c.requests) return r;
    paged_request(c, b, &r.start, &r.T, &r.L);
    const int rows = r.T * c.group;
    if (r.T > 0 && (cut.route == 0 || (rows <= cut.few) == (cut.route == 1))) {
        r.tiles = (rows + (1 << cut.row_shift) - 1) >> cut.row_shift;
        r.units = paged_units(r.T, min(r.L - 1, cap) + 1, cut, c.window, c.sinks);
    }
    return r;
}

// Item `want` of the call, found by every wave on its own: the lengths are known
// on the GPU alone, and 64 requests cost two scans.  No LDS, no barrier.
__device__ __forceinline__ PagedItem paged_find(const PagedCall& c, const PagedCut& cut, int want) {
    const int lane = __lane_id(), cap = paged_key_cap(c);
    PagedLane at = paged_lane(c, cut, cap, lane);
    int chunk = 0x7fffffff;  // the units a split takes
    if (cut.split) {
        unsigned long long total = (unsigned long long)at.tiles * at.units;
        for (int b = 64; b < c.requests; b += 64) {
            const PagedLane more = paged_lane(c, cut, cap, b + lane);
            total += (unsigned long long)more.tiles * more.units;
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) total += __shfl_xor(total, d, 64);
        const unsigned long long per = (total * c.kv_heads + (1u << cut.target_shift) - 1) >> cut.target_shift;
        chunk = (int)min(per > (unsigned)cut.unit_min ? per : (unsigned long long)cut.unit_min, 0x7fffffffull);
    }
    // every field is the same in all lanes: readlane keeps them scalar
    PagedItem it;
    it.found = false;
    it.b = it.T = it.L = it.start = it.tile = it.split = it.splits = it.group_index = 0;
    it.chunk = __builtin_amdgcn_readfirstlane(chunk);
    int items_before = 0, tiles_before = 0;
    for (int b0 = 0; b0 < c.requests && !it.found; b0 += 64) {
        if (b0) at = paged_lane(c, cut, cap, b0 + lane);
        const int splits = at.units <= chunk ? 1 : (int)(((unsigned)at.units + (unsigned)chunk - 1) / (unsigned)chunk);
        const int items = at.tiles * splits;
        const int ie = items_before + paged_scan(items), te = tiles_before + paged_scan(at.tiles);
        const unsigned long long hit = __ballot(want < ie && want >= ie - items);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            it.found = true;
            it.b = b0 + src;
            it.start = __builtin_amdgcn_readlane(at.start, src);
            it.T = __builtin_amdgcn_readlane(at.T, src);
            it.L = __builtin_amdgcn_readlane(at.L, src);
            it.splits = __builtin_amdgcn_readlane(splits, src);
            it.first = __builtin_amdgcn_readlane(ie - items, src);
            it.tile = (want - it.first) / it.splits;
            it.first += it.tile * it.splits;
            it.split = want - it.first;
            it.group_index = __builtin_amdgcn_readlane(te - at.tiles, src) + it.tile;
        }
        items_before = __builtin_amdgcn_readlane(ie, 63);
        tiles_before = __builtin_amdgcn_readlane(te, 63);
    }
    return it;
}

// One workgroup's part of a (tile, key head) that several share is written: true
// in the one that comes last, which then sees the others' parts.  Its counter
// is zero before and after.
__device__ __forceinline__ bool paged_last(int* counter, int splits) {
    __shared__ int came;
    __syncthreads();
    if (threadIdx.x == 0) {
        came = __hip_atomic_fetch_add(counter, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        if (came == splits - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return came == splits - 1;
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
