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

#include <type_traits>

#include "kq_common.hpp"

namespace lloom {

constexpr int PAGED_MAX_REQUESTS = 4096;
constexpr int PAGED_JOINS = 2048;
// The least reference of a row that has seen a key: so a row's reference is -inf exactly
// where it has seen none, and its sums are zero there.  A row whose scores are all -inf
// or NaN has this reference, and sums that make it NaN.
constexpr float PAGED_LOWEST = -3.402823466e38f;

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
    // Over 64 requests: where a launch before (k_paged_index) left the splits' length
    // and every request's sums, of route 1 behind the others'; 64 requests fit a wave,
    // which finds them itself.
    const int* index;
};

// How a kernel cuts its requests: 2^row_shift rows of a request and 2^unit_shift
// keys at a time; a tile with more units of keys than a 2^target_shift-th of the
// call's, and than `unit_min`, is split among several items.  A tile's last token
// is at most `more` past its first.
// route: 0 every request, 1 those with few rows (paged_few), 2 the others.
struct PagedCut {
    int row_shift, unit_shift, unit_min, target_shift, more, route;
    int slots;  // workgroups that the card holds at once, two a CU; 0: not told
};
// integers of a cut: chunk, whether the call is refused, then from 16 on items and splits summed
constexpr int PAGED_INDEX = 16 + 2 * PAGED_MAX_REQUESTS;
// Whether a request is one of few rows, which are served 16 at a time, each 16
// reading its keys.  Measured with 16 requests of lengths up to 8191 (heads of 128, 4
// key heads of 4, f16), the kernel of few rows against that of many: 16 rows each
// 18 and 28 us, 64 22 and 37; two of 30000 tokens, 64 rows 53 and 86, 128 rows 93 and
// 173, 192 rows 233 and 125; eight of 900, 96 rows 16 and 30, 256 rows 34 and 36, 400
// rows 50 and 38; eight of 300, 128 rows 11 and 17, 256 rows 19.5 and 19.0.  In f32
// and with heads of 64 and 96 the first is ahead by more; with heads of 256 from 192
// rows on by none (0.8 to 0.9 of it the other).  Sixteen requests that all have 8191
// tokens are served better by the other from 32 rows on (77 and 62 us; 96 rows 122
// and 77; heads of 64 37 and 33, of 256 141 and 113): they fill the card with either.
constexpr int PAGED_FEW = 96, PAGED_FEW_SHORT = 256, PAGED_SHORT = 1024;
__host__ __device__ inline bool paged_few(int64_t rows, int64_t length) {
    return rows <= PAGED_FEW || (rows <= PAGED_FEW_SHORT && length <= PAGED_SHORT);
}

// A split tile has more units than a 2^target_shift-th of all, so that there are
// under 2^target_shift of them and under twice as many items of theirs; where
// shorter splits fit there are no more than `slots` items.
__host__ __device__ inline int paged_parts(int target_shift) { return 2 << target_shift; }

// The keys that rows at positions lo .. see, up to key hi: [first, hi] and the
// first `sink` tokens before it, as steps of `step` keys.  Step i of the list is
// step i of the cache while i < sink_steps, then step skip + i.
struct PagedSpan {
    int first, sink_steps, skip, steps;
};
__host__ __device__ inline PagedSpan paged_span(int lo, int hi, int window, int sinks, int step) {
    PagedSpan s;
    s.first = window > 0 && lo >= window ? lo - window + 1 : 0;
    // no keys past hi, where a length passes its table
    const int keys = hi < 0 ? 0 : hi + 1, before = keys < s.first ? keys : s.first, sink = sinks < before ? sinks : before;
    const int fs = s.first / step;
    s.sink_steps = sink / step + (sink % step != 0);
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

// The most items a call has: its tiles, and the splits of the longest ones, of
// which there are no more than the tables have units of keys for.
inline int64_t paged_items_most(const PagedCall& c, const PagedCut& cut) {
    const int64_t rows = (int64_t)1 << cut.row_shift, some = c.requests < c.tokens ? c.requests : c.tokens;
    int64_t tiles = ((int64_t)c.tokens * c.group >> cut.row_shift) + some;
    if (cut.route == 1 && tiles > some * (PAGED_FEW_SHORT / rows)) tiles = some * (PAGED_FEW_SHORT / rows);
    tiles *= c.kv_heads;
    const int64_t keys = (int64_t)c.max_blocks << c.page_shift, units = (keys + (1 << cut.unit_shift) - 1) >> cut.unit_shift;
    int64_t all = tiles + ((int64_t)1 << cut.target_shift);
    if (all < cut.slots) all = cut.slots;  // where shorter splits fit
    return units < all && units * tiles < all ? units * tiles : all;
}

#if defined(__HIPCC__)

// One item: rows of tile `tile` of request b, split `split` of `splits` of its keys.
struct PagedItem {
    int b, T, L, start, tile, split, splits;
    int part;   // split 0's number among the items of split tiles
    int joint;  // the tile's number among them
    bool found;
    bool refused;  // q_start falls or is negative: the call has no items
};

// False where its rows' ends are in no order: rows that two requests own were cut
// into more items than the grid is sized for, and a split that no workgroup serves
// would never be counted.  Rows past the call's are left out, as if the request ended
// with the last one that there is.
__device__ __forceinline__ bool paged_request(const PagedCall& c, int b, int* start, int* T, int* L) {
    int s = c.q_start[b], e = c.q_start[b + 1];
    const bool order = s >= 0 && e >= s;
    const int past = order ? e - max(s, min(e, c.tokens)) : 0;
    s = min(max(s, 0), c.tokens);
    e = min(max(e, s), c.tokens);
    *start = s;
    *T = e - s;
    *L = max(c.seq_lens[b], 0) - past;
    return order;
}
// The last key that a table has a place for; two steps of keys past it are in 32 bits too.
__device__ __forceinline__ int paged_key_cap(const PagedCall& c) {
    return (int)min(((int64_t)c.max_blocks << c.page_shift) - 1, (int64_t)0x7fffffff - 128);
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

// Inclusive sums over the wave, in 6 DPP additions (shuffles: 6 passes through LDS).
template <class T>
__device__ __forceinline__ T paged_scan(T v) {
    const auto from = [](T x, auto ctrl, auto rows) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
    };
    using std::integral_constant;
    using All = integral_constant<int, 0xf>;
    v += from(v, integral_constant<int, 0x111>(), All());  // row_shr:1
    v += from(v, integral_constant<int, 0x112>(), All());
    v += from(v, integral_constant<int, 0x114>(), All());
    v += from(v, integral_constant<int, 0x118>(), All());
    v += from(v, integral_constant<int, 0x142>(), integral_constant<int, 0xa>());  // row_bcast:15
    v += from(v, integral_constant<int, 0x143>(), integral_constant<int, 0xc>());  // row_bcast:31
    return v;
}
__device__ __forceinline__ int paged_sum(int v) { return __builtin_amdgcn_readlane(paged_scan(v), 63); }

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ half8_t as_half8(uint4 v) { return __builtin_bit_cast(half8_t, v); }

// x as hi + lo, two halves: exact to 2^-22 of x where x is in half's normal range.
__device__ __forceinline__ void split8(const float (&x)[8], half8_t& hi, half8_t& lo) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const _Float16 h = (_Float16)x[i];
        hi[i] = h;
        lo[i] = (_Float16)(x[i] - (float)h);
    }
}

// Queries are scaled so that a row's largest is in 2^Q_SHIFT * [1, 2): halves then
// hold the others exactly to 2^-22 of them or 2^-38 of the largest.
constexpr int Q_SHIFT = 14;
// Keys may be infinite: lo has x's sign and is not zero, or the two products would be
// infinities of both signs, or NaN.  hi is x towards zero for that, and lo half's least
// number more than the rest, 2^-38 of the row's largest.
__device__ __forceinline__ void split8_query(const float (&x)[8], half8_t& hi, half8_t& lo) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const auto h = __builtin_amdgcn_cvt_pkrtz(x[i], x[i + 1]);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            hi[i + j] = (_Float16)h[j];
            lo[i + j] = (_Float16)(x[i + j] - (float)h[j] + __builtin_copysignf(0x1p-24f, x[i + j]));
        }
    }
}

// Bit j: an infinity or a NaN at key j of 8 keys' values.  An exponent of all ones and
// 1 more is the sign's bit.
__device__ __forceinline__ uint32_t odd_keys(uint4 v) {
    uint32_t odd = 0;
    const uint32_t* w = (const uint32_t*)&v;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t at = ((w[j] & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
        odd |= (at >> 15 & 1) << (2 * j) | (at >> 31) << (2 * j + 1);
    }
    return odd;
}
// Zeroes the values of the keys whose bit is not set.
__device__ __forceinline__ void keep8(uint4& v, uint32_t bits) {
    uint32_t* w = (uint32_t*)&v;
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] &= (bits >> (2 * j) & 1) * 0xffffu | (bits >> (2 * j + 1) & 1) * 0xffff0000u;
}

// A lane's request: its rows' tiles, and the units of keys of one.
struct PagedLane {
    int start, T, L, tiles, units;
    bool order;
};
__device__ __forceinline__ PagedLane paged_lane(const PagedCall& c, const PagedCut& cut, int cap, int b) {
    PagedLane r{0, 0, 0, 0, 0, true};
    if (b >= c.requests) return r;
    r.order = paged_request(c, b, &r.start, &r.T, &r.L);
    const int rows = r.T * c.group;
    if (r.T > 0 && (cut.route == 0 || paged_few(rows, r.L) == (cut.route == 1))) {
        r.tiles = (rows + (1 << cut.row_shift) - 1) >> cut.row_shift;
        r.units = paged_units(r.T, min(r.L - 1, cap) + 1, cut, c.window, c.sinks);
    }
    return r;
}

template <bool F32>
__device__ __forceinline__ void paged_store4(void* out, int64_t at, float x, float y, float z, float w) {
    if constexpr (F32) {
        *(float4*)((float*)out + at) = make_float4(x, y, z, w);
    } else {
        *(uint2*)((uint16_t*)out + at) = make_uint2(f32_to_f16(x) | (uint32_t)f32_to_f16(y) << 16,
                                                    f32_to_f16(z) | (uint32_t)f32_to_f16(w) << 16);
    }
}

// What the requests of a wave's lanes are cut into: items, and items and tiles of
// split tiles.
struct PagedCount {
    int splits, items, split;
};
__device__ __forceinline__ PagedCount paged_count(const PagedLane& at, int chunk) {
    PagedCount n;
    n.splits = at.units <= chunk ? 1 : (int)(((unsigned)at.units + (unsigned)chunk - 1) / (unsigned)chunk);
    n.items = at.tiles * n.splits;
    n.split = n.splits > 1 ? n.items << 16 | at.tiles : 0;
    return n;
}
// The units a split takes, from all requests' tiles x units: in f32, which is exact
// under 2^24, and rounded up from there.
__device__ __forceinline__ int paged_chunk(const PagedCall& c, const PagedCut& cut, float total) {
    total *= c.kv_heads;
    if (total >= 16777216.0f) total *= 1.0f + 1.0f / 65536;
    return max((int)__builtin_fminf(__builtin_ceilf(__builtin_ldexpf(total, -cut.target_shift)), 1e9f), cut.unit_min);
}

// Item `want` of the call, found by every wave on its own: the lengths are known
// on the GPU alone.  No LDS, no barrier.
__device__ __forceinline__ PagedItem paged_find(const PagedCall& c, const PagedCut& cut, int want) {
    const int lane = __lane_id(), cap = paged_key_cap(c);
    PagedItem it;
    it.found = it.refused = false;
    it.b = it.T = it.L = it.start = it.tile = it.split = it.splits = it.part = it.joint = 0;
    int b0 = 0, ie = 0, se = 0, chunk = 0;  // the lanes' first request; their sums
    if (c.index) {
        const int* index = c.index + (cut.route == 1 ? PAGED_INDEX : 0);
        const int *sums = index + 16, last = c.requests - 1;
        const int end = 64 * lane <= last ? sums[min(64 * lane + 63, last)] : 0x7fffffff;
        const unsigned long long past = __ballot(want < end && end != 0x7fffffff);
        b0 = past ? 64 * __builtin_ctzll(past) : c.requests;
        chunk = index[0];
        ie = sums[min(b0 + lane, last)];
        se = sums[PAGED_MAX_REQUESTS + min(b0 + lane, last)];
    }
    // the one place of both ways: with two, the f32 tiles spilled 8 registers and not 5
    // (128.1 against 125.8 us for 50 GFLOP)
    const PagedLane at = paged_lane(c, cut, cap, b0 + lane);
    it.refused = c.index ? c.index[1] != 0 : __any(!at.order);
    if (it.refused) return it;
    if (!c.index) {
        const float total = paged_scan((float)at.tiles * at.units);
        chunk = paged_chunk(c, cut, __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, total), 63)));
        // Shorter ones, down to half of that, if every item still starts at once: a second
        // round of a few items takes as long as the first.
        if (cut.slots && paged_sum(at.tiles) * c.kv_heads < cut.slots) {
            int less = max((chunk + 1) / 2, cut.unit_min);
            while (less < chunk) {
                const int items = paged_sum(at.tiles * (int)(((unsigned)at.units + less - 1) / (unsigned)less)) * c.kv_heads;
                if (items <= cut.slots) break;
                less += max(less / 8, (int)((int64_t)less * (items - cut.slots) / cut.slots)) + 1;
            }
            chunk = min(chunk, less);
        }
    }
    const PagedCount n = paged_count(at, __builtin_amdgcn_readfirstlane(chunk));
    if (!c.index) {
        ie = paged_scan(n.items);
        se = paged_scan(n.split);
        if (cut.slots) {
            // Two workgroups a CU, and the longest items come first: the second ones in
            // turn, so that the longest of them is not with the longest of the first.
            const int all = __builtin_amdgcn_readlane(ie, 63), first = (cut.slots / 2) / c.kv_heads;
            if (all * c.kv_heads <= cut.slots && want >= first && want < all) want = first + all - 1 - want;
        }
    }
    const unsigned long long hit = __ballot(want < ie && want >= ie - n.items);
    if (hit) {
        // every field is the same in all lanes: readlane keeps them scalar
        const int src = __builtin_ctzll(hit);
        it.found = true;
        it.b = b0 + src;
        it.start = __builtin_amdgcn_readlane(at.start, src);
        it.T = __builtin_amdgcn_readlane(at.T, src);
        it.L = __builtin_amdgcn_readlane(at.L, src);
        it.splits = __builtin_amdgcn_readlane(n.splits, src);
        const int in = want - __builtin_amdgcn_readlane(ie - n.items, src), tile = it.splits == 1 ? in : in < it.splits ? 0 : in / it.splits;
        const int before = __builtin_amdgcn_readlane(se - n.split, src);
        it.split = in - tile * it.splits;
        it.part = (before >> 16) + tile * it.splits;
        it.joint = (before & 0xffff) + tile;
        // the last tokens, which see the most, first
        it.tile = __builtin_amdgcn_readlane(at.tiles, src) - 1 - tile;
    }
    return it;
}

// The parts of a tile that several workgroups share are stored and loaded at the
// agent's scope: past the L2, which each XCD has one of.  A release of ordinary
// stores writes the whole L2 back instead (537 MB of one request's cache 106 us that
// way, 100 this).
__device__ __forceinline__ void part_store(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void part_store4(float* p, float x, float y, float z, float w) {
    uint64_t* q = (uint64_t*)p;
    const auto two = [](float a, float b) { return (uint64_t)__builtin_bit_cast(uint32_t, b) << 32 | __builtin_bit_cast(uint32_t, a); };
    __hip_atomic_store(q, two(x, y), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(q + 1, two(z, w), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float part_load(const float* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float4 part_load4(const float* p) {
    const uint64_t a = __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint64_t b = __hip_atomic_load((const uint64_t*)p + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float4(__builtin_bit_cast(float, (uint32_t)a), __builtin_bit_cast(float, (uint32_t)(a >> 32)),
                       __builtin_bit_cast(float, (uint32_t)b), __builtin_bit_cast(float, (uint32_t)(b >> 32)));
}

// A workgroup's part is stored: true in the last of them to come, which then loads
// the others'.  Every wave waits until its stores are done before any of them is
// counted.  The counter is zero before and after.
__device__ __forceinline__ bool paged_last(int* counter, int splits) {
    __shared__ int came;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        came = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (came == splits - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    asm volatile("" ::: "memory");
    return came == splits - 1;
}

// The last of a tile's splits joins their parts, each m [ROWS], l [ROWS] and
// o [ROWS][D] at the reference m: a thread takes 4 dimensions of QN rows in every
// `slices`-th split, QN x SN loads in flight, then the slices are joined in their
// order.  `lds`: 24 bytes a thread.
template <int D, bool F32, int ROWS, int THREADS, int QN, int SN, class Place>
__device__ __forceinline__ void paged_join(const float* all, int64_t apart, int splits, int nrows, void* lds, void* out,
                                           Place place) {
    float4* sum4 = (float4*)lds;
    float2* stat2 = (float2*)(sum4 + THREADS);
    const int quads = nrows * (D / 4), slices = max(min(THREADS / quads, splits), 1);
    for (int q0 = 0; q0 < quads; q0 += QN * THREADS) {
        const int slice = slices > 1 ? threadIdx.x / quads : 0, e0 = slices > 1 ? threadIdx.x % quads : q0 + threadIdx.x;
        const bool on = slice < slices && e0 < quads;
        float4 a[QN];
        float top[QN], sum[QN];
#pragma unroll
        for (int i = 0; i < QN; i++) a[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f), top[i] = -INFINITY, sum[i] = 0.0f;
        for (int s0 = slice; on && s0 < splits; s0 += SN * slices) {
            float ms[QN][SN], ls[QN][SN];
            float4 vs[QN][SN];
#pragma unroll
            for (int i = 0; i < QN; i++)
#pragma unroll
                for (int j = 0; j < SN; j++) {
                    const int e = min(e0 + i * THREADS, quads - 1), rr = e / (D / 4);
                    const float* p = all + min(s0 + j * slices, splits - 1) * apart;
                    ms[i][j] = part_load(p + rr);
                    ls[i][j] = part_load(p + ROWS + rr);
                    vs[i][j] = part_load4(p + 2 * ROWS + 4 * e);
                }
#pragma unroll
            for (int i = 0; i < QN; i++) {
                float now = top[i];
#pragma unroll
                for (int j = 0; j < SN; j++) {
                    if (s0 + j * slices >= splits) ms[i][j] = -INFINITY;
                    now = __builtin_fmaxf(now, ms[i][j]);
                }
                const float base = now == -INFINITY ? 0.0f : now, less = __builtin_amdgcn_exp2f(top[i] - base);
                top[i] = now;
                a[i].x *= less, a[i].y *= less, a[i].z *= less, a[i].w *= less, sum[i] *= less;
#pragma unroll
                for (int j = 0; j < SN; j++) {
                    if (ms[i][j] == -INFINITY) continue;  // saw no key, or is no split
                    const float w = __builtin_amdgcn_exp2f(ms[i][j] - base);
                    a[i].x += w * vs[i][j].x, a[i].y += w * vs[i][j].y, a[i].z += w * vs[i][j].z, a[i].w += w * vs[i][j].w;
                    sum[i] += w * ls[i][j];
                }
            }
        }
        if (slices > 1) {  // then one quad a thread
            __syncthreads();
            sum4[threadIdx.x] = a[0];
            stat2[threadIdx.x] = make_float2(top[0], sum[0]);
            __syncthreads();
            if (threadIdx.x >= quads) continue;
            for (int i = 1; i < slices; i++) top[0] = __builtin_fmaxf(top[0], stat2[i * quads + e0].x);
            const float base = top[0] == -INFINITY ? 0.0f : top[0];
            a[0] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            sum[0] = 0.0f;
            for (int i = 0; i < slices; i++) {
                const float2 st = stat2[i * quads + e0];
                const float4 v = sum4[i * quads + e0];
                const float w = __builtin_amdgcn_exp2f(st.x - base);
                a[0].x += w * v.x, a[0].y += w * v.y, a[0].z += w * v.z, a[0].w += w * v.w, sum[0] += w * st.y;
            }
        }
#pragma unroll
        for (int i = 0; i < QN; i++) {
            const int e = e0 + i * THREADS;
            if (!on || e >= quads) continue;
            const float inv = 1.0f / sum[i];
            const bool none = top[i] == -INFINITY;
            paged_store4<F32>(out, place(e / (D / 4)) + 4 * (e % (D / 4)), none ? 0.0f : a[i].x * inv, none ? 0.0f : a[i].y * inv,
                              none ? 0.0f : a[i].z * inv, none ? 0.0f : a[i].w * inv);
        }
    }
}

// Rows of out that no request owns are zero: those before the first's and past the last's,
// and all of a refused call's.  Reports that, and requests with rows past the call's.
template <bool F32>
__device__ __forceinline__ void paged_zero_rest(const PagedCall& c, int dim, int wg, int wgs, int first, int last, bool refused) {
    if ((refused || last > c.tokens) && wg == 0 && threadIdx.x == 0) c.flags[0] = 1;
    if (refused) first = last = c.tokens;
    const int head = min(max(first, 0), c.tokens), end = min(max(last, head), c.tokens);
    const int per = c.kv_heads * c.group * dim, rest = c.tokens - (end - head);
    for (int n = wg; n < rest; n += wgs) {
        const int64_t row = n < head ? n : n + (end - head);
        for (int i = threadIdx.x; i < per; i += blockDim.x) {
            if (F32) ((float*)c.out)[row * per + i] = 0.0f;
            else ((uint16_t*)c.out)[row * per + i] = 0;
        }
    }
}

#endif

}  // namespace lloom
