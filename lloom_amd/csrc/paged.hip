// paged.hip -- block tables and slot maps from request lengths, and the
// writes of new k and v rows into the pages of the cache (paged.hpp).
#include "paged_launch.hpp"
#include "kq_common.hpp"
#include "paged.hpp"

namespace lloom {

// ------------------------------------------------------------------ plan --
// With c = cached, n = new tokens and P = page:
//   q_start = exclusive sum of n,  seq = c + n,  held = ceil(c / P),
//   taken = ceil(seq / P) - held,  off = exclusive sum of taken.
// Token t of request b is at pos = c + t; its page is tables[b][pos / P] where
// pos / P < held, else free[off + pos / P - held], which the page's first
// token (pos % P = 0) stores in the table.  No token waits for another's
// store, so one launch does it all: every workgroup sums the lengths itself
// (4 KB for 512 requests, from the L2) and then serves its own tokens.  A launch and
// three loads in a row: 4.0 us for 64 requests, 4.6 for 224 with 12000 tokens.
constexpr int PLAN_WG = 256;

// Exclusive scan over the workgroup of one 64-bit value a thread; *total its sum.
__device__ __forceinline__ int64_t wg_scan(int64_t v, int64_t* part, int64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(s, d, 64);
        if (lane >= d) s += o;
    }
    if (lane == 63) part[wave] = s;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < PLAN_WG / 64; w++) {
        before += w < wave ? part[w] : 0;
        all += part[w];
    }
    __syncthreads();
    *total = all;
    return before + s - v;
}

struct PlanArgs {
    const int *cached, *fresh, *free;
    int *tables, *q_start, *seq_lens, *positions, *taken;
    int64_t* slots;
    int* flags;
    int64_t table_stride;
    int requests, tokens, max_blocks, free_count, page_shift;
};

__device__ __forceinline__ int sat31(int64_t v) { return (int)min(v, (int64_t)0x7fffffff); }

__global__ __launch_bounds__(PLAN_WG) void k_paged_plan(PlanArgs a) {
    extern __shared__ int lds[];  // starts [requests], off [requests]
    __shared__ int64_t part[PLAN_WG / 64];
    int *starts = lds, *offs = lds + a.requests;
    const int tid = threadIdx.x, page = 1 << a.page_shift;
    const int per = (a.requests + PLAN_WG - 1) / PLAN_WG, b0 = tid * per, b1 = min(b0 + per, a.requests);
    bool bad = false;
    int64_t sum_n = 0, sum_t = 0;
    for (int b = b0; b < b1; b++) {
        const int64_t c = max(a.cached[b], 0), n = max(a.fresh[b], 0);
        bad |= a.cached[b] < 0 || a.fresh[b] < 0 || c + n > ((int64_t)a.max_blocks << a.page_shift);
        sum_n += n;
        sum_t += ((c + n + page - 1) >> a.page_shift) - ((c + page - 1) >> a.page_shift);
    }
    int64_t all_n, all_t;
    int64_t at_n = wg_scan(sum_n, part, &all_n), at_t = wg_scan(sum_t, part, &all_t);
    for (int b = b0; b < b1; b++) {
        const int64_t c = max(a.cached[b], 0), n = max(a.fresh[b], 0);
        starts[b] = sat31(at_n);
        offs[b] = sat31(at_t);
        if (blockIdx.x == 0) {
            a.q_start[b] = sat31(at_n);
            a.seq_lens[b] = sat31(c + n);
        }
        at_n += n;
        at_t += ((c + n + page - 1) >> a.page_shift) - ((c + page - 1) >> a.page_shift);
    }
    if (blockIdx.x == 0) {
        if (tid == 0) {
            a.q_start[a.requests] = sat31(all_n);
            a.taken[0] = sat31(all_t);
            bad |= all_n > a.tokens || all_t > a.free_count;
        }
        if (bad) a.flags[0] = 1;
    }
    __syncthreads();
    const int n = blockIdx.x * PLAN_WG + tid;
    if (n >= a.tokens) return;
    if (n >= all_n) {  // a padded batch's rows
        a.positions[n] = 0;
        a.slots[n] = -1;
        return;
    }
    // the last request that starts at or before n
    int lo = 0, hi = a.requests - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (starts[mid] <= n) lo = mid;
        else hi = mid - 1;
    }
    const int64_t c = max(a.cached[lo], 0), pos = c + n - starts[lo];
    const int64_t blk = pos >> a.page_shift, held = (c + page - 1) >> a.page_shift;
    int pg = -1;
    if (blk < a.max_blocks) {
        int* entry = a.tables + lo * a.table_stride + blk;
        if (blk < held) {
            pg = *entry;
        } else {
            const int64_t f = offs[lo] + blk - held;
            if (f < a.free_count) pg = a.free[f];
            if ((pos & (page - 1)) == 0) *entry = pg;  // -1 where no page is left: attention passes such a page over
        }
    }
    if (pg < 0) a.flags[0] = 1;
    a.positions[n] = sat31(pos);
    a.slots[n] = pg < 0 ? -1 : ((int64_t)pg << a.page_shift) + (pos & (page - 1));
}

hipError_t launch_paged_plan(const int* cached, const int* fresh, int requests, int tokens, int* tables,
                             int64_t table_stride, int max_blocks, const int* free, int free_count, int page_shift,
                             int* q_start, int* seq_lens, int* positions, int64_t* slots, int* taken, int* flags,
                             hipStream_t s) {
    PlanArgs a{cached, fresh, free, tables, q_start, seq_lens, positions, taken, slots, flags, table_stride,
               requests, tokens, max_blocks, free_count, page_shift};
    const int wgs = tokens > 0 ? (tokens + PLAN_WG - 1) / PLAN_WG : 1;
    hipLaunchKernelGGL(k_paged_plan, dim3(wgs), dim3(PLAN_WG), 2 * requests * sizeof(int), s, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------- append --
// A workgroup takes 64 tokens of one head (8 where there are few).  K rows are
// copied as they are.  V goes to the page's other order: a run of 8 tokens
// whose slots follow each other from a multiple of 8 is stored as one 16-byte
// piece a dimension, through LDS; the tokens that no run holds (a decode step's,
// or the ends of a prompt) as single halves.  8192 tokens of 8 x 128 in f16 (67 MB)
// take 16 us, 4.2 TB/s where a large copy reaches 4.9, in f32 (101 MB) 22, 4.5 TB/s; 64
// tokens 3.4, a launch.
struct AppendArgs {
    const void *k, *v;
    uint16_t *kc, *vc;
    const int64_t* slots;
    int* flags;
    int64_t k_stride, v_stride, slot_count;
    int tokens, kv_heads, dim, page_shift;
};

template <bool F32>
__device__ __forceinline__ uint4 half8(const void* p, int64_t i) {
    if constexpr (!F32) {
        return *(const uint4*)((const uint16_t*)p + i);
    } else {
        const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
        uint4 r;
        r.x = f32_to_f16(a.x) | (uint32_t)f32_to_f16(a.y) << 16;
        r.y = f32_to_f16(a.z) | (uint32_t)f32_to_f16(a.w) << 16;
        r.z = f32_to_f16(b.x) | (uint32_t)f32_to_f16(b.y) << 16;
        r.w = f32_to_f16(b.z) | (uint32_t)f32_to_f16(b.w) << 16;
        return r;
    }
}

template <bool F32, int TOK>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
    // rows of V as f16, a dword more than the row apart
    extern __shared__ uint32_t rows[];
    __shared__ int64_t slot[TOK];
    __shared__ unsigned long long runs[2];
    const int tid = threadIdx.x, n0 = blockIdx.x * TOK, h = blockIdx.y, pitch = a.dim / 2 + 1;
    const int page = 1 << a.page_shift;
    if (tid < 64) {
        int64_t s = -1;
        bool bad = false;
        if (tid < TOK && n0 + tid < a.tokens) {
            s = a.slots[n0 + tid];
            bad = s >= a.slot_count;
            if (bad) s = -1;
        }
        if (bad) a.flags[0] = 1;
        if (tid < TOK) slot[tid] = s;
        // lane i: tokens i .. i + 7 fill an aligned 16-byte piece
        const int64_t next = __shfl_down(s, 1, 64);
        const unsigned long long follow = __ballot(tid < 63 && s >= 0 && next == s + 1);
        unsigned long long r = follow & (follow >> 1);
        r &= r >> 2;
        r &= (follow >> 4) & (follow >> 5) & (follow >> 6);
        r &= __ballot(s >= 0 && (s & 7) == 0);
        unsigned long long held = r | (r << 1);
        held |= held << 2;
        held |= held << 4;
        if (tid == 0) {
            runs[0] = r;
            runs[1] = held;
        }
    }
    __syncthreads();
    const int pieces = a.dim / 8;
    for (int i = tid; i < TOK * pieces; i += 256) {
        const int t = i / pieces, p = i % pieces;
        const int64_t s = slot[t];
        if (s < 0) continue;
        const int64_t at = (int64_t)(n0 + t);
        const uint4 kv = half8<F32>(a.k, at * a.k_stride + h * a.dim + 8 * p);
        const uint4 vv = half8<F32>(a.v, at * a.v_stride + h * a.dim + 8 * p);
        const int64_t base = (((s >> a.page_shift) * a.kv_heads + h) * a.dim) << a.page_shift;
        *(uint4*)(a.kc + base + (s & (page - 1)) * a.dim + 8 * p) = kv;
        uint32_t* row = rows + t * pitch + 4 * p;
        row[0] = vv.x;
        row[1] = vv.y;
        row[2] = vv.z;
        row[3] = vv.w;
    }
    __syncthreads();
    const uint16_t* half = (const uint16_t*)rows;
    // runs: a lane a dimension, 16 bytes each
    for (unsigned long long r = runs[0]; r; r &= r - 1) {
        const int t = __builtin_ctzll(r);
        const int64_t s = slot[t];
        const int64_t base = ((((s >> a.page_shift) * a.kv_heads + h) * a.dim) << a.page_shift) + (s & (page - 1));
        for (int d = tid; d < a.dim; d += 256) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                w[j] = half[(t + 2 * j) * 2 * pitch + d] | (uint32_t)half[(t + 2 * j + 1) * 2 * pitch + d] << 16;
            *(uint4*)(a.vc + base + ((int64_t)d << a.page_shift)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    // the rest: a lane a token
    const unsigned long long held = runs[1];
    for (int i = tid; i < TOK * a.dim; i += 256) {
        const int t = i % TOK, d = i / TOK;
        const int64_t s = slot[t];
        if (s < 0 || (held >> t & 1)) continue;
        a.vc[((((s >> a.page_shift) * a.kv_heads + h) * a.dim + d) << a.page_shift) + (s & (page - 1))] =
            half[t * 2 * pitch + d];
    }
}

template <bool F32, int TOK>
static void append_as(const AppendArgs& a, hipStream_t s) {
    const size_t lds = (size_t)TOK * (a.dim / 2 + 1) * sizeof(uint32_t);
    hipLaunchKernelGGL((k_paged_append<F32, TOK>), dim3((a.tokens + TOK - 1) / TOK, a.kv_heads), dim3(256), lds, s, a);
}

hipError_t launch_paged_append(int act, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                               const int64_t* slots, int tokens, void* kc, void* vc, int pages, int kv_heads, int dim,
                               int page_shift, int* flags, hipStream_t s) {
    AppendArgs a{k, v, (uint16_t*)kc, (uint16_t*)vc, slots, flags, k_stride, v_stride, (int64_t)pages << page_shift,
                 tokens, kv_heads, dim, page_shift};
    // heads of 128 in f16, 8 tokens a workgroup against 64: 64 tokens of 8 heads 3.3 and
    // 6.9 us, 2048 7.5 and 8.6, 4096 11.9 and 10.7, 8192 21.4 and 16.6; f32 8.7 and 9.9,
    // 14.6 and 12.9, 26.0 and 21.3.  Heads of 64, 96 and 256 turn between the same two, in
    // both types (2048 and 4096 tokens of 64 in f16: 5.7 and 6.1, 8.7 and 7.3; of 256 in
    // f32: 14.4 and 15.2, 27.8 and 22.2).
    const bool few = (int64_t)tokens * kv_heads < 20480;
    if (act == T_F32) few ? append_as<true, 8>(a, s) : append_as<true, 64>(a, s);
    else few ? append_as<false, 8>(a, s) : append_as<false, 64>(a, s);
    return hipGetLastError();
}

}  // namespace lloom
