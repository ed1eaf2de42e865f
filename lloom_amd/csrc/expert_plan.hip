// expert_plan.hip -- planes (token, slot) in the order of their experts: a
// stable counting sort in one launch.
#include "fp8.hpp"

namespace lloom {

// A workgroup an expert (the last one's also has the planes of none, which follow
// its own: one workgroup more than CUs is 15 us for 10), and each for itself: a
// wave has a run of planes, counts in it those of smaller experts, and lists its
// own in LDS, a ballot ranking a row of 64; with the counts of all waves it knows
// where its own go.  No atomics, so the order is the planes' own, and nothing passes
// between workgroups; what it costs is that each reads all ids.  ROWS rows of 64
// are loaded at a time, the next ones under those in work.  A wave whose list is
// too short (over PLAN_LIST planes of one expert in its run) goes through its run
// again, a list at a time.  Rows without a plane of the expert are skipped: 800000
// planes 73 us, 77 without.  128 experts, 256 planes 2.8 us (a launch), 16384 5.2, 65536
// 9.9 (12.7 with a first time that only counts), 256 experts 9.8; 4096 experts, 16000
// planes 35.5.
constexpr int PLAN_LIST = 1024;

// Keys of a wave's next rows from plane p on: an id (CLAMP: `none` for one of no
// expert), -1 past the last.
template <bool CLAMP, int ROWS>
__device__ __forceinline__ void plan_keys(const int* __restrict__ ids, int p, int last, uint32_t none, uint32_t (&key)[ROWS]) {
    const int at = p + (int)__lane_id();
    if (p + 64 * ROWS <= last) {
#pragma unroll
        for (int i = 0; i < ROWS; i++) key[i] = CLAMP ? min((uint32_t)ids[at + 64 * i], none) : (uint32_t)ids[at + 64 * i];
    } else {
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            key[i] = at + 64 * i < last ? (uint32_t)ids[at + 64 * i] : ~0u;
            if (CLAMP && at + 64 * i < last) key[i] = min(key[i], none);
        }
    }
}

// Lists a wave's planes with key `mine` from rows of keys (the first of them plane
// `off` of the run), `found` of them being there.
template <int ROWS>
__device__ __forceinline__ void plan_list(const uint32_t (&key)[ROWS], uint32_t mine, int off, uint16_t* list, int& found) {
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const uint64_t m = __ballot(key[i] == mine);
        if (m == 0) continue;
        const int at = found + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        if (key[i] == mine && at < PLAN_LIST) list[at] = (uint16_t)(off + 64 * i + (int)__lane_id());
        found += __builtin_popcountll(m);
    }
}

template <int ROWS>
__global__ __launch_bounds__(1024) void k_expert_plan(const int* __restrict__ ids, int planes, uint64_t per_topk,
                                                      int experts, int* __restrict__ starts, int* __restrict__ sorted,
                                                      int* __restrict__ tokens, int* __restrict__ flags) {
    __shared__ int s_less[16], s_same[16];
    __shared__ uint16_t s_list[16][PLAN_LIST];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t mine = blockIdx.x, none = (uint32_t)experts;
    const int run = ((planes + waves - 1) / waves + 63) & ~63, first = min(planes, wave * run), last = min(planes, first + run);
    uint16_t* list = s_list[wave];
    int less = 0, same = 0;
    uint32_t key[ROWS], next[ROWS];
    plan_keys<false>(ids, first, last, none, key);
    for (int p = first; p < last; p += 64 * ROWS) {
        plan_keys<false>(ids, p + 64 * ROWS, last, none, next);
        plan_list(key, mine, p - first, list, same);
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            less += key[i] < mine;
            key[i] = next[i];
        }
    }
    less = __builtin_amdgcn_readlane(wave_scan(less), 63);
    if (lane == 0) s_less[wave] = less, s_same[wave] = same;
    __syncthreads();
    int at = 0, before = 0, all = 0, others = 0;  // planes: own ahead, of smaller experts, own, of none ahead
    for (int w = 0; w < waves; w++) {
        const int count = s_same[w], smaller = s_less[w];
        before += smaller;
        all += count;
        if (w < wave) at += count, others += run - count - smaller;  // the runs ahead are whole
    }
    if (threadIdx.x == 0) starts[mine] = before;
    at += before;
    bool bad = false;
    auto place = [&](int from, int count, uint32_t whose) {  // a wave's own list: its LDS operations are in order
        for (int i = lane; i < count; i += 64) {
            const int plane = from + list[i];
            sorted[at + i] = plane;
            tokens[at + i] = (int)((uint64_t)plane * per_topk >> 40);
            if (whose == none) bad |= ids[plane] >= experts;
        }
        at += count;
    };
    auto again = [&](uint32_t whose) {
        static_assert(64 * ROWS <= PLAN_LIST, "rows loaded at a time fit the list");
        for (int p = first; p < last; p += 64 * ROWS) {
            int found = 0;
            plan_keys<true>(ids, p, last, none, key);
            plan_list(key, whose, 0, list, found);
            place(p, found, whose);
        }
    };
    if (same <= PLAN_LIST && run <= 65536) place(first, same, mine);
    else again(mine);
    if (mine + 1 == none) {
        if (threadIdx.x == 0) starts[none] = before + all;
        if (before + all < planes) {
            at = before + all + min(others, planes);
            again(none);
        }
    }
    if (bad) flags[0] = 1;
}

hipError_t launch_expert_plan(const int* ids, int64_t planes, int topk, int experts, int* starts, int* sorted,
                              int* tokens, int* flags, hipStream_t s) {
    // planes < 2^24 and topk <= 2^12: the quotient by 2^40 / topk + 1 is exact
    const uint64_t per = (1ull << 40) / (uint32_t)topk + 1;
    const int p = (int)planes;
    if (planes <= 1024)
        k_expert_plan<4><<<experts, 256, 0, s>>>(ids, p, per, experts, starts, sorted, tokens, flags);
    else if (planes <= 4096)
        k_expert_plan<4><<<experts, 1024, 0, s>>>(ids, p, per, experts, starts, sorted, tokens, flags);
    else
        k_expert_plan<16><<<experts, 1024, 0, s>>>(ids, p, per, experts, starts, sorted, tokens, flags);
    return hipGetLastError();
}

}  // namespace lloom
