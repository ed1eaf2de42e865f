// expert_plan.hip -- planes (token, slot) in the order of their experts: a
// stable counting sort in one launch.
#include "fp8.hpp"

namespace lloom {

// A workgroup an expert (the last one: planes of none), and each for itself: a
// wave has a run of planes, counts in it those of smaller experts and those of
// its own, and with the counts of all waves knows where its own go; a ballot
// ranks a row of 64.  No atomics, so the order is the planes' own, and nothing
// passes between workgroups; what it costs is that each reads all ids.  ROWS rows
// of 64 are loaded at a time, the next ones under those in work, and what they hold
// goes to a list in LDS first, so that stores have full waves.  ONCE: a run is no
// longer than that and is kept for the second time.  128 experts, 256 planes 2.7 us,
// 16384 4.8, 65536 12.7 (22.5 with a load at a time and stores of what each row
// holds): the ids pass 256 KB a workgroup twice, and five VALU operations each.  Two
// workgroups an expert, half of the second part each: 12.6, of 256 experts 18.6
// against 13.0.
// Keys of a wave's next rows from plane p on: an id, `none` for one of no expert,
// -1 past the last.
template <int ROWS>
__device__ __forceinline__ void plan_keys(const int* __restrict__ ids, int p, int last, uint32_t none, uint32_t (&key)[ROWS]) {
    const int at = p + (int)__lane_id();
    if (p + 64 * ROWS <= last) {
#pragma unroll
        for (int i = 0; i < ROWS; i++) key[i] = min((uint32_t)ids[at + 64 * i], none);
    } else {
#pragma unroll
        for (int i = 0; i < ROWS; i++) key[i] = at + 64 * i < last ? min((uint32_t)ids[at + 64 * i], none) : ~0u;
    }
}

template <int ROWS, bool ONCE>
__global__ __launch_bounds__(1024) void k_expert_plan(const int* __restrict__ ids, int planes, uint64_t per_topk,
                                                      int experts, int* __restrict__ starts, int* __restrict__ sorted,
                                                      int* __restrict__ tokens, int* __restrict__ flags) {
    __shared__ int s_less[16], s_same[16];
    __shared__ uint16_t s_list[16][64 * ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const uint32_t mine = blockIdx.x, none = (uint32_t)experts;
    const int run = ((planes + waves - 1) / waves + 63) & ~63, first = min(planes, wave * run), last = min(planes, first + run);
    int less = 0, same = 0;
    uint32_t key[ROWS], next[ROWS];
    plan_keys(ids, first, last, none, key);
    for (int p = first; p < last; p += 64 * ROWS) {
        if (!ONCE) plan_keys(ids, p + 64 * ROWS, last, none, next);
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            less += key[i] < mine;
            same += key[i] == mine;
            if (!ONCE) key[i] = next[i];
        }
    }
    less = __builtin_amdgcn_readlane(wave_scan(less), 63);
    same = __builtin_amdgcn_readlane(wave_scan(same), 63);
    if (lane == 0) s_less[wave] = less, s_same[wave] = same;
    __syncthreads();
    int at = 0, before = 0;
    for (int w = 0; w < waves; w++) {
        before += s_less[w];
        if (w < wave) at += s_same[w];
    }
    if (threadIdx.x == 0) starts[mine] = before;
    at += before;
    if (!same) return;
    uint16_t* list = s_list[wave];
    bool bad = false;
    if (!ONCE) plan_keys(ids, first, last, none, key);
    for (int p = first; p < last; p += 64 * ROWS) {
        if (!ONCE) plan_keys(ids, p + 64 * ROWS, last, none, next);
        int found = 0;
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            const uint64_t m = __ballot(key[i] == mine);
            if (key[i] == mine)
                list[found + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0))] =
                    (uint16_t)(64 * i + lane);
            found += __builtin_popcountll(m);
            if (!ONCE) key[i] = next[i];
        }
        // a wave's own list: its LDS operations are in order
        for (int i = lane; i < found; i += 64) {
            const int plane = p + list[i];
            sorted[at + i] = plane;
            tokens[at + i] = (int)((uint64_t)plane * per_topk >> 40);
            if (mine == none) bad |= ids[plane] >= experts;
        }
        at += found;
    }
    if (bad) flags[0] = 1;
}

hipError_t launch_expert_plan(const int* ids, int64_t planes, int topk, int experts, int* starts, int* sorted,
                              int* tokens, int* flags, hipStream_t s) {
    // planes < 2^24 and topk <= 2^12: the quotient by 2^40 / topk + 1 is exact
    const uint64_t per = (1ull << 40) / (uint32_t)topk + 1;
    const int p = (int)planes;
    if (planes <= 1024)
        k_expert_plan<4, true><<<experts + 1, 256, 0, s>>>(ids, p, per, experts, starts, sorted, tokens, flags);
    else if (planes <= 4096)
        k_expert_plan<4, true><<<experts + 1, 1024, 0, s>>>(ids, p, per, experts, starts, sorted, tokens, flags);
    else if (planes <= 16384)
        k_expert_plan<16, true><<<experts + 1, 1024, 0, s>>>(ids, p, per, experts, starts, sorted, tokens, flags);
    else
        k_expert_plan<16, false><<<experts + 1, 1024, 0, s>>>(ids, p, per, experts, starts, sorted, tokens, flags);
    return hipGetLastError();
}

}  // namespace lloom
