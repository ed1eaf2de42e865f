// expert_plan.hip -- planes (token, slot) in the order of their experts: a
// stable counting sort in one launch.
#include "fp8.hpp"

namespace lloom {

// A workgroup an expert (the last one: planes of none), and each for itself: a
// wave has a run of planes, counts in it those of smaller experts and those of
// its own, and with the counts of all waves knows where its own go; a ballot
// ranks a row of 64.  No atomics, so the order is the planes' own, and nothing
// passes between workgroups; what it costs is that each reads all ids twice.
__global__ __launch_bounds__(1024) void k_expert_plan(const int* __restrict__ ids, int planes, uint64_t per_topk,
                                                      int experts, int* __restrict__ starts, int* __restrict__ sorted,
                                                      int* __restrict__ tokens, int* __restrict__ flags) {
    __shared__ int s_less[16], s_same[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const uint32_t mine = blockIdx.x, none = (uint32_t)experts;
    const int run = ((planes + waves - 1) / waves + 63) & ~63, first = min(planes, wave * run), last = min(planes, first + run);
    int less = 0, same = 0;
    bool bad = false;
#pragma unroll 4
    for (int p = first + lane; p < last; p += 64) {
        const int id = ids[p];
        const uint32_t key = min((uint32_t)id, none);
        less += key < mine;
        same += key == mine;
        bad |= id >= experts;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        less += __shfl_xor(less, o, 64);
        same += __shfl_xor(same, o, 64);
    }
    if (lane == 0) s_less[wave] = less, s_same[wave] = same;
    if (mine == none && __ballot(bad) && lane == 0) flags[0] = 1;
    __syncthreads();
    int at = 0, before = 0;
    for (int w = 0; w < waves; w++) {
        before += s_less[w];
        if (w < wave) at += s_same[w];
    }
    if (threadIdx.x == 0) starts[mine] = before;
    at += before;
    if (!same) return;
    for (int p = first; p < last; p += 64) {
        const bool ours = p + lane < last && min((uint32_t)ids[min(p + lane, last - 1)], none) == mine;
        const uint64_t m = __ballot(ours);
        if (ours) {
            const int to = at + __builtin_popcountll(m & ((1ull << lane) - 1));
            sorted[to] = p + lane;
            tokens[to] = (int)((uint64_t)(p + lane) * per_topk >> 40);
        }
        at += __builtin_popcountll(m);
    }
}

hipError_t launch_expert_plan(const int* ids, int64_t planes, int topk, int experts, int* starts, int* sorted,
                              int* tokens, int* flags, hipStream_t s) {
    // planes < 2^24 and topk <= 2^12: the quotient by 2^40 / topk + 1 is exact
    const uint64_t per = (1ull << 40) / (uint32_t)topk + 1;
    k_expert_plan<<<experts + 1, planes <= 2048 ? 256 : 1024, 0, s>>>(ids, (int)planes, per, experts, starts, sorted,
                                                                      tokens, flags);
    return hipGetLastError();
}

}  // namespace lloom
