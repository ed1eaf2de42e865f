// paged_tile.hip -- attention of chunks of new tokens over the paged cache.
//
// A workgroup takes 128 rows of a request and a key head.  Its waves are 4 groups
// of 32 rows times KG groups of keys; a step of the workgroup is KG * STEP keys,
// whose K and V come into LDS by global_load_lds a step ahead of their use.
// Both products run transposed on 32x32x16 MFMAs, S^T = K Q^T (A: 32 keys x 16
// dims) and O^T = V^T P^T (A: 32 dims x 16 keys).  A lane of S^T's result holds
// of one row the keys 8 (j / 4) + 4 half + j % 4, j = 0 .. 15; with K's rows taken
// in the order that makes them 16 (j / 8) + 8 half + j % 8 they are the second
// product's B operand as they stand, and P never leaves its lane.
#include "kernels.hpp"
#include "kq_common.hpp"
#include "paged.hpp"

namespace lloom {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void lds_void;

__device__ __forceinline__ f32x16 mfma32(half8_t a, half8_t b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ void lds_load16(const void* g, uint8_t* lds_piece) {
    __builtin_amdgcn_global_load_lds(g, (lds_void*)lds_piece, 16, 0, 0);
}

template <int D, bool F32>
struct PagedTile {
    static constexpr int ROWS = 128, RG = 4;             // rows, and groups of 32 of them
    static constexpr int STEP = D <= 128 ? 64 : 32;      // keys of a wave in a step
    static constexpr int KG = D == 256 && F32 ? 1 : 2;   // groups of keys
    static constexpr int WAVES = RG * KG, THREADS = 64 * WAVES;
    static constexpr int KEYS = KG * STEP, KEY_SHIFT = KEYS == 128 ? 7 : KEYS == 64 ? 6 : 5;
    static constexpr int PIECES = D == 96 ? 16 : D / 8;  // 16-byte pieces of a row of K in LDS (96: a quarter unused)
    static constexpr int K_BYTES = KEYS * PIECES * 16, V_BYTES = KEYS * D * 2, STAGE = K_BYTES + V_BYTES;
    static constexpr int GROUPS = KEYS / 16, SHARE = WAVES / GROUPS;  // waves that load 16 keys together
    static constexpr int K_LOADS = PIECES / 4 / SHARE, V_LOADS = D / 32;
    static constexpr int V_EACH = (V_LOADS + SHARE - 1) / SHARE;
    static constexpr int JOIN = RG * (D / 32) * 16 * 64 * 4 + RG * 64 * 8;  // the second key group's sums
    static constexpr int LDS = 2 * STAGE > JOIN ? 2 * STAGE : JOIN;
    static constexpr int PART = ROWS * (D + 2);
    // p is kept times 2^SHIFT, and the reference it is relative to stands until a
    // row's largest passes it by 2^SLACK: rescaling the sums is then rare.  Halves
    // hold 2^(SHIFT + SLACK) and, as normal numbers, down to 2^-(14 + SHIFT).
    static constexpr float SHIFT = F32 ? 12.0f : 8.0f, SLACK = F32 ? 3.0f : 7.0f;
    static_assert(GROUPS * SHARE == WAVES && (PIECES / 4) % SHARE == 0, "loads by 16 keys");
};

template <int D, bool F32>
__global__ __launch_bounds__((PagedTile<D, F32>::THREADS)) void k_paged_tile(PagedCall c, PagedCut cut, float* parts) {
    using C = PagedTile<D, F32>;
    constexpr int DC = D / 16, DT = D / 32, ST = C::STEP / 32;
    __shared__ __align__(16) uint8_t lds[C::LDS];
    __shared__ int bad_group[2][C::GROUPS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, half = lane >> 5, rg = wave % C::RG, kg = wave / C::RG;
    if (cut.route == 0) paged_zero_tail<F32>(c, D, blockIdx.x, gridDim.x);
    const PagedItem it = paged_find(c, cut, blockIdx.x / c.kv_heads);
    if (!it.found) return;
    const int h = blockIdx.x % c.kv_heads, page = 1 << c.page_shift;

    const int row0 = it.tile * C::ROWS, nrows = min(it.T * c.group - row0, C::ROWS);
    const int tok0 = row0 / c.group, row = row0 - tok0 * c.group;  // the tile's first token, and its row 0 from there
    const int pos0 = it.L - it.T + tok0;
    // row i's place in out
    const auto place = [&](int i) {
        const int t = paged_token(c, row + i);
        return ((int64_t)(it.start + tok0 + t) * c.kv_heads * c.group + h * c.group + row + i - t * c.group) * D;
    };
    const int cap = paged_key_cap(c), key_last = min(pos0 + paged_token(c, row + nrows - 1), cap);
    const auto reach = [&](int p) { return c.window > 0 ? max(max(p, 0) - c.window + 1, 0) : 0; };
    // the lane's row, and the wave's rows
    const int mine = min(32 * rg + r, nrows - 1), tok = paged_token(c, row + mine), pos = pos0 + tok;
    const int tile_lo = reach(pos0);
    const bool any_rows = 32 * rg < nrows;
    const int pos_lo = pos0 + paged_token(c, row + min(32 * rg, nrows - 1));
    const int pos_hi = pos0 + paged_token(c, row + min(32 * rg + 31, nrows - 1));
    const int pos_key = min(pos, cap), wave_last = min(pos_hi, cap), win = reach(pos), win_lo = reach(pos_lo), win_hi = reach(pos_hi);

    // q as B operands, dims 16 c + 8 half .., its sign turned where the scale is negative
    half8_t qh[DC], ql[F32 ? DC : 1];
    float factor = __builtin_fabsf(c.scale);
    const int64_t qi = (int64_t)(it.start + tok0 + tok) * c.q_stride + (int64_t)(h * c.group + row + mine - tok * c.group) * D + 8 * half;
    if constexpr (F32) {
        // times a power of two of the row's own, so that its largest is in [1, 2)
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < DC; i++) {
            const float4 a = *(const float4*)((const float*)c.q + qi + 16 * i);
            const float4 b = *(const float4*)((const float*)c.q + qi + 16 * i + 4);
            const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 8; j++) top = __builtin_fmaxf(top, __builtin_fabsf(v[j]));
        }
        top = __builtin_fmaxf(top, partner32(top));
        int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
        e = min(max(e, -100), 100);  // a zero, subnormal or infinite row
        const float down = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23) * (c.scale < 0.0f ? -1.0f : 1.0f);
        factor *= __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
#pragma unroll
        for (int i = 0; i < DC; i++) {
            const float4 a = *(const float4*)((const float*)c.q + qi + 16 * i);
            const float4 b = *(const float4*)((const float*)c.q + qi + 16 * i + 4);
            const float v[8] = {a.x * down, a.y * down, a.z * down, a.w * down, b.x * down, b.y * down, b.z * down, b.w * down};
            split8(v, qh[i], ql[i]);
        }
    } else {
        const uint32_t turn = c.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
        for (int i = 0; i < DC; i++) {
            uint4 v = *(const uint4*)((const uint16_t*)c.q + qi + 16 * i);
            v.x ^= turn, v.y ^= turn, v.z ^= turn, v.w ^= turn;
            qh[i] = as_half8(v);
        }
    }
    factor = __builtin_fmaxf(factor, 1e-30f);  // a scale of zero: -inf times it stays what it is

    const PagedSpan span = paged_span(pos0, key_last, c.window, c.sinks, C::KEYS);
    const int per = (span.steps + it.splits - 1) / it.splits;
    const int s0 = it.split * per, s_end = min(span.steps, s0 + per);
    const int* table = c.tables + it.b * c.table_stride;
    const int64_t head_off = (int64_t)h * D << c.page_shift, page_size = (int64_t)c.kv_heads * D << c.page_shift;
    bool bad_page = it.L - 1 > cap;
    const auto first_key = [&](int i) { return C::KEYS * (i < span.sink_steps ? i : span.skip + i); };

    // This wave's loads of a step: K and V of 16 keys (a share of them).  In LDS, K
    // [key][piece ^ key's low bits] and V [16 keys][dim][the two runs of 8 keys, in
    // turn every 8 dims]: 16 lanes that read one piece of 16 keys, or one run of 16
    // dims, hit all banks once.
    const int group = wave / C::SHARE, share = wave % C::SHARE;
    uint32_t k_off[C::K_LOADS], v_off[C::V_EACH];
#pragma unroll
    for (int i = 0; i < C::K_LOADS; i++) {
        const int at = (share * C::K_LOADS + i) * 64 + lane, key = at / C::PIECES;
        int piece = (at % C::PIECES) ^ (C::PIECES == 8 ? key >> 1 & 7 : key & 15);
        if (piece >= D / 8) piece -= 4;  // a head of 96: any other
        k_off[i] = key * D * 2 + piece * 16;
    }
#pragma unroll
    for (int i = 0; i < C::V_EACH; i++) {
        const int dim = min(share * C::V_EACH + i, C::V_LOADS - 1) * 32 + (lane >> 1);
        v_off[i] = (uint32_t)(dim << (c.page_shift + 1)) + ((lane & 1) ^ (dim >> 3 & 1)) * 16;
    }
    const auto page_of = [&](int s) { return table[min(first_key(s) + 16 * group, key_last) >> c.page_shift]; };
    const auto load = [&](int s, int pg, int buf) {
        const int key = first_key(s) + 16 * group;
        pg = __builtin_amdgcn_readfirstlane(pg);
        // a page that no row sees may be none
        const bool seen = key <= key_last && (key + 15 >= tile_lo || key < c.sinks);
        const bool bad = (unsigned)pg >= (unsigned)c.pages && seen;
        if ((unsigned)pg >= (unsigned)c.pages) pg = 0;
        bad_page |= bad;
        if (lane == 0) bad_group[buf][group] = bad;
        const uint8_t* k = (const uint8_t*)(c.k + pg * page_size + head_off + (int64_t)(key & (page - 1)) * D);
        const uint8_t* v = (const uint8_t*)(c.v + pg * page_size + head_off + (key & (page - 1)));
        uint8_t* to = lds + buf * C::STAGE;
#pragma unroll
        for (int i = 0; i < C::K_LOADS; i++)
            lds_load16(k + k_off[i], to + (group * (C::PIECES / 4) + share * C::K_LOADS + i) * 1024);
#pragma unroll
        for (int i = 0; i < C::V_EACH; i++)
            if (share * C::V_EACH + i < C::V_LOADS)
                lds_load16(v + v_off[i], to + C::K_BYTES + (group * C::V_LOADS + share * C::V_EACH + i) * 1024);
    };

    f32x16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) o[i][j] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    // where this lane reads its operands: key 16 (r / 16) + 8 (r / 4 & 1) + 4 (r / 8 & 1)
    // + r % 4 of a tile of K, dim r of a tile of V
    const int kkey = (r & 16) + (r >> 2 & 1) * 8 + (r >> 3 & 1) * 4 + (r & 3);
    const uint32_t k_turn = ((uint32_t)(half ^ (C::PIECES == 8 ? kkey >> 1 & 7 : kkey & 15))) << 4;
    const uint32_t k_base = (uint32_t)(kg * C::STEP + kkey) * C::PIECES * 16;
    const uint32_t v_base = C::K_BYTES + (uint32_t)kg * C::STEP * D * 2 + (r * 2 + (half ^ (r >> 3 & 1))) * 16;

    // One step of this wave's keys; EDGE: some row does not see some of them.
    const auto step = [&](const uint8_t* at, int key0, uint32_t bad, auto edge_c) {
        constexpr bool EDGE = decltype(edge_c)::value;
        f32x16 z[ST];
#pragma unroll
        for (int t = 0; t < ST; t++) {
#pragma unroll
            for (int j = 0; j < 16; j++) z[t][j] = 0.0f;
#pragma unroll
            for (int i = 0; i < DC; i++) {
                const half8_t k = as_half8(*(const uint4*)(at + k_base + (k_turn ^ (i << 5)) + t * 32 * C::PIECES * 16));
                z[t] = mfma32(k, qh[i], z[t]);
                if constexpr (F32) z[t] = mfma32(k, ql[i], z[t]);
            }
        }
        uint32_t any[2 * ST];  // keys that some row of the wave sees: the others' v may hold anything
        if constexpr (EDGE) {
#pragma unroll
            for (int g = 0; g < 2 * ST; g++) {
                const int key = key0 + 16 * g + 8 * half;
                const bool out = bad >> g & 1;
                const uint32_t seen = out ? 0u : paged_seen8(key, win, pos_key, c.sinks);
                any[g] = out ? 0u : paged_seen8(key, win_lo, wave_last, c.sinks);
#pragma unroll
                for (int j = 0; j < 8; j++) z[g >> 1][8 * (g & 1) + j] = seen >> j & 1 ? z[g >> 1][8 * (g & 1) + j] : -INFINITY;
            }
        }
        float top = z[0][0];
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int j = 0; j < 16; j++) top = __builtin_fmaxf(top, z[t][j]);
        top = __builtin_fmaxf(top, partner32(top)) * factor;
        if (__any(top > m + C::SLACK)) {
            const float now = __builtin_fmaxf(m, top);
            const float less = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= less;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int j = 0; j < 16; j++) o[i][j] *= less;
        }
        const float base = m == -INFINITY ? 0.0f : m - C::SHIFT;
#pragma unroll
        for (int g = 0; g < 2 * ST; g++) {
            float p[8];
            half8_t ph, pl;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[g >> 1][8 * (g & 1) + j], factor, -base));
                l += p[j];
            }
            if constexpr (F32) {
                split8(p, ph, pl);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) ph[j] = (_Float16)p[j];
            }
            uint32_t odd = 0;
#pragma unroll
            for (int i = 0; i < DT; i++) {
                uint4 v = *(const uint4*)(at + v_base + g * D * 32 + i * 1024);
                if constexpr (EDGE) {
                    keep8(v, any[g]);
                    // values that are no numbers, where other rows do not see them: they
                    // leave the product (0 times them is no zero) and are added below
                    if (pos_lo != pos_hi) odd |= take_odd(v);
                }
                o[i] = mfma32(as_half8(v), ph, o[i]);
                if constexpr (F32) o[i] = mfma32(as_half8(v), pl, o[i]);
            }
            if constexpr (EDGE) {
                if (!__any(odd)) continue;
#pragma unroll 1
                for (int k = 0; k < 16; k++) {
                    const unsigned long long who = __ballot(odd >> (k & 7) & 1);
                    if (!(who >> (32 * (k >> 3)) & 0xffffffffu)) continue;
                    float pk = 0.0f, zk = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        pk = e == (k & 7) ? p[e] : pk;
                        zk = e == (k & 7) ? z[g >> 1][8 * (g & 1) + e] : zk;
                    }
                    pk = __shfl(pk, (k >> 3) * 32 + r, 64);
                    zk = __shfl(zk, (k >> 3) * 32 + r, 64);
#pragma unroll
                    for (int i = 0; i < DT; i++) {
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const int dim = 8 * (j >> 2) + 4 * half + (j & 3);
                            const uint16_t x = *(const uint16_t*)(at + C::K_BYTES + (kg * C::STEP + 16 * g) * D * 2 + i * 1024 +
                                                                  (dim * 2 + ((k >> 3) ^ (dim >> 3 & 1))) * 16 + (k & 7) * 2);
                            const bool add = ((x & 0x7c00) == 0x7c00) & (zk != -INFINITY);
                            o[i][j] += add ? pk * f16_to_f32(x) : 0.0f;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    };

    int pg = s0 < s_end ? page_of(s0) : 0;
    if (s0 < s_end) {
        load(s0, pg, 0);
        if (s0 + 1 < s_end) pg = page_of(s0 + 1);
    }
    for (int s = s0; s < s_end; s++) {
        const int buf = (s - s0) & 1;
        __syncthreads();  // step s is in LDS, and no wave reads the other buffer any more
        if (s + 1 < s_end) {
            load(s + 1, pg, buf ^ 1);
            if (s + 2 < s_end) pg = page_of(s + 2);
        }
        const int key0 = first_key(s) + kg * C::STEP, key_end = key0 + C::STEP - 1;
        // keys that no row of the wave sees
        if (!any_rows || key0 > wave_last || (c.window > 0 && key_end < win_lo && key0 >= c.sinks)) continue;
        uint32_t bad = 0;
#pragma unroll
        for (int g = 0; g < 2 * ST; g++) bad |= (uint32_t)bad_group[buf][kg * (C::STEP / 16) + g] << g;
        bad = __builtin_amdgcn_readfirstlane(bad);
        const uint8_t* at = lds + buf * C::STAGE;
        const bool edge = key_end > min(pos_lo, cap) || (c.window > 0 && key0 < win_hi && key_end >= c.sinks) || bad;
        if (edge) step(at, key0, bad, std::integral_constant<bool, true>());
        else step(at, key0, 0u, std::integral_constant<bool, false>());
    }
    if (bad_page && lane == 0) c.flags[0] = 1;

    // the halves of a row's sum, and the two key groups' sums
    l += partner32(l);
    if constexpr (C::KG == 2) {
        float4* sums = (float4*)lds + (rg * DT * 4) * 64 + lane;
        float2* stat = (float2*)(lds + C::RG * DT * 4 * 64 * 16) + rg * 64 + lane;
        __syncthreads();
        if (kg == 1) {
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    sums[(i * 4 + a) * 64] = make_float4(o[i][4 * a], o[i][4 * a + 1], o[i][4 * a + 2], o[i][4 * a + 3]);
            *stat = make_float2(m, l);
        }
        __syncthreads();
        if (kg == 0) {
            const float2 other = *stat;
            const float top = __builtin_fmaxf(m, other.x), base = top == -INFINITY ? 0.0f : top;
            const float e0 = __builtin_amdgcn_exp2f(m - base), e1 = __builtin_amdgcn_exp2f(other.x - base);
            m = top;
            l = l * e0 + other.y * e1;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int a = 0; a < 4; a++) {
                    const float4 v = sums[(i * 4 + a) * 64];
                    o[i][4 * a] = o[i][4 * a] * e0 + v.x * e1;
                    o[i][4 * a + 1] = o[i][4 * a + 1] * e0 + v.y * e1;
                    o[i][4 * a + 2] = o[i][4 * a + 2] * e0 + v.z * e1;
                    o[i][4 * a + 3] = o[i][4 * a + 3] * e0 + v.w * e1;
                }
        }
    }
    if (kg == 0 && 32 * rg + r < nrows) {
        if (it.splits > 1) {
            float* part = parts + ((int64_t)(it.part + it.split) * c.kv_heads + h) * C::PART;
            if (half == 0) {
                part[32 * rg + r] = m;
                part[C::ROWS + 32 * rg + r] = l;
            }
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    *(float4*)(part + 2 * C::ROWS + (32 * rg + r) * D + 32 * i + 8 * a + 4 * half) =
                        make_float4(o[i][4 * a], o[i][4 * a + 1], o[i][4 * a + 2], o[i][4 * a + 3]);
        } else {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const bool none = l == 0.0f;
            const int64_t to = place(32 * rg + r) + 4 * half;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    paged_store4<F32>(c.out, to + 32 * i + 8 * a, none ? 0.0f : o[i][4 * a] * inv, none ? 0.0f : o[i][4 * a + 1] * inv,
                                      none ? 0.0f : o[i][4 * a + 2] * inv, none ? 0.0f : o[i][4 * a + 3] * inv);
        }
    }
    if (it.splits > 1 && paged_last(c.joins + it.joint * c.kv_heads + h, it.splits))
        paged_join<D, F32, C::ROWS, C::THREADS>(parts + ((int64_t)it.part * c.kv_heads + h) * C::PART,
                                                (int64_t)c.kv_heads * C::PART, it.splits, nrows, lds, c.out, place);
}

// Workgroups that the card holds at once.
constexpr int TILE_TARGET_SHIFT = 8, TILE_UNIT_MIN = 4;

template <int D, bool F32>
static hipError_t tiles_as(const PagedCall& c, int route, int few, float* parts, hipStream_t s) {
    using C = PagedTile<D, F32>;
    const PagedCut cut{7, C::KEY_SHIFT, TILE_UNIT_MIN, TILE_TARGET_SHIFT, (C::ROWS - 1) / c.group + 1, route, few};
    hipLaunchKernelGGL((k_paged_tile<D, F32>), dim3((unsigned)paged_items_most(c, cut)), dim3(C::THREADS), 0, s, c, cut, parts);
    return hipGetLastError();
}

hipError_t launch_paged_tiles(int act, int dim, const PagedCall& c, int route, int few, void* ws, hipStream_t s) {
    float* parts = (float*)ws;
    switch (dim) {
        case 64: return act == T_F32 ? tiles_as<64, true>(c, route, few, parts, s) : tiles_as<64, false>(c, route, few, parts, s);
        case 96: return act == T_F32 ? tiles_as<96, true>(c, route, few, parts, s) : tiles_as<96, false>(c, route, few, parts, s);
        case 128: return act == T_F32 ? tiles_as<128, true>(c, route, few, parts, s) : tiles_as<128, false>(c, route, few, parts, s);
        case 256: return act == T_F32 ? tiles_as<256, true>(c, route, few, parts, s) : tiles_as<256, false>(c, route, few, parts, s);
    }
    return hipErrorInvalidValue;
}

size_t paged_tiles_workspace_bytes(int kv_heads, int dim) {
    return ((size_t)paged_parts(TILE_TARGET_SHIFT) + kv_heads) * 128 * (dim + 2) * sizeof(float);
}

// Requests of at most this many rows go to the kernel of few rows.
constexpr int PAGED_FEW = 32;

size_t paged_attention_workspace_bytes(int64_t tokens, int64_t requests, int kv_heads, int group, int dim, int max_new) {
    (void)requests;
    const int64_t longest = max_new > 0 && max_new < tokens ? max_new : tokens;
    const size_t rows = paged_rows_workspace_bytes(kv_heads, dim);
    return longest * group <= PAGED_FEW ? rows : rows + paged_tiles_workspace_bytes(kv_heads, dim);
}

hipError_t launch_paged_attention(int act, int dim, const PagedCall& c, int max_new, void* ws, hipStream_t s) {
    const int64_t longest = max_new > 0 && max_new < c.tokens ? max_new : c.tokens;
    if (longest * c.group <= PAGED_FEW) return launch_paged_rows(act, dim, c, 0, 0, ws, s);
    void* tiles_ws = (char*)ws + paged_rows_workspace_bytes(c.kv_heads, dim);
    if (c.requests == 1) return launch_paged_tiles(act, dim, c, 0, 0, tiles_ws, s);
    const hipError_t e = launch_paged_rows(act, dim, c, 1, PAGED_FEW, ws, s);
    return e != hipSuccess ? e : launch_paged_tiles(act, dim, c, 2, PAGED_FEW, tiles_ws, s);
}

}  // namespace lloom
