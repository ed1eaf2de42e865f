// paged_attn.hip -- attention of few rows a request (decode) over the paged
// cache.
//
// out[n] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - max), over the
// keys j <= pos(n) with window = 0, j > pos(n) - window or j < sinks.
//
// Both products run transposed: S^T = K Q^T (A: 16 keys x 32 dims, B: 32 dims x
// 16 rows) and O^T = V^T P^T (A: 16 dims x 32 keys, B: 32 keys x 16 rows).  A
// lane of S^T's result holds 4 consecutive keys of one row; taking K's rows in
// the order key = 8 (r / 4) + 4 t + r % 4 (row r of tile t) makes the two tiles
// of a 32-key step leave 8 consecutive keys in a lane, which is B's operand of
// the second product as it stands: P never leaves its lane, and K and V come
// straight from the cache in 16-byte pieces, with no LDS.
#include "kernels.hpp"
#include "kq_common.hpp"
#include "paged.hpp"

namespace lloom {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// p is kept times 2^14: halves then hold it down to 2^-38 of the row's largest.
constexpr float P_SHIFT = 14.0f;
constexpr int ATT_WAVES = 4, ATT_ROWS = 16, ATT_STEP = 32;

__device__ __forceinline__ f32x4 mfma16(half8_t a, half8_t b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
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

// Zeroes the infinities and NaN among N pieces of 8 keys; bit j of the result:
// there was one at key j.
template <int N>
__device__ __forceinline__ uint32_t take_odd(uint4 (&v)[N]) {
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        uint32_t* w = (uint32_t*)&v[i];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if ((w[j] & 0x7c00u) == 0x7c00u) {
                odd |= 1u << (2 * j);
                w[j] &= 0xffff0000u;
            }
            if ((w[j] & 0x7c000000u) == 0x7c000000u) {
                odd |= 2u << (2 * j);
                w[j] &= 0xffffu;
            }
        }
    }
    return odd;
}

template <int D, bool F32>
__global__ __launch_bounds__(64 * ATT_WAVES) void k_paged_rows(PagedCall c, PagedCut cut, float* parts) {
    constexpr int DC = D / 32, DT = D / 16, PITCH = D + 4;
    __shared__ float acc[ATT_WAVES][ATT_ROWS][PITCH];
    __shared__ float stat[ATT_WAVES][2][ATT_ROWS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g4 = lane >> 4;
    if (cut.route != 2) paged_zero_tail<F32>(c, D, blockIdx.x, gridDim.x);
    const PagedItem it = paged_find<false>(c, cut, blockIdx.x / c.kv_heads);
    if (!it.found) return;
    const int h = blockIdx.x % c.kv_heads, page = 1 << c.page_shift;

    // the lane's row: token and head in group
    const int row0 = it.tile * ATT_ROWS, nrows = min(it.T * c.group - row0, ATT_ROWS);
    const int row = row0 + min(r, nrows - 1), tok = row / c.group, head = h * c.group + row % c.group;
    const int pos = it.L - it.T + tok;
    const int pos_lo = it.L - it.T + row0 / c.group, pos_hi = it.L - it.T + (row0 + nrows - 1) / c.group;

    // q as B operands: dims 32 c + 8 g4 ..
    half8_t qh[DC], ql[F32 ? DC : 1];
    float factor = c.scale;
    const int64_t qi = (int64_t)(it.start + tok) * c.q_stride + (int64_t)head * D + 8 * g4;
    if constexpr (F32) {
        // times a power of two of the row's own, so that its largest is in [1, 2)
        float x[DC][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < DC; i++) {
            const float4 a = *(const float4*)((const float*)c.q + qi + 32 * i);
            const float4 b = *(const float4*)((const float*)c.q + qi + 32 * i + 4);
            const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[i][j] = v[j];
                top = __builtin_fmaxf(top, __builtin_fabsf(v[j]));
            }
        }
        top = __builtin_fmaxf(top, partner16(top));
        top = __builtin_fmaxf(top, partner32(top));
        int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127;
        e = min(max(e, -100), 100);  // a zero, subnormal or infinite row
        const float down = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
        factor *= __builtin_bit_cast(float, (uint32_t)(127 + e) << 23);
#pragma unroll
        for (int i = 0; i < DC; i++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[i][j] *= down;
            split8(x[i], qh[i], ql[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < DC; i++) qh[i] = as_half8(*(const uint4*)((const uint16_t*)c.q + qi + 32 * i));
    }

    const int cap = paged_key_cap(c), key_last = min(pos_hi, cap), pos_key = min(pos, cap);
    // the first key of the lane's window, and of the window that reaches furthest back
    const int win = c.window > 0 ? pos - c.window + 1 : 0, win_lo = c.window > 0 ? pos_lo - c.window + 1 : 0;
    const PagedSpan span = paged_span(pos_lo, key_last, c.window, c.sinks, ATT_STEP);
    const int per = it.splits > 1 ? it.chunk * ATT_WAVES : span.steps;
    const int s_end = (int)min((int64_t)span.steps, (int64_t)(it.split + 1) * per);
    int s = it.split * per + wave;

    f32x4 o[DT];
#pragma unroll
    for (int i = 0; i < DT; i++) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    const int* table = c.tables + it.b * c.table_stride;
    const int kk = 8 * (r >> 2) + (r & 3), vk = 8 * g4;  // this lane's key of K tile 0, and its first of V, in a step
    const int64_t head_off = (int64_t)h * D << c.page_shift, page_size = (int64_t)c.kv_heads * D << c.page_shift;
    bool bad_page = it.L - 1 > cap;

    for (; s < s_end; s += ATT_WAVES) {
        const int key0 = ATT_STEP * (s < span.sink_steps ? s : span.skip + s);
        // the pages of the lane's keys; past the last key that one's page, masked below
        const int k8 = key0 + (kk & ~7), v8 = key0 + vk;
        int kp = table[min(k8, key_last) >> c.page_shift], vp = table[min(v8, key_last) >> c.page_shift];
        const bool bad = (unsigned)vp >= (unsigned)c.pages;
        if ((unsigned)kp >= (unsigned)c.pages) kp = 0;
        if (bad) vp = 0;
        bad_page |= bad;
        const uint16_t* kptr = c.k + kp * page_size + head_off + (int64_t)((key0 + kk) & (page - 1)) * D + 8 * g4;
        const uint16_t* vptr = c.v + vp * page_size + head_off + ((int64_t)r << c.page_shift) + (v8 & (page - 1));
        half8_t kr[2][DC];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int i = 0; i < DC; i++) kr[t][i] = as_half8(*(const uint4*)(kptr + 4 * t * D + 32 * i));
        uint4 vraw[DT];
#pragma unroll
        for (int i = 0; i < DT; i++) vraw[i] = *(const uint4*)(vptr + ((int64_t)(16 * i) << c.page_shift));

        float z[8];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            f32x4 a = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < DC; i++) {
                a = mfma16(kr[t][i], qh[i], a);
                if constexpr (F32) a = mfma16(kr[t][i], ql[i], a);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) z[4 * t + j] = a[j] * factor;
        }
        // a step that some row does not see whole
        const bool edge = key0 + ATT_STEP - 1 > min(pos_lo, cap) ||
                          (c.window > 0 && key0 <= pos_hi - c.window && key0 + ATT_STEP > c.sinks) || __any(bad);
        if (edge) {
            uint32_t any = 0;  // keys that some row sees: the others' v may hold anything
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int key = v8 + j;
                // bitwise: hipcc 7.2 lost the first key's assignment among the branches of && and ||
                const bool seen = !bad & (key <= pos_key) & ((key >= win) | (key < c.sinks));
                z[j] = seen ? z[j] : -INFINITY;
                const bool some = !bad & (key <= key_last) & ((key >= win_lo) | (key < c.sinks));
                any |= (uint32_t)some << j;
            }
            uint32_t keep[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                keep[j] = ((any >> (2 * j) & 1) ? 0xffffu : 0u) | ((any >> (2 * j + 1) & 1) ? 0xffff0000u : 0u);
#pragma unroll
            for (int i = 0; i < DT; i++) {
                vraw[i].x &= keep[0];
                vraw[i].y &= keep[1];
                vraw[i].z &= keep[2];
                vraw[i].w &= keep[3];
            }
        }
        // values that are no numbers, in a step that not every row sees whole: they
        // leave the product (0 times them is no zero) and are added by hand below
        uint32_t odd = 0;
        if (edge) odd = take_odd<DT>(vraw);
        const bool any_odd = edge && __any(odd != 0);
        float top = z[0];
#pragma unroll
        for (int j = 1; j < 8; j++) top = __builtin_fmaxf(top, z[j]);
        top = __builtin_fmaxf(top, partner16(top));
        top = __builtin_fmaxf(top, partner32(top));
        if (__any(top > m)) {
            const float now = __builtin_fmaxf(m, top);
            const float less = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= less;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[i][j] *= less;
        }
        const float base = m == -INFINITY ? 0.0f : m - P_SHIFT;
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            p[j] = __builtin_amdgcn_exp2f(z[j] - base);
            l += p[j];
        }
        half8_t ph, pl;
        if constexpr (F32) {
            split8(p, ph, pl);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) ph[j] = (_Float16)p[j];
        }
#pragma unroll
        for (int i = 0; i < DT; i++) {
            o[i] = mfma16(as_half8(vraw[i]), ph, o[i]);
            if constexpr (F32) o[i] = mfma16(as_half8(vraw[i]), pl, o[i]);
        }
        if (any_odd) {
#pragma unroll 1
            for (int j = 0; j < 8; j++) {
                const unsigned long long who = __ballot(odd >> j & 1);
                float pj = 0.0f, zj = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    pj = e == j ? p[e] : pj;
                    zj = e == j ? z[e] : zj;
                }
#pragma unroll 1
                for (int g = 0; g < 4; g++) {
                    if (!(who >> (16 * g) & 0xffff)) continue;
                    const float pr = __shfl(pj, 16 * g + r, 64), zr = __shfl(zj, 16 * g + r, 64);
                    const int pg = __shfl(vp, 16 * g, 64);
                    const uint16_t* src = c.v + pg * page_size + head_off + ((key0 + 8 * g + j) & (page - 1));
#pragma unroll
                    for (int i = 0; i < DT; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint16_t x = src[(int64_t)(16 * i + 4 * g4 + e) << c.page_shift];
                            const bool add = ((x & 0x7c00) == 0x7c00) & (zr != -INFINITY);
                            o[i][e] += add ? pr * f16_to_f32(x) : 0.0f;
                        }
                }
            }
        }
    }
    if (__any(bad_page) && lane == 0) c.flags[0] = 1;

    // the waves' sums, joined at the largest of their maxima
    l += partner16(l);
    l += partner32(l);
    if (g4 == 0) {
        stat[wave][0][r] = m;
        stat[wave][1][r] = l;
    }
#pragma unroll
    for (int i = 0; i < DT; i++) *(f32x4*)&acc[wave][r][16 * i + 4 * g4] = o[i];
    __syncthreads();
    float* part = parts + (int64_t)blockIdx.x * ATT_ROWS * (D + 2);
    for (int i = threadIdx.x; i < nrows * D; i += 64 * ATT_WAVES) {
        const int rr = i / D, d = i % D;
        float top = stat[0][0][rr];
#pragma unroll
        for (int w = 1; w < ATT_WAVES; w++) top = __builtin_fmaxf(top, stat[w][0][rr]);
        const float base = top == -INFINITY ? 0.0f : top;
        float v = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < ATT_WAVES; w++) {
            const float e = __builtin_amdgcn_exp2f(stat[w][0][rr] - base);
            v += acc[w][rr][d] * e;
            sum += stat[w][1][rr] * e;
        }
        if (it.splits > 1) {
            part[2 * ATT_ROWS + i] = v;
            if (d == 0) {
                part[rr] = top;
                part[ATT_ROWS + rr] = sum;
            }
        } else {
            const int gr = row0 + rr, t = gr / c.group, hd = h * c.group + gr % c.group;
            const int64_t oi = ((int64_t)(it.start + t) * c.kv_heads * c.group + hd) * D + d;
            const float y = sum == 0.0f ? 0.0f : v / sum;
            if constexpr (F32) ((float*)c.out)[oi] = y;
            else ((uint16_t*)c.out)[oi] = f32_to_f16(y);
        }
    }
}

// The splits of a (request, tile, key head) joined, in their order.
template <int D, bool F32>
__global__ __launch_bounds__(256) void k_paged_join(PagedCall c, PagedCut cut, const float* parts) {
    const PagedItem it = paged_find<true>(c, cut, blockIdx.x / c.kv_heads);
    if (!it.found || it.splits <= 1) return;
    const int h = blockIdx.x % c.kv_heads;
    const int row0 = it.tile * cut.rows, nrows = min(it.T * c.group - row0, cut.rows);
    const int64_t size = (int64_t)cut.rows * (D + 2);
    for (int i = threadIdx.x; i < nrows * D; i += 256) {
        const int rr = i / D;
        const float* p = parts + ((int64_t)it.split * c.kv_heads + h) * size;
        float top = -INFINITY;
        for (int s = 0; s < it.splits; s++) top = __builtin_fmaxf(top, p[s * c.kv_heads * size + rr]);
        const float base = top == -INFINITY ? 0.0f : top;
        float v = 0.0f, sum = 0.0f;
        for (int s = 0; s < it.splits; s++) {
            const float* q = p + s * c.kv_heads * size;
            const float e = __builtin_amdgcn_exp2f(q[rr] - base);
            v += q[2 * cut.rows + i] * e;
            sum += q[cut.rows + rr] * e;
        }
        const int gr = row0 + rr, t = gr / c.group, hd = h * c.group + gr % c.group;
        const int64_t oi = ((int64_t)(it.start + t) * c.kv_heads * c.group + hd) * D + i % D;
        const float y = sum == 0.0f ? 0.0f : v / sum;
        if constexpr (F32) ((float*)c.out)[oi] = y;
        else ((uint16_t*)c.out)[oi] = f32_to_f16(y);
    }
}

// About two rounds of the workgroups that the card holds at once.
constexpr int ATT_TARGET = 1024;

static int64_t tiles_most(int64_t tokens, int64_t requests, int group, int rows) {
    return tokens * group / rows + (requests < tokens ? requests : tokens);
}

static PagedCut rows_cut(const PagedCall& c, int route, int few) {
    PagedCut cut{ATT_ROWS, ATT_STEP * ATT_WAVES, 2, ATT_TARGET, route, few, 0};
    cut.split = tiles_most(c.tokens, c.requests, c.group, ATT_ROWS) * c.kv_heads < ATT_TARGET;
    return cut;
}

size_t paged_attention_workspace_bytes(int64_t tokens, int64_t requests, int kv_heads, int group, int dim,
                                       int max_new) {
    (void)max_new;
    const int64_t tiles = tiles_most(tokens, requests, group, ATT_ROWS) * kv_heads;
    if (tiles >= ATT_TARGET) return 0;
    return (size_t)(ATT_TARGET + tiles) * ATT_ROWS * (dim + 2) * sizeof(float);
}

template <int D, bool F32>
static hipError_t rows_as(const PagedCall& c, const PagedCut& cut, float* parts, hipStream_t s) {
    const int64_t tiles = tiles_most(c.tokens, c.requests, c.group, ATT_ROWS) * c.kv_heads;
    const int64_t grid = cut.split ? ATT_TARGET + tiles : tiles;
    hipLaunchKernelGGL((k_paged_rows<D, F32>), dim3((unsigned)grid), dim3(64 * ATT_WAVES), 0, s, c, cut, parts);
    if (cut.split) hipLaunchKernelGGL((k_paged_join<D, F32>), dim3((unsigned)tiles), dim3(256), 0, s, c, cut, parts);
    return hipGetLastError();
}

hipError_t launch_paged_attention(int act, int dim, const PagedCall& c, int max_new, void* ws, hipStream_t s) {
    (void)max_new;
    const PagedCut cut = rows_cut(c, 0, 0);
    float* parts = (float*)ws;
    switch (dim) {
        case 64: return act == T_F32 ? rows_as<64, true>(c, cut, parts, s) : rows_as<64, false>(c, cut, parts, s);
        case 96: return act == T_F32 ? rows_as<96, true>(c, cut, parts, s) : rows_as<96, false>(c, cut, parts, s);
        case 128: return act == T_F32 ? rows_as<128, true>(c, cut, parts, s) : rows_as<128, false>(c, cut, parts, s);
        case 256: return act == T_F32 ? rows_as<256, true>(c, cut, parts, s) : rows_as<256, false>(c, cut, parts, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace lloom
