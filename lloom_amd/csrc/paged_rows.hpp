// paged_rows.hpp -- attention of few rows a request (decode) over the paged
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
//
// Bound by reading the cache: one request of 131072 tokens (8 key heads of 128, 537
// MB) takes 100 us, 5.4 TB/s where a large read reaches 6.4.  With less to read,
// latencies in a row are what it takes: of the 10 us of one request of 641 tokens
// (1.3 MB) the search for the item is 1.2, the page table and a wave's first K and
// V 2, the second four waves' another 1.7 (a CU's 32 KB of L1 hold what is in
// flight: 24 B a clock), the waves' sums 0.5, the counter 0.8, the parts' join 1.5,
// the launch the rest.  Loads a step ahead of the products are there already: eight
// waves' 16 KB each.
// Heads of 256 in f32 hold more than the registers: 43 are spilled (31 us for 16 requests
// of up to 8191 tokens, 66 MB, where f16 takes 21).
//
// The weights are two halves (2^-22 of them) for f16 queries too: rounded to one, an
// output was off by 2.19e-4 of 64 bits and not by the 2.07e-4 of its own rounding (32
// requests, 62 MB), for 0.1 of 17.8 us less; 0 to 2 % in other calls.
#pragma once

#include "paged_launch.hpp"
#include "kq_common.hpp"
#include "paged.hpp"

namespace lloom {

// p is kept times 2^14: halves then hold it down to 2^-38 of the row's largest.
constexpr float P_SHIFT = 14.0f;
constexpr int ATT_ROWS = 16, ATT_STEP = 32;

__device__ __forceinline__ f32x4 mfma16(half8_t a, half8_t b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// LDS of a workgroup of W waves.
template <int D, int W>
struct RowsLds {
    float acc[W][ATT_ROWS][D + 4];
    float stat[W][2][ATT_ROWS];
};

// Workgroup `wg` of `wgs`, of W waves.
template <int D, bool F32, int W>
__device__ __forceinline__ void paged_rows(const PagedCall& c, const PagedCut& cut, float* parts, int wg, int wgs,
                                           float (&acc)[W][ATT_ROWS][D + 4], float (&stat)[W][2][ATT_ROWS], int* joins) {
    constexpr int DC = D / 32, DT = D / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g4 = lane >> 4;
    const int first = c.q_start[0], last = c.q_start[c.requests];
    const PagedItem it = paged_find(c, cut, wg / c.kv_heads);
    paged_zero_rest<F32>(c, D, wg, wgs, first, last, it.refused);
    if (!it.found) return;
    const int h = wg % c.kv_heads, page = 1 << c.page_shift;

    // the lane's row: token and head in group
    const int row0 = it.tile * ATT_ROWS, nrows = min(it.T * c.group - row0, ATT_ROWS);
    const int tok0 = row0 ? row0 / c.group : 0, row = row0 - tok0 * c.group;  // the tile's first token, and its row 0 from there
    const int tok = paged_token(c, row + min(r, nrows - 1)), head = h * c.group + row + min(r, nrows - 1) - tok * c.group;
    const int pos_lo = it.L - it.T + tok0, pos = pos_lo + tok, pos_hi = pos_lo + paged_token(c, row + nrows - 1);
    // row i's place in out
    const auto place = [&](int i) {
        const int t = paged_token(c, row + i);
        return ((int64_t)(it.start + tok0 + t) * c.kv_heads * c.group + h * c.group + row + i - t * c.group) * D;
    };

    // q as B operands: dims 32 c + 8 g4 ..
    half8_t qh[DC], ql[F32 ? DC : 1];
    float factor = c.scale;
    const int64_t qi = (int64_t)(it.start + tok0 + tok) * c.q_stride + (int64_t)head * D + 8 * g4;
    if constexpr (F32) {
        // times a power of two of the row's own, so that its largest is in 2^Q_SHIFT * [1, 2)
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
        e = min(max(e, Q_SHIFT - 126), 127);  // a zero, subnormal or infinite row; both powers are normal
        const float down = __builtin_bit_cast(float, (uint32_t)(127 + Q_SHIFT - e) << 23);
        factor *= __builtin_bit_cast(float, (uint32_t)(127 - Q_SHIFT + e) << 23);
#pragma unroll
        for (int i = 0; i < DC; i++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[i][j] *= down;
            split8_query(x[i], qh[i], ql[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < DC; i++) qh[i] = as_half8(*(const uint4*)((const uint16_t*)c.q + qi + 32 * i));
    }

    const int cap = paged_key_cap(c), key_last = min(pos_hi, cap), pos_key = min(pos, cap);
    // the first key of the lane's window, and of the window that reaches furthest back
    const auto reach = [&](int p) { return c.window > 0 ? max(max(p, 0) - c.window + 1, 0) : 0; };
    const int win = reach(pos), win_lo = reach(pos_lo);
    const PagedSpan span = paged_span(pos_lo, key_last, c.window, c.sinks, ATT_STEP);
    const int per = (span.steps + it.splits - 1) / it.splits;
    const int s_end = (int)min((int64_t)span.steps, (int64_t)(it.split + 1) * per);
    int s = it.split * per + wave;

    f32x4 o[DT];
#pragma unroll
    for (int i = 0; i < DT; i++) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    const int* table = c.tables + it.b * c.table_stride;
    const int kk = 8 * (r >> 2) + (r & 3), vk = 8 * g4;  // this lane's key of K tile 0, and its first of V, in a step
    const int64_t head_off = (int64_t)h * D << c.page_shift, page_size = (int64_t)c.kv_heads * D << c.page_shift;
    const int64_t v_apart = (int64_t)16 << c.page_shift;
    bool bad_page = it.L - 1 > cap;

    // the pages of the lane's keys in a step, read a step ahead; past the last key
    // that one's page, masked below
    const auto first_key = [&](int i) { return ATT_STEP * (i < span.sink_steps ? i : span.skip + i); };
    const auto page_of = [&](int key) { return table[min(key, key_last) >> c.page_shift]; };
    int key0 = first_key(s), kp = 0, vp = 0;
    if (s < s_end) kp = page_of(key0 + (kk & ~7)), vp = page_of(key0 + vk);

    for (; s < s_end; s += W) {
        const int v8 = key0 + vk;
        // a page that no row sees may be none
        const bool bad = (unsigned)vp >= (unsigned)c.pages && v8 <= key_last && (v8 + 7 >= win_lo || v8 < c.sinks);
        if ((unsigned)kp >= (unsigned)c.pages) kp = 0;
        if ((unsigned)vp >= (unsigned)c.pages) vp = 0;
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
        for (int i = 0; i < DT; i++) {
            vraw[i] = *(const uint4*)vptr;
            vptr += v_apart;
        }

        int key1 = 0, kp1 = 0, vp1 = 0;
        if (s + W < s_end) {
            key1 = first_key(s + W);
            kp1 = page_of(key1 + (kk & ~7)), vp1 = page_of(key1 + vk);
        }

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
        uint32_t odd = 0, seen = 0xffu;
        if (edge) {
            seen = bad ? 0u : paged_seen8(v8, win, pos_key, c.sinks);
            // keys that some row sees: the others' v may hold anything
            const uint32_t any = bad ? 0u : paged_seen8(v8, win_lo, key_last, c.sinks);
#pragma unroll
            for (int j = 0; j < 8; j++) z[j] = seen >> j & 1 ? z[j] : -INFINITY;
#pragma unroll
            for (int i = 0; i < DT; i++) keep8(vraw[i], any);
            // 0 times an infinity or a NaN is no zero: where rows of other tokens do not see
            // them, keys that hold such values leave the product and are added by hand below
            if (pos_lo != pos_hi) {
#pragma unroll
                for (int i = 0; i < DT; i++) odd |= odd_keys(vraw[i]);
                if (__any(odd != 0)) {
#pragma unroll
                    for (int d = 1; d < 16; d <<= 1) odd |= __shfl_xor(odd, d, 64);
#pragma unroll
                    for (int i = 0; i < DT; i++) keep8(vraw[i], ~odd);
                }
            }
        }
        float top = seen ? PAGED_LOWEST : -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; j++) top = __builtin_fmaxf(top, z[j]);
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
        split8(p, ph, pl);
#pragma unroll
        for (int i = 0; i < DT; i++) {
            o[i] = mfma16(as_half8(vraw[i]), ph, o[i]);
            o[i] = mfma16(as_half8(vraw[i]), pl, o[i]);
        }
        if (__any(odd != 0)) {
#pragma unroll 1
            for (int j = 0; j < 8; j++) {
                const unsigned long long who = __ballot(odd >> j & 1);
                float zj = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) zj = e == j ? z[e] : zj;
#pragma unroll 1
                for (int g = 0; g < 4; g++) {
                    if (!(who >> (16 * g) & 0xffff)) continue;
                    const float pr = __builtin_amdgcn_exp2f(__shfl(zj, 16 * g + r, 64) - base);
                    const bool sees = __shfl(seen, 16 * g + r, 64) >> j & 1;  // zero times it is no zero either
                    const int pg = __shfl(vp, 16 * g, 64);
                    int shift = c.page_shift;
                    asm volatile("" : "+s"(shift));  // or the main loop carries these loads' addresses
                    const uint16_t* src = c.v + pg * page_size + head_off + ((key0 + 8 * g + j) & (page - 1)) +
                                          ((int64_t)(4 * g4) << shift);
#pragma unroll
                    for (int i = 0; i < DT; i++) {
                        const uint16_t* at = src;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            o[i][e] += sees ? pr * f16_to_f32(*at) : 0.0f;
                            at += 1 << shift;
                        }
                        src += 16 << shift;
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
        key0 = key1, kp = kp1, vp = vp1;
    }
    if (__any(bad_page) && lane == 0) c.flags[0] = 1;

    // the waves' sums, joined at the largest of their maxima
    l += partner16(l);
    l += partner32(l);
    if (g4 == 0) {
        stat[wave][0][r] = m;
        stat[wave][1][r] = l;
    }
    if (r < nrows) {
#pragma unroll
        for (int i = 0; i < DT; i++) *(f32x4*)&acc[wave][r][16 * i + 4 * g4] = o[i];
    }
    __syncthreads();
    constexpr int PART = ATT_ROWS * (D + 2);
    float* part = parts + ((int64_t)(it.part + it.split) * c.kv_heads + h) * PART;
    for (int i = threadIdx.x; i < nrows * D; i += 64 * W) {
        const int rr = i / D, d = i % D;
        float top = stat[0][0][rr];
#pragma unroll
        for (int w = 1; w < W; w++) top = __builtin_fmaxf(top, stat[w][0][rr]);
        const float base = top == -INFINITY ? 0.0f : top;
        float v = 0.0f, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float e = __builtin_amdgcn_exp2f(stat[w][0][rr] - base);
            v += acc[w][rr][d] * e;
            sum += stat[w][1][rr] * e;
        }
        if (it.splits > 1) {
            part_store(part + 2 * ATT_ROWS + i, v);
            if (d == 0) {
                part_store(part + rr, top);
                part_store(part + ATT_ROWS + rr, sum);
            }
        } else {
            const int64_t oi = place(rr) + d;
            const float y = top == -INFINITY ? 0.0f : v / sum;
            if constexpr (F32) ((float*)c.out)[oi] = y;
            else ((uint16_t*)c.out)[oi] = f32_to_f16(y);
        }
    }
    if (it.splits > 1 && paged_last(joins + it.joint * c.kv_heads + h, it.splits))
        paged_join<D, F32, ATT_ROWS, 64 * W, 1, 8>(parts + ((int64_t)it.part * c.kv_heads + h) * PART,
                                                     (int64_t)c.kv_heads * PART, it.splits, nrows, acc, c.out, place);
}

}  // namespace lloom
