// paged_tile.hip -- attention of chunks of new tokens over the paged cache.
//
// A workgroup takes 128 rows of a request and a key head, 32 a wave; a step is 64
// keys, whose K and V come into LDS by global_load_lds a step ahead of their use.
// Both products run transposed on 32x32x16 MFMAs, S^T = K Q^T (A: 32 keys x 16
// dims) and O^T = V^T P^T (A: 32 dims x 16 keys).  A lane of S^T's result holds
// of one row the keys 8 (j / 4) + 4 half + j % 4, j = 0 .. 15; with K's rows taken
// in the order that makes them 16 (j / 8) + 8 half + j % 8 they are the second
// product's B operand as they stand, and P never leaves its lane.
//
// Two workgroups a CU: the one's waits and prologue run beside the other's products
// (one of 8 waves, which share a step's 128 keys: 119 against 116 us for a prompt of
// 4096 tokens, 16 heads of 128 in f16, and 100 against 64 for two chunks of 2048 with
// a window of 1024).  The prompt runs at 640 TFLOP/s in 107 us, a large library
// product at 1300; with f32 q and p in two halves each, so twice the matrix
// instructions, four chunks of 509 over 8000 take 125 us (795 TFLOP/s of them).  f32
// spills 5 registers with heads of 128, and 23 with heads of 256 (two chunks of 1500 over
// 1000: 172 us, 101 in f16).
// Issue and waits bound it, no unit: a step of a wave is 32 MFMAs (1024 clocks) among
// 370 instructions, and a long tile that is left alone on its CU takes 3900 clocks
// for it.  Left out by turns, loads are 24 us of the prompt's 111 (without the check
// of the reference, which is 10), the products with V 13, the weights 13.
#include "paged_launch.hpp"
#include "kq_common.hpp"
#include "paged_rows.hpp"

namespace lloom {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;

__device__ __forceinline__ f32x16 mfma32(half8_t a, half8_t b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ void lds_load16(const void* g, uint8_t* lds_piece) {
    __builtin_amdgcn_global_load_lds(g, (lds_void*)lds_piece, 16, 0, 0);
}

template <int D, bool F32>
struct PagedTile {
    static constexpr int ROWS = 128, WAVES = 4, THREADS = 64 * WAVES;
    static constexpr int KEYS = 64, KEY_SHIFT = 6;       // of a step
    static constexpr int PIECES = D == 96 ? 16 : D / 8;  // 16-byte pieces of a row of K in LDS (96: a quarter unused)
    static constexpr int K_BYTES = KEYS * PIECES * 16, V_BYTES = KEYS * D * 2, STAGE = K_BYTES + V_BYTES;
    static constexpr int K_LOADS = PIECES / 4, V_LOADS = D / 32;  // of 1 KB a wave: 16 keys of K; 8 dims of V each
    // operands read ahead: tiles of 32 keys of K, runs of 16 keys of V
    static constexpr int K_AHEAD = F32 || D == 256 ? 1 : 2, V_AHEAD = F32 || D == 256 ? 2 : 4;
    static constexpr int PART = ROWS * (D + 2);
    // p is kept times 2^SHIFT, and the reference it is relative to stands until a
    // row's largest passes it by 2^SLACK: rescaling the sums is then rare.  Halves
    // hold 2^(SHIFT + SLACK), and below 2^-(14 + SHIFT) of the reference they are off
    // by 2^-33 of it at most.
    static constexpr float SHIFT = 8.0f, SLACK = 7.0f;
};

// Workgroup `wg`; lds: two stages, then bad_group.
template <int D, bool F32>
__device__ __forceinline__ void paged_tile(const PagedCall& c, const PagedCut& cut, float* parts, int wg, uint8_t* lds,
                                           int (*bad_group)[4]) {
    using C = PagedTile<D, F32>;
    constexpr int DC = D / 16, DT = D / 32, ST = 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, half = lane >> 5;
    const PagedItem it = paged_find(c, cut, wg / c.kv_heads);
    if (!it.found) return;
    const int h = wg % c.kv_heads, page = 1 << c.page_shift;

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
    const int mine = min(32 * wave + r, nrows - 1), tok = paged_token(c, row + mine), pos = pos0 + tok;
    const int tile_lo = reach(pos0);
    const bool any_rows = 32 * wave < nrows;
    const int pos_lo = pos0 + paged_token(c, row + min(32 * wave, nrows - 1));
    const int pos_hi = pos0 + paged_token(c, row + min(32 * wave + 31, nrows - 1));
    const int pos_key = min(pos, cap), wave_last = min(pos_hi, cap), win = reach(pos), win_lo = reach(pos_lo), win_hi = reach(pos_hi);

    // q as B operands, dims 16 c + 8 half .., its sign turned where the scale is negative
    half8_t qh[DC], ql[F32 ? DC : 1];
    float factor = __builtin_fabsf(c.scale);
    const int64_t qi = (int64_t)(it.start + tok0 + tok) * c.q_stride + (int64_t)(h * c.group + row + mine - tok * c.group) * D + 8 * half;
    if constexpr (F32) {
        // times a power of two of the row's own, so that its largest is in 2^Q_SHIFT * [1, 2)
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
        e = min(max(e, Q_SHIFT - 126), 127);  // a zero, subnormal or infinite row; both powers are normal
        const float down = __builtin_bit_cast(float, (uint32_t)(127 + Q_SHIFT - e) << 23) * (c.scale < 0.0f ? -1.0f : 1.0f);
        factor *= __builtin_bit_cast(float, (uint32_t)(127 - Q_SHIFT + e) << 23);
#pragma unroll
        for (int i = 0; i < DC; i++) {
            const float4 a = *(const float4*)((const float*)c.q + qi + 16 * i);
            const float4 b = *(const float4*)((const float*)c.q + qi + 16 * i + 4);
            const float v[8] = {a.x * down, a.y * down, a.z * down, a.w * down, b.x * down, b.y * down, b.z * down, b.w * down};
            split8_query(v, qh[i], ql[i]);
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

    // This wave's loads of a step.  In LDS, K [key][piece ^ key's low bits] and V
    // [64 keys][dim][run of 8 keys ^ dim / 2's low bits]: 16 lanes that read one piece
    // of 16 keys, or one run of 16 dims, hit all banks once.  A load of V takes whole
    // runs of 64 keys of a dim from one page, or from as many as hold them: a lane's
    // run is one of two, by whether its 8 dims are an even or an odd 8.
    uint32_t k_off[C::K_LOADS];
#pragma unroll
    for (int i = 0; i < C::K_LOADS; i++) {
        const int at = i * 64 + lane, key = at / C::PIECES;
        int piece = (at % C::PIECES) ^ (C::PIECES == 8 ? key >> 1 & 7 : key & 15);
        if (piece >= D / 8) piece -= 4;  // a head of 96: any other
        k_off[i] = key * D * 2 + piece * 16;
    }
    const int v_first = wave * C::V_LOADS;           // its first 8 dims of V
    const int run = 8 * ((lane & 7) ^ (lane >> 4));  // its run in an even 8 dims; 32 keys off in an odd 8
    const uint32_t v_row = (uint32_t)(lane >> 3) << (c.page_shift + 1);
    struct Pages {
        int k, v[2];
    };
    const auto pages_of = [&](int s) {
        const int key = first_key(s);
        const auto of = [&](int k) { return table[min(key + k, key_last) >> c.page_shift]; };
        return Pages{of(16 * wave), {of(run), of(run ^ 32)}};
    };
    const auto load = [&](int s, const Pages& pg, uint8_t* to, int* bad_to) __attribute__((always_inline)) {
        const int key0 = first_key(s), key = key0 + 16 * wave;
        int kp = __builtin_amdgcn_readfirstlane(pg.k);
        // a page that no row sees may be none
        const bool seen = key <= key_last && (key + 15 >= tile_lo || key < c.sinks);
        const bool bad = (unsigned)kp >= (unsigned)c.pages && seen;
        if ((unsigned)kp >= (unsigned)c.pages) kp = 0;
        bad_page |= bad;
        if (lane == 0) bad_to[wave] = bad;
        const uint8_t* k = (const uint8_t*)(c.k + kp * page_size + head_off + (int64_t)(key & (page - 1)) * D);
#pragma unroll
        for (int i = 0; i < C::K_LOADS; i++)
            lds_load16(k + k_off[i], to + (wave * C::K_LOADS + i) * 1024);
        int shift = c.page_shift;
        asm volatile("" : "+s"(shift));  // or every load's offset is held in scalar registers
        const uint8_t* v[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int vp = (unsigned)pg.v[i] >= (unsigned)c.pages ? 0 : pg.v[i];
            v[i] = (const uint8_t*)(c.v + vp * page_size + head_off + ((key0 + (run ^ (32 * i))) & (page - 1))) + v_row +
                   ((uint32_t)(i ? v_first | 1 : (v_first + 1) & ~1) << (shift + 4));
        }
#pragma unroll
        for (int i = 0; i < C::V_LOADS; i++) {
            const int par = (v_first + i) & 1;
            lds_load16(par ? v[1] : v[0], to + C::K_BYTES + (v_first + i) * 1024);
            (par ? v[1] : v[0]) += 32 << shift;
        }
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
    const uint32_t k_base = (uint32_t)kkey * C::PIECES * 16;
    const uint32_t v_turn = (uint32_t)(half ^ (r >> 1 & 7)) << 4, v_base = C::K_BYTES + r * 128;
    const auto v_at = [&](const uint8_t* at, int g, int i) { return *(const uint4*)(at + v_base + (v_turn ^ (g << 5)) + i * 4096); };

    const auto k_at = [&](const uint8_t* at, int t, int i) {
        return as_half8(*(const uint4*)(at + k_base + (k_turn ^ (i << 5)) + t * 32 * C::PIECES * 16));
    };
    const auto largest = [&](const f32x16 (&z)[ST]) {
        float top = z[0][0];
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int j = 0; j < 16; j++) top = __builtin_fmaxf(top, z[t][j]);
        return __builtin_fmaxf(top, partner32(top)) * factor;
    };

    // z = K Q^T of a step.
    const auto scores = [&](const uint8_t* at, f32x16 (&z)[ST]) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < ST; t++)
#pragma unroll
            for (int j = 0; j < 16; j++) z[t][j] = 0.0f;
#pragma unroll
        for (int t0 = 0; t0 < ST; t0 += C::K_AHEAD) {
            half8_t kf[C::K_AHEAD][DC];
#pragma unroll
            for (int i = 0; i < DC; i++)
#pragma unroll
                for (int t = 0; t < C::K_AHEAD; t++) kf[t][i] = k_at(at, t0 + t, i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < DC; i++)
#pragma unroll
                for (int t = 0; t < C::K_AHEAD; t++) {
                    z[t0 + t] = mfma32(kf[t][i], qh[i], z[t0 + t]);
                    if constexpr (F32) z[t0 + t] = mfma32(kf[t][i], ql[i], z[t0 + t]);
                }
        }
    };
    // The weights of 16 keys, added to l, as B operands.
    const auto weights = [&](const f32x16 (&z)[ST], int g, float base, half8_t& ph, half8_t& pl) __attribute__((always_inline)) {
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[g >> 1][8 * (g & 1) + j], factor, -base));
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < 8; j++) l += p[j];
            split8(p, ph, pl);
        } else {
            // Rounded to halves, and summed as rounded, which is what the values are summed
            // with.  Two halves as for f32 cost half the matrix instructions again: 139
            // against 113 us for a prompt of 4096 tokens (73 and 61 for two chunks of 2048
            // with a window), for outputs off by 2.06e-4 of 64 bits, what their own
            // rounding leaves, and not by 2.43e-4.
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const half2_t two = {(_Float16)p[j], (_Float16)p[j + 1]}, one = {(_Float16)1.0f, (_Float16)1.0f};
                ph[j] = two[0], ph[j + 1] = two[1];
                l = __builtin_amdgcn_fdot2(two, one, l, false);
            }
        }
    };

    // x, or -inf where bit j is not set (two instructions, and no lane mask held in
    // scalar registers).
    const auto hide = [](float x, uint32_t bits, int j) {
        const uint32_t keep = (uint32_t)((int32_t)(bits << (31 - j)) >> 31);
        return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & keep) | (0xff800000u & ~keep));
    };

    // Any step; edge: some row does not see some of its keys.
    const auto any_step = [&](const uint8_t* at, int key0, uint32_t bad, bool edge) __attribute__((always_inline)) {
        f32x16 z[ST];
        scores(at, z);
        float low = PAGED_LOWEST;
        if (edge) {
            uint32_t some = 0;
#pragma unroll
            for (int g = 0; g < 2 * ST; g++) {
                const uint32_t seen = bad >> g & 1 ? 0u : paged_seen8(key0 + 16 * g + 8 * half, win, pos_key, c.sinks);
#pragma unroll
                for (int j = 0; j < 8; j++) z[g >> 1][8 * (g & 1) + j] = hide(z[g >> 1][8 * (g & 1) + j], seen, j);
                some |= seen;
            }
            low = some ? PAGED_LOWEST : -INFINITY;
            low = __builtin_fmaxf(low, partner32(low));
        }
        const float now = __builtin_fmaxf(__builtin_fmaxf(m, low), largest(z));
        const float less = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - now);
        m = now;
        l *= less;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int j = 0; j < 16; j++) o[i][j] *= less;
        const float base = m == -INFINITY ? 0.0f : m - C::SHIFT;
        // Values that some row does not see may be anything, and 0 times an infinity or a
        // NaN is no zero.  Zero times all the values tells whether there are such ones;
        // if so, keys that no row sees, and keys that hold such values, leave the product,
        // and the latter are added by hand to the rows that see them.
        uint32_t odd = 0, keep = 0xffffffffu;  // bit 8 g + j: key 16 g + 8 half + j
        if (edge) {
            f32x16 none;
#pragma unroll
            for (int j = 0; j < 16; j++) none[j] = 0.0f;
            const half8_t zero = as_half8(make_uint4(0, 0, 0, 0));
#pragma unroll
            for (int g = 0; g < 2 * ST; g++)
#pragma unroll
                for (int i = 0; i < DT; i++) none = mfma32(as_half8(v_at(at, g, i)), zero, none);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; j++) sum += none[j];
            if (__any(sum != 0.0f)) {  // a NaN is not zero
#pragma unroll 1
                for (int g = 0; g < 2 * ST; g++) {
                    const uint32_t any = bad >> g & 1 ? 0u : paged_seen8(key0 + 16 * g + 8 * half, win_lo, wave_last, c.sinks);
                    uint32_t marks = 0;
#pragma unroll 1
                    for (int i = 0; i < DT; i++) marks |= odd_keys(v_at(at, g, i));
                    odd |= (marks & any) << (8 * g);
                    keep &= ~((~any & 0xffu) << (8 * g));
                }
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) odd |= __shfl_xor(odd, d, 64);
                keep &= ~odd;
            }
        }
#pragma unroll
        for (int g = 0; g < 2 * ST; g++) {
            half8_t ph, pl;
            weights(z, g, base, ph, pl);
#pragma unroll
            for (int i = 0; i < DT; i++) {
                uint4 v = v_at(at, g, i);
                if (edge) keep8(v, keep >> (8 * g));
                o[i] = mfma32(as_half8(v), ph, o[i]);
                if constexpr (F32) o[i] = mfma32(as_half8(v), pl, o[i]);
            }
        }
        const uint32_t odd2[2] = {(uint32_t)__builtin_amdgcn_readlane(odd, 0), (uint32_t)__builtin_amdgcn_readlane(odd, 32)};
        for (int side = 0; side < 2; side++) {
#pragma unroll 1
            for (uint32_t left = side ? odd2[1] : odd2[0]; left; left &= left - 1) {
                const int bit = __builtin_ctz(left), k = 16 * (bit >> 3) + 8 * side + (bit & 7);
                float zk = 0.0f;
#pragma unroll
                for (int e = 0; e < 16 * ST; e++) zk = e == bit ? z[e >> 4][e & 15] : zk;
                zk = __shfl(zk, side * 32 + r, 64);
                const float pk = __builtin_amdgcn_exp2f(__builtin_fmaf(zk, factor, -base));
                // zero times it is no zero either
                if (key0 + k > pos_key || (key0 + k < win && key0 + k >= c.sinks)) continue;
                int side4 = 4 * half;
                asm volatile("" : "+v"(side4));  // or the main loop carries these reads' addresses
                const uint8_t* from = at + C::K_BYTES + (k & 7) * 2;
#pragma unroll
                for (int i = 0; i < DT; i++) {
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const int dim = 32 * i + 8 * (j >> 2) + side4 + (j & 3);
                        const uint16_t x = *(const uint16_t*)(from + dim * 128 + (k >> 3 ^ (dim >> 1 & 7)) * 16);
                        o[i][j] += pk * f16_to_f32(x);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    };

    const auto bad_of = [&](const int* from) {
        const uint32_t bad = from[0] | from[1] << 1 | from[2] << 2 | from[3] << 3;
        return (uint32_t)__builtin_amdgcn_readfirstlane(bad);
    };
    // steps fast0 .. fast1 - 1 of this wave: every row sees all their keys
    const int whole = min(pos_lo, cap) + 1 - C::KEYS;
    const int fast0 = max(span.sink_steps, ((win_hi + C::KEYS - 1) >> C::KEY_SHIFT) - span.skip);
    const int fast1 = any_rows && whole >= 0 ? min(s_end - 1, (whole >> C::KEY_SHIFT) - span.skip + 1) : 0;
    Pages pg{0, {0, 0}};
    int s = s0;
    if (s < s_end) {
        load(s, pages_of(s), lds, bad_group[0]);
        pg = pages_of(s + 1);
    }
    // a wave's own loads, which a barrier does not wait for, then everyone's
    const auto arrive = [&]() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    bool there = false;  // step s is in LDS, and no wave reads the other stage any more
    while (s < s_end) {
        // any step
        const int odd = (s - s0) & 1, key0 = first_key(s), key_end = key0 + C::KEYS - 1;
        if (!there) arrive();
        there = false;
        if (s + 1 < s_end) {
            load(s + 1, pg, lds + (odd ^ 1) * C::STAGE, bad_group[odd ^ 1]);
            pg = pages_of(s + 2);
        }
        // one with keys that some row of the wave sees
        if (any_rows && key0 <= wave_last && (c.window <= 0 || key_end >= win_lo || key0 < c.sinks)) {
            const uint32_t bad = bad_of(bad_group[odd]);
            any_step(lds + odd * C::STAGE, key0, bad,
                     bad || key_end > min(pos_lo, cap) || (c.window > 0 && key0 < win_hi && key_end >= c.sinks));
        }
        s++;
        if (s < fast0) continue;
        // Steps whose keys every row of the wave sees, up to one where a row's largest
        // passes its reference by more than the slack.  The sums change at the end alone:
        // else they were held, and moved, in two sets of registers.  The next step's
        // loads follow this one's last read, as the compiler has every read of LDS wait
        // for the loads before it.
        while (s < fast1) {
            const int now = (s - s0) & 1;
            const uint8_t* at = lds + now * C::STAGE;
            arrive();
            there = true;
            if (bad_of(bad_group[now])) break;
            f32x16 z[ST];
            scores(at, z);
            half8_t vf[C::V_AHEAD][DT];
#pragma unroll
            for (int g = 0; g < C::V_AHEAD; g++)
#pragma unroll
                for (int i = 0; i < DT; i++) vf[g][i] = as_half8(v_at(at, g, i));
            __builtin_amdgcn_sched_barrier(0);
            if (__any(__builtin_fmaxf(largest(z), PAGED_LOWEST) > m + C::SLACK)) break;
            const float base = m - C::SHIFT;  // m is not -inf: the lowest passes such a reference
#pragma unroll
            for (int g0 = 0; g0 < 2 * ST; g0 += C::V_AHEAD) {
                if (g0) {
#pragma unroll
                    for (int g = 0; g < C::V_AHEAD; g++)
#pragma unroll
                        for (int i = 0; i < DT; i++) vf[g][i] = as_half8(v_at(at, g0 + g, i));
                }
                if (g0 + C::V_AHEAD == 2 * ST) {
                    __builtin_amdgcn_sched_barrier(0);
                    load(s + 1, pg, lds + (now ^ 1) * C::STAGE, bad_group[now ^ 1]);
                    pg = pages_of(s + 2);
                }
#pragma unroll
                for (int g = 0; g < C::V_AHEAD; g++) {
                    half8_t ph, pl;
                    weights(z, g0 + g, base, ph, pl);
#pragma unroll
                    for (int i = 0; i < DT; i++) {
                        o[i] = mfma32(vf[g][i], ph, o[i]);
                        if constexpr (F32) o[i] = mfma32(vf[g][i], pl, o[i]);
                    }
                }
            }
            there = false;
            s++;
        }
    }
    if (bad_page && lane == 0) c.flags[0] = 1;

    l += partner32(l);  // the halves of a row's sum
    if (32 * wave + r < nrows) {
        if (it.splits > 1) {
            float* part = parts + ((int64_t)(it.part + it.split) * c.kv_heads + h) * C::PART;
            if (half == 0) {
                part_store(part + 32 * wave + r, m);
                part_store(part + C::ROWS + 32 * wave + r, l);
            }
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    part_store4(part + 2 * C::ROWS + (32 * wave + r) * D + 32 * i + 8 * a + 4 * half, o[i][4 * a], o[i][4 * a + 1],
                                o[i][4 * a + 2], o[i][4 * a + 3]);
        } else {
            const float inv = 1.0f / l;
            const bool none = m == -INFINITY;
            const int64_t to = place(32 * wave + r) + 4 * half;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int a = 0; a < 4; a++)
                    paged_store4<F32>(c.out, to + 32 * i + 8 * a, none ? 0.0f : o[i][4 * a] * inv, none ? 0.0f : o[i][4 * a + 1] * inv,
                                      none ? 0.0f : o[i][4 * a + 2] * inv, none ? 0.0f : o[i][4 * a + 3] * inv);
        }
    }
    if (it.splits > 1 && paged_last(c.joins + it.joint * c.kv_heads + h, it.splits))
        paged_join<D, F32, C::ROWS, C::THREADS, 4, 2>(parts + ((int64_t)it.part * c.kv_heads + h) * C::PART,
                                                (int64_t)c.kv_heads * C::PART, it.splits, nrows, lds, c.out, place);
}

// The tiles of the requests with many rows, and after them in the same launch the
// requests with few, whose splits count themselves with the other half of the
// counters.
template <int D, bool F32>
__global__ __launch_bounds__((PagedTile<D, F32>::THREADS), D == 256 ? 1 : 2) void k_paged_tile(PagedCall c, PagedCut tiles, float* tile_parts,
                                                                                            PagedCut rows, float* row_parts, int tile_wgs) {
    using C = PagedTile<D, F32>;
    union Lds {
        struct {
            uint8_t stages[2 * C::STAGE];
            int bad_group[2][4];
        } t;
        RowsLds<D, C::WAVES> r;
    };
    __shared__ __align__(16) Lds lds;
    const int wg = blockIdx.x;
    if (wg < tile_wgs) paged_tile<D, F32>(c, tiles, tile_parts, wg, lds.t.stages, lds.t.bad_group);
    else paged_rows<D, F32, C::WAVES>(c, rows, row_parts, wg - tile_wgs, gridDim.x - tile_wgs, lds.r.acc, lds.r.stat, c.joins + PAGED_JOINS / 2);
}

// A tile is split past what a CU would take of the whole call (two workgroups').
// Splits of tiles that fill the card by themselves cost more than they level (two
// parts for each of 512 tiles: 64 -> 116 us).
constexpr int TILE_TARGET_SHIFT = 8, TILE_UNIT_MIN = 8;
// Rows beside tiles: two workgroups of 4 waves a CU.
constexpr int ROWS_TARGET_SHIFT = 8;

template <int D, bool F32>
static hipError_t tiles_as(PagedCall c, int* index, float* tile_parts, float* row_parts, hipStream_t s) {
    using C = PagedTile<D, F32>;
    const PagedCut cuts[2] = {{7, C::KEY_SHIFT, TILE_UNIT_MIN, TILE_TARGET_SHIFT, (C::ROWS - 1) / c.group + 1, 2, D == 256 ? 256 : 512},
                              {4, 7, 2, ROWS_TARGET_SHIFT, (ATT_ROWS - 1) / c.group + 1, 1, 0}};
    if (const hipError_t e = launch_paged_index(c, cuts, 2, index, s)) return e;
    const int tile_wgs = (int)paged_items_most(c, cuts[0]), row_wgs = (int)paged_items_most(c, cuts[1]);
    hipLaunchKernelGGL((k_paged_tile<D, F32>), dim3(tile_wgs + row_wgs), dim3(C::THREADS), 0, s, c, cuts[0], tile_parts, cuts[1], row_parts, tile_wgs);
    return hipGetLastError();
}

hipError_t launch_paged_tiles(int act, int dim, const PagedCall& c, int* index, void* tile_ws, void* row_ws, hipStream_t s) {
    float *t = (float*)tile_ws, *r = (float*)row_ws;
    switch (dim) {
        case 64: return act == T_F32 ? tiles_as<64, true>(c, index, t, r, s) : tiles_as<64, false>(c, index, t, r, s);
        case 96: return act == T_F32 ? tiles_as<96, true>(c, index, t, r, s) : tiles_as<96, false>(c, index, t, r, s);
        case 128: return act == T_F32 ? tiles_as<128, true>(c, index, t, r, s) : tiles_as<128, false>(c, index, t, r, s);
        case 256: return act == T_F32 ? tiles_as<256, true>(c, index, t, r, s) : tiles_as<256, false>(c, index, t, r, s);
    }
    return hipErrorInvalidValue;
}

size_t paged_tiles_workspace_bytes(int kv_heads, int dim) {
    return ((size_t)paged_parts(TILE_TARGET_SHIFT) + kv_heads) * 128 * (dim + 2) * sizeof(float);
}

// Few rows in every request, as far as the host can see.
static bool all_few(int64_t tokens, int64_t group, int64_t max_new, int64_t keys) {
    return paged_few((max_new > 0 && max_new < tokens ? max_new : tokens) * group, keys);
}

size_t paged_attention_workspace_bytes(int64_t tokens, int64_t requests, int kv_heads, int group, int dim, int max_new) {
    const size_t rows = paged_index_workspace_bytes(requests) + paged_rows_workspace_bytes(kv_heads, dim);
    return all_few(tokens, group, max_new, PAGED_SHORT + 1) ? rows : rows + paged_tiles_workspace_bytes(kv_heads, dim);
}

hipError_t launch_paged_attention(int act, int dim, const PagedCall& c, int max_new, void* ws, hipStream_t s) {
    char* row_ws = (char*)ws + paged_index_workspace_bytes(c.requests);
    if (all_few(c.tokens, c.group, max_new, (int64_t)c.max_blocks << c.page_shift)) return launch_paged_rows(act, dim, c, (int*)ws, row_ws, s);
    return launch_paged_tiles(act, dim, c, (int*)ws, row_ws + paged_rows_workspace_bytes(c.kv_heads, dim), row_ws, s);
}

}  // namespace lloom
