// fp8.hpp -- products with e4m3 weights that have a scale for each block of
// 128 x 128 (fp8_rows.hip, fp8_few.hip, fp8_tile.hip, fp8_api.hip): the calls'
// launchers and what their kernels share.
//
//   y[m][n] = sum_b sx[m][b] sw[n / 128][b] sum_{k in b} qx[m][k] qw[n][k]
//
// over blocks b of 128 values of k, q the e4m3 numbers.  A block's inner sum is
// formed on the matrix cores, the scales meet it in f32.
#pragma once

#include "kernels.hpp"
#include "kq_common.hpp"

namespace lloom {

// Type ids beside those of kq_common.hpp: BF16 is GGUF's, E4M3 has none there.
constexpr int T_BF16 = 30, T_E4M3 = 100;

// A product's operands.  Rows of x are x_stride elements apart, its scales
// (e4m3 x) at [row * xs_row + block * xs_block].  starts (null: one group of
// all m rows): row i of group e, starts[e] <= i < starts[e + 1], is row
// gather[i] of x (null: i) and is stored at row scatter[i] of y (null: i).
struct Fp8Call {
    const uint8_t* w;
    const float* ws;
    const void* x;
    const float* xs;
    void* y;
    const int *starts, *gather, *scatter;
    int* flags;  // [0]: rows, starts or ids out of range
    int64_t x_stride, xs_row, xs_block;
    int n, k, kb, nb, m, x_rows, y_rows, experts, y_type;
    bool cut;  // halves of many rows by the 8-bit matrix instructions, whose sums are cut
};

// fp8_rows.hip: rows of x (F32, F16, BF16; x_stride elements apart) into e4m3 q
// [rows][k] and scales [block * scales_stride + row]; `up` (or null): of
// silu(x) * up.
hipError_t launch_fp8_rows(int type, const void* x, int64_t x_stride, const void* up, int64_t up_stride, int64_t rows,
                           int64_t k, void* q, float* scales, int64_t scales_stride, hipStream_t s);
// Weights [planes][n][k] into q and scales [planes][n / 128][k / 128].
hipError_t launch_fp8_weights(int type, const void* w, int64_t planes, int64_t n, int64_t k, void* q, float* scales,
                              hipStream_t s);
// expert_plan.hip
hipError_t launch_expert_plan(const int* ids, int64_t planes, int topk, int experts, int* starts, int* sorted,
                              int* tokens, int* flags, hipStream_t s);
// Whether fp8_few.hip serves a call (else fp8_tile.hip).  Its workgroups' tiles
// meet no other's, so it keeps all CUs busy with small outputs.  us of the two: 64 rows
// of [4096, 4096] 10.9 / 17.0, 128 14.9 / 17.2, 256 25.9 / 17.8; 32 of [8192, 8192] 21 / 32, 64 30.6 / 32.3,
// 128 52 / 33; 64 of [8192, 2048] 9.6 / 10.5, 96 15.2 / 10.9, 64 of [8192, 512] 5.4 / 5.8, 96 7.0 / 6.0;
// 256 of [2048, 8192] 25 / 30 (by MMA_FP8 the other is up to a tenth faster at the limit, 128 of [4096,
// 4096] 13.6).  Grouped, with 4, 6 and 8 rows an expert on average: [128, 1536, 2048] 67, 71, 77
// against 73, 74, 75, [128, 2048, 768] 4: 41.7 / 40.6; of small outputs 4 experts of 64 rows by 264
// 8.6 / 11.1, 64 of 8 by 256 12.9 / 12.5, by 512 19.7 / 16.1, 16 of 10 by 2048 13.1 / 11.0.
inline bool fp8_few_rows(int64_t rows, int64_t n, int64_t experts, bool grouped) {
    return rows <= 16 || (grouped ? rows <= 4 * experts || rows * n <= 128 * 1024 : rows * n <= 128 * 4096);
}
// fp8_few.hip: x E4M3, or any type where fp8_few_fuses (it is brought into 8 bits
// by each workgroup; only calls that fp8_few_rows gives to it).
bool fp8_few_fuses(int x_type, int64_t rows, int64_t k, int64_t experts, bool grouped);
hipError_t launch_fp8_few(int x_type, const Fp8Call& c, hipStream_t s);
// fp8_tile.hip: x E4M3.
hipError_t launch_fp8_tile(const Fp8Call& c, hipStream_t s);
// Whether such a launch has fewer threads than the 2^32 that one may have (of a call
// its sizes and y_type, cut, and whether it has starts).
constexpr int64_t FP8_THREADS = (int64_t)1 << 32;
bool fp8_few_fits(int x_type, const Fp8Call& c);
bool fp8_tile_fits(const Fp8Call& c);

#if defined(__HIP_DEVICE_COMPILE__) || defined(__HIPCC__)

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int fp8_v4i __attribute__((ext_vector_type(4)));
typedef float fp8_f4 __attribute__((ext_vector_type(4)));
typedef float fp8_f16v __attribute__((ext_vector_type(16)));
typedef _Float16 fp8_h2 __attribute__((ext_vector_type(2)));
typedef _Float16 fp8_h8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------- a block's scale --
// 2^e with the least e >= -126 for which a block's largest finite size is at
// most 448 * 2^e (448: the largest e4m3 number, 1.75 * 2^8), 1 for zeros.  The
// biased e is the size's own exponent less 8, and one more where its fraction
// passes .75.  The division by it is exact, so each value goes to the e4m3
// number that is nearest to it, whatever the arithmetic.
__device__ __forceinline__ uint32_t fp8_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t fp8_size(float v) {
    const uint32_t u = fp8_bits(v);
    return u < 0x7f800000u ? u : 0u;  // what is no number, or infinite, has no say
}
// Largest size of N values: as bits, and value by value only where some are no
// numbers (theirs are the largest bits).
template <int N>
__device__ __forceinline__ uint32_t fp8_largest(const float (&v)[N]) {
    uint32_t u = 0;
#pragma unroll
    for (int i = 0; i < N; i++) u = max(u, fp8_bits(v[i]));
    if (__builtin_expect(u >= 0x7f800000u, 0)) {
        u = 0;
#pragma unroll
        for (int i = 0; i < N; i++) u = max(u, fp8_size(v[i]));
    }
    return u;
}
__device__ __forceinline__ int fp8_exponent(uint32_t size) {
    return size ? max((int)((size + 0x1fffffu) >> 23) - 8, 1) : 127;
}
__device__ __forceinline__ float fp8_scale(int biased) { return __builtin_bit_cast(float, biased << 23); }
__device__ __forceinline__ float fp8_inverse(int biased) { return __builtin_bit_cast(float, (254 - biased) << 23); }

// Largest of the lanes that are 16 apart, in all of them.
__device__ __forceinline__ uint32_t column_max(uint32_t v) {
    v = max(v, __builtin_bit_cast(uint32_t, partner16(__builtin_bit_cast(float, v))));
    return max(v, __builtin_bit_cast(uint32_t, partner32(__builtin_bit_cast(float, v))));
}
// Largest of the 16 lanes of a row, in all of them.
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
    v = max(v, (uint32_t)dppi<DPP_XOR1>((int)v));
    v = max(v, (uint32_t)dppi<DPP_XOR2>((int)v));
    v = max(v, (uint32_t)dppi<DPP_HALF_MIRROR>((int)v));
    return max(v, (uint32_t)dppi<DPP_ROW_MIRROR>((int)v));
}

// Four values, scaled, to four e4m3 numbers (nearest, ties to even; NaN and
// infinities to NaN: the values themselves never pass 448).
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// Eight e4m3 numbers as halves (exact: they are in 2^-9 .. 448).
__device__ __forceinline__ fp8_h8 fp8_halves(uint32_t lo, uint32_t hi) {
    const fp8_h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    const fp8_h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const fp8_h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    const fp8_h2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return fp8_h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ---------------------------------------------------------------- types --
// Eight values from element i (16-byte aligned) as f32.
template <int TYPE>
__device__ __forceinline__ void fp8_load8(const void* p, int64_t i, float (&v)[8]) {
    if constexpr (TYPE == T_F32) {
        const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 a = *(const uint4*)((const uint16_t*)p + i);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if constexpr (TYPE == T_F16) {
                v[2 * j] = f16_to_f32(w[j] & 0xffffu);
                v[2 * j + 1] = f16_to_f32(w[j] >> 16);
            } else {
                v[2 * j] = __builtin_bit_cast(float, w[j] << 16);
                v[2 * j + 1] = __builtin_bit_cast(float, w[j] & 0xffff0000u);
            }
        }
    }
}

// f32 rounded to y's type (nearest even), its bits.
template <int TYPE>
__device__ __forceinline__ uint16_t fp8_half_bits(float v) {
    if constexpr (TYPE == T_F16) return f32_to_f16(v);
    return __builtin_bit_cast(uint16_t, (__bf16)v);
}
// Stores of 8 and 16 bytes wherever a row's values are: rows of y begin where n has
// them begin, and memory takes stores at any place (5184 rows into 3102 halves 63
// us, 79 where such rows are stored one value at a time).
typedef uint32_t fp8_at4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t fp8_at2 __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ void fp8_store16(void* p, const uint4& v) { *(fp8_at4*)p = fp8_at4{v.x, v.y, v.z, v.w}; }
__device__ __forceinline__ void fp8_store8(void* p, uint32_t x, uint32_t y) { *(fp8_at2*)p = fp8_at2{x, y}; }
// Four neighbours of a row, `count` of which are there.
template <int TYPE>
__device__ __forceinline__ void fp8_store4(void* y, int64_t i, const float (&v)[4], int count) {
    if constexpr (TYPE == T_F32) {
        float* p = (float*)y + i;
        if (count >= 4) {
            fp8_store16(p, __builtin_bit_cast(uint4, make_float4(v[0], v[1], v[2], v[3])));
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j < count) p[j] = v[j];
        }
    } else {
        uint16_t* p = (uint16_t*)y + i;
        uint16_t b[4];
#pragma unroll
        for (int j = 0; j < 4; j++) b[j] = fp8_half_bits<TYPE>(v[j]);
        if (count >= 4) {
            fp8_store8(p, b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j < count) p[j] = b[j];
        }
    }
}

// --------------------------------------------------------------- buffers --
// Operands are read through buffers of 2^31 bytes from a tile's own first: what is
// not there (rows past the operand's or a tile's, bytes past k) gets an offset
// that no buffer holds, which reads zeros and nothing of memory.
constexpr uint32_t FP8_OUT = 0x80000000u;
__device__ __forceinline__ fp8_v4i fp8_buffer(const void* p) {
    const uint64_t a = (uint64_t)p;
    return fp8_v4i{(int)__builtin_amdgcn_readfirstlane((int)a),
                   (int)__builtin_amdgcn_readfirstlane((int)(a >> 32) & 0xffff), (int)FP8_OUT, 0x00020000};
}

// ---------------------------------------------------------- tiles of rows --
// Tile t of a call whose groups are cut into tiles of up to 2^SHIFT rows, in
// the groups' order, then the rows past the last group (`zero`: no group owns
// them, y is 0 there).  Every wave looks for itself: a
// lane has a group, a scan its first tile.  Where starts do not begin with 0,
// fall, or pass m, no row has a group (and flags[0] is set).
struct Fp8Tile {
    int group, first, count;
    bool zero;
};
// Inclusive sums over the lanes, by DPP alone: within rows of 16 (row_shr), then
// the last lane of a row to the next (row_bcast15) and of the first half to the
// second (row_bcast31).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
// 256 groups from `base` on, four a lane: their first rows, rows, and tiles up to
// and with each, `before` tiles being ahead of them.
template <int SHIFT>
struct Fp8Groups {
    int at[4], count[4], upto[4];
    // returns the tiles up to the last of them
    __device__ __forceinline__ int read(const Fp8Call& c, int base, int before, bool& bad) {
        int next[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int e = base + 64 * i + (int)__lane_id();
            at[i] = e <= c.experts ? c.starts[e] : c.m;
            next[i] = e < c.experts ? c.starts[e + 1] : c.m;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            count[i] = next[i] - at[i];
            upto[i] = before;
            if (base + 64 * i > c.experts) continue;
            bad |= at[i] < 0 || at[i] > c.m || count[i] < 0;
            upto[i] += wave_scan(tiles(i));
            before = lane_value(upto[i], 63);
        }
        return before;
    }
    __device__ __forceinline__ int tiles(int i) const { return (int)(((uint32_t)count[i] + (1 << SHIFT) - 1) >> SHIFT); }
};
// The tile of a workgroup: place(tiles that there are) says which one, -1: none.
template <int SHIFT, class Place>
__device__ __forceinline__ Fp8Tile fp8_tile(const Fp8Call& c, Place place) {
    constexpr int ROWS = 1 << SHIFT;
    const int E = c.experts, cut = (int)(((uint32_t)c.m + ROWS - 1) >> SHIFT);  // tiles of rows that no group cuts
    if (!c.starts) {
        const int t = place(cut);
        return {0, t << SHIFT, t < 0 ? 0 : min(ROWS, c.m - (t << SHIFT)), false};
    }
    Fp8Groups<SHIFT> g;
    int tiles = 0;
    bool bad = c.starts[0] != 0;
    for (int base = 0; base <= E; base += 256) tiles = g.read(c, base, tiles, bad);
    if (__ballot(bad)) {
        const int t = place(cut);
        if (t == 0) c.flags[0] = 1;
        return {0, t << SHIFT, t < 0 ? 0 : min(ROWS, c.m - (t << SHIFT)), true};
    }
    const int t = place(tiles);
    Fp8Tile r = {0, 0, 0, true};
    if (t < 0 || t >= tiles) return r;
    int before = 0;
    for (int base = 0; base <= E; base += 256) {
        if (E >= 256) before = g.read(c, base, before, bad);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint64_t hit = __ballot(t < g.upto[i] && t >= g.upto[i] - g.tiles(i));
            if (hit) {  // the lanes past the last group have no tiles
                const int j = __builtin_ctzll(hit), e = base + 64 * i + j;
                const int in = (t - (lane_value(g.upto[i], j) - lane_value(g.tiles(i), j))) << SHIFT;
                r = {e, lane_value(g.at[i], j) + in, min(ROWS, lane_value(g.count[i], j) - in), e == E};
            }
        }
    }
    return r;
}
// Tiles there can be: one that is not full a group, and one of no group.
inline int64_t fp8_tiles(const Fp8Call& c, int rows) {
    if (!c.starts) return ((int64_t)c.m + rows - 1) / rows;
    return c.m / rows + (c.experts < c.m ? c.experts : c.m) + 1;
}
// Row i's row of x and of y, -1 where there is none (flags[0] is set).
__device__ __forceinline__ int fp8_x_row(const Fp8Call& c, int i) {
    if (!c.gather) return i;
    const int r = c.gather[i];
    if ((uint32_t)r < (uint32_t)c.x_rows) return r;
    c.flags[0] = 1;
    return -1;
}
__device__ __forceinline__ int fp8_y_row(const Fp8Call& c, int i) {
    if (!c.scatter) return i;
    const int r = c.scatter[i];
    if ((uint32_t)r < (uint32_t)c.y_rows) return r;
    c.flags[0] = 1;
    return -1;
}

#endif

}  // namespace lloom
