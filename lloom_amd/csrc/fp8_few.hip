// fp8_few.hip -- products with e4m3 weights for few rows of x.
#include "fp8.hpp"

namespace lloom {

#pragma clang fp contract(off)

// A workgroup has NT tiles of 16 weight rows and a tile of up to 16 rows of x;
// its W waves take blocks of 128 of k in turn, the loads of the next D under way,
// and meet in LDS.  The e4m3 numbers go to the matrix cores as halves
// (v_mfma_f32_16x16x32_f16), whose products are exact and whose sums are f32: the
// 8-bit instructions add groups of eight products with 14 bits.  Lane (g, r)
// holds bytes 16 g .. + 15 and 64 + 16 g .. + 15 of a block of row r, of the
// weight and of x alike, so a load is 64 bytes of each of 16 rows; which bytes
// meet in which instruction does not matter.  x of another type is brought into
// 8 bits in LDS by each workgroup, under the first weights' loads.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t few_buffer(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)FP8_OUT, 0x00020000);
}
__device__ __forceinline__ uint4 few_load(__amdgpu_buffer_rsrc_t b, uint32_t off) {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0));
}

template <int XT, int W, int NT, int D>
__global__ __launch_bounds__(64 * W) void k_fp8_few(const Fp8Call c, int nblocks) {
    constexpr bool FUSED = XT != T_E4M3;
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r16 = lane & 15;
    const int t = blockIdx.x / nblocks, n0 = 16 * NT * (blockIdx.x - t * nblocks);
    const Fp8Tile tile = fp8_tile<4>(c, t);
    if (tile.count <= 0) return;  // the same in all waves
    const int i = tile.first + r16;
    const bool mine = r16 < tile.count;
    fp8_f4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) acc[j] = fp8_f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (!tile.zero) {
        const __amdgpu_buffer_rsrc_t wbuf = few_buffer(c.w + ((int64_t)tile.group * c.n + n0) * c.k);
        // the 16 NT rows are of one row of blocks
        const float* ws = c.ws + ((int64_t)tile.group * c.nb + (n0 >> 7)) * c.kb;
        uint32_t wrow[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) wrow[j] = n0 + 16 * j + r16 < c.n ? (uint32_t)(16 * j + r16) * (uint32_t)c.k : FP8_OUT;
        const int64_t x0 = c.gather ? 0 : tile.first;
        const int from = mine && !FUSED ? fp8_x_row(c, i) : -1, xr = from < 0 ? -1 : from - (int)x0;
        const __amdgpu_buffer_rsrc_t xbuf = few_buffer((const uint8_t*)c.x + x0 * c.x_stride);
        const float* xs = FUSED ? nullptr : c.xs + (x0 + max(xr, 0)) * c.xs_row;
        const uint32_t xrow = xr >= 0 ? (uint32_t)xr * (uint32_t)c.x_stride : FP8_OUT;

        uint4 q[D][NT][2], x[D][2];
        float sw[D], sx[D];
        auto load = [&](int b, int u) {
            const uint32_t o = 128u * b + 16u * g;
            const bool in0 = o < (uint32_t)c.k, in1 = o + 64 < (uint32_t)c.k;
#pragma unroll
            for (int j = 0; j < NT; j++) {
                q[u][j][0] = few_load(wbuf, in0 ? wrow[j] + o : FP8_OUT);
                q[u][j][1] = few_load(wbuf, in1 ? wrow[j] + o + 64 : FP8_OUT);
            }
            const int there = min(b, c.kb - 1);
            sw[u] = ws[there];
            if constexpr (!FUSED) {
                x[u][0] = few_load(xbuf, in0 ? xrow + o : FP8_OUT);
                x[u][1] = few_load(xbuf, in1 ? xrow + o + 64 : FP8_OUT);
                sx[u] = xs[there * c.xs_block];
            }
        };
#pragma unroll
        for (int u = 0; u < D; u++) load(wave + W * u, u);
        // x [row][pitch] e4m3 (a pitch of 16 odd pieces: rows fall on all banks),
        // then scales [row][block]
        const int pitch = (c.k + 127) / 128 * 128 + 16;
        float* s_scale = (float*)(smem + tile.count * pitch);
        if constexpr (FUSED) {
            for (int b = wave * 4 + g; b < tile.count * c.kb; b += 4 * W) {
                const int row = b / c.kb, blk = b - row * c.kb, col = 128 * blk + 8 * r16;
                const int from = fp8_x_row(c, tile.first + row);
                float v[8] = {};
                if (col < c.k && from >= 0) fp8_load8<XT>(c.x, from * c.x_stride + col, v);
                const int e = fp8_exponent(row16_max(fp8_largest(v)));
                const float f = fp8_inverse(e);
                *(uint2*)(smem + row * pitch + col) = make_uint2(fp8_pack4(v[0] * f, v[1] * f, v[2] * f, v[3] * f),
                                                                 fp8_pack4(v[4] * f, v[5] * f, v[6] * f, v[7] * f));
                if (r16 == 0) s_scale[b] = fp8_scale(e);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
        }
        const int xl = min(r16, tile.count - 1);  // lanes of no row repeat the last: their sums are not stored
        for (int b0 = wave; b0 < c.kb; b0 += W * D) {
#pragma unroll
            for (int u = 0; u < D; u++) {
                const int b = b0 + W * u;
                if (FUSED) {
                    const uint8_t* p = smem + xl * pitch + 128 * min(b, c.kb - 1) + 16 * g;
                    x[u][0] = *(const uint4*)p;
                    x[u][1] = *(const uint4*)(p + 64);
                    sx[u] = s_scale[xl * c.kb + min(b, c.kb - 1)];
                }
                fp8_h8 xh[4];
#pragma unroll
                for (int p = 0; p < 2; p++) {
                    xh[2 * p] = fp8_halves(x[u][p].x, x[u][p].y);
                    xh[2 * p + 1] = fp8_halves(x[u][p].z, x[u][p].w);
                }
                const float f = b < c.kb ? sx[u] * sw[u] : 0.0f;
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    fp8_f4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        const uint4 v = q[u][j][p];
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp8_halves(v.x, v.y), xh[2 * p], d, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(fp8_halves(v.z, v.w), xh[2 * p + 1], d, 0, 0, 0);
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[j][r] = __builtin_fmaf(d[r], f, acc[j][r]);
                }
                load(b + W * D, u);
            }
        }
    }
    __syncthreads();  // the sums take x's place
    float4* s_sum = (float4*)smem;
#pragma unroll
    for (int j = 0; j < NT; j++) s_sum[(wave * NT + j) * 64 + lane] = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
    __syncthreads();
    if (wave >= NT || !mine) return;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < W; u++) {
        const float4 p = s_sum[(u * NT + wave) * 64 + lane];
        v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
    }
    const int yr = fp8_y_row(c, i), col = n0 + 16 * wave + 4 * g;
    if (yr < 0) return;
    const int64_t at = (int64_t)yr * c.n + col;
    const bool wide = c.n % 4 == 0;
    if (c.y_type == T_F32) fp8_store4<T_F32>(c.y, at, v, c.n - col, wide);
    else if (c.y_type == T_F16) fp8_store4<T_F16>(c.y, at, v, c.n - col, wide);
    else fp8_store4<T_BF16>(c.y, at, v, c.n - col, wide);
}

static int64_t few_lds(int64_t rows, int64_t k) {
    const int64_t kb = (k + 127) / 128;
    return (rows < 16 ? rows : 16) * (kb * 128 + 16 + kb * 4);
}

// One row of few blocks, and the few rows of a grouped call, each of which meets
// few of them in a tile, are cheaper brought into 8 bits by every workgroup than
// in a launch before (2.3 us): m = 1 on [6144, 2048] 5.9 against 8.0 us, 16 rows
// 8.7 against 8.5, 32 tokens of 128 experts (16 rows at once in LDS) 84 against 58.
bool fp8_few_fuses(int x_type, int64_t rows, int64_t k, bool grouped) {
    if (x_type == T_E4M3 || rows > 16) return false;
    return few_lds(rows, k) <= 65536 && (grouped || rows * ((k + 127) / 128) <= 64);
}

template <int XT, int W, int NT, int D>
static hipError_t few_of(const Fp8Call& c, hipStream_t s) {
    const int nblocks = (c.n + 16 * NT - 1) / (16 * NT);
    int lds = W * NT * 64 * 16;
    if (XT != T_E4M3 && few_lds(c.m, c.k) > lds) lds = (int)few_lds(c.m, c.k);
    k_fp8_few<XT, W, NT, D><<<dim3((uint32_t)(fp8_tiles(c, 16) * nblocks)), 64 * W, lds, s>>>(c, nblocks);
    return hipGetLastError();
}

// How many weight rows a workgroup has, by how many there are and how many rows
// of x read them.  us by (W, NT, D): [6144, 2048] 1 row (8, 1, 2) 6.0, (4, 2, 2)
// 5.9, (4, 4, 1) 8.1, 16 rows 7.2, 6.2, 7.9; [2048, 8192] 1 row 7.6, 12.1, 19.6;
// [8192, 8192] 1 row 15.9, 18.1, 24.5, 16 rows 20.7, 15.9, 23.1; 32 tokens top 8 of
// 128 experts, [1536, 2048] 85, 57, 55 and [2048, 768] 76, 43, 33; 4 tokens (29
// experts, [1536, 2048]) 24.3, 20.0, 22.7.
template <int XT>
static hipError_t few_with(const Fp8Call& c, hipStream_t s) {
    const int64_t tiles = (c.starts ? (c.experts < c.m ? c.experts : c.m) : 1) * ((c.n + 15) / 16);
    if (tiles >= 4096) return few_of<XT, 4, 4, 1>(c, s);
    if (tiles >= 1024 || (tiles >= 256 && c.m > 4)) return few_of<XT, 4, 2, 2>(c, s);
    return few_of<XT, 8, 1, 2>(c, s);
}

hipError_t launch_fp8_few(int x_type, const Fp8Call& c, hipStream_t s) {
    switch (x_type) {
        case T_F32: return few_with<T_F32>(c, s);
        case T_F16: return few_with<T_F16>(c, s);
        case T_BF16: return few_with<T_BF16>(c, s);
        default: return few_with<T_E4M3>(c, s);
    }
}

}  // namespace lloom
