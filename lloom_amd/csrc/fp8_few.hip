// fp8_few.hip -- products with e4m3 weights for few rows of x.
#include "fp8.hpp"

namespace lloom {

#pragma clang fp contract(off)

// A workgroup has NT tiles of 16 weight rows and MT of 16 rows of x; its W waves
// take blocks of 128 of k in turn, the loads of the next D under way, and meet in
// LDS.  The e4m3 numbers go to the matrix cores as halves
// (v_mfma_f32_16x16x32_f16), whose products are exact and whose sums are f32: the
// 8-bit instructions add groups of eight products with 14 bits.  Lane (g, r)
// holds bytes 16 g .. + 15 and 64 + 16 g .. + 15 of a block of row r, of the
// weight and of x alike, so a load is 64 bytes of each of 16 rows; which bytes
// meet in which instruction does not matter.  x of another type is brought into
// 8 bits in LDS by each workgroup, under the first weights' loads.
//
// One row is bound by what a launch and a few loads in a row take (12.6 MB in 6 us),
// a decode step's experts by the read (276 MB in 46 to 51 us), 17 rows and more by the
// caches, from which each tile reads its rows of x again (32 of [8192, 8192] 21 us for
// 67 MB; more waves, more loads under way 20 to 24).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t few_buffer(const void* p) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)FP8_OUT, 0x00020000);
}
__device__ __forceinline__ float few_load4(__amdgpu_buffer_rsrc_t b, uint32_t off) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(b, off, 0, 0));
}
__device__ __forceinline__ uint4 few_load(__amdgpu_buffer_rsrc_t b, uint32_t off) {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0));
}

template <int XT, int W, int MT, int NT, int D>
__global__ __launch_bounds__(64 * W) void k_fp8_few(const Fp8Call c, int nblocks) {
    constexpr bool FUSED = XT != T_E4M3;
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r16 = lane & 15;
    const int t = blockIdx.x / nblocks, n0 = 16 * NT * (blockIdx.x - t * nblocks);
    const Fp8Tile tile = fp8_tile<MT == 1 ? 4 : 5>(c, [&](int) { return t; });
    if (tile.count <= 0) return;  // the same in all waves
    fp8_f4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int a = 0; a < MT; a++) acc[j][a] = fp8_f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (!tile.zero) {
        const __amdgpu_buffer_rsrc_t wbuf = few_buffer(c.w + ((int64_t)tile.group * c.n + n0) * c.k);
        // the 16 NT rows are of one row of blocks
        const float* ws = c.ws + ((int64_t)tile.group * c.nb + (n0 >> 7)) * c.kb;
        uint32_t wrow[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) wrow[j] = n0 + 16 * j + r16 < c.n ? (uint32_t)(16 * j + r16) * (uint32_t)c.k : FP8_OUT;
        const int64_t x0 = c.gather ? 0 : tile.first;
        const __amdgpu_buffer_rsrc_t xbuf = few_buffer((const uint8_t*)c.x + x0 * c.x_stride);
        const __amdgpu_buffer_rsrc_t sbuf = few_buffer(c.xs + x0 * c.xs_row);
        uint32_t xrow[MT], srow[MT];
#pragma unroll
        for (int a = 0; a < MT; a++) {
            const int row = 16 * a + r16, from = !FUSED && row < tile.count ? fp8_x_row(c, tile.first + row) : -1;
            xrow[a] = from >= 0 ? (uint32_t)(from - (int)x0) * (uint32_t)c.x_stride : FP8_OUT;
            srow[a] = from >= 0 ? (uint32_t)(from - (int)x0) * (uint32_t)c.xs_row * 4u : FP8_OUT;
        }

        uint4 q[D][NT][2], x[D][MT][2];
        float sw[D], sx[D][MT];
        auto load = [&](int b, int u) {
            const uint32_t o = 128u * b + 16u * g;
            const bool in0 = o < (uint32_t)c.k, in1 = o + 64 < (uint32_t)c.k;
#pragma unroll
            for (int j = 0; j < NT; j++) {
                q[u][j][0] = few_load(wbuf, in0 ? wrow[j] + o : FP8_OUT);
                q[u][j][1] = few_load(wbuf, in1 ? wrow[j] + o + 64 : FP8_OUT);
            }
            sw[u] = ws[min(b, c.kb - 1)];
            if constexpr (!FUSED) {
#pragma unroll
                for (int a = 0; a < MT; a++) {
                    x[u][a][0] = few_load(xbuf, in0 ? xrow[a] + o : FP8_OUT);
                    x[u][a][1] = few_load(xbuf, in1 ? xrow[a] + o + 64 : FP8_OUT);
                    sx[u][a] = few_load4(sbuf, b < c.kb ? srow[a] + (uint32_t)b * (uint32_t)c.xs_block * 4u : FP8_OUT);
                }
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
                    x[u][0][0] = *(const uint4*)p;
                    x[u][0][1] = *(const uint4*)(p + 64);
                    sx[u][0] = s_scale[xl * c.kb + min(b, c.kb - 1)];
                }
                fp8_h8 xh[MT][4];
                float f[MT];
#pragma unroll
                for (int a = 0; a < MT; a++) {
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        xh[a][2 * p] = fp8_halves(x[u][a][p].x, x[u][a][p].y);
                        xh[a][2 * p + 1] = fp8_halves(x[u][a][p].z, x[u][a][p].w);
                    }
                    f[a] = b < c.kb ? sx[u][a] * sw[u] : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    fp8_f4 d[MT];
#pragma unroll
                    for (int a = 0; a < MT; a++) d[a] = fp8_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        const uint4 v = q[u][j][p];
                        const fp8_h8 lo = fp8_halves(v.x, v.y), hi = fp8_halves(v.z, v.w);
#pragma unroll
                        for (int a = 0; a < MT; a++) {
                            d[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, xh[a][2 * p], d[a], 0, 0, 0);
                            d[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, xh[a][2 * p + 1], d[a], 0, 0, 0);
                        }
                    }
#pragma unroll
                    for (int a = 0; a < MT; a++)
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[j][a][r] = __builtin_fmaf(d[a][r], f[a], acc[j][a][r]);
                }
                load(b + W * D, u);
            }
        }
    }
    __syncthreads();  // the sums take x's place
    float4* s_sum = (float4*)smem;
#pragma unroll
    for (int j = 0; j < NT; j++)
#pragma unroll
        for (int a = 0; a < MT; a++) {
            const fp8_f4& d = acc[j][a];
            s_sum[((wave * NT + j) * MT + a) * 64 + lane] = make_float4(d[0], d[1], d[2], d[3]);
        }
    __syncthreads();
    for (int p = wave; p < NT * MT; p += W) {
        const int j = p / MT, row = 16 * (p - j * MT) + r16;
        if (row >= tile.count) continue;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < W; u++) {
            const float4 s = s_sum[(u * NT * MT + p) * 64 + lane];
            v[0] += s.x, v[1] += s.y, v[2] += s.z, v[3] += s.w;
        }
        const int yr = fp8_y_row(c, tile.first + row), col = n0 + 16 * j + 4 * g;
        if (yr < 0) continue;
        const int64_t at = (int64_t)yr * c.n + col;
        if (c.y_type == T_F32) fp8_store4<T_F32>(c.y, at, v, c.n - col);
        else if (c.y_type == T_F16) fp8_store4<T_F16>(c.y, at, v, c.n - col);
        else fp8_store4<T_BF16>(c.y, at, v, c.n - col);
    }
}

static int64_t few_lds(int64_t rows, int64_t k) {
    const int64_t kb = (k + 127) / 128;
    return (rows < 16 ? rows : 16) * (kb * 128 + 16 + kb * 4);
}

// One row of few blocks, and a grouped call's rows where an expert has no more than
// one on average, are cheaper brought into 8 bits by every workgroup than in a
// launch before (2.3 us): one row of [6144, 2048] 5.9 against 8.0 us, 16 rows 8.7
// against 8.5; top 8 of 128 experts, [1536, 2048], 4 tokens 19.8 / 21.0, 16 47.2 / 46.7,
// 32 60 / 57, 64 77 / 68; 32 tokens top 2 of 64, [1024, 1024], 12.0 / 14.6.
bool fp8_few_fuses(int x_type, int64_t rows, int64_t k, int64_t experts, bool grouped) {
    if (x_type == T_E4M3) return false;
    if (grouped) return (rows <= 16 || rows <= experts) && few_lds(rows, k) <= 40960;
    return rows <= 16 && rows * ((k + 127) / 128) <= 64 && few_lds(rows, k) <= 65536;
}

// W waves, MT tiles of 16 rows of x, NT of the weight, loads of D blocks under way.
template <int W_, int MT_, int NT_, int D_>
struct FewCfg {
    static constexpr int W = W_, MT = MT_, NT = NT_, D = D_;
};
template <int XT, class C>
static hipError_t few_of(const Fp8Call& c, hipStream_t s) {
    constexpr int W = C::W, MT = C::MT, NT = C::NT;
    const int nblocks = (c.n + 16 * NT - 1) / (16 * NT);
    int lds = W * NT * MT * 64 * 16;
    if (XT != T_E4M3 && few_lds(c.m, c.k) > lds) lds = (int)few_lds(c.m, c.k);
    k_fp8_few<XT, W, MT, NT, C::D><<<dim3((uint32_t)(fp8_tiles(c, 16 * MT) * nblocks)), 64 * W, lds, s>>>(c, nblocks);
    return hipGetLastError();
}

// A workgroup's tile: as large as leaves about 200 of them, since each tile reads
// its rows of x and of the weight again, from the caches.  us by (rows of x, of
// the weight) a tile:
//   (16, 16) with 8 waves / (16, 32): 1 row of [2048, 8192] 7.6 / 12.1, of [8192,
//     8192] 15.9 / 18.1; 16 rows of [6144, 2048] 7.2 / 6.2, of [8192, 8192] 20.7 / 15.9
//   (16, 32) / (32, 32) / (32, 64) / (64, 64): 32 rows of [4096, 4096] 8.9 / 10.7 /
//     14.7 / 16.7; 64 of [2048, 8192] 14.0 / 17.5 / 24.9 / 32.7, of [8192, 2048]
//     15.1 / 10.9 / 9.7 / 12.1; 128 of [2048, 2048] 8.9 / 7.2 / 9.3 / 11.9; 96 of
//     [8192, 8192] 70 / 51 / 48 / 35
//   grouped, (16, 16) / (16, 32) / (16, 64): 32 tokens top 8 of 128 experts, [1536,
//     2048] 85 / 57 / 55 and [2048, 768] 76 / 43 / 33; 4 tokens (29 experts) 24 / 20 /
//     23; (32, 64) is slower (67), most tiles being far from full
template <bool E4M3, class F>
static auto few_choice(const Fp8Call& c, F with) {
    const int64_t groups = c.starts ? (c.experts < c.m ? c.experts : c.m) : 1, tiles = groups * ((c.n + 15) / 16);
    if constexpr (E4M3) {
        if (!c.starts && c.m > 16) {
            auto enough = [&](int rows, int cols) {
                return (int64_t)((c.m + rows - 1) / rows) * ((c.n + cols - 1) / cols) >= 200;
            };
            if (enough(32, 64)) return with(FewCfg<4, 2, 4, 1>{});
            if (enough(32, 32)) return with(FewCfg<4, 2, 2, 1>{});
            return with(FewCfg<4, 1, 2, 2>{});
        }
    }
    if (tiles >= 4096) return with(FewCfg<4, 1, 4, 1>{});
    if (tiles >= 1024 || (tiles >= 256 && c.m > 4)) return with(FewCfg<4, 1, 2, 2>{});
    return with(FewCfg<8, 1, 1, 2>{});
}

template <int XT>
static hipError_t few_with(const Fp8Call& c, hipStream_t s) {
    return few_choice<XT == T_E4M3>(c, [&](auto cfg) { return few_of<XT, decltype(cfg)>(c, s); });
}

bool fp8_few_fits(int x_type, const Fp8Call& c) {
    auto fits = [&](auto cfg) {
        typedef decltype(cfg) C;
        return fp8_tiles(c, 16 * C::MT) * ((c.n + 16 * C::NT - 1) / (16 * C::NT)) < FP8_THREADS / (64 * C::W);
    };
    return x_type == T_E4M3 ? few_choice<true>(c, fits) : few_choice<false>(c, fits);
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
