// fp8_tile.hip -- products with e4m3 weights for many rows of x: tiles through
// LDS.  Built with the MFMA results in VGPRs (-amdgpu-mfma-vgpr-form): a block's
// sum is read by the VALU right away.
#include "fp8.hpp"
#include "kq_gemm.hpp"

namespace lloom {

#pragma clang fp contract(off)

// A workgroup has BM rows of x and BN of the weight, WM x WN waves with 32 MF x 32
// NF of them each; k moves a block (128) a step through S LDS stages,
//   W [BN][128] e4m3, piece p (16 bytes) of row r at p ^ swizzle(r)
//   X [BM][128] likewise
//   scales [BM] f32 of the block's rows
// every byte by buffer_load .. lds: what is out of the operands (rows past a
// tile's, a last block's bytes past k) has an offset out of the buffer's range
// and arrives as zeros.  Lane (g, c) of a wave takes the same pieces of row c of
// both operands; which bytes meet in which instruction does not matter.  The
// weight is the matrix instructions' A: a lane's sums are of one row of x, so one
// factor (its scale times the weight block's) serves them all.
//
// Where there are few tiles, KS parts of k are summed side by side, each by its own
// waves in its own stages, and meet in LDS at the end.  A step is a wave's way from a
// barrier through its reads to its products, about 0.5 us whatever the tile and
// the stages; two waves a SIMD go it at once.
//
// The numbers go as halves to v_mfma_f32_32x32x16_f16 (EXACT), whose products are
// exact and whose sums are f32, into every type of y.  All 8-bit instructions of
// this chip add groups of eight products with 14 bits from the group's largest on:
// what is under 2^-13 of that is cut, so that where 448 * 448 and its negative meet,
// neighbours of up to 24 vanish.  They have twice the rate (8192^3: 483 us and 961), and
// a caller who would rather have that for F16 and BF16 y says so (MMA_FP8): a block of
// a 16 x 16 tile is then one v_mfma_f32_16x16x128_f8f6f4, the groups and the blocks
// are added in f32, and it is 1.5e-5 of the result in the 2-norm for normal values,
// where F16's own rounding is 2.1e-4 and BF16's 1.7e-3.  Tiles of 32 x 32 for it: 543 us
// for 527, their sums waiting for two chained instructions.
//
// 8192^3 is 1130 TFLOP/s, the MFMA pipe busy 58 % and the VALU with the conversions 62 %;
// by MMA_FP8 2090 to 2280: without the loads 424 us, without LDS and
// barriers too 382, with zeros for data 493, 354 and 301: the clock falls with the
// data's bits, and the loads cost a fifth, nearly all of it though every tile come
// from one place of the L2 (490).
template <int WM_, int WN_, int MF_, int NF_, int S_, int KS_ = 1>
struct Fp8Cfg {
    static constexpr int WM = WM_, WN = WN_, MF = MF_, NF = NF_, S = S_, KS = KS_;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES * KS;  // WAVES: of a part of k
    static constexpr int BM = 32 * WM * MF, BN = 32 * WN * NF;
    static constexpr int SHIFT = BM == 32 ? 5 : BM == 64 ? 6 : BM == 128 ? 7 : 8;
    static constexpr int W = BN * 128, X = BM * 128, XS = BM * 4 < 256 ? 256 : BM * 4, STAGE = W + X + XS;
    static constexpr int W_LOADS = BN / 8 / WAVES, X_LOADS = BM / 8 / WAVES;
    static constexpr int XS_LOADS = (BM / 64 + WAVES - 1) / WAVES < 1 ? 1 : (BM / 64 + WAVES - 1) / WAVES;
    static constexpr int PITCH = 32 * NF * 4 + 16;  // a row of a wave's part of y on its way out, f32 at most
    static constexpr int OUT = WAVES * 32 * PITCH, RING = S * STAGE, SUMS = (KS - 1) * BM * BN * 4;
    static constexpr int LDS = KS * RING + BM * 4 > OUT + SUMS ? KS * RING + BM * 4 : OUT + SUMS;
    static_assert(BM == 1 << SHIFT && W_LOADS * WAVES * 8 == BN && X_LOADS * WAVES * 8 == BM, "whole loads");
    static_assert(128 % (32 * NF) == 0, "a wave's weight rows share their scales");
    static constexpr int DMA = W_LOADS + X_LOADS + XS_LOADS;  // a wave's loads of a stage
    static_assert((S - 1) * DMA <= 63 && LDS <= 160 * 1024, "counts and LDS");
};

__device__ __forceinline__ void fp8_dma16(fp8_v4i b, uint32_t voff, uint32_t soff, uint32_t lds) {
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(b), "s"(soff), "{m0}"(lds) : "memory");
}
__device__ __forceinline__ void fp8_dma4(fp8_v4i b, uint32_t voff, uint32_t soff, uint32_t lds) {
    asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds" ::"v"(voff), "s"(b), "s"(soff), "{m0}"(lds) : "memory");
}
// A load and its wait in one: left to the compiler, the loop would wait for
// it, and so for the whole next stage, in every step.
__device__ __forceinline__ float fp8_load_now(const float* p) {
    float v;
    asm volatile("global_load_dword %0, %1, off\n\ts_waitcnt vmcnt(0)" : "=&v"(v) : "v"(p) : "memory");
    return v;
}
__device__ __forceinline__ int fp8_swizzle(int row) { return (row >> 1) & 7; }
// This wave's reads of LDS are done, and all its loads but the last N.
template <int N>
__device__ __forceinline__ void fp8_landed() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}
// Keeps a tile's sums in the place of the program where they are written: the
// compiler would gather a step's at its end, and spill.
template <class V>
__device__ __forceinline__ void fp8_here(V& v) {
    asm volatile("" : "+v"(v));
}

// A lane's 64 bytes of a row of a stage.
struct Fp8Row {
    uint4 p[4];
};
__device__ __forceinline__ Fp8Row fp8_read(const uint8_t* rows, int row, int h) {
    Fp8Row r;
    const int at = row * 128 + 16 * (h ^ fp8_swizzle(row));
#pragma unroll
    for (int i = 0; i < 4; i++) r.p[i] = *(const uint4*)(rows + (at ^ 32 * i));
    return r;
}
// The same for tiles of 16 x 16: lane (g, c) takes pieces g and g + 4.
__device__ __forceinline__ v8i fp8_read16(const uint8_t* rows, int row, int g) {
    const int at = row * 128 + 16 * (g ^ fp8_swizzle(row));
    const uint4 a = *(const uint4*)(rows + at), b = *(const uint4*)(rows + (at ^ 64));
    return v8i{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

// Place of a workgroup among a grouped call's tiles: a run of them an XCD, walked
// in groups of four, as tile_of walks another call's: what an XCD's workgroups
// have in flight then shares rows of x and of the weight in its L2 (MMA_FP8, 8192 tokens top
// 8 of 64 experts, [2048, 2048]: 389 us in launch order, 377 so; smaller tiles have
// fewer rows of one expert to share, (128, 128) 129 and 140).  t is -1 where none is
// left.
__device__ __forceinline__ void fp8_grouped_place(int tiles, int nbn, int& t, int& bn) {
    const int all = tiles * nbn, each = all >> 3, more = all & 7;
    const int xcd = blockIdx.x & 7, i = blockIdx.x >> 3;
    const int pid = xcd * each + min(xcd, more) + i;
    const int per = 4 * nbn, group = pid / per, in = pid - group * per, size = min(tiles - 4 * group, 4);
    const bool none = i >= each + (xcd < more ? 1 : 0);
    t = none ? -1 : 4 * group + in % size;
    bn = none ? 0 : in / size;
}

template <bool EXACT>
struct Fp8Sums {
    typedef fp8_f16v V;
};
template <>
struct Fp8Sums<false> {
    typedef fp8_f4 V;
};

template <class C, bool EXACT, int YT>
__global__ __launch_bounds__(C::THREADS) void k_fp8_tile(const Fp8Call c, int nbn) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part_k = C::KS > 1 ? wave / C::WAVES : 0, wv = wave - part_k * C::WAVES, wm = wv / C::WN, wn = wv % C::WN;
    int t, bn;
    const Fp8Tile tile = fp8_tile<C::SHIFT>(c, [&](int tiles) {
        if (!c.starts) tile_of(tiles, nbn, t, bn);
        else if (C::BM >= 256) fp8_grouped_place(tiles, nbn, t, bn);
        else t = blockIdx.x / nbn, bn = blockIdx.x - t * nbn;
        return t;
    });
    if (tile.count <= 0) return;
    // block s of this part of k is block `base + s` of the rows; parts are of one
    // length, and what the last has past kb is zeros
    const int n0 = bn * C::BN, steps = tile.zero ? 0 : (c.kb + C::KS - 1) / C::KS, base = part_k * steps;

    const uint8_t* wbase = c.w + ((int64_t)tile.group * c.n + n0) * c.k;
    const fp8_v4i wbuf = fp8_buffer(wbase);
    const int64_t x0 = c.gather ? 0 : tile.first;
    const fp8_v4i xbuf = fp8_buffer((const uint8_t*)c.x + x0 * c.x_stride);
    const fp8_v4i sbuf = fp8_buffer(c.xs + x0 * c.xs_row);
    // A wave's loads of an operand are WAVES * 8 rows apart, so its lanes' pieces
    // are alike in all of them.  Rows of x are looked up in LDS, where they wait
    // for their step (-1: none): held in registers their offsets would spill.
    int* s_from = (int*)(smem + C::KS * C::RING);
    for (int row = threadIdx.x; row < C::BM; row += C::THREADS)
        s_from[row] = row < tile.count && steps ? fp8_x_row(c, tile.first + row) - (int)x0 : -1;
    __syncthreads();
    const int row0 = 8 * wv + (lane >> 3), byte = 16 * ((lane & 7) ^ fp8_swizzle(row0));
    const uint32_t wlast = (uint32_t)min(C::BN, c.n - n0) - 1;
    uint8_t* ring = smem + part_k * C::RING;
    const uint32_t lds0 = lds_addr(ring);
    constexpr int XS_PARTS = C::BM < 64 ? 1 : C::BM / 64;
    struct From {
        int x[C::X_LOADS], s[C::XS_LOADS];
    };
    auto look = [&](From& from) {
#pragma unroll
        for (int i = 0; i < C::X_LOADS; i++) from.x[i] = s_from[row0 + 8 * C::WAVES * i];
#pragma unroll
        for (int i = 0; i < C::XS_LOADS; i++) from.s[i] = s_from[(64 * ((wv + C::WAVES * i) % XS_PARTS) + lane) % C::BM];
    };
    // loads lo .. hi - 1 of the wave's share of a stage
    auto issue = [&](int s, int slot, const From& from, int lo, int hi) {
        const uint32_t st = lds0 + slot * C::STAGE, block = base + s, at = 128u * block;
        const bool past = (int)at + byte >= c.k;  // the last block's pieces past the end of the rows
#pragma unroll
        for (int j = 0; j < C::DMA; j++) {
            if (j < lo || j >= hi) continue;
            if (j < C::X_LOADS) {
                const int i = j, r = from.x[i];
                fp8_dma16(xbuf, past || r < 0 ? FP8_OUT : (uint32_t)r * (uint32_t)c.x_stride + byte, at,
                          st + C::W + 1024 * (wv + C::WAVES * i));
            } else if (j < C::X_LOADS + C::XS_LOADS) {
                const int i = j - C::X_LOADS, r = from.s[i];
                const bool none = r < 0 || (C::KS > 1 && block >= (uint32_t)c.kb);
                const uint32_t sb = C::KS > 1 ? min(block, (uint32_t)c.kb - 1) : block;
                fp8_dma4(sbuf, none ? FP8_OUT : (uint32_t)r * (uint32_t)c.xs_row * 4u, sb * (uint32_t)c.xs_block * 4u,
                         st + C::W + C::X + 256 * ((wv + C::WAVES * i) % XS_PARTS));
            } else {
                const int i = j - C::X_LOADS - C::XS_LOADS;
                const uint32_t off = min((uint32_t)(row0 + 8 * C::WAVES * i), wlast) * (uint32_t)c.k + byte;
                fp8_dma16(wbuf, past ? FP8_OUT : off, at, st + 1024 * (wv + C::WAVES * i));
            }
        }
    };

    // tiles of 32 x 32 (EXACT) or 16 x 16
    constexpr int T = EXACT ? 32 : 16, MT = C::MF * 32 / T, NT = C::NF * 32 / T;
    typedef typename Fp8Sums<EXACT>::V Sums;
    const int ct = lane % T, ht = lane / T;
    Sums acc[NT][MT];
#pragma unroll
    for (int b = 0; b < NT; b++)
#pragma unroll
        for (int a = 0; a < MT; a++) acc[b][a] = Sums{};

    const float* ws = c.ws + ((int64_t)tile.group * c.nb + min((n0 + wn * 32 * C::NF) >> 7, c.nb - 1)) * c.kb;
    float wscale = 0.0f;  // lane l: of block 64 i + l
    auto weight_scale = [&](int s) {
        if ((s & 63) == 0) {
            wscale = fp8_load_now(ws + min(base + s + lane, c.kb - 1));
            if (C::KS > 1 && base + s + lane >= c.kb) wscale = 0.0f;
        }
        return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wscale), s & 63));
    };
    auto read_s = [&](int slot, int a) {
        return *(const float*)(ring + slot * C::STAGE + C::W + C::X + 4 * ((wm * MT + a) * T + ct));
    };
    // Everything of a step's stage is read before its last weight rows are
    // multiplied: there the next stage has had S - 1 steps' time to land, a barrier
    // frees the slot for the one S steps on, and the next step's first operands
    // are read under the products that are left.  That one's loads are issued in
    // parts between those products where a CU has one workgroup: a wave waits at
    // each for its place in the queue (8192^3: all at once 550 us, 536 so; 2048
    // tokens top 8 of 64 experts on (128, 128) tiles 136 and 143).
    From from;
    constexpr int PARTS = C::BM >= 256 ? C::DMA : 1, PART = (C::DMA + PARTS - 1) / PARTS;
    auto bring = [&](int s, int slot, int part) {
        if (s + C::S < steps) issue(s + C::S, slot, from, part * PART, (part + 1) * PART);
    };
    auto turn = [&](int s, int slot) {
        look(from);
        __builtin_amdgcn_sched_barrier(0);
        if (C::S > 2 && s + C::S - 1 < steps) fp8_landed<(C::S - 2) * C::DMA>();
        else fp8_landed<0>();
        __builtin_amdgcn_s_barrier();
        bring(s, slot, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    if (steps) {
        look(from);
#pragma unroll
        for (int i = 0; i < C::S; i++)
            if (i < steps) issue(i, i, from, 0, C::DMA);
        if (steps >= C::S) fp8_landed<(C::S - 1) * C::DMA>();
        else fp8_landed<0>();
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        float f[MT], next[MT];
#pragma unroll
        for (int a = 0; a < MT; a++) f[a] = read_s(0, a);
        int slot = 0;
        if constexpr (EXACT) {
            auto read_w = [&](int slot, int b) { return fp8_read(ring + slot * C::STAGE, (wn * NT + b) * 32 + ct, ht); };
            auto read_x = [&](int slot, int a) { return fp8_read(ring + slot * C::STAGE + C::W, (wm * MT + a) * 32 + ct, ht); };
            Fp8Row x[MT], w = read_w(0, 0);
#pragma unroll
            for (int a = 0; a < MT; a++) x[a] = read_x(0, a);
            for (int s = 0; s < steps; s++) {
                const int after = slot + 1 < C::S ? slot + 1 : 0;
                const float sw = weight_scale(s);
                fp8_h8 xh[MT][8];
#pragma unroll
                for (int a = 0; a < MT; a++) {
                    f[a] *= sw;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        xh[a][2 * i] = fp8_halves(x[a].p[i].x, x[a].p[i].y);
                        xh[a][2 * i + 1] = fp8_halves(x[a].p[i].z, x[a].p[i].w);
                    }
                }
#pragma unroll
                for (int b = 0; b < NT; b++) {
                    const Fp8Row ahead = b < NT - 1 ? read_w(slot, b + 1) : read_w(after, 0);
                    fp8_f16v d[MT];
#pragma unroll
                    for (int a = 0; a < MT; a++) d[a] = fp8_f16v{};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const fp8_h8 w0 = fp8_halves(w.p[i].x, w.p[i].y), w1 = fp8_halves(w.p[i].z, w.p[i].w);
#pragma unroll
                        for (int a = 0; a < MT; a++) {
                            d[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w0, xh[a][2 * i], d[a], 0, 0, 0);
                            d[a] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w1, xh[a][2 * i + 1], d[a], 0, 0, 0);
                        }
                    }
                    if (b == NT - 2) {
                        fp8_here(d[MT - 1]);
                        turn(s, slot);
                    }
#pragma unroll
                    for (int a = 0; a < MT; a++) {
                        if (b == NT - 1) x[a] = read_x(after, a), next[a] = read_s(after, a);
#pragma unroll
                        for (int r = 0; r < 16; r++) acc[b][a][r] = __builtin_fmaf(d[a][r], f[a], acc[b][a][r]);
                        fp8_here(acc[b][a]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                    w = ahead;
                }
#pragma unroll
                for (int a = 0; a < MT; a++) f[a] = next[a];
                slot = after;
            }
        } else {
            // a wave's tiles in turn, the sums of the one LAG before brought home
            // under a tile's products; weight rows are read two tiles' rows ahead
            constexpr int LAG = 2, TILES = NT * MT, TURN = (NT - 3) * MT;
            auto read_w = [&](int slot, int b) { return fp8_read16(ring + slot * C::STAGE, (wn * NT + b) * 16 + ct, ht); };
            auto read_x = [&](int slot, int a) { return fp8_read16(ring + slot * C::STAGE + C::W, (wm * MT + a) * 16 + ct, ht); };
            v8i x[MT], w[3] = {read_w(0, 0), read_w(0, 1), v8i{}};
#pragma unroll
            for (int a = 0; a < MT; a++) x[a] = read_x(0, a);
            for (int s = 0; s < steps; s++) {
                const int after = slot + 1 < C::S ? slot + 1 : 0;
                const float sw = weight_scale(s);
#pragma unroll
                for (int a = 0; a < MT; a++) f[a] *= sw;
                fp8_f4 d[LAG + 1];
#pragma unroll
                for (int t = 0; t < TILES + LAG; t++) {
                    const int b = t / MT, a = t % MT;
                    if (t < TILES) {
                        if (a == 0) w[2] = b + 2 < NT ? read_w(slot, b + 2) : read_w(after, b + 2 - NT);
                        d[t % (LAG + 1)] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[0], x[a], fp8_f4{}, 0, 0, 0, 0, 0, 0);
                        if (t == TURN) {
                            fp8_here(d[t % (LAG + 1)]);
                            turn(s, slot);
                        } else if (C::BM >= 256 && t > TURN && t - TURN < PARTS) {
                            bring(s, slot, t - TURN);
                        }
                        if (b == NT - 1) x[a] = read_x(after, a), next[a] = read_s(after, a);
                        if (a == MT - 1) w[0] = w[1], w[1] = w[2];
                    }
                    if (t >= LAG) {
                        const int u = t - LAG;
                        fp8_f4& v = acc[u / MT][u % MT];
#pragma unroll
                        for (int r = 0; r < 4; r++) v[r] = __builtin_fmaf(d[u % (LAG + 1)][r], f[u % MT], v[r]);
                        fp8_here(v);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int a = 0; a < MT; a++) f[a] = next[a];
                slot = after;
            }
        }
    }
    // every wave has read its last operands before y passes through the ring
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();

    // the parts' sums meet in the first's waves
    if constexpr (C::KS > 1) {
        constexpr int QUADS = T * T / 256;
        float4* sums = (float4*)(smem + C::OUT) + wv * 64 + lane;
        auto at = [&](int p, int b, int a, int r) { return (((p * NT + b) * MT + a) * QUADS + r) * 64 * C::WAVES; };
#pragma unroll
        for (int b = 0; b < NT; b++)
#pragma unroll
            for (int a = 0; a < MT; a++)
#pragma unroll
                for (int r = 0; r < QUADS; r++) {
                    const Sums& v = acc[b][a];
                    if (part_k) sums[at(part_k - 1, b, a, r)] = make_float4(v[4 * r], v[4 * r + 1], v[4 * r + 2], v[4 * r + 3]);
                }
        __syncthreads();
        if (part_k) return;
#pragma unroll
        for (int p = 0; p < C::KS - 1; p++)
#pragma unroll
            for (int b = 0; b < NT; b++)
#pragma unroll
                for (int a = 0; a < MT; a++)
#pragma unroll
                    for (int r = 0; r < QUADS; r++) {
                        const float4 d = sums[at(p, b, a, r)];
                        Sums& v = acc[b][a];
                        v[4 * r] += d.x, v[4 * r + 1] += d.y, v[4 * r + 2] += d.z, v[4 * r + 3] += d.w;
                    }
    }

    // y: a wave's 32 rows at a time through LDS, so that stores run along n
    constexpr int SIZE = YT == T_F32 ? 4 : 2, PER = 16 / SIZE, LANES = 32 * C::NF / PER, ROWS = 64 / LANES;
    uint8_t* part = smem + wv * 32 * C::PITCH;
    const int col0 = n0 + wn * 32 * C::NF, cl = lane % LANES * PER;
#pragma unroll
    for (int a = 0; a < C::MF; a++) {
#pragma unroll
        for (int b = 0; b < NT; b++)
#pragma unroll
            for (int q = 0; q < MT / C::MF; q++)
#pragma unroll
                for (int r = 0; r < T * T / 64; r += 4) {
                    const Sums& v = acc[b][a * (MT / C::MF) + q];
                    uint8_t* p = part + (T * q + ct) * C::PITCH + SIZE * (T * b + 2 * r + 4 * ht);
                    if constexpr (YT == T_F32) {
                        *(float4*)p = make_float4(v[r], v[r + 1], v[r + 2], v[r + 3]);
                    } else {
                        *(uint2*)p =
                            make_uint2(fp8_half_bits<YT>(v[r]) | (uint32_t)fp8_half_bits<YT>(v[r + 1]) << 16,
                                       fp8_half_bits<YT>(v[r + 2]) | (uint32_t)fp8_half_bits<YT>(v[r + 3]) << 16);
                    }
                }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < 32; i += ROWS) {
            const int lr = i + lane / LANES, row = (wm * C::MF + a) * 32 + lr, col = col0 + cl;
            const uint4 v = *(const uint4*)(part + lr * C::PITCH + SIZE * cl);
            if (row >= tile.count || col >= c.n) continue;
            const int yr = fp8_y_row(c, tile.first + row);
            if (yr < 0) continue;
            uint8_t* y = (uint8_t*)c.y + ((int64_t)yr * c.n + col) * SIZE;
            if (col + PER <= c.n) {
                fp8_store16(y, v);
            } else {
                const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < PER; j++) {
                    if (col + j >= c.n) break;
                    if constexpr (YT == T_F32) ((uint32_t*)y)[j] = e[j];
                    else ((uint16_t*)y)[j] = (uint16_t)(e[j >> 1] >> (16 * (j & 1)));
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <class C, bool EXACT, int YT>
static hipError_t tile_of_type(const Fp8Call& c, hipStream_t s) {
    const int nbn = (c.n + C::BN - 1) / C::BN;
    const hipError_t e = set_lds_limit((const void*)k_fp8_tile<C, EXACT, YT>, C::LDS);
    if (e != hipSuccess) return e;
    k_fp8_tile<C, EXACT, YT><<<dim3((uint32_t)(fp8_tiles(c, C::BM) * nbn)), C::THREADS, C::LDS, s>>>(c, nbn);
    return hipGetLastError();
}

template <class C>
static hipError_t tile_with(const Fp8Call& c, hipStream_t s) {
    if constexpr (C::BM < 256) {  // the large tile's sums and halves of both operands would not fit the registers
        if (c.y_type == T_F32) return tile_of_type<C, true, T_F32>(c, s);
        if (!c.cut) return c.y_type == T_F16 ? tile_of_type<C, true, T_F16>(c, s) : tile_of_type<C, true, T_BF16>(c, s);
    }
    return c.y_type == T_F16 ? tile_of_type<C, false, T_F16>(c, s) : tile_of_type<C, false, T_BF16>(c, s);
}

// The largest tile that is mostly full and leaves workgroups for all CUs; where the
// small ones are one round, k in two parts.  The rule is one for all types of y and
// for grouped calls, whose groups' last tiles are taken as half full (a group's rows
// are known on the GPU alone).  us by (rows of x, of the weight) a tile, into bf16:
//   (32, 128) / two parts / (64, 128) / two parts / (128, 128) / two parts:
//     256 rows of [4096, 4096] 25.9 / 17.8 / 26.0 / 22.0 / 36 / 31, 509 36 / 33 / 27.5 / 24.3 / 37 / 32,
//     1000 67 / 63 / 43 / 45 / 40 / 36; 384 of [8192, 8192] 110 / 89 / 77 / 80 / 71 / 65; 96 of [8192,
//     2048] 14.7 / 10.9 / 15.0 / 13.4 / 20.6 / 18.5, 509 37 / 38 / 24.2 / 27.2 / 23.6 / 22.1, 1200 83 /
//     90 / 53 / 64 / 54 / 58, 2048 133 / 150 / 80 / 106 / 71 / 83; 96 of [8192, 512] 6.2 / 6.0 / 6.6 /
//     7.0 / 8.5 / 8.8; 2000 of [264, 2048] 14.6 / 10.8 / 14.9 / 13.2 / 20.6 / 18.5, 44000 of [112, 1264] 42 /
//     52 / 28 / 38 / 30 / 37, 20000 of [300, 4096] 126 / 131 / 79 / 91 / 70 / 78; long outputs of few
//     rows: 32 of [65536, 4096] 64 / 54 / 67 / 60 / 70 / -, 64 76 / 75 / 68 / 64 / 74 / -, 96 104 / 105 /
//     86 / 102 / 77 / -, 64 of [128256, 2048] 83 / 96 / 59 / 71 / 75 / -, 20 of [32768, 8192] 63 / 67 / 70 / 68 / 75 / -
//   grouped, the same: top 8 of 128 experts [1536, 2048], 8, 32 and 128 rows an expert on
//     average, 75 / 84 / 75 / 92 / 98 / 114, 100 / 116 / 91 / 110 / 111 / 132, 241 / 295 / 167 / 222 /
//     172 / 209; of 64 [2048, 2048], 1024 rows 1098 / 1326 / 636 / 860 / 580 / 693; of 4
//     [264, 2048], 256 rows 15.4 / 11.7 / 15.9 / 13.9 / 21.5 / 19.4, 2048 38 / 41 / 24.5 / 29 / 24.6 /
//     22.8; of 8 [1024, 1024], 128 rows 12.8 / 14.5 / 10.5 / 10.1 / 13.6 / 13.4, [512, 4096], 512 rows
//     57 / 53 / 40 / 46 / 39 / 36; of 64 [512, 2048], 8 rows 17.6 / 16.1 / 20.0 / 17.5 / - / -
// With MMA_FP8, and (256, 256) where its rounds of 256 are full by 5 / 8 on average:
//   (64, 128) / (128, 128) / (256, 256): 1200 rows of [8192, 2048] 34 / 35 / 34, 1400 40 / 39 / 34,
//     2304 (288 large tiles) 65 / 61 / 63, 3000 77 / 69 / 66, 4160 (544 of them) 109 / 99 / 94,
//     4400 110 / 97 / 98, 6200 154 / 136 / 131, 8192^3 704 / 601 / 483; grouped, of 8 experts, 2048
//     rows by 2048, [512, 2048] 36 / 39 / 36, [1024, 2048] (272 tiles) 64 / 61 / 63, [1536, 2048] 94 /
//     84 / 70; of 64 [2048, 2048], 1024 rows 462 / 405 / 346
template <class F>
static auto tile_choice(const Fp8Call& c, F with) {
    const int64_t groups = c.experts < c.m ? c.experts : c.m, each = c.starts ? c.m / c.experts : c.m;
    auto count = [&](int rows, int cols) {
        const int64_t tiles = c.starts ? c.m / rows + (groups + 1) / 2 : (c.m + rows - 1) / rows;
        return tiles * ((c.n + cols - 1) / cols);
    };
    const int64_t large = count(256, 256), rounds = (large + 255) / 256;
    // enough rows for tiles of 256, of 128, of 64
    const bool whole = c.starts ? each >= 512 : each > 128, full = c.starts ? each >= 96 : each > 64,
               half = c.starts ? each >= 10 : each > 32;
    if (c.cut && c.nb > 1 && whole && 8 * large >= 5 * 256 * rounds) return with(Fp8Cfg<4, 2, 2, 4, 2>{});
    if (full && count(128, 128) >= 300) return with(Fp8Cfg<2, 2, 2, 2, 2>{});
    if (full && count(64, 128) > 256 && count(128, 128) <= 256 && c.kb >= (c.cut ? 32 : 16))
        return with(Fp8Cfg<2, 2, 2, 2, 2, 2>{});
    const bool parts = c.kb >= 8;
    if (half && count(64, 128) > (parts ? 256 : 128)) return with(Fp8Cfg<2, 2, 1, 2, 2>{});
    if (!parts || count(64, 128) > 256) return with(Fp8Cfg<1, 2, 1, 2, 3>{});
    if (half && count(64, 128) > 128) return with(Fp8Cfg<2, 2, 1, 2, 3, 2>{});
    return with(Fp8Cfg<1, 2, 1, 2, 3, 2>{});
}

hipError_t launch_fp8_tile(const Fp8Call& c, hipStream_t s) {
    if (!c.xs && c.x_rows) return hipErrorInvalidValue;  // rows that are not in 8 bits
    return tile_choice(c, [&](auto cfg) { return tile_with<decltype(cfg)>(c, s); });
}

bool fp8_tile_fits(const Fp8Call& c) {
    return tile_choice(c, [&](auto cfg) {
        typedef decltype(cfg) C;
        return fp8_tiles(c, C::BM) * ((c.n + C::BN - 1) / C::BN) < FP8_THREADS / C::THREADS;
    });
}

}  // namespace lloom
