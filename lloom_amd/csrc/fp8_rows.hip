// fp8_rows.hip -- rows of activations, and weights, into e4m3 numbers with a
// scale a block (fp8.hpp says how a scale is chosen).
#include "fp8.hpp"

namespace lloom {

#pragma clang fp contract(off)

// v / (1 + exp(-v)) of N values, the quotient as IEEE division rounds it: from -80
// on neither 1 / d nor v / d is near the ends of f32, and one correction of v (1 / d)
// by its residual (Markstein) rounds right: the same as division for every f32 from -80
// on, by trial of all of them (an infinite v gives NaN for infinity; both are NaN in
// e4m3).  27 instructions to 20.
template <int N>
__device__ __forceinline__ void fp8_silu(float (&v)[N]) {
    float least = v[0];
#pragma unroll
    for (int i = 1; i < N; i++) least = fminf(least, v[i]);
    if (__builtin_expect(least < -80.0f, 0)) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = v[i] / (1.0f + expf(-v[i]));
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float d = 1.0f + expf(-v[i]), r = __builtin_amdgcn_rcpf(d), q = v[i] * r;
        v[i] = __builtin_fmaf(-__builtin_fmaf(d, q, -v[i]), r, q);  // so signed, -0 stays -0
    }
}

// ------------------------------------------------------------------- rows --
// A wave takes four blocks (512 values) of a row, 16 lanes and 8 values a lane
// each, of R rows; a workgroup 4 R rows.  The scales go out block by block,
// the rows of a block side by side, as the products read them.  Four rows where
// that leaves workgroups for all CUs several times over.  8192 rows of 4096, f16: 21
// us through the calls (4.8 TB/s read and written; a copy reaches 5.15), the gate 35
// (4.8 TB/s; 42 with IEEE division, when the VALU bound it).
template <int TYPE, bool GATE, int R>
__global__ __launch_bounds__(256) void k_fp8_rows(const void* __restrict__ x, int64_t xs, const void* __restrict__ up,
                                                  int64_t us, int rows, int k, int groups, uint8_t* __restrict__ q,
                                                  float* __restrict__ scales, int64_t ss) {
    __shared__ float s_scale[4][4 * R];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rg = blockIdx.x / groups, g = blockIdx.x - rg * groups;
    const int col = 512 * g + 8 * lane, r0 = 4 * R * rg + R * wave;
    const bool in = col < k;  // k is a multiple of 16: all eight or none
    float v[R][8];
#pragma unroll
    for (int i = 0; i < R; i++) {
        if (in && r0 + i < rows) {
            fp8_load8<TYPE>(x, (r0 + i) * xs + col, v[i]);
            if constexpr (GATE) {
                float u[8];
                fp8_load8<TYPE>(up, (r0 + i) * us + col, u);
                fp8_silu(v[i]);
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] *= u[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] = 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int e = fp8_exponent(row16_max(fp8_largest(v[i])));
        const float f = fp8_inverse(e);
        if (in && r0 + i < rows)
            *(uint2*)(q + (int64_t)(r0 + i) * k + col) =
                make_uint2(fp8_pack4(v[i][0] * f, v[i][1] * f, v[i][2] * f, v[i][3] * f),
                           fp8_pack4(v[i][4] * f, v[i][5] * f, v[i][6] * f, v[i][7] * f));
        if ((lane & 15) == 0) s_scale[lane >> 4][R * wave + i] = fp8_scale(e);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * R; i += 256) {
        const int b = i / (4 * R), r = i - b * (4 * R);
        if (512 * g + 128 * b < k && 4 * R * rg + r < rows) scales[(4 * g + b) * ss + 4 * R * rg + r] = s_scale[b][r];
    }
}

template <int TYPE, bool GATE>
static hipError_t rows_of(const void* x, int64_t xs, const void* up, int64_t us, int64_t rows, int64_t k, void* q,
                          float* scales, int64_t ss, hipStream_t s) {
    const int64_t groups = (k + 511) / 512;
    if (rows * groups >= 8192) {
        k_fp8_rows<TYPE, GATE, 4><<<dim3((uint32_t)(groups * ((rows + 15) / 16))), 256, 0, s>>>(
            x, xs, up, us, (int)rows, (int)k, (int)groups, (uint8_t*)q, scales, ss);
    } else {
        k_fp8_rows<TYPE, GATE, 1><<<dim3((uint32_t)(groups * ((rows + 3) / 4))), 256, 0, s>>>(
            x, xs, up, us, (int)rows, (int)k, (int)groups, (uint8_t*)q, scales, ss);
    }
    return hipGetLastError();
}

hipError_t launch_fp8_rows(int type, const void* x, int64_t x_stride, const void* up, int64_t up_stride, int64_t rows,
                           int64_t k, void* q, float* scales, int64_t scales_stride, hipStream_t s) {
#define ROWS(T)                                                                                               \
    return up ? rows_of<T, true>(x, x_stride, up, up_stride, rows, k, q, scales, scales_stride, s)            \
              : rows_of<T, false>(x, x_stride, nullptr, 0, rows, k, q, scales, scales_stride, s)
    switch (type) {
        case T_F32: ROWS(T_F32);
        case T_F16: ROWS(T_F16);
        default: ROWS(T_BF16);
    }
#undef ROWS
}

// ---------------------------------------------------------------- weights --
// A workgroup a block of 128 x 128: 16 lanes a row, 16 rows at once, 8 times.
template <int TYPE>
__global__ __launch_bounds__(256) void k_fp8_weights(const void* __restrict__ w, int n, int k, int nb, int kb,
                                                     uint8_t* __restrict__ q, float* __restrict__ scales) {
    __shared__ uint32_t s_size[4];
    const int64_t id = blockIdx.x;
    const int b = (int)(id % kb), o = (int)(id / kb % nb);
    const int64_t plane = id / ((int64_t)kb * nb);
    const int col = 128 * b + 8 * (threadIdx.x & 15), row0 = 128 * o + (threadIdx.x >> 4);
    float v[8][8];
    uint32_t size = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int row = row0 + 16 * i;
        if (row < n && col < k) {
            fp8_load8<TYPE>(w, (plane * n + row) * k + col, v[i]);
            size = max(size, fp8_largest(v[i]));
        }
    }
    size = column_max(row16_max(size));
    if ((threadIdx.x & 63) == 0) s_size[threadIdx.x >> 6] = size;
    __syncthreads();
    const int e = fp8_exponent(max(max(s_size[0], s_size[1]), max(s_size[2], s_size[3])));
    const float f = fp8_inverse(e);
    if (threadIdx.x == 0) scales[id] = fp8_scale(e);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int row = row0 + 16 * i;
        if (row < n && col < k)
            *(uint2*)(q + (plane * n + row) * k + col) =
                make_uint2(fp8_pack4(v[i][0] * f, v[i][1] * f, v[i][2] * f, v[i][3] * f),
                           fp8_pack4(v[i][4] * f, v[i][5] * f, v[i][6] * f, v[i][7] * f));
    }
}

hipError_t launch_fp8_weights(int type, const void* w, int64_t planes, int64_t n, int64_t k, void* q, float* scales,
                              hipStream_t s) {
    const int64_t nb = (n + 127) / 128, kb = (k + 127) / 128;
    const dim3 grid((uint32_t)(planes * nb * kb));
    switch (type) {
        case T_F32: k_fp8_weights<T_F32><<<grid, 256, 0, s>>>(w, (int)n, (int)k, (int)nb, (int)kb, (uint8_t*)q, scales); break;
        case T_F16: k_fp8_weights<T_F16><<<grid, 256, 0, s>>>(w, (int)n, (int)k, (int)nb, (int)kb, (uint8_t*)q, scales); break;
        default: k_fp8_weights<T_BF16><<<grid, 256, 0, s>>>(w, (int)n, (int)k, (int)nb, (int)kb, (uint8_t*)q, scales); break;
    }
    return hipGetLastError();
}

}  // namespace lloom
