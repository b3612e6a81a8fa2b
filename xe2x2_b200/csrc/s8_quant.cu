// s8_quant.cu -- per-token s8 quantisation with the MLP's activation in the same pass.
//
// Contract (w4_quant_s8): y = fn(x) in f32, s = max|y| / 127 (1 if 0),
// q = clamp(rint(y / s), -127, 127), the arithmetic of w4_rmsnorm_quant_s8 without its norm
// (kernels/epilogue_quant/rmsnorm_epilogue.cpp:56-70).
#include "tma_util.cuh"
#include "w4_common.cuh"
#include "w4_internal.h"

namespace w4 {
namespace s8q {

constexpr uint32_t kInfBits = 0x7F800000u;

// Eight consecutive values of a row, 16-byte loads.
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const uint4 a = ld_nc_v4(p), b = ld_nc_v4(p + 4);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    } else {
        const uint4 a = ld_nc_v4(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = Conv<T>::to_f2(w[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

template <typename T, int FN>
__device__ __forceinline__ void load_y(const T *xr, int K, int j, float (&y)[8]) {
    load8(xr + j, y);
    if constexpr (FN == W4_FN_SILU_MUL) {
        float u[8];
        load8(xr + K + j, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __fdiv_rn(y[i], 1.f + expf(-y[i])) * u[i];
    } else if constexpr (FN == W4_FN_RELU2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] < 0.f ? 0.f : y[i] * y[i];  // NaN stays NaN
    }
}

__device__ __forceinline__ uint32_t code(float y, float s) {
    const float q = fminf(fmaxf(rintf(__fdiv_rn(y, s)), -127.f), 127.f);
    return (uint32_t)(uint8_t)(int8_t)(int)q;
}

// One CTA per row; the row is read twice (the second time from cache).
template <typename T, int FN>
__global__ void __launch_bounds__(256) quant_s8_kernel(const T *__restrict__ x, int8_t *__restrict__ q,
                                                       float *__restrict__ scale, int K) {
    __shared__ uint32_t sh[8];
    grid_dep_launch();
    grid_dep_wait();
    const int row = blockIdx.x;
    const T *xr = x + (size_t)row * K * (FN == W4_FN_SILU_MUL ? 2 : 1);
    // max over the bit patterns of |y|: they order as the values do, infinity and NaN above all
    uint32_t top = 0;
    for (int j = threadIdx.x * 8; j < K; j += 256 * 8) {
        float y[8];
        load_y<T, FN>(xr, K, j, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(y[i]) & 0x7FFFFFFFu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, sh[i]);
    float s = __fdiv_rn(__uint_as_float(top), 127.f);
    if (s <= 0.f) s = 1.f;
    if (threadIdx.x == 0) scale[row] = s;
    for (int j = threadIdx.x * 8; j < K; j += 256 * 8) {
        uint32_t w[2] = {0u, 0u};
        if (top < kInfBits) {
            float y[8];
            load_y<T, FN>(xr, K, j, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i >> 2] |= code(y[i], s) << (8 * (i & 3));
        }
        *reinterpret_cast<uint2 *>(q + (size_t)row * K + j) = make_uint2(w[0], w[1]);
    }
}

template <typename T>
static int launch(const void *x, int fn, int8_t *q, float *scale, int M, int K, cudaStream_t st) {
    auto kern = fn == W4_FN_SILU_MUL ? quant_s8_kernel<T, W4_FN_SILU_MUL>
                : fn == W4_FN_RELU2  ? quant_s8_kernel<T, W4_FN_RELU2>
                                     : quant_s8_kernel<T, W4_FN_NONE>;
    W4_CUDA_TRY(launch_decode(kern, dim3(M), dim3(256), 0, st, 1, static_cast<const T *>(x), q, scale, K));
    return W4_OK;
}

}  // namespace s8q

int quant_s8(const void *x, int x_dtype, int fn, int8_t *q, float *scale, int M, int K, cudaStream_t st) {
    if (x_dtype == W4_F32) return s8q::launch<float>(x, fn, q, scale, M, K, st);
    if (x_dtype == W4_BF16) return s8q::launch<__nv_bfloat16>(x, fn, q, scale, M, K, st);
    return s8q::launch<__half>(x, fn, q, scale, M, K, st);
}

}  // namespace w4
