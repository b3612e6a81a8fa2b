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

// Eight consecutive values of a row: 16-byte loads, and their values.
template <typename T> struct Raw8 {
    static constexpr int W = 2 * (int)sizeof(T);  // 32-bit words
    uint32_t w[W];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const uint4 u = ld_nc_v4(reinterpret_cast<const uint32_t *>(p) + i);
            w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(w[i]);
            } else {
                const float2 f = Conv<T>::to_f2(w[i / 2]);
                v[i] = i & 1 ? f.y : f.x;
            }
        }
    }
};

// g / (1 + exp(-g)) with the hardware's base-2 exponential (relative error 2^-22, and that of its rounded
// argument, |g| 2^-24) and reciprocal (2^-23; 0 where the exponential is infinite or near it): about
// 6e-7 for |g| up to 8, a thousandth of a code.  expf and a division made this kernel bound by its
// instructions (37 a value, 60 us where this takes 45).
__device__ __forceinline__ float silu(float g) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return g * r;
}

// Eight inputs of fn (with SwiGLU: of the gate and of the up half) and fn of them.
template <typename T, int FN> struct In8 {
    Raw8<T> a, b;
    __device__ __forceinline__ void load(const T *xr, int K, int j) {
        a.load(xr + j);
        if constexpr (FN == W4_FN_SILU_MUL) b.load(xr + K + j);
    }
    __device__ __forceinline__ void zero() {
        a.zero();
        if constexpr (FN == W4_FN_SILU_MUL) b.zero();
    }
    __device__ __forceinline__ void values(float (&y)[8]) const {
        a.values(y);
        if constexpr (FN == W4_FN_SILU_MUL) {
            float u[8];
            b.values(u);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = silu(y[i]) * u[i];
        } else if constexpr (FN == W4_FN_RELU2) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = y[i] < 0.f ? 0.f : y[i] * y[i];  // NaN stays NaN
        }
    }
};

// max(|a|, |b|, |c|), NaN if one is.
__device__ __forceinline__ float absmax3(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float absmax8(const float (&y)[8], float top) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) top = absmax3(top, y[i], y[i + 1]);
    return top;
}

// rint(y / s) as eight signed bytes.  y * (1 / s) is within 2 roundings of the quotient (1.5e-5 at
// 127), so its nearest whole number is the quotient's unless it lies that close to a half; then the
// division decides.  Adding 1.5 * 2^23 rounds to the nearest whole number, ties to even, and leaves it
// in the low bits.
__device__ __forceinline__ uint2 codes8(const float (&y)[8], float s, float inv) {
    constexpr float kRound = 12582912.f;
    float r[8], off[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        r[i] = fmaf(y[i], inv, kRound);
        off[i] = fmaf(y[i], inv, kRound - r[i]);
    }
    if (absmax8(off, 0.f) > 0.4999f) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (fabsf(off[i]) > 0.4999f) r[i] = __fdiv_rn(y[i], s) + kRound;
    }
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(r[i]);
    return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

struct Scale {
    float s, inv;
    bool finite;
};
// From the largest bit pattern of |y|: they order as the values do, infinity and NaN above all.
__device__ __forceinline__ Scale scale_of(uint32_t top) {
    Scale r;
    r.s = __fdiv_rn(__uint_as_float(top), 127.f);
    if (r.s <= 0.f) r.s = 1.f;
    r.inv = __fdiv_rn(1.f, r.s);
    r.finite = top < kInfBits;
    return r;
}
__device__ __forceinline__ uint2 quant8(const float (&y)[8], const Scale &c) {
    if (!c.finite) return make_uint2(0u, 0u);
    if (c.s >= 1e-30f) return codes8(y, c.s, c.inv);
    // A scale whose reciprocal may overflow: the same quotients, both sides times 2^100.  A subnormal scale
    // may have rounded down by more than the last code's half: the quotient is held to 127.
    const float s = c.s * 0x1p100f, most = 127.f * s;
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = fminf(fmaxf(y[i] * 0x1p100f, -most), most);
    return codes8(z, s, __fdiv_rn(1.f, s));
}

// A row on TPR threads, held in registers from the one read to the store: VPT vectors of eight values a
// thread.  CTAs loop over rows, and a row's loads are issued before the row ahead of it is reduced
// (not with 1024 threads, whose registers are taken).  Bound by memory (5 bytes a value with SwiGLU)
// and the instructions per value about equally; at 24,576 x 1856, bf16 -> 45 us, 5.0 TB/s, where
// one CTA a row with a second read and a division per value took 139.
template <typename T, int FN, int TPR, int VPT>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR)
quant_s8_kernel(const T *__restrict__ x, int8_t *__restrict__ q, float *__restrict__ scale, int M, int K) {
    constexpr int RPC = TPR < 256 ? 256 / TPR : 1;  // rows of a CTA
    constexpr bool AHEAD = TPR < 1024;
    __shared__ uint32_t sh[2][RPC][TPR / 32];
    grid_dep_launch();
    grid_dep_wait();
    const int rl = threadIdx.x / TPR, t = threadIdx.x % TPR;
    const size_t width = (size_t)K * (FN == W4_FN_SILU_MUL ? 2 : 1);
    In8<T, FN> in[VPT];
    auto fetch = [&](long row) {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int j = (v * TPR + t) * 8;
            if (row < M && j < K) in[v].load(x + row * width, K, j);
            else in[v].zero();
        }
    };
    long row = (long)blockIdx.x * RPC + rl;
    if (AHEAD) fetch(row);
    // all rows of the CTA take the same number of turns
    for (int turn = 0; row - rl < M; row += (long)gridDim.x * RPC, turn ^= 1) {
        if (!AHEAD) fetch(row);
        float y[VPT][8], most = 0.f;
#pragma unroll
        for (int v = 0; v < VPT; ++v) in[v].values(y[v]);
        if (AHEAD) fetch(row + (long)gridDim.x * RPC);
#pragma unroll
        for (int v = 0; v < VPT; ++v) most = absmax8(y[v], most);
        uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
        if constexpr (TPR > 32) {
            if ((t & 31) == 0) sh[turn][rl][t / 32] = top;
            __syncthreads();
            top = __reduce_max_sync(0xffffffffu, (t & 31) < TPR / 32 ? sh[turn][rl][t & 31] : 0u);
        }
        if (row >= M) continue;
        const Scale c = scale_of(top);
        if (t == 0) scale[row] = c.s;
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const int j = (v * TPR + t) * 8;
            if (j < K) *reinterpret_cast<uint2 *>(q + (size_t)row * K + j) = quant8(y[v], c);
        }
    }
}

// Rows too long for the registers of a CTA: read twice, the second time from cache.
template <typename T, int FN>
__global__ void __launch_bounds__(1024)
quant_s8_long_kernel(const T *__restrict__ x, int8_t *__restrict__ q, float *__restrict__ scale, int K) {
    __shared__ uint32_t sh[32];
    grid_dep_launch();
    grid_dep_wait();
    const size_t row = blockIdx.x;
    const T *xr = x + row * K * (FN == W4_FN_SILU_MUL ? 2 : 1);
    float most = 0.f;
    for (int j = threadIdx.x * 8; j < K; j += 1024 * 8) {
        float y[8];
        In8<T, FN> in;
        in.load(xr, K, j);
        in.values(y);
        most = absmax8(y, most);
    }
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, sh[threadIdx.x & 31]);
    const Scale c = scale_of(top);
    if (threadIdx.x == 0) scale[row] = c.s;
    for (int j = threadIdx.x * 8; j < K; j += 1024 * 8) {
        float y[8];
        In8<T, FN> in;
        in.load(xr, K, j);
        in.values(y);
        *reinterpret_cast<uint2 *>(q + row * K + j) = quant8(y, c);
    }
}

template <typename T, int FN, int TPR, int VPT>
static int launch(const T *x, int8_t *q, float *scale, int M, int K, cudaStream_t st) {
    constexpr int CTA = TPR < 256 ? 256 : TPR, RPC = CTA / TPR;
    const int ctas = (M + RPC - 1) / RPC, room = num_sms() * (1536 / CTA);  // 1024 threads an SM: 49 us, 1536: 45
    W4_CUDA_TRY(launch_decode(quant_s8_kernel<T, FN, TPR, VPT>, dim3(ctas < room || TPR == 1024 ? ctas : room), dim3(CTA),
                              0, st, 1, x, q, scale, M, K));
    return W4_OK;
}

// Threads a row: a power of two with at most two vectors a thread up to 1024 threads, then three or four.
template <typename T, int FN>
static int launch_fn(const void *xv, int8_t *q, float *scale, int M, int K, cudaStream_t st) {
    const T *x = static_cast<const T *>(xv);
    const int nvec = K / 8;
    if (nvec <= 64) return launch<T, FN, 32, 2>(x, q, scale, M, K, st);
    if (nvec <= 128) return launch<T, FN, 64, 2>(x, q, scale, M, K, st);
    if (nvec <= 256) return launch<T, FN, 128, 2>(x, q, scale, M, K, st);
    if (nvec <= 512) return launch<T, FN, 256, 2>(x, q, scale, M, K, st);
    if (nvec <= 1024) return launch<T, FN, 512, 2>(x, q, scale, M, K, st);
    if (nvec <= 2048) return launch<T, FN, 1024, 2>(x, q, scale, M, K, st);
    if (nvec <= 3 * 1024) return launch<T, FN, 1024, 3>(x, q, scale, M, K, st);
    if (nvec <= 4096) return launch<T, FN, 1024, 4>(x, q, scale, M, K, st);
    W4_CUDA_TRY(launch_decode(quant_s8_long_kernel<T, FN>, dim3(M), dim3(1024), 0, st, 1, x, q, scale, K));
    return W4_OK;
}

template <typename T>
static int launch_t(const void *x, int fn, int8_t *q, float *scale, int M, int K, cudaStream_t st) {
    if (fn == W4_FN_SILU_MUL) return launch_fn<T, W4_FN_SILU_MUL>(x, q, scale, M, K, st);
    if (fn == W4_FN_RELU2) return launch_fn<T, W4_FN_RELU2>(x, q, scale, M, K, st);
    return launch_fn<T, W4_FN_NONE>(x, q, scale, M, K, st);
}

}  // namespace s8q

int quant_s8(const void *x, int x_dtype, int fn, int8_t *q, float *scale, int M, int K, cudaStream_t st) {
    if (x_dtype == W4_F32) return s8q::launch_t<float>(x, fn, q, scale, M, K, st);
    if (x_dtype == W4_BF16) return s8q::launch_t<__nv_bfloat16>(x, fn, q, scale, M, K, st);
    return s8q::launch_t<__half>(x, fn, q, scale, M, K, st);
}

}  // namespace w4
