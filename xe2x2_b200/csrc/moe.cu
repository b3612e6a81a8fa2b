// moe.cu -- the parts of a mixture-of-experts layer around the grouped GEMMs: the router with the
// batch's order by expert (w4_moe_route), and the weighted sum of the experts' outputs
// (w4_moe_combine).
#include <float.h>

#include "tma_util.cuh"
#include "w4_common.cuh"
#include "w4_internal.h"

namespace w4 {
namespace moe {

// ---------------------------------------------------------------------------- routing
//
// One warp per token.  Lane l holds experts [l * EPL, (l + 1) * EPL), so the lowest lane (and the
// lowest slot in it) with the largest key is the lowest expert: ties need no extra work.  Keys
// are unsigned integers that order as the values do, 0 for an expert that cannot be chosen, and
// the warp's maximum is one redux (32-bit keys) or two (64-bit).  Without a bias the order of the
// scores is the order of the logits and the key is the logit, exact in 32 bits.  With one the key
// is score + bias in 64 bits: the k-th and the next score of a few thousand tokens come closer
// than 32 bits tell apart, and the choice would then depend on how exp was rounded.
//
// The order by expert is a counting sort without atomics whose order matters: a token takes an
// expert at most once, so a bit mask over a chunk's tokens for each expert gives counts (popc) and
// ranks (popc below the token's bit).
constexpr int kThreads = 512, kWarps = kThreads / 32;

struct RouteArgs {
    const void *logits;
    const float *bias;
    int dtype, T, E, k, softmax, groups, topk_group, top2, renorm;
    float scaling;
    int *ids;
    float *weights;
    int *offsets, *rows, *slots;  // null: no plan
    int *counts;                  // [chunks][E], null with one chunk
    int chunk;                    // tokens per CTA, a multiple of 32
};

__device__ __forceinline__ float load_logit(const void *p, int dt, size_t i) {
    if (dt == W4_F32) return static_cast<const float *>(p)[i];
    if (dt == W4_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}

// Unsigned integers in the order of the values; above 0 for every value but -NaN.
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ double score_of(float l, bool softmax, float top) {
    return softmax ? exp((double)l - (double)top) : 1.0 / (1.0 + exp(-(double)l));
}

// Bit mask of the groups whose experts may be chosen: lane g sums up group g.
__device__ __forceinline__ uint32_t kept_groups(const double *base, const RouteArgs &a, int lane) {
    const int size = a.E / a.groups;
    double first = -HUGE_VAL, second = -HUGE_VAL;
    if (lane < a.groups)
        for (int i = 0; i < size; ++i) {
            const double v = base[lane * size + i];
            if (v > first) {
                second = first;
                first = v;
            } else if (v > second) {
                second = v;
            }
        }
    const double total = a.top2 && second > -HUGE_VAL ? first + second : first;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
        const double o = __shfl_sync(0xffffffffu, total, g);
        rank += o > total || (o == total && g < lane);
    }
    return __ballot_sync(0xffffffffu, lane < a.groups && rank < a.topk_group);
}

template <int EPL, typename KeyT>
__device__ __forceinline__ void route_token(const RouteArgs &a, int t, double *base, uint32_t *mask, int words,
                                            int t_local) {
    const int lane = threadIdx.x & 31;
    constexpr bool kWide = sizeof(KeyT) == 8;
    float l[EPL];
    bool nan = false;
    uint32_t top_key = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const int e = lane * EPL + i;
        float v = e < a.E ? load_logit(a.logits, a.dtype, (size_t)t * a.E + e) : -INFINITY;
        if (v != v) {
            nan = true;
            v = -INFINITY;
        }
        l[i] = v + 0.f;  // -0 orders as 0
        if (v > -INFINITY) top_key = max(top_key, ordered(fminf(l[i], FLT_MAX)));
    }
    nan = __any_sync(0xffffffffu, nan);
    top_key = warp_max(top_key);
    const bool live = top_key != 0;
    const float top = live ? __uint_as_float(top_key & 0x80000000u ? top_key & 0x7FFFFFFFu : ~top_key) : 0.f;

    KeyT key[EPL];
    double z = 0.0;  // sum of the softmax
    if constexpr (kWide) {
        double s[EPL];
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            s[i] = l[i] > -INFINITY ? score_of(fminf(l[i], FLT_MAX), a.softmax, top) : 0.0;
            z += s[i];
        }
        z = warp_sum(z);
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = lane * EPL + i;
            const double p = a.softmax && live ? s[i] / z : s[i];
            double v = a.bias ? (e < a.E ? p + (double)a.bias[e] : 0.0) : (double)l[i];
            const bool off = !(l[i] > -INFINITY) || !(v > -HUGE_VAL);
            key[i] = off ? 0 : ordered(v);
            if (a.groups > 1 && e < a.E) base[e] = off ? -HUGE_VAL : a.top2 && !a.bias ? p : v;
        }
    } else {
        float zf = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = lane * EPL + i;
            if (a.softmax && !a.renorm && l[i] > -INFINITY) zf += expf(fminf(l[i], FLT_MAX) - top);
            key[i] = l[i] > -INFINITY ? ordered(l[i]) : 0;
            if (a.groups > 1 && e < a.E) base[e] = (double)l[i];
        }
        z = warp_sum((double)zf);
    }
    if (a.groups > 1) {
        __syncwarp();
        const uint32_t kept = kept_groups(base, a, lane);
        const int size = a.E / a.groups;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = lane * EPL + i;
            if (e < a.E && !(kept >> (e / size) & 1)) key[i] = 0;
        }
        __syncwarp();  // base is rewritten for the next token
    }

    int my_e = -1;
    float my_l = 0.f;
    for (int j = 0; j < a.k; ++j) {
        KeyT best = 0;
        int at = 0;
        float bl = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; ++i)
            if (key[i] > best) {
                best = key[i];
                at = i;
                bl = l[i];
            }
        const KeyT m = warp_max(best);
        if (m == 0) break;  // nothing left to choose
        const int win = __ffs(__ballot_sync(0xffffffffu, best == m)) - 1;
        const int e = __shfl_sync(0xffffffffu, lane * EPL + at, win);
        const float wl = __shfl_sync(0xffffffffu, bl, win);
        if (lane == j) {
            my_e = e;
            my_l = wl;
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i)
            if (lane * EPL + i == e) key[i] = 0;
    }

    double w = my_e >= 0 ? score_of(fminf(my_l, FLT_MAX), a.softmax, top) : 0.0;
    const double sum = warp_sum(w);
    if (a.renorm) w = sum > 0.0 ? w / sum : 0.0;
    else if (a.softmax && live) w /= z;
    if (lane < a.k) {
        const size_t o = (size_t)t * a.k + lane;
        a.ids[o] = my_e;
        a.weights[o] = nan ? __int_as_float(0x7fc00000) : (float)(w * (double)a.scaling);
        if (a.offsets && my_e >= 0) atomicOr(&mask[my_e * words + (t_local >> 5)], 1u << (t_local & 31));
    }
}

// Exclusive prefix sum of v over the CTA's threads; the last one's inclusive sum in *total.
__device__ __forceinline__ int block_scan(int v, int *sh, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
    }
    if (lane == 31) sh[warp] = inc;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kWarps; ++w) {
        const int u = sh[w];
        if (w < warp) before += u;
        all += u;
    }
    __syncthreads();
    *total = all;
    return before + inc - v;
}

// Offsets, rows and slots of one chunk from its masks, the experts' totals and the counts of the
// chunks before it (thread e: expert e).
__device__ __forceinline__ void place(const RouteArgs &a, const uint32_t *mask, int words, int *base, int *sh, int t0,
                                      int n, int total, int before) {
    int all = 0;
    const int start = block_scan(total, sh, &all);
    if ((int)threadIdx.x < a.E) {
        base[threadIdx.x] = start + before;
        if (blockIdx.x == 0) a.offsets[threadIdx.x] = start;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[a.E] = all;
    __syncthreads();
    for (int i = threadIdx.x; i < n * a.k; i += kThreads) {
        const int tl = i / a.k;
        const size_t o = (size_t)t0 * a.k + i;
        const int e = a.ids[o];
        int pos = -1;
        if (e >= 0) {
            pos = base[e];
            for (int w = 0; w < tl >> 5; ++w) pos += __popc(mask[e * words + w]);
            pos += __popc(mask[e * words + (tl >> 5)] & ((1u << (tl & 31)) - 1));
            a.rows[pos] = t0 + tl;
        }
        a.slots[o] = pos;
    }
    const long end = (long)a.T * a.k;  // rows behind the last expert's
    for (long i = (long)all + (long)blockIdx.x * kThreads + threadIdx.x; i < end; i += (long)gridDim.x * kThreads)
        a.rows[i] = -1;
}

template <int EPL, typename KeyT>
__global__ void __launch_bounds__(kThreads) route_kernel(const RouteArgs a) {
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ int base_sh[kMaxMoeExperts], scan_sh[kWarps];
    const int words = a.chunk / 32;
    uint32_t *mask = reinterpret_cast<uint32_t *>(sm);
    double *base = reinterpret_cast<double *>(sm + (((size_t)(a.offsets ? a.E * words : 0) * 4 + 15) & ~size_t(15))) +
                   (size_t)(threadIdx.x >> 5) * a.E;
    grid_dep_launch();
    if (a.offsets)
        for (int i = threadIdx.x; i < a.E * words; i += kThreads) mask[i] = 0;
    __syncthreads();
    grid_dep_wait();
    const int t0 = blockIdx.x * a.chunk, n = min(a.chunk, a.T - t0);
    for (int i = threadIdx.x >> 5; i < n; i += kWarps) route_token<EPL, KeyT>(a, t0 + i, base, mask, words, i);
    if (!a.offsets) return;
    __syncthreads();
    int count = 0;
    if ((int)threadIdx.x < a.E)
        for (int w = 0; w < words; ++w) count += __popc(mask[threadIdx.x * words + w]);
    if (a.counts) {
        if ((int)threadIdx.x < a.E) a.counts[(size_t)blockIdx.x * a.E + threadIdx.x] = count;
    } else {
        place(a, mask, words, base_sh, scan_sh, t0, n, count, 0);
    }
}

__global__ void __launch_bounds__(kThreads) place_kernel(const RouteArgs a) {
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ int base_sh[kMaxMoeExperts], scan_sh[kWarps];
    const int words = a.chunk / 32;
    uint32_t *mask = reinterpret_cast<uint32_t *>(sm);
    grid_dep_launch();
    for (int i = threadIdx.x; i < a.E * words; i += kThreads) mask[i] = 0;
    __syncthreads();
    grid_dep_wait();
    const int t0 = blockIdx.x * a.chunk, n = min(a.chunk, a.T - t0);
    for (int i = threadIdx.x; i < n * a.k; i += kThreads) {
        const int e = a.ids[(size_t)t0 * a.k + i], tl = i / a.k;
        if (e >= 0) atomicOr(&mask[e * words + (tl >> 5)], 1u << (tl & 31));
    }
    int total = 0, before = 0;
    if ((int)threadIdx.x < a.E)
#pragma unroll 8
        for (int c = 0; c < (int)gridDim.x; ++c) {
            const int v = a.counts[(size_t)c * a.E + threadIdx.x];
            total += v;
            if (c < (int)blockIdx.x) before += v;
        }
    __syncthreads();
    place(a, mask, words, base_sh, scan_sh, t0, n, total, before);
}

// Tokens per CTA: one CTA up to 64 tokens, else about one chunk per SM; at most 1024 (the masks
// are E * chunk / 8 bytes of shared memory).
static int chunk_of(int T) {
    if (T <= 64) return 64;
    const int per = (T + num_sms() - 1) / num_sms();
    const int c = (per + 31) / 32 * 32;
    return c < 32 ? 32 : c > 1024 ? 1024 : c;
}

template <typename KeyT>
static cudaError_t launch_route(const RouteArgs &a, int chunks, size_t smem, cudaStream_t st) {
    auto kern = a.E <= 32    ? route_kernel<1, KeyT>
                : a.E <= 64  ? route_kernel<2, KeyT>
                : a.E <= 128 ? route_kernel<4, KeyT>
                : a.E <= 256 ? route_kernel<8, KeyT>
                             : route_kernel<16, KeyT>;
    if (smem > 40960) {  // above the default limit less the static arrays
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
    }
    return launch_decode(kern, dim3(chunks), dim3(kThreads), smem, st, 1, a);
}

// ---------------------------------------------------------------------------- combine
// out[t] = add[t] + sum_j weights[t, j] * y[slots[t, j]], in f32, j in order.
template <typename T>
__device__ __forceinline__ float as_f(T v) {
    if constexpr (sizeof(T) == 4) return v;
    else return Conv<T>::to_f(v);
}
template <typename T>
__device__ __forceinline__ T from_f(float v) {
    if constexpr (sizeof(T) == 4) return v;
    else return Conv<T>::from_f(v);
}

template <typename T, int N>
__device__ __forceinline__ void load_n(const T *p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = as_f<T>(*p);
    } else {
        constexpr int W = N * (int)sizeof(T) / 4;  // 32-bit words, a multiple of 2
        uint32_t w[W];
#pragma unroll
        for (int i = 0; i < W; i += W % 4 ? 2 : 4) {
            if constexpr (W % 4 == 0) {
                const uint4 u = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
                w[i] = u.x, w[i + 1] = u.y, w[i + 2] = u.z, w[i + 3] = u.w;
            } else {
                const uint2 u = *reinterpret_cast<const uint2 *>(reinterpret_cast<const uint32_t *>(p) + i);
                w[i] = u.x, w[i + 1] = u.y;
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(w[i]);
            } else {
                const float2 f = Conv<T>::to_f2(w[i / 2]);
                v[i] = i & 1 ? f.y : f.x;
            }
        }
    }
}

// N channels a thread (16 bytes of y, or one where rows cannot be read that way), eight choices' rows
// in flight.  Bound by memory: top_k + 1 rows a token.
constexpr int kCombineThreads = 128;
template <typename TY, typename TO, int N>
__global__ void __launch_bounds__(kCombineThreads)
combine_kernel(const TY *__restrict__ y, int rows, const int *__restrict__ slots, const float *__restrict__ weights,
               const TO *add, TO *out, int k, int H) {
    grid_dep_launch();
    grid_dep_wait();
    const size_t t = blockIdx.x;
    const int h = (blockIdx.y * kCombineThreads + threadIdx.x) * N;
    if (h >= H) return;
    float acc[N] = {};
    if (add) load_n<TO, N>(add + t * H + h, acc);
    for (int j0 = 0; j0 < k; j0 += 8) {
        float v[8][N], w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool on = j0 + j < k;
            const int s = on ? slots[t * k + j0 + j] : -1;
            w[j] = on ? weights[t * k + j0 + j] : 0.f;
            if (s >= 0 && s < rows) {
                load_n<TY, N>(y + (size_t)s * H + h, v[j]);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) v[j][i] = 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] = fmaf(w[j], v[j][i], acc[i]);
    }
    TO *dst = out + t * H + h;
    if constexpr (N == 1) {
        *dst = from_f<TO>(acc[0]);
    } else {
        __align__(16) TO r[N];
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = from_f<TO>(acc[i]);
        if constexpr (N * sizeof(TO) % 16 == 0) {
#pragma unroll
            for (int i = 0; i < N * (int)sizeof(TO) / 16; ++i)
                reinterpret_cast<uint4 *>(dst)[i] = reinterpret_cast<const uint4 *>(r)[i];
        } else {
            *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(r);
        }
    }
}

template <typename TY, typename TO>
static int launch_combine(const void *y, int rows, const int *slots, const float *weights, const void *add, void *out,
                          int T, int k, int H, cudaStream_t st) {
    constexpr int N = 16 / (int)sizeof(TY);
    const bool wide = H % N == 0 && aligned(y, 16) && aligned(out, 16) && aligned(add, 16);
    const int per = kCombineThreads * (wide ? N : 1), gy = (H + per - 1) / per;
    W4_REQUIRE(gy <= 65535, W4_ERR_UNSUPPORTED, "H=%d is too long", H);
    W4_CUDA_TRY(launch_decode(wide ? combine_kernel<TY, TO, N> : combine_kernel<TY, TO, 1>, dim3(T, gy),
                              dim3(kCombineThreads), 0, st, 1, static_cast<const TY *>(y), rows, slots, weights,
                              static_cast<const TO *>(add), static_cast<TO *>(out), k, H));
    return W4_OK;
}

template <typename TY>
static int combine_out(const void *y, int rows, const int *slots, const float *weights, const void *add, void *out,
                       int out_dtype, int T, int k, int H, cudaStream_t st) {
    if (out_dtype == W4_F32) return launch_combine<TY, float>(y, rows, slots, weights, add, out, T, k, H, st);
    if (out_dtype == W4_BF16) return launch_combine<TY, __nv_bfloat16>(y, rows, slots, weights, add, out, T, k, H, st);
    return launch_combine<TY, __half>(y, rows, slots, weights, add, out, T, k, H, st);
}

}  // namespace moe

size_t moe_route_workspace(int T, int E) {
    const int c = moe::chunk_of(T);
    return T <= c ? 0 : ((size_t)((T + c - 1) / c) * E * 4 + 255) & ~size_t(255);
}

int moe_route(const void *logits, int dtype, const float *bias, int T, int E, int k, int score, int groups,
              int topk_group, int group_score, int renorm, float scaling, int *ids, float *weights, int *offsets,
              int *rows, int *slots, void *workspace, cudaStream_t st) {
    using namespace moe;
    RouteArgs a;
    a.logits = logits;
    a.bias = bias;
    a.dtype = dtype;
    a.T = T;
    a.E = E;
    a.k = k;
    a.softmax = score == W4_SCORE_SOFTMAX;
    a.groups = groups;
    a.topk_group = topk_group;
    a.top2 = group_score == W4_GROUP_TOP2;
    a.renorm = renorm != 0;
    a.scaling = scaling;
    a.ids = ids;
    a.weights = weights;
    a.offsets = offsets;
    a.rows = rows;
    a.slots = slots;
    a.chunk = chunk_of(T);
    const int chunks = T > a.chunk ? (T + a.chunk - 1) / a.chunk : 1;
    a.counts = chunks > 1 && offsets ? static_cast<int *>(workspace) : nullptr;
    const size_t masks = offsets ? (size_t)E * (a.chunk / 32) * 4 : 0;
    const size_t smem = ((masks + 15) & ~size_t(15)) + (groups > 1 ? (size_t)kWarps * E * 8 : 0);
    // 64-bit keys where scores are compared, not logits
    const bool wide = bias || (groups > 1 && a.top2);
    W4_CUDA_TRY(wide ? launch_route<uint64_t>(a, chunks, smem, st) : launch_route<uint32_t>(a, chunks, smem, st));
    if (a.counts) {
        if (masks > 40960)
            W4_CUDA_TRY(cudaFuncSetAttribute(place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)masks));
        W4_CUDA_TRY(launch_decode(place_kernel, dim3(chunks), dim3(kThreads), masks, st, 1, a));
    }
    return W4_OK;
}

int moe_combine(const void *y, int y_dtype, int rows, const int *slots, const float *weights, const void *add,
                void *out, int out_dtype, int T, int k, int H, cudaStream_t st) {
    if (y_dtype == W4_F32) return moe::combine_out<float>(y, rows, slots, weights, add, out, out_dtype, T, k, H, st);
    if (y_dtype == W4_BF16)
        return moe::combine_out<__nv_bfloat16>(y, rows, slots, weights, add, out, out_dtype, T, k, H, st);
    return moe::combine_out<__half>(y, rows, slots, weights, add, out, out_dtype, T, k, H, st);
}

}  // namespace w4
