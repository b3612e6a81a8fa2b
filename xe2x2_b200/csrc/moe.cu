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
// is score + bias, and the k-th and the next score of a few thousand tokens come closer than 32 bits
// tell apart: the choice would depend on how exp was rounded.  So a token is first chosen for in 32
// bits, with one rank more than asked for, and where two neighbours (or the last group kept and the
// next) are closer than the 32-bit errors, it is chosen for again in 64 (under 1 % of the tokens; all
// in 64 bits took 61 us for 8192 x 256, top 8 of 4 in 8 groups, where this takes 21).
//
// The order by expert is a counting sort without atomics whose order matters: a token takes an
// expert at most once, so a bit mask over a chunk's tokens for each expert gives counts (popc) and
// ranks (popc below the token's bit).

struct RouteArgs {
    const void *logits;
    const float *bias;
    int dtype, T, E, k, softmax, groups, topk_group, top2, renorm;
    int whole;  // lanes of a group, where that is a whole power of two, else 0
    float scaling;
    int *ids;
    float *weights;
    int *offsets, *rows, *slots;  // null: no plan
    uint16_t *counts;             // [chunks / 8, rounded up][E][8], zeros behind the last; null with one chunk
    int chunk, words;             // tokens per CTA, and words of their bit masks
    bool vec, vec_bias;           // a lane's logits, its biases, are aligned to their size or 16
};

__device__ __forceinline__ float load_logit(const void *p, int dt, size_t i) {
    if (dt == W4_F32) return static_cast<const float *>(p)[i];
    if (dt == W4_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}

__device__ __forceinline__ float logit_of(const RouteArgs &a, int t, int e) {
    return load_logit(a.logits, a.dtype, (size_t)t * a.E + e);
}

// Unsigned integers in the order of the values; above 0 for every value but -NaN.
__device__ __forceinline__ uint32_t ordered(float v) {
    const int b = __float_as_int(v);
    return (uint32_t)(b ^ ((b >> 31) | (int)0x80000000));
}
__device__ __forceinline__ uint64_t ordered(double v) {
    const long long b = __double_as_longlong(v);
    return (uint64_t)(b ^ ((b >> 63) | (long long)0x8000000000000000ull));
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

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// exp(l - top) or 1 / (1 + exp(-l)): in 64 bits, and in 32 with the hardware's base-2 exponential and
// reciprocal.
__device__ __forceinline__ double score_of(float l, bool softmax, float top, double) {
    return softmax ? exp((double)l - (double)top) : 1.0 / (1.0 + exp(-(double)l));
}
__device__ __forceinline__ float score_of(float l, bool softmax, float top, float) {
    constexpr float kLog2e = 1.4426950408889634f;
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((softmax ? l - top : -l) * kLog2e));
    if (softmax) return e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return r;
}
// Two values further apart than this are in order although their scores were taken in 32 bits.  A sigmoid
// of 32 bits is within 2e-7 of the exact one (2^-22 of the exponential times at most a quarter, 2^-23 of
// the reciprocal).  Two terms of a softmax, d = l - top below the largest, are each within 2^-22 of the
// exponential and |d| 2^-23 of its argument, which rounds twice (log2(e) itself is common to both, but
// for |d| 2^-26); the sum of up to 512 terms, 2.4e-6, scales both alike: 3e-6 + 2.6e-7 |d| of the larger
// one together, and |d| is at most -log(score).  `score` is the larger score (or sum of scores) of the
// two; their values round once or twice more.
__device__ __forceinline__ float close_to(bool softmax, float score, float value) {
    return (softmax ? (4e-6f - 3e-7f * __logf(fmaxf(score, 1e-38f))) * score : 1e-6f) + 5e-7f * fabsf(value);
}

// What a warp knows of one token: its logits (-inf where an expert is off), the largest one (finite), and
// the logits' keys (0 where an expert is off).
template <int EPL> struct Token {
    float l[EPL], top;
    uint32_t key[EPL];
    bool live, nan;
    int t;
};
struct Choice {
    int e;     // lane j: the j-th expert, -1 if there is none
    double z;  // the softmax's sum, where it was needed
};

__device__ __forceinline__ int padded(int e) { return e + (e >> 5); }  // apart in the banks from group to group

// The two largest values of `n` neighbouring lanes (a power of two), from each lane's two.
template <typename V>
__device__ __forceinline__ void merge_top2(V &first, V &second, int n) {
    for (int o = 1; o < n; o <<= 1) {
        const V f = __shfl_xor_sync(0xffffffffu, first, o), s = __shfl_xor_sync(0xffffffffu, second, o);
        const V least = first < f ? first : f;
        second = f > first ? s : second;
        first = f > first ? f : first;
        second = second > least ? second : least;
    }
}
template <typename V>
__device__ __forceinline__ void add_top2(V &first, V &second, V v) {
    const V least = v < first ? v : first;
    first = v > first ? v : first;
    second = least > second ? least : second;
}

// Whether this lane's group (lpg neighbouring lanes hold one, with its two best values) is among those
// whose experts may be chosen.  *close: whether 32-bit errors could have swapped the last group in for
// the first one out.
template <typename V>
__device__ __forceinline__ bool group_kept(const RouteArgs &a, V first, V second, int lpg, int lane, bool *close) {
    const int g = lane / lpg;
    const V total = a.top2 && second > (V)-INFINITY ? first + second : first;
    int rank = 0;
    for (int o = 0; o < a.groups; ++o) {
        const V v = __shfl_sync(0xffffffffu, total, o * lpg);
        rank += v > total || (v == total && o < g);
    }
    if (close && a.topk_group < a.groups) {
        const bool lead = lane % lpg == 0 && g < a.groups;
        const int in = __ffs(__ballot_sync(0xffffffffu, lead && rank == a.topk_group - 1)) - 1;
        const int out = __ffs(__ballot_sync(0xffffffffu, lead && rank == a.topk_group)) - 1;
        const float x = (float)__shfl_sync(0xffffffffu, total, in), y = (float)__shfl_sync(0xffffffffu, total, out);
        // the values' errors are of their size, not of the sum's: two large ones may cancel
        const float size = (float)(fabs(first) + (a.top2 && second > (V)-INFINITY ? fabs(second) : (V)0));
        const float most = fmaxf(__shfl_sync(0xffffffffu, size, in), __shfl_sync(0xffffffffu, size, out));
        *close = y > -INFINITY && x - y <= 2 * close_to(a.softmax, 1.f, most);
    }
    return g < a.groups && rank < a.topk_group;
}

// The largest key of the warp: its expert in every lane, and the key taken off.  0: none left.
template <int EPL, typename KeyT>
__device__ __forceinline__ KeyT take_best(KeyT (&key)[EPL], int lane, int *e) {
    KeyT best = key[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) best = max(best, key[i]);
    const KeyT m = warp_max(best);
    if (m == 0) return 0;
    const int win = __ffs(__ballot_sync(0xffffffffu, best == m)) - 1;
    int at = 0;
#pragma unroll
    for (int i = EPL - 1; i > 0; --i)
        if (key[i] == m) at = i;
    if (key[0] == m) at = 0;
    *e = __shfl_sync(0xffffffffu, lane * EPL + at, win);
#pragma unroll
    for (int i = 0; i < EPL; ++i)
        if (lane * EPL + i == *e) key[i] = 0;
    return m;
}

// EPL floats in a row, in 16-byte loads (aligned to their size or 16).
template <int EPL>
__device__ __forceinline__ void load_f32(const float *p, float (&v)[EPL]) {
    if constexpr (EPL >= 4) {
#pragma unroll
        for (int i = 0; i < EPL; i += 4) {
            const float4 u = *reinterpret_cast<const float4 *>(p + i);
            v[i] = u.x, v[i + 1] = u.y, v[i + 2] = u.z, v[i + 3] = u.w;
        }
    } else if constexpr (EPL == 2) {
        const float2 u = *reinterpret_cast<const float2 *>(p);
        v[0] = u.x, v[1] = u.y;
    } else {
        v[0] = *p;
    }
}

// A warp's scratch for select32: the lanes' maxima, candidates and the order (key, expert).
struct Pick {
    uint32_t best[32];
    uint2 cand[32], out[32];
};

// The kk <= 32 largest keys in order, the j-th to lane j (*m = 0 where there is none), in a fixed number
// of steps: the kk-th largest of the lanes' maxima bounds the kk-th largest key from below, and the
// few keys from there on are ranked against each other (all *count of them, down to *from, are left in
// order in p->out).  False if those are more than 32.
template <int EPL>
__device__ __forceinline__ bool select32(const uint32_t (&key)[EPL], int kk, int lane, Pick *p, int *e, uint32_t *m,
                                         int *count, uint32_t *from) {
    uint32_t best = key[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) best = max(best, key[i]);
    p->best[lane] = best;
    __syncwarp();
    int above = 0;
#pragma unroll
    for (int o = 0; o < 32; o += 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p->best + o);
        above += (v.x > best) + (v.y > best) + (v.z > best) + (v.w > best);
    }
    const uint32_t least = max(__reduce_min_sync(0xffffffffu, above < kk ? best : 0xffffffffu), 1u);
    int n = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const bool in = key[i] >= least;
        const uint32_t b = __ballot_sync(0xffffffffu, in);
        const int pos = n + __popc(b & ((1u << lane) - 1));
        if (in && pos < 32) p->cand[pos] = make_uint2(key[i], lane * EPL + i);
        n += __popc(b);
    }
    __syncwarp();
    *count = n;
    *from = least;
    if (n > 32) return false;
    const uint2 mine = lane < n ? p->cand[lane] : make_uint2(0u, 0u);
    int rank = 0;
#pragma unroll 4
    for (int c = 0; c < n; ++c) {
        const uint2 o = p->cand[c];
        rank += o.x > mine.x || (o.x == mine.x && o.y < mine.y);
    }
    if (lane < n) p->out[rank] = mine;
    __syncwarp();
    const bool on = lane < n && lane < kk;
    const uint2 r = on ? p->out[lane] : make_uint2(0u, 0u);
    *m = r.x;
    *e = on ? (int)r.y : -1;
    return true;
}

// Choose for a token with values of type V (float or double).  False: too close to call in 32 bits.
template <int EPL, typename V, typename KeyT>
__device__ __forceinline__ bool choose(const RouteArgs &a, const Token<EPL> &k, V *base, int lpg, Pick *pick, int lane,
                                       Choice *c) {
    constexpr bool NARROW = sizeof(V) == 4;
    const bool scored = a.bias || (a.groups > 1 && a.top2);  // values that are compared are not all logits
    const bool doubt = NARROW && scored;
    KeyT key[EPL];
    V val[EPL];  // what groups are scored by
    if (!scored) {
        if (a.softmax && !a.renorm) {  // the weights need the sum
            V z = 0;
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (k.key[i]) z += score_of(fminf(k.l[i], FLT_MAX), true, k.top, V());
            c->z = (double)warp_sum(z);
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i) key[i] = k.key[i];
#pragma unroll
        for (int i = 0; i < EPL; ++i) val[i] = (V)k.l[i];
    } else {
        V (&s)[EPL] = val, z = 0;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            s[i] = 0;
            if (k.key[i]) s[i] = score_of(fminf(k.l[i], FLT_MAX), a.softmax, k.top, V());
            z += s[i];
        }
        if (a.softmax) {
            z = warp_sum(z);
            c->z = (double)z;
            if (k.live) {
                const V iz = (V)1 / z;
#pragma unroll
                for (int i = 0; i < EPL; ++i) s[i] = NARROW ? s[i] * iz : s[i] / z;
            }
        }
        if (a.bias) {
            float b[EPL];
            if (a.vec_bias && lane * EPL < a.E) {
                load_f32<EPL>(a.bias + lane * EPL, b);
            } else {
#pragma unroll
                for (int i = 0; i < EPL; ++i) b[i] = lane * EPL + i < a.E ? a.bias[lane * EPL + i] : 0.f;
            }
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                s[i] += (V)b[i];
                key[i] = k.key[i] && s[i] > (V)-INFINITY ? ordered(s[i] + (V)0) : 0;
            }
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i)  // -0 orders as 0, as in the 32-bit keys
                key[i] = NARROW ? k.key[i] : k.key[i] ? ordered((V)k.l[i] + (V)0) : 0;
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i) val[i] = key[i] ? s[i] : (V)-INFINITY;
    }
    if (a.groups > 1) {
        const V low = (V)-INFINITY;
        V first = low, second = low;
        bool close = false;
        if (a.whole) {  // a group is a power of two of whole lanes
#pragma unroll
            for (int i = 0; i < EPL; ++i) add_top2(first, second, val[i]);
            merge_top2(first, second, a.whole);
            const bool kept = group_kept<V>(a, first, second, a.whole, lane, doubt ? &close : nullptr);
            if (close) return false;
#pragma unroll
            for (int i = 0; i < EPL; ++i) key[i] = kept ? key[i] : 0;
        } else {
#pragma unroll
            for (int i = 0; i < EPL; ++i)
                if (lane * EPL + i < a.E) base[padded(lane * EPL + i)] = val[i];
            __syncwarp();
            const int size = a.E / a.groups, mine = lane / lpg;
            if (mine < a.groups)
                for (int i = lane % lpg; i < size; i += lpg) add_top2(first, second, base[padded(mine * size + i)]);
            __syncwarp();  // base is rewritten later
            merge_top2(first, second, lpg);
            const bool in = group_kept<V>(a, first, second, lpg, lane, doubt ? &close : nullptr);
            const uint32_t kept = __ballot_sync(0xffffffffu, in);
            if (close) return false;
            int g = lane * EPL / size, r = lane * EPL % size;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                if (lane * EPL + i < a.E && !(kept >> (g * lpg) & 1)) key[i] = 0;
                if (++r == size) {
                    r = 0;
                    ++g;
                }
            }
        }
    }
    c->e = -1;
    KeyT mine = 0;  // lane j: the j-th key; in doubt also the one behind the last
    uint32_t last = 0, from = 0;
    int last_e = -1, n = 0;
    bool done = false;
    if constexpr (NARROW) {
        const int kk = a.k + (doubt && a.bias ? 1 : 0);
        if (kk <= 32 && select32<EPL>(key, kk, lane, pick, &c->e, &mine, &n, &from)) {
            done = true;
            last = __shfl_sync(0xffffffffu, mine, a.k & 31);
            last_e = __shfl_sync(0xffffffffu, c->e, a.k & 31);
            if (kk == a.k) last = 0;
        }
    }
    if (!done) {
        for (int j = 0; j <= a.k; ++j) {
            int e = -1;
            const KeyT m = take_best<EPL, KeyT>(key, lane, &e);
            if (m == 0) break;  // nothing left to choose
            if (j == a.k) {
                last = (uint32_t)m;
                last_e = e;
            } else if (lane == j) {
                c->e = e;
                mine = m;
            }
        }
    }
    if (lane >= a.k) c->e = -1;
    if constexpr (NARROW) {
        if (a.bias) {  // are all neighbours in the order, the one behind it included, clearly apart?
            const int be = __shfl_down_sync(0xffffffffu, c->e, 1);
            const uint32_t bm = __shfl_down_sync(0xffffffffu, mine, 1);
            const int e2 = lane == a.k - 1 ? last_e : be;
            const uint32_t m2 = lane == a.k - 1 ? last : bm;
            bool near = false, tie = false;
            if (lane < a.k && c->e >= 0 && m2 != 0 && e2 >= 0) {
                const float x = from_ordered(mine), y = from_ordered(m2), bx = a.bias[c->e], by = a.bias[e2];
                // equal logits and biases are a tie in any precision
                if (x - y <= close_to(a.softmax, fmaxf(x - bx, y - by), x)) {
                    near = bx != by || logit_of(a, k.t, c->e) != logit_of(a, k.t, e2);
                    tie = !near && lane == a.k - 1;
                }
            }
            if (__any_sync(0xffffffffu, tie)) {
                // The last one chosen ties with the one behind it, which says nothing of those behind that: each
                // is compared with the last one here, and the largest of those that were not ranked.
                const int le = __shfl_sync(0xffffffffu, c->e, a.k - 1);
                const float x = from_ordered(__shfl_sync(0xffffffffu, mine, a.k - 1)), bx = a.bias[le];
                uint32_t rest = 0;
#pragma unroll
                for (int i = 0; i < EPL; ++i) rest = max(rest, key[i] < from ? key[i] : 0u);
                rest = warp_max(rest);
                near |= !done || (rest != 0 && x - from_ordered(rest) <= close_to(a.softmax, 1.f, x));
                if (done && lane > a.k && lane < n) {
                    const uint2 o = pick->out[lane];
                    const float y = from_ordered(o.x), by = a.bias[o.y];
                    if (x - y <= close_to(a.softmax, fmaxf(x - bx, y - by), x))
                        near |= bx != by || logit_of(a, k.t, le) != logit_of(a, k.t, o.y);
                }
            }
            if (__any_sync(0xffffffffu, near)) {
                // A sigmoid needs no other expert: if every key that could reach the top_k is among those
                // that were ranked, these are ranked again by score + bias in 64 bits, one a lane.
                const uint32_t kth = __shfl_sync(0xffffffffu, mine, a.k - 1);
                const float x = from_ordered(kth);
                if (!done || a.softmax || (kth != 0 && x - from_ordered(from) <= 2 * close_to(false, 0.f, x))) return false;
                const int e = lane < n ? (int)pick->out[lane].y : -1;
                double v = -HUGE_VAL;
                if (e >= 0) v = score_of(fminf(logit_of(a, k.t, e), FLT_MAX), false, 0.f, 0.0) + (double)a.bias[e];
                int rank = 0;
                for (int o = 0; o < n; ++o) {
                    const double u = __shfl_sync(0xffffffffu, v, o);
                    const int oe = __shfl_sync(0xffffffffu, e, o);
                    rank += u > v || (u == v && oe < e);
                }
                if (lane < n) pick->cand[rank] = make_uint2(0u, e);
                __syncwarp();
                c->e = lane < n && lane < a.k ? (int)pick->cand[lane].y : -1;
                __syncwarp();
            }
        }
    }
    return true;
}

// Logits of a lane, EPL in a row: in one or a few wide loads where rows allow it.
template <int EPL>
__device__ __forceinline__ void load_logits(const RouteArgs &a, int t, int lane, float (&l)[EPL]) {
    const size_t o = (size_t)t * a.E + lane * EPL;
    if (a.vec && lane * EPL < a.E) {
        if (a.dtype == W4_F32) {
            load_f32<EPL>(static_cast<const float *>(a.logits) + o, l);
            return;
        }
        if constexpr (EPL >= 2) {
            const uint16_t *p = static_cast<const uint16_t *>(a.logits) + o;
            uint32_t w[EPL / 2];
            if constexpr (EPL >= 8) {
#pragma unroll
                for (int i = 0; i < EPL / 8; ++i) {
                    const uint4 u = reinterpret_cast<const uint4 *>(p)[i];
                    w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
                }
            } else if constexpr (EPL == 4) {
                const uint2 u = *reinterpret_cast<const uint2 *>(p);
                w[0] = u.x, w[1] = u.y;
            } else {
                w[0] = *reinterpret_cast<const uint32_t *>(p);
            }
#pragma unroll
            for (int i = 0; i < EPL / 2; ++i) {
                const float2 f = a.dtype == W4_BF16 ? Conv<__nv_bfloat16>::to_f2(w[i]) : Conv<__half>::to_f2(w[i]);
                l[2 * i] = f.x;
                l[2 * i + 1] = f.y;
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) l[i] = lane * EPL + i < a.E ? load_logit(a.logits, a.dtype, o + i) : -INFINITY;
}

template <int EPL>
__device__ __forceinline__ void route_token(const RouteArgs &a, int t, const float (&logits)[EPL], double *base, int lpg,
                                            Pick *pick, uint32_t *mask, int words, int t_local) {
    const int lane = threadIdx.x & 31;
    Token<EPL> k;
    k.t = t;
    bool nan = false;
    uint32_t top_key = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        nan |= logits[i] != logits[i];
        const bool on = logits[i] > -INFINITY;  // not for NaN
        k.l[i] = on ? logits[i] : -INFINITY;
        k.key[i] = on ? ordered(logits[i] + 0.f) : 0u;  // -0 orders as 0
        top_key = max(top_key, k.key[i]);
    }
    k.nan = __any_sync(0xffffffffu, nan);
    top_key = warp_max(top_key);
    k.live = top_key != 0;
    k.top = k.live ? fminf(from_ordered(top_key), FLT_MAX) : 0.f;

    Choice c;
    if (!choose<EPL, float, uint32_t>(a, k, reinterpret_cast<float *>(base), lpg, pick, lane, &c))
        choose<EPL, double, uint64_t>(a, k, base, lpg, pick, lane, &c);

    // Weights in 32 bits (expf and the quotient within an ulp) unless a score is so small that it, or the
    // sum, would be lost.  A softmax that is not renormalised divides by the sum that choose() took, of
    // base-2 exponentials of the hardware: within 2.4e-6 of itself (see close_to).
    const float l = c.e >= 0 ? fminf(logit_of(a, t, c.e), FLT_MAX) : 0.f;
    const float f = a.softmax ? expf(l - k.top) : __fdiv_rn(1.f, 1.f + expf(-l));
    float w = c.e >= 0 ? f : 0.f;
    if (__any_sync(0xffffffffu, c.e >= 0 && !(f > 1e-30f))) {
        double d = c.e >= 0 ? score_of(l, a.softmax, k.top, 0.0) : 0.0;
        if (a.renorm) {
            const double sum = warp_sum(d);
            d = sum > 0.0 ? d / sum : 0.0;
        } else if (a.softmax && k.live) {
            d /= c.z;
        }
        w = (float)(d * (double)a.scaling);
    } else {
        if (a.renorm) {
            const float sum = warp_sum(w);
            w = sum > 0.f ? __fdiv_rn(w, sum) : 0.f;
        } else if (a.softmax && k.live) {
            w = __fdiv_rn(w, (float)c.z);
        }
        w *= a.scaling;
    }
    if (lane < a.k) {
        const size_t o = (size_t)t * a.k + lane;
        a.ids[o] = c.e;
        a.weights[o] = k.nan ? __int_as_float(0x7fc00000) : w;
        if (a.offsets && c.e >= 0) atomicOr(&mask[c.e * words + (t_local >> 5)], 1u << (t_local & 31));
    }
}

// Exclusive prefix sum of v over the CTA's threads; the last one's inclusive sum in *total.
template <int KT>
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
    for (int w = 0; w < KT / 32; ++w) {
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
template <int KT>
__device__ __forceinline__ void place(const RouteArgs &a, const uint32_t *mask, int words, int *base, int *sh, int t0,
                                      int n, int total, int before) {
    int all = 0;
    const int start = block_scan<KT>(total, sh, &all);
    if ((int)threadIdx.x < a.E) {
        base[threadIdx.x] = start + before;
        if (blockIdx.x == 0) a.offsets[threadIdx.x] = start;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[a.E] = all;
    __syncthreads();
    for (int i = threadIdx.x; i < n * a.k; i += KT) {
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
    for (long i = (long)all + (long)blockIdx.x * KT + threadIdx.x; i < end; i += (long)gridDim.x * KT)
        a.rows[i] = -1;
}

template <int EPL, int KT>
__global__ void __launch_bounds__(KT) route_kernel(const RouteArgs a) {
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ int base_sh[kMaxMoeExperts], scan_sh[(KT / 32)];
    __shared__ __align__(16) Pick pick_sh[(KT / 32)];
    const int words = a.words;
    uint32_t *mask = reinterpret_cast<uint32_t *>(sm);
    double *base = reinterpret_cast<double *>(sm + (((size_t)(a.offsets ? a.E * words : 0) * 4 + 15) & ~size_t(15))) +
                   (size_t)(threadIdx.x >> 5) * padded(a.E);
    int lpg = 32;  // lanes that sum up a group: as many as every group can have
    while (lpg * a.groups > 32) lpg >>= 1;
    grid_dep_launch();
    if (a.offsets)
        for (int i = threadIdx.x; i < a.E * words; i += KT) mask[i] = 0;
    __syncthreads();
    grid_dep_wait();
    const int t0 = blockIdx.x * a.chunk, n = min(a.chunk, a.T - t0);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float l[EPL], ahead[EPL];  // a token's logits are on their way while the one before it is chosen for
    if (warp < n) load_logits<EPL>(a, t0 + warp, lane, ahead);
    for (int i = warp; i < n; i += (KT / 32)) {
#pragma unroll
        for (int u = 0; u < EPL; ++u) l[u] = ahead[u];
        if (i + (KT / 32) < n) load_logits<EPL>(a, t0 + i + (KT / 32), lane, ahead);
        route_token<EPL>(a, t0 + i, l, base, lpg, &pick_sh[warp], mask, words, i);
    }
    if (!a.offsets) return;
    __syncthreads();
    int count = 0;
    if ((int)threadIdx.x < a.E)
        for (int w = 0; w < words; ++w) count += __popc(mask[threadIdx.x * words + w]);
    if (a.counts) {
        if ((int)threadIdx.x < a.E) {
            uint16_t *eight = a.counts + ((size_t)(blockIdx.x / 8) * a.E + threadIdx.x) * 8;
            eight[blockIdx.x % 8] = (uint16_t)count;  // at most 1024
            if (blockIdx.x == gridDim.x - 1)
                for (int c = blockIdx.x % 8 + 1; c < 8; ++c) eight[c] = 0;
        }
    } else {
        place<KT>(a, mask, words, base_sh, scan_sh, t0, n, count, 0);
    }
}

template <int KT>
__global__ void __launch_bounds__(KT) place_kernel(const RouteArgs a) {
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ int base_sh[kMaxMoeExperts], scan_sh[(KT / 32)];
    const int words = a.words;
    uint32_t *mask = reinterpret_cast<uint32_t *>(sm);
    grid_dep_launch();
    for (int i = threadIdx.x; i < a.E * words; i += KT) mask[i] = 0;
    __syncthreads();
    grid_dep_wait();
    const int t0 = blockIdx.x * a.chunk, n = min(a.chunk, a.T - t0);
    for (int i = threadIdx.x; i < n * a.k; i += KT) {
        const int e = a.ids[(size_t)t0 * a.k + i], tl = i / a.k;
        if (e >= 0) atomicOr(&mask[e * words + (tl >> 5)], 1u << (tl & 31));
    }
    // every chunk's counts, eight in 16 bytes: P threads an expert, then one
    __shared__ int part_sh[2][KT];
    int width = 32;
    while (width < a.E) width <<= 1;  // at most KT
    const int P = KT / width, e = threadIdx.x % width, c8 = (gridDim.x + 7) / 8;
    unsigned total = 0, before = 0;
    if (e < a.E) {
        const uint4 *col = reinterpret_cast<const uint4 *>(a.counts) + e;  // neighbours in 16 bytes each
        const int part = threadIdx.x / width, mine = blockIdx.x / 8;  // mine: the eight that hold this chunk
#pragma unroll 8
        for (int i = part; i < c8; i += P) {
            const uint4 v = col[(size_t)i * a.E];
            total = __dp2a_lo(v.w, 0x0101u, __dp2a_lo(v.z, 0x0101u, __dp2a_lo(v.y, 0x0101u, __dp2a_lo(v.x, 0x0101u, total))));
            if (i < mine) before = total;
        }
        if (mine % P == part) {
            const uint4 v = col[(size_t)mine * a.E];
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            const int in = blockIdx.x % 8;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                before = __dp2a_lo(w[u], (2 * u < in ? 1u : 0u) | (2 * u + 1 < in ? 0x100u : 0u), before);
        }
    }
    part_sh[0][threadIdx.x] = total;
    part_sh[1][threadIdx.x] = before;
    __syncthreads();
    total = before = 0;
    if ((int)threadIdx.x < a.E)
        for (int i = 0; i < P; ++i) {
            total += part_sh[0][i * width + threadIdx.x];
            before += part_sh[1][i * width + threadIdx.x];
        }
    place<KT>(a, mask, words, base_sh, scan_sh, t0, n, total, before);
}

// Threads and tokens of a CTA.  Up to 32 tokens one CTA does everything.  Up to 16 an SM: 16 warps, a token
// each (148 tokens: 8.4 us, with 32 warps 11.6).  More: one CTA of 32 warps an SM (8192 tokens: 25 us where
// two of 16 warps took 28, since every CTA of the second kernel reads all counts; 21 us since); at most 1024
// tokens (the masks are E * chunk / 8 bytes of shared memory).
struct Shape {
    int threads, chunk;
};
static Shape shape_of(int T, int E) {
    if (T <= 32) return {512, 32};
    const int per = (T + num_sms() - 1) / num_sms();
    if (per <= 16) return {512, 16};
    return {E > 256 ? 512 : 1024, per > 1024 ? 1024 : per};  // 16 experts a lane take the registers of 512
}

static int experts_per_lane(int E) { return E <= 32 ? 1 : E <= 64 ? 2 : E <= 128 ? 4 : E <= 256 ? 8 : 16; }

template <int KT>
static cudaError_t launch_route(const RouteArgs &a, int chunks, size_t masks, size_t smem, cudaStream_t st) {
    void (*kern)(RouteArgs) = nullptr;
    switch (experts_per_lane(a.E)) {
        case 1: kern = route_kernel<1, KT>; break;
        case 2: kern = route_kernel<2, KT>; break;
        case 4: kern = route_kernel<4, KT>; break;
        case 8: kern = route_kernel<8, KT>; break;
        default: kern = route_kernel<16, 512>;
    }
    // Above the default limit less the static arrays: what any call takes, so that a smaller call from
    // another thread does not lower the limit before this one's launch.
    constexpr int kMost = kMaxMoeExperts * 1024 / 8 + 16 + 32 * (256 + 8) * 8;
    static_assert(16 * (kMaxMoeExperts + kMaxMoeExperts / 32) <= 32 * (256 + 8), "512 threads above 256 experts");
    if (smem > 16384) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
        if (e != cudaSuccess) return e;
    }
    cudaError_t e = launch_decode(kern, dim3(chunks), dim3(KT), smem, st, 1, a);
    if (e != cudaSuccess || !a.counts) return e;
    if (masks > 32768)
        e = cudaFuncSetAttribute(place_kernel<KT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kMaxMoeExperts * 1024 / 8);
    return e != cudaSuccess ? e : launch_decode(place_kernel<KT>, dim3(chunks), dim3(KT), masks, st, 1, a);
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

// STREAM: memory that is read once and not written meanwhile.
template <typename T, int N, bool STREAM>
__device__ __forceinline__ void load_n(const T *p, float (&v)[N]) {
    if constexpr (N == 1) {
        v[0] = as_f<T>(*p);
    } else {
        constexpr int W = N * (int)sizeof(T) / 4;  // 32-bit words, a multiple of 2
        uint32_t w[W];
#pragma unroll
        for (int i = 0; i < W; i += W % 4 ? 2 : 4) {
            if constexpr (W % 4 == 0) {
                const uint4 *q = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i);
                const uint4 u = STREAM ? ld_stream_v4(q) : *q;
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
// in flight.  Bound by memory: top_k + 1 rows a token; 8192 x 8 x 4096 bf16 takes 104 us, 5.8 TB/s (110
// without the streaming loads and stores, 158 with 256 threads a CTA).
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
    if (add) load_n<TO, N, false>(add + t * H + h, acc);
    for (int j0 = 0; j0 < k; j0 += 8) {
        float v[8][N], w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool on = j0 + j < k;
            const int s = on ? slots[t * k + j0 + j] : -1;
            w[j] = on ? weights[t * k + j0 + j] : 0.f;
            if (s >= 0 && s < rows) {
                load_n<TY, N, true>(y + (size_t)s * H + h, v[j]);
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
                __stcs(reinterpret_cast<uint4 *>(dst) + i, reinterpret_cast<const uint4 *>(r)[i]);
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
    const int c = moe::shape_of(T, E).chunk;
    const size_t chunks = (T + c - 1) / c;
    return T <= c ? 0 : ((chunks + 7) / 8 * 8 * E * 2 + 255) & ~size_t(255);
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
    const Shape sh = shape_of(T, E);
    a.chunk = sh.chunk;
    a.words = (a.chunk + 31) / 32;
    const int chunks = T > a.chunk ? (T + a.chunk - 1) / a.chunk : 1;
    a.counts = chunks > 1 && offsets ? static_cast<uint16_t *>(workspace) : nullptr;
    const int epl = experts_per_lane(E), es = dtype == W4_F32 ? 4 : 2, width = epl * es < 16 ? epl * es : 16;
    a.vec = E % epl == 0 && E * es % width == 0 && aligned(logits, width);
    const int size = E / groups, lanes = size / epl;
    a.whole = size % epl == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    a.vec_bias = E % epl == 0 && aligned(bias, epl * 4 < 16 ? epl * 4 : 16);
    const size_t masks = offsets ? (size_t)E * a.words * 4 : 0;
    const size_t smem = ((masks + 15) & ~size_t(15)) +
                        (groups > 1 && !a.whole ? (size_t)(sh.threads / 32) * (E + E / 32) * 8 : 0);
    W4_CUDA_TRY(sh.threads == 1024 ? launch_route<1024>(a, chunks, masks, smem, st)
                                   : launch_route<512>(a, chunks, masks, smem, st));
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
