// s8_gemm.cu -- W8A8 GEMM on the 5th-generation tensor cores (tcgen05.mma kind::i8, sm_100a), for
// one matrix and for a batch sorted by expert.
//
// Contract: w4_s8_gemm / w4_s8_gemm_grouped,
//   C[m, n] = f(sum_k A[m, k] * W[n, k]) * a_scale[m] * w_scale[n] + bias[n]
// with the integer sum exact (s32 in TMEM; |sum| <= 2^14 K < 2^31) and every step behind it in f32.
//
// The weights are the MMA's M side (128 output channels a tile) and the tokens its N side, so that
// one kernel serves every batch: N is 16 for a decode step and 256 for a prompt, and the MMA's N
// follows the rows that a tile has.  Both operands are K-major 128-byte lines, 128-byte swizzle,
// fetched by TMA; K is padded with zeros by the copy itself.  Warp 0 produces, warp 1 issues the
// MMAs, warps 2 to 5 or 9 read the sums out of TMEM (two accumulators: one fills while the other is read),
// scale and store.  Token rows that are gathered through an index come by 16-byte cp.async from
// four more warps: TMA's tile::gather4 (four rows a copy) took 55 to 75 cycles a copy, which made a
// batch of 4096 tokens x 6 of 64 experts (K 2688, N 3712) 1.12 ms; it takes 0.26 now.
// Every wait is bounded; no copy names more than one CTA.
#include <atomic>
#include <mutex>
#include <type_traits>

#include "tma_util.cuh"
#include "w4_common.cuh"
#include "w4_internal.h"

namespace w4 {

static __device__ unsigned int g_s8_timeout;  // a bounded wait expired (sticky until read)

namespace s8g {

constexpr int BN = 128, BK = 128;  // output channels and bytes of K in a stage
constexpr int kGather = 4;  // gather warps
// Epilogue warps (from warp 2 on): two to a lane quarter for the widest tile (M = 24,576, K = 2688,
// N = 3712: f32 262 -> 215 us, bf16 within 4 %).
constexpr int epi_warps(int bt) { return bt == 256 ? 8 : 4; }
constexpr uint32_t W_BYTES = BN * BK;

enum Mode { kDense = 0, kGrouped = 1, kGathered = 2 };
constexpr int threads_of(int bt, int mode) { return 32 * (2 + epi_warps(bt) + (mode == kGathered ? kGather : 0)); }

struct Args {
    const int8_t *a;  // gathered rows only (TMA has its map)
    const float *a_scale, *w_scale, *bias;
    const int *offsets, *src;
    void *c;
    int c_dtype, M, a_rows, N, K, E;
    int bt, box;  // token rows of a tile (a multiple of 16), of one token copy
    int ntn;      // column tiles
    bool pairs;   // 16-bit rows of C can be stored four bytes at a time (N even, c aligned)
    bool wide;    // and eight
};

// BT token rows at most, S stages, two accumulators of BT columns.  PAIR: two CTAs (a cluster) on one
// tile of 256 channels; each holds its 128 channels and half of the token rows.
template <int BT, bool PAIR> struct Cfg {
    static constexpr int EPI = epi_warps(BT);
    static constexpr uint32_t T_BYTES = (PAIR ? BT / 2 : BT) * BK, STAGE = W_BYTES + T_BYTES;
    static constexpr int S = STAGE > 40960 ? 4 : STAGE > 28672 ? 6 : STAGE > 20480 ? 8 : 5;
    static constexpr uint32_t TMEM_COLS = 2 * BT < 32 ? 32 : 2 * BT;
    static constexpr uint32_t BAR_OFF = S * STAGE, AS_OFF = BAR_OFF + (2 * S + 5) * 8 / 16 * 16 + 16,
                              MISC_OFF = AS_OFF + 2 * BT * 4, TILE_OFF = MISC_OFF + 16;
    static constexpr uint32_t LD = BT < 32 ? BT : 32;  // columns of one TMEM read
    static constexpr size_t smem(int E) { return TILE_OFF + (size_t)2 * (E + 1) * 4 + 1024; }
    static_assert(TILE_OFF + 2 * (kMaxMoeExperts + 1) * 4 + 1024 <= 227 * 1024, "shared memory plan");
};

// cta_group::2 forms (PAIR) are executed by one warp of each CTA of the pair.
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t *slot, uint32_t ncols) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)),
                     "r"(ncols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)),
                     "r"(ncols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    if constexpr (PAIR)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// The same barrier in CTA `rank` of the cluster, as a shared::cluster address; an arrival there.  The
// default scope (the CTA): such an arrival passes on that the tensor core has finished with a stage or an
// accumulator, or that a read of TMEM has (tcgen05.commit, tcgen05.wait), and nothing that threads wrote.
// Rows that threads wrote go by publish_rows / observe_rows.
__device__ __forceinline__ uint32_t bar_of(uint64_t *bar, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(bar)), "r"(rank));
    return a;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ int4 ld_cluster_v4(const void *p, uint32_t rank) {
    uint32_t a;
    int4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(a));
    return v;
}
// Arrival on this CTA's barrier when the MMAs issued so far are complete (a pair's: on both SMs).
template <bool PAIR>
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                     : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (PAIR)
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc)
            : "memory");
    else
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc)
            : "memory");
}
// TMA loads into this CTA whose bytes count on a barrier of the pair's first CTA.
__device__ __forceinline__ void pair_load_2d(void *dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void pair_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
// 16 bytes global -> shared, asynchronously; zeros where n is 0.
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void *src, uint32_t n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
// 32 lanes x NC columns of 32 bits, lane quarter in the address's upper half.
template <int NC>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&v)[NC]) {
    static_assert(NC == 16 || NC == 32, "16 or 32 columns");
    if constexpr (NC == 32) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
            "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
              "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
              "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
              "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
            : "r"(taddr));
    } else {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
            "%15}, [%16];"
            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
              "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
            : "r"(taddr));
    }
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// K-major operand, 128-byte swizzle, 8-row groups 1024 bytes apart, version 1.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::i8: s32 accumulator (2 at bit 4), signed A and B (1 at bits 7 and 10), N>>3 at 17, M>>4 at 24.
__device__ __forceinline__ uint32_t idesc_for(int n, int m) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Token rows that threads of one CTA copied into its shared memory, read by MMAs that a thread of the other
// CTA issues: the arrival and the wait that see each other need cluster scope, and so does the order around
// them.  The fences' .sync_restrict forms order accesses to shared memory alone, which is all there is:
// 4096 tokens x 6 of 64 experts, K = 2688, N = 3712 take 257 us; with .release.cluster on the arrival
// and .acquire.cluster on the wait 314, with fence.acq_rel.cluster behind the wait 573.
__device__ __forceinline__ void publish_rows(uint32_t addr) {
    asm volatile(
        "fence.release.sync_restrict::shared::cta.cluster;\n\t"
        "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr)
        : "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, "
        "p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ void observe_rows() {
    asm volatile("fence.acquire.sync_restrict::shared::cluster.cluster;" ::: "memory");
}

// Bounded wait.  The clock is read only after some tries: reading it costs about as much as a stage
// of the decode GEMM takes.  CLUSTER: see publish_rows.
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_s8(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    const uint32_t b = smem_u32(bar);
    auto done = [&] { return CLUSTER ? try_wait_cluster(b, parity) : mbar_try_wait(b, parity); };
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
        if (done()) return true;
    const unsigned long long t0 = global_ns();
    while (!done()) {
        if (*abort_flag) return false;
        if (global_ns() - t0 > kWaitLimitNs) {
            *abort_flag = 1;
            atomicExch(&g_s8_timeout, 1u);
            return false;
        }
    }
    return true;
}

// One lane of a converged warp, in the form from which the compiler knows that it is one: a copy or an
// MMA inside needs no loop over the lanes that might execute it.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}

// A tile: rows [row0, row0 + rows) of C (and of A, unless gathered), channels from n0 of expert e.
struct Tile {
    int e, row0, rows, n0;
};

// Token columns of a tile's MMA (M = 128: a multiple of 16; M = 256: of 32, half from each CTA).
template <bool PAIR> __device__ __forceinline__ int mma_cols(int rows) {
    return PAIR ? (rows + 31) & ~31 : (rows + 15) & ~15;
}

// Tile t.  Grouped: first[e] tiles before expert e, off[e] its first row; the offsets come from
// device memory and were clamped to [0, M] and to ascending order when they were read.
template <int MODE, bool PAIR>
__device__ __forceinline__ Tile tile_of(const Args &a, int t, const int *first, const int *off) {
    Tile r;
    int lo = 0, row_begin = 0, row_end = a.M, q = t;
    if constexpr (MODE != kDense) {
        int hi = a.E;  // the last expert with first[e] <= t has tile t (first[e + 1] > t)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= t) lo = mid;
            else hi = mid;
        }
        row_begin = off[lo];
        row_end = off[lo + 1];
        q = t - first[lo];
    }
    const int mt = (row_end - row_begin + a.bt - 1) / a.bt;
    r.e = lo;
    r.n0 = q / mt * (PAIR ? 2 * BN : BN);
    r.row0 = row_begin + q % mt * a.bt;
    r.rows = min(a.bt, row_end - r.row0);
    return r;
}

__device__ __forceinline__ void store_c(const Args &a, size_t o, float v) { store_out(a.c, a.c_dtype, o, v); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// LD token columns of a warp's 32 channels, as 16-bit rows of C: neighbouring lanes exchange a pair of
// tokens, and each stores two channels of one of them (4 bytes, 64 in a row to a half warp).  Through
// shared memory, 16 bytes a store, the epilogue took a share of the bandwidth that the copies and the
// MMAs use up (128 bytes a cycle at 256 x 256): M = 24,576, N = 3712 at K = 1024 took 114 us, not 96 (at
// K = 2688 178 and 182).
template <int LD, typename T>
__device__ __forceinline__ void store_rows(const Args &a, const uint32_t (&v)[LD], const float *as, float ws, float bs,
                                           int row, int rows, int n, int lane) {
    const int odd = lane & 1;
    const uint32_t sel = odd ? 0x3276u : 0x5410u;
    T *dst = static_cast<T *>(a.c) + (size_t)(row + odd) * a.N + (n & ~1);
    const bool in = n < a.N;  // N is even
#pragma unroll
    for (int i = 0; i < LD / 4; ++i) {
        const float4 s = *reinterpret_cast<const float4 *>(as + 4 * i);
        const uint32_t p = pack2<T>(fmaf((float)(int)v[4 * i] * s.x, ws, bs), fmaf((float)(int)v[4 * i + 1] * s.y, ws, bs));
        const uint32_t q =
            pack2<T>(fmaf((float)(int)v[4 * i + 2] * s.z, ws, bs), fmaf((float)(int)v[4 * i + 3] * s.w, ws, bs));
        const uint32_t w0 = __byte_perm(p, __shfl_xor_sync(0xffffffffu, p, 1), sel);
        const uint32_t w1 = __byte_perm(q, __shfl_xor_sync(0xffffffffu, q, 1), sel);
        if (in && 4 * i + odd < rows) *reinterpret_cast<uint32_t *>(dst) = w0;
        if (in && 4 * i + 2 + odd < rows) *reinterpret_cast<uint32_t *>(dst + 2 * (size_t)a.N) = w1;
        dst += 4 * (size_t)a.N;
    }
}

// A gather warp's finished stage: every lane orders its copies into its own CTA's shared memory before
// the tensor core's reads (the .shared::cluster form of the fence took more than twice as long for the whole
// kernel), then one arrival (on the first CTA's barrier, where the pair's MMAs are issued).
template <bool PAIR>
__device__ __forceinline__ void hand_over(uint64_t *bar, uint32_t lead, int lane) {
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) {
        if constexpr (PAIR) publish_rows(bar_of(bar, lead));
        else mbar_arrive(bar);
    }
}

// The same column by column, for rows that cannot be stored in pairs (f32, odd N): a warp's 32
// channels of one token are one store.
template <int LD, typename T>
__device__ __forceinline__ void store_cols(const Args &a, const uint32_t (&v)[LD], const float *as, float ws, float bs,
                                           int row, int rows, int n) {
    T *dst = static_cast<T *>(a.c) + (size_t)row * a.N + n;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
        if (i < rows) {
            const float y = fmaf((float)(int)v[i] * as[i], ws, bs);
            if constexpr (sizeof(T) == 4) *dst = y;
            else *dst = Conv<T>::from_f(y);
        }
        dst += a.N;
    }
}

// This CTA's share of a split tile's rows: the sums of the ks CTAs (KS, where it is known) added up, a warp
// a row, four channels a lane, four rows in flight.
template <bool PAIR, int KS>
__device__ __forceinline__ void finish_split(const Args &a, const Tile &tl, const uint8_t *sm, const float *as_sh,
                                             const float (&ws)[4], const float (&bs)[4], int rank, int kr, int ks) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int n = tl.n0 + rank * BN + 4 * lane, r1 = tl.rows * (kr + 1) / ks;
    for (int r0 = tl.rows * kr / ks + warp; r0 < r1; r0 += 4 * warps) {
        int v[4][4] = {};
        const int zs = KS ? KS : ks;
#pragma unroll(KS ? KS : 2)
        for (int z = 0; z < zs; ++z)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = min(r0 + i * warps, r1 - 1);
                const uint8_t *at = sm + (row * BN + 4 * lane) * 4;
                const int4 p = z == kr ? *reinterpret_cast<const int4 *>(at)
                                       : ld_cluster_v4(at, PAIR ? 2 * z + rank : z);
                v[i][0] += p.x;
                v[i][1] += p.y;
                v[i][2] += p.z;
                v[i][3] += p.w;
            }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = r0 + i * warps;
            if (row >= r1 || n >= a.N) continue;
            const float as = as_sh[row];
            float y[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) y[u] = fmaf((float)v[i][u] * as, ws[u], bs[u]);
            const size_t o = (size_t)(tl.row0 + row) * a.N + n;
            if (a.wide && a.c_dtype == W4_BF16) {
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.c) + o) =
                    make_uint2(pack2<__nv_bfloat16>(y[0], y[1]), pack2<__nv_bfloat16>(y[2], y[3]));
            } else if (a.wide && a.c_dtype == W4_F16) {
                *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.c) + o) =
                    make_uint2(pack2<__half>(y[0], y[1]), pack2<__half>(y[2], y[3]));
            } else {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (n + u < a.N) store_c(a, o + u, y[u]);
            }
        }
    }
}

template <int BT, int MODE, bool PAIR>
__global__ void __launch_bounds__(threads_of(BT, MODE), 1)
s8_gemm_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap a_map, const Args a) {
    using C_ = Cfg<BT, PAIR>;
    constexpr int S = C_::S, EPI = C_::EPI;
    extern __shared__ uint8_t smem_dyn[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(sm + C_::BAR_OFF);
    uint64_t *empty = full + S;
    uint64_t *acc_full = empty + S;  // [2]
    uint64_t *acc_empty = acc_full + 2;
    uint64_t *drain = acc_empty + 2;
    float *as_sh = reinterpret_cast<float *>(sm + C_::AS_OFF);  // [2][BT] token scales
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(sm + C_::MISC_OFF);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(sm + C_::MISC_OFF + 4);
    int *first = reinterpret_cast<int *>(sm + C_::TILE_OFF);  // [E + 1] tiles before each expert
    int *off = first + a.E + 1;                                // [E + 1] its first row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nkb_all = (a.K + BK - 1) / BK;
    // The cluster: a pair's two CTAs along x, and along z a K split, where this CTA (or pair) sums
    // blocks [kb0, kb1) of its one tile.
    const int rank = PAIR ? blockIdx.x & 1 : 0;
    const uint32_t lead = 2 * blockIdx.z;  // the pair's first CTA
    const int t0 = PAIR ? blockIdx.x >> 1 : blockIdx.x, tstep = PAIR ? gridDim.x >> 1 : gridDim.x;
    const int ks = gridDim.z, kr = blockIdx.z;
    const int kb0 = (int)((long)nkb_all * kr / ks), kb1 = (int)((long)nkb_all * (kr + 1) / ks);

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], MODE == kGathered ? (PAIR ? 3 : 2) : 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], PAIR ? 2 * EPI : EPI);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
        prefetch_tensormap(&w_map);
        prefetch_tensormap(&a_map);
    }
    if (warp == 1) tmem_alloc<PAIR>(tmem_slot, C_::TMEM_COLS);
    grid_dep_wait();
    int ntiles;
    if constexpr (MODE == kDense) {
        ntiles = (a.M + a.bt - 1) / a.bt * a.ntn;
    } else {
        if (warp == 0) {  // prefix over the experts, 32 at a time
            int tiles = 0, row = min(max(a.offsets[0], 0), a.M);
            for (int e0 = 0; e0 < a.E; e0 += 32) {
                const int e = e0 + lane;
                int end = e < a.E ? min(max(a.offsets[e + 1], 0), a.M) : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {  // ascending whatever the memory holds
                    const int u = __shfl_up_sync(0xffffffffu, end, o);
                    if (lane >= o) end = max(end, u);
                }
                end = max(end, row);
                int begin = __shfl_up_sync(0xffffffffu, end, 1);
                if (lane == 0) begin = row;
                int n = e < a.E ? (end - begin + a.bt - 1) / a.bt * a.ntn : 0;
                int inc = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += u;
                }
                if (e < a.E) {
                    first[e] = tiles + inc - n;
                    off[e] = begin;
                    if (e == a.E - 1) {
                        first[a.E] = tiles + inc;
                        off[a.E] = end;
                    }
                }
                tiles += __shfl_sync(0xffffffffu, inc, 31);
                row = __shfl_sync(0xffffffffu, end, 31);
            }
        }
        ntiles = 0;
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();  // both CTAs' barriers exist
    tc_fence_after();
    if constexpr (MODE != kDense) ntiles = first[a.E];
    const uint32_t tmem = *tmem_slot;

    // Warps 0 and 1 leave their loops to one lane (elect_one): a wait by all 32 lanes costs 190 cycles
    // on a barrier that is complete already, and inside a branch on the lane number each MMA cost
    // another 105 of register moves; a stage took 780 cycles whatever its N, where the tensor work of
    // 128 k is 512 at N = 256 and 32 at N = 16.
    if (warp == 0 && elect_one()) {
        // ---------------- producer ----------------
        int g = 0, s = 0;    // k-blocks issued, their stage
        uint32_t phase = 1;  // a fresh barrier's "previous" phase counts as complete
        bool ok = true;
        for (int t = t0; t < ntiles && ok; t += tstep) {
            const Tile tl = tile_of<MODE, PAIR>(a, t, first, off);
            const int cols = mma_cols<PAIR>(tl.rows), mine = PAIR ? cols / 2 : cols;  // this CTA's token rows
            const int boxes = MODE == kGathered ? 0 : (mine + a.box - 1) / a.box;
            const uint32_t tx = (PAIR ? 2 : 1) * (W_BYTES + (uint32_t)(boxes * a.box) * BK);
            for (int kb = kb0; kb < kb1; ++kb, ++g) {
                if (!wait_s8(&empty[s], phase, abort_flag)) {
                    ok = false;
                    break;
                }
                uint8_t *w_dst = sm + s * C_::STAGE, *t_dst = w_dst + W_BYTES;
                // the MMAs' commit reaches the first CTA's barrier; it tells the other one
                if (PAIR && rank == 0 && g >= S) mbar_arrive_cluster(bar_of(&empty[s], lead + 1));
                if (rank == 0) mbar_arrive_expect_tx(&full[s], tx);  // of both CTAs
                if constexpr (PAIR) {
                    const uint32_t bar = bar_of(&full[s], lead);
                    pair_load_3d(w_dst, &w_map, kb * BK, tl.n0 + rank * BN, tl.e, bar);
                    for (int b = 0; b < boxes; ++b)
                        pair_load_2d(t_dst + b * a.box * BK, &a_map, kb * BK, tl.row0 + rank * mine + b * a.box, bar);
                } else {
                    tma_load_3d(w_dst, &w_map, kb * BK, tl.n0, tl.e, &full[s]);
                    for (int b = 0; b < boxes; ++b)
                        tma_load_2d(t_dst + b * a.box * BK, &a_map, kb * BK, tl.row0 + b * a.box, &full[s]);
                }
                if (++s == S) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        // after a wait that gave up, nothing of this CTA's copies may still be in flight at its end
        if (*abort_flag && rank == 0)
            for (int i = g > S ? g - S : 0; i < g; ++i) mbar_wait_bounded(&full[i % S], (uint32_t)((i / S) & 1));
    } else if (warp == 1 && rank == 0 && elect_one()) {
        // ---------------- MMA issuer ----------------
        constexpr bool ROWS_BY_THREADS = PAIR && MODE == kGathered;  // those of the other CTA too
        const uint64_t d0 = sw128_desc(smem_u32(sm));
        int s = 0, j = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = t0; t < ntiles && ok; t += tstep, ++j) {
            const Tile tl = tile_of<MODE, PAIR>(a, t, first, off);
            const uint32_t idesc = idesc_for(mma_cols<PAIR>(tl.rows), PAIR ? 2 * BN : BN);
            const uint32_t acc = tmem + (uint32_t)(j & 1) * BT;
            if (j >= 2 && !wait_s8(&acc_empty[j & 1], (uint32_t)((j / 2 - 1) & 1), abort_flag)) break;
            tc_fence_after();
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!wait_s8<ROWS_BY_THREADS>(&full[s], phase, abort_flag)) {
                    ok = false;
                    break;
                }
                if constexpr (ROWS_BY_THREADS) observe_rows();
                tc_fence_after();
                const uint64_t wd = d0 + (uint64_t)(s * (C_::STAGE >> 4)), td = wd + (W_BYTES >> 4);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)  // 32 k a step; zeros behind K
                    mma_i8<PAIR>(acc, wd + 2 * kk, td + 2 * kk, idesc, kb > kb0 || kk > 0);
                tc_commit<PAIR>(&empty[s]);
                if (++s == S) {
                    s = 0;
                    phase ^= 1;
                }
            }
            if (ok) tc_commit<PAIR>(&acc_full[j & 1]);
        }
        if (*abort_flag) {  // let the MMAs in flight end before TMEM is freed
            tc_commit<PAIR>(drain);
            mbar_wait_bounded(drain, 0u);
        }
    } else if (warp < 2) {
        // the other lanes wait at the end
    } else if (MODE == kGathered && warp >= 2 + EPI) {
        // ---------------- gather: token rows through the index, 16 bytes a lane and copy ----------------
        // The warps take the stages in turn.  Lane (r, c) of four rows a copy: chunk c of row r lies at
        // c ^ (r % 8) of its 128-byte line.  Row numbers are spread over the lanes, 32 a register.
        // S >= kGather: a warp that waits for stage g's last use to end knows that use g - kGather - S has
        // ended, and the parity it waits for means the right phase only if use g - 2 S is no later.
        // (Handing a stage over only after the next one's copies were issued: slower by a fifth.)
        static_assert(S >= kGather, "stage parity");
        constexpr int ROWS = PAIR ? BT / 2 : BT;
        const int r0 = lane >> 3, c = lane & 7;
        int g = 0;
        bool ok = true;
        for (int t = t0; t < ntiles && ok; t += tstep) {
            const Tile tl = tile_of<MODE, PAIR>(a, t, first, off);
            const int half = mma_cols<PAIR>(tl.rows) / 2, begin = rank * half;  // this CTA's first row
            const int mine = PAIR && rank == 0 ? min(tl.rows, half) : tl.rows - begin;
            int src[(ROWS + 31) / 32];
#pragma unroll
            for (int i = 0; i < (ROWS + 31) / 32; ++i) {
                const int r = 32 * i + lane;
                src[i] = r < mine ? a.src[tl.row0 + begin + r] : 0;
                if (src[i] < 0 || src[i] >= a.a_rows) src[i] = 0;  // scaled by 0
            }
            for (int kb = kb0; kb < kb1; ++kb, ++g) {
                if (g % kGather != warp - (2 + EPI)) continue;
                const int s = g % S;
                if (g >= S && !__all_sync(0xffffffffu, wait_s8(&empty[s], (uint32_t)((g / S - 1) & 1), abort_flag))) {
                    ok = false;
                    break;
                }
                const int x = kb * BK + c * 16;
                const uint32_t n = x < a.K ? 16u : 0u, line = smem_u32(sm + s * C_::STAGE + W_BYTES) + r0 * BK;
                const int8_t *col = a.a + (n ? x : 0);
#pragma unroll
                for (int i = 0; i < ROWS / 4; ++i) {
                    const int r = 4 * i + r0;
                    const int row = __shfl_sync(0xffffffffu, src[i / 8], r & 31);
                    if (r < mine) cp_async16_zfill(line + i * 4 * BK + ((c ^ (r & 7)) << 4), col + (size_t)row * a.K, n);
                }
                cp_async_commit();
                cp_async_wait<0>();
                hand_over<PAIR>(&full[s], lead, lane);
            }
        }
    } else {
        // ---------------- epilogue: lane quarter warp % 4 ----------------
        const int q = warp & 3, ew = warp - 2;
        bool ok = true;
        int j = 0;
        for (int t = t0; t < ntiles; t += tstep, ++j) {
            const Tile tl = tile_of<MODE, PAIR>(a, t, first, off);
            float *as = as_sh + (j & 1) * BT;
            for (int i = threadIdx.x - 64; i < tl.rows; i += EPI * 32) {
                int r = tl.row0 + i;
                if constexpr (MODE == kGathered) r = a.src[r];
                as[i] = MODE != kGathered || (r >= 0 && r < a.a_rows) ? a.a_scale[r] : 0.f;
            }
            const int n0 = tl.n0 + rank * BN, n = n0 + 32 * q + lane;
            const bool in = n < a.N;
            const float ws = in ? a.w_scale[(size_t)tl.e * a.N + n] : 0.f;
            const float bs = in && a.bias ? a.bias[(size_t)tl.e * a.N + n] : 0.f;
            // as[] is complete (and the other one read).  A warp whose wait gave up still comes here for
            // every tile, so that the others are never left waiting.
            asm volatile("bar.sync 1, %0;" ::"r"(EPI * 32) : "memory");
            ok = ok && __all_sync(0xffffffffu, wait_s8(&acc_full[j & 1], (uint32_t)((j / 2) & 1), abort_flag));
            if (!ok) continue;
            if (PAIR && rank == 0 && ew == 0 && lane == 0) mbar_arrive_cluster(bar_of(&acc_full[j & 1], lead + 1));
            tc_fence_after();
            const uint32_t acc = tmem + (uint32_t)(j & 1) * BT + ((uint32_t)(32 * q) << 16);
            for (int c0 = ew / 4 * C_::LD; c0 < tl.rows; c0 += EPI / 4 * C_::LD) {
                uint32_t v[C_::LD];
                tmem_ld<C_::LD>(acc + c0, v);
                if (ks > 1) {  // raw sums, summed over the cluster below
                    int *red = reinterpret_cast<int *>(sm) + c0 * BN + 32 * q + lane;
#pragma unroll
                    for (int i = 0; i < (int)C_::LD; ++i) red[i * BN] = (int)v[i];
                } else if (a.pairs && a.c_dtype == W4_BF16) {
                    store_rows<C_::LD, __nv_bfloat16>(a, v, as + c0, ws, bs, tl.row0 + c0, tl.rows - c0, n, lane);
                } else if (a.pairs && a.c_dtype == W4_F16) {
                    store_rows<C_::LD, __half>(a, v, as + c0, ws, bs, tl.row0 + c0, tl.rows - c0, n, lane);
                } else if (in) {
                    if (a.c_dtype == W4_F32)
                        store_cols<C_::LD, float>(a, v, as + c0, ws, bs, tl.row0 + c0, tl.rows - c0, n);
                    else if (a.c_dtype == W4_BF16)
                        store_cols<C_::LD, __nv_bfloat16>(a, v, as + c0, ws, bs, tl.row0 + c0, tl.rows - c0, n);
                    else store_cols<C_::LD, __half>(a, v, as + c0, ws, bs, tl.row0 + c0, tl.rows - c0, n);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(bar_of(&acc_empty[j & 1], lead));
                else mbar_arrive(&acc_empty[j & 1]);
            }
        }
    }
    // Not before: the next grid's CTAs would take what slots are free, unevenly (M = 16, K = N = 5120: 8.9 us
    // where this takes 7.6).
    grid_dep_launch();
    // What the end of a split tile needs, on its way while the others finish.
    float ws[4] = {}, bs[4] = {};
    Tile last = {};
    if (ks > 1 && t0 < ntiles) {
        last = tile_of<MODE, PAIR>(a, t0, first, off);
        const int n = last.n0 + rank * BN + 4 * lane;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (n + u < a.N) ws[u] = a.w_scale[(size_t)last.e * a.N + n + u];
            if (n + u < a.N && a.bias) bs[u] = a.bias[(size_t)last.e * a.N + n + u];
        }
    }
    tc_fence_before();
    __syncthreads();
    // a pair is done with its TMEM and each other's barriers; the CTAs of a split have stored their sums
    if (PAIR || ks > 1) cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<PAIR>(tmem, C_::TMEM_COLS);
    }
    // The CTAs along z hold their parts of one tile's sums (s32: the order does not matter) where their
    // stages were; each finishes an equal share of the rows.
    switch (ks) {
        case 1: break;
        case 2: finish_split<PAIR, 2>(a, last, sm, as_sh, ws, bs, rank, kr, ks); break;
        case 3: finish_split<PAIR, 3>(a, last, sm, as_sh, ws, bs, rank, kr, ks); break;
        case 4: finish_split<PAIR, 4>(a, last, sm, as_sh, ws, bs, rank, kr, ks); break;
        default: finish_split<PAIR, 0>(a, last, sm, as_sh, ws, bs, rank, kr, ks);
    }
    if (PAIR || ks > 1) cluster_sync_all();  // nobody leaves while its sums are read
}

// Clusters of a dense kernel with K split ks that the current device runs at once.
template <int BT, bool PAIR>
static int clusters_at_once(int ks) {
    const void *kern = (const void *)s8_gemm_kernel<BT, kDense, PAIR>;
    const size_t smem = Cfg<BT, PAIR>::smem(0);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = PAIR ? 2 : 1;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = ks;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(PAIR ? 2 : 1, 1, ks);
    cfg.blockDim = dim3(threads_of(BT, kDense));
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
        (void)cudaGetLastError();
        n = num_sms() / (ks * (PAIR ? 2 : 1)) / 2;  // a careful guess
    }
    return n > 0 ? n : 1;
}
// The same by plan: tile c (16, 64, 128, 256, pair); asked of the runtime once a device.
static int dense_clusters(int dev, int c, int ks) {
    static std::atomic<int> cache[16][5][9];
    std::atomic<int> *at = dev < 16 ? &cache[dev][c][ks] : nullptr;
    int n = at ? at->load(std::memory_order_relaxed) : 0;
    if (n > 0) return n;
    n = c == 0   ? clusters_at_once<16, false>(ks)
        : c == 1 ? clusters_at_once<64, false>(ks)
        : c == 2 ? clusters_at_once<128, false>(ks)
        : c == 3 ? clusters_at_once<256, false>(ks)
                 : clusters_at_once<256, true>(ks);
    if (at) at->store(n, std::memory_order_relaxed);
    return n;
}

template <int BT, int MODE, bool PAIR = false>
static int launch(const CUtensorMap &w_map, const CUtensorMap &a_map, const Args &a, int grid, int ks,
                  cudaStream_t st) {
    const size_t smem = Cfg<BT, PAIR>::smem(MODE == kDense ? 0 : a.E);
    auto kern = s8_gemm_kernel<BT, MODE, PAIR>;
    {
        static std::mutex mu;
        static int set_dev[128] = {};
        int dev = 0;
        W4_CUDA_TRY(cudaGetDevice(&dev));
        std::lock_guard<std::mutex> lk(mu);
        if (dev >= 128 || set_dev[dev] < (int)smem) {
            W4_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            if (dev < 128) set_dev[dev] = (int)smem;
        }
    }
    W4_CUDA_TRY(launch_cluster(kern, dim3(PAIR ? 2 * grid : grid, 1, ks), dim3(threads_of(BT, MODE)), smem, st,
                               dim3(PAIR ? 2 : 1, 1, ks), w_map, a_map, a));
    return W4_OK;
}

template <int MODE>
static int launch_bt(int BT, bool pair, const CUtensorMap &w_map, const CUtensorMap &a_map, const Args &a, int grid,
                     int ks, cudaStream_t st) {
    if (pair) return launch<256, MODE, true>(w_map, a_map, a, grid, ks, st);
    switch (BT) {
        case 16: return launch<16, MODE>(w_map, a_map, a, grid, ks, st);
        case 64: return launch<64, MODE>(w_map, a_map, a, grid, ks, st);
        case 128: return launch<128, MODE>(w_map, a_map, a, grid, ks, st);
        default: return launch<256, MODE>(w_map, a_map, a, grid, ks, st);
    }
}

// Tile of a call: capacity BT (with PAIR for two CTAs), bt token rows used of it, K split ks.
struct Plan {
    int BT, bt, ks, ntn;
    bool pair;
    long tiles;
};

// The plan with the least estimated cycles, from measured times of the plans on some 30 shapes of 1 to
// 8192 tokens.  A k-block of 128 takes 2 bt tensor cycles, or longer to arrive (128 channels and bt rows
// at 58 bytes a cycle and SM; a pair's CTA has half of the rows and gets 64), and 500 at least; tiles go
// in waves over the SMs; a pair costs 4500 for its barriers and fill; a K split (a cluster of at most 8
// CTAs, four k-blocks each at least, one tile a cluster, all clusters at once) costs its exchange; and
// nothing is faster than memory.  Against the best of all plans on 30 shapes: within 4 % but for four
// short calls of 128 to 2050 tokens, 13 to 24 % off (128 x 2048 x 2048: 6.9 us where 16-row tiles take 5.5).
static Plan plan_for(int M, int N, int K, int dev, int nsm) {
    const int nkb = (K + BK - 1) / BK;
    Plan best = {};
    double least = 0;
    const double memory = ((double)N * K + (double)M * K + 2.0 * M * N) / 3500;  // cycles at 6.5 TB/s
    for (int c = 0; c < 5; ++c) {
        Plan p;
        p.BT = c == 0 ? 16 : c == 1 ? 64 : c == 2 ? 128 : 256;
        p.pair = c == 4;
        if (c > 0 && c < 4 && M <= p.BT / 4) continue;  // far wider than the batch
        const int step = p.pair ? 32 : 16, mt = (M + p.BT - 1) / p.BT;
        p.bt = ((M + mt - 1) / mt + step - 1) / step * step;  // equal tiles of rows
        p.ntn = p.pair ? (N + 2 * BN - 1) / (2 * BN) : (N + BN - 1) / BN;
        p.tiles = (long)((M + p.bt - 1) / p.bt) * p.ntn;
        const int slots = p.pair ? nsm / 2 : nsm;
        double per_kb = p.pair ? (256 + p.bt > 2 * p.bt ? 256 + p.bt : 2 * p.bt) : 1.1 * (256 + 2 * p.bt);
        per_kb = per_kb > 500 ? per_kb : 500;
        for (p.ks = 1; p.ks <= (p.pair ? 4 : 8); ++p.ks) {
            if (p.ks > 1 && (p.tiles * p.ks > slots || nkb / p.ks < 4 || p.tiles > dense_clusters(dev, c, p.ks))) break;
            const double waves = p.ks > 1 ? 1 : (double)((p.tiles + slots - 1) / slots);
            double t = waves * ((nkb + p.ks - 1) / p.ks) * per_kb;
            t = (t > memory ? t : memory) + 10.0 * p.bt + (p.pair ? 4500 : 0) +
                (p.ks > 1 ? 1500 + 400 * p.ks + 34.0 * p.bt : 0);
            if (least == 0 || t < least) {
                least = t;
                best = p;
            }
        }
    }
    return best;
}

static int map_failed() {
    set_error("s8 GEMM: the tensor map of an operand was refused (shape or alignment)");
    return W4_ERR_UNSUPPORTED;
}

}  // namespace s8g

int s8_gemm(const int8_t *a, const float *a_scale, const int8_t *w, const float *w_scale, const float *bias, void *c,
            int c_dtype, int M, int N, int K, cudaStream_t st) {
    using namespace s8g;
    int dev = 0;
    W4_CUDA_TRY(cudaGetDevice(&dev));
    const int nsm = num_sms();
    const Plan p = plan_for(M, N, K, dev, nsm);
    const Args g = {a, a_scale, w_scale, bias, nullptr, nullptr, c, c_dtype, M, M, N, K, 1, p.bt,
                    p.pair ? p.bt / 2 : p.bt, p.ntn, N % 2 == 0 && aligned(c, 4), N % 4 == 0 && aligned(c, 8)};
    CUtensorMap w_map, a_map;
    if (!make_map_3d(&w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, K, N, 1, K, (uint64_t)N * K, BK, BN,
                     CU_TENSOR_MAP_SWIZZLE_128B) ||
        !make_map_2d(&a_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, a, K, M, K, BK, g.box, CU_TENSOR_MAP_SWIZZLE_128B))
        return map_failed();
    W4_REQUIRE(p.tiles < (1L << 30), W4_ERR_UNSUPPORTED, "s8 GEMM: %ld tiles", p.tiles);
    const int slots = p.pair ? nsm / 2 : nsm;
    return launch_bt<kDense>(p.BT, p.pair, w_map, a_map, g, (int)(p.tiles < slots ? p.tiles : slots), p.ks, st);
}

int s8_gemm_grouped(const int8_t *a, int a_rows, const float *a_scale, const int8_t *w, const float *w_scale,
                    const float *bias, const int *offsets, const int *src, int E, void *c, int c_dtype, int R, int N,
                    int K, cudaStream_t st) {
    using namespace s8g;
    // The counts are on the device: capacity for about twice the average expert's rows.
    const long rows = 2L * R / E;
    const int BT = rows <= 16 ? 16 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    const bool pair = BT == 256 && N > BN;
    const Args g = {a, a_scale, w_scale, bias, offsets, src, c, c_dtype, R, a_rows, N, K, E, BT, BT < 32 ? BT : 32,
                    pair ? (N + 2 * BN - 1) / (2 * BN) : (N + BN - 1) / BN, N % 2 == 0 && aligned(c, 4), N % 4 == 0 && aligned(c, 8)};
    CUtensorMap w_map, a_map;
    if (!make_map_3d(&w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, K, N, E, K, (uint64_t)N * K, BK, BN,
                     CU_TENSOR_MAP_SWIZZLE_128B) ||
        !make_map_2d(&a_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, a, K, a_rows, K, BK, g.box, CU_TENSOR_MAP_SWIZZLE_128B))
        return map_failed();
    const long most = ((long)R / g.bt + (R < E ? R : E)) * g.ntn;  // tiles at most, whatever the counts
    W4_REQUIRE(most < (1L << 30), W4_ERR_UNSUPPORTED, "s8 GEMM: %ld tiles", most);
    const int nsm = num_sms(), slots = pair ? nsm / 2 : nsm, grid = (int)(most < slots ? most : slots);
    return src ? launch_bt<kGathered>(BT, pair, w_map, a_map, g, grid, 1, st)
               : launch_bt<kGrouped>(BT, pair, w_map, a_map, g, grid, 1, st);
}

int take_s8_wait_status() {
    unsigned int v = 0;
    W4_CUDA_TRY(cudaMemcpyFromSymbol(&v, g_s8_timeout, sizeof(v)));
    if (v) {
        const unsigned int zero = 0;
        W4_CUDA_TRY(cudaMemcpyToSymbol(g_s8_timeout, &zero, sizeof(zero)));
        set_error("a device-side wait expired in the s8 GEMM");
        return W4_ERR_TIMEOUT;
    }
    return W4_OK;
}

}  // namespace w4
