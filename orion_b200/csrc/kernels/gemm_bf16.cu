// bfloat16 GEMM with either operand in either memory order, for the gradient side of the transformer clients:
//
//   C[b][m, n] = alpha * sum_k A[b][m, k] * B[b][n, k]  (+ bias[n])          b = batch_outer x batch_inner problems
//
// A lies in memory as [M, K] rows (K-major) or as [K, M] rows (MN-major); B as [N, K] rows or as [K, N] rows; row and
// batch strides are free (multiples of 8 elements).  That covers, without a transposed copy of anything,
//   dX = dY . W          (B = W [out, in]: the reduction index `out` is the slow one  -> B MN-major)
//   dW = dY^T . X        (both operands [tokens, features]: the reduction index is the slow one of both -> A and B MN-major)
//   attention:  P.V, dV = P^T.dO, dP = dO.V^T, dQ = dS.K, dK = dS^T.Q straight on the fused projection's [B, S, 3, H, 64]
// which the reference replays as cublasSgemm / cublasSgemmStridedBatched with transpose flags
// (reference src/scheduler/utils_sched.cpp:490-513; rows of benchmarking/model_kernels/bert_8_fb1).
//
// One CTA = 128 x BN output tile per work unit, persistent over units; or a pair of CTAs (a cluster on the two SMs of a TPC,
// cta_group::2) = 256 x BN, each CTA staging its 128 rows of A and half of B, so that an SM takes 32 KB instead of 48 KB of
// operands from L2 per 128 x 256 x 64 product of its own.  Operand traffic is what bounds the single CTA (about 64 bytes a clock
// and SM): decoder feed-forward 8192 x 4096 x 1024 57.9 -> 50.3 us (1.37 PFLOP/s), vocabulary projection 8192 x 32000 x 1024
// 505 -> 411 us.  Warp 0 issues TMA copies (4-D tensor maps:
// inner, outer, batch_inner, batch_outer; out-of-range elements read as zero, so ragged M, N, K need no special path),
// warp 1 issues tcgen05.mma kind::f16 into one of two tensor-memory accumulators, warps 2-5 (more for the epilogues that compute) drain the other one:
// tcgen05.ld (one output row per thread), alpha / bias / residual in registers, 32 rows x 128 bytes staged in a swizzled
// shared-memory slab per warp and written by a TMA store (two slabs per warp in flight; the tensor map clips ragged edges;
// outputs whose rows are not 16-byte multiples take per-thread stores).  An MN-major operand is declared as such in the instruction
// descriptor; its stage is filled by boxes of 64 reduction rows x 128 bytes, which is the canonical layout (atoms of
// 8 rows x 128 bytes, 1024 bytes apart along the reduction, 8192 bytes apart along M / N).
// Split-K (few output tiles, long reduction: the weight gradients) writes float32 partial matrices that a second
// kernel sums in split order, so the result does not depend on timing or on the CTA count.  Causal attention: `tri` modes
// skip the score tiles above the diagonal and cut the reductions over keys / queries at it.  The kernel is launched as a
// programmatic dependent: its set-up overlaps the tail of the kernel before it in the stream.
// Every wait is bounded; on expiry the kernel sets the status word, frees tensor memory and returns.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>

#include <type_traits>

#include "elastic.h"
#include "fast_gelu.cuh"
#include "gemm_call.h"
#include "philox.cuh"
#include "sm100_primitives.cuh"

namespace ob200 {

constexpr int GM_BM = 128;
constexpr int GM_BK = 64;
// Warp 0: TMA, warp 1: MMA + tensor memory, the others: epilogue.  Four of them, or sixteen (four for each 32 rows, each a share of the
// columns) where a turn of the epilogue is a long chain of latencies: bias + GELU of 8192 x 4096 x 1024.  Eight for the loss: over a
// short reduction the exponentials bound it (4096 x 16384 x 256: row maxima and sums 57 us in four warps, 44 in eight; over 1024 deep
// no difference), and sixteen for its gradient take the stages that a deep one needs (2048 x 32000 x 1024: 475 us in eight, 486).
__host__ __device__ constexpr int gm_epi_warps(int epi) {
    if (epi == GM_EPI_ACT || epi == GM_EPI_ACT_SLOPE || epi == GM_EPI_ACT_ANY) return 16;
    return epi == GM_EPI_LSE || epi == GM_EPI_DLOGITS ? 8 : 4;
}
__host__ __device__ constexpr int gm_threads(int epi) { return 64 + 32 * gm_epi_warps(epi); }
constexpr int GM_A_BYTES = GM_BM * 128;

// CG CTAs (1, or a pair) share a tile of CG * 128 rows: each stages its 128 rows of A and BN / CG rows of B.
template <int BN, int CG, int EPI>
struct GemmCfg {
    static constexpr int STAGE_BYTES = GM_A_BYTES + BN / CG * 128;
    static constexpr bool WIDE = gm_epi_warps(EPI) == 16;
    static constexpr int STAGES = STAGE_BYTES == 49152 ? (WIDE ? 3 : 4) : STAGE_BYTES == 32768 ? (WIDE ? 5 : 6) : WIDE ? 6 : 8;
    static constexpr int EPI_BYTES = WIDE ? 16 * 4096 : 32768;   // per epilogue warp two slabs of 32 rows x 64 (x 128) bytes for the TMA stores
    static constexpr int SMEM = STAGES * STAGE_BYTES + EPI_BYTES + 1024 + 512;   // + alignment, barriers
    static constexpr int TMEM_COLS = 2 * BN < 32 ? 32 : 2 * BN;
};

struct GemmParams {
    void* c;
    float* slabs;            // split-K partial matrices [splits][batch][M][N], or null
    const float* bias;
    const __nv_bfloat16* bias_bf16;   // the same addend given in bfloat16 (a parameter of a bfloat16 model)
    const __nv_bfloat16* residual;    // optional bfloat16 tensor laid out like C, added in float32 before rounding
    int* status;
    int M, N, K;
    int batch, nb_inner;
    long long ldc, c_si, c_so;
    int out_f32;
    int a_mn, b_mn;
    int tiles_m, tiles_n, kblocks, splits, kb_per_split;
    int vec_ok;              // C rows and batch offsets are 16-byte aligned
    int c_tma;               // C is written by TMA stores from swizzled shared-memory slabs (tmap_c)
    int tri;                 // causal attention: 1 = only output tiles that touch n <= m are computed (the rest is left unwritten),
                             // 2 = A[m, k] is zero for k > m (reduction stops behind the tile's last row),
                             // 3 = A[m, k] is zero for k < m (reduction starts at the tile's first row)
    float alpha;
    const int* live;         // packed rows: how many count, or null
    int live_k;              // they are the reduction (of a dual launch's second product in any case)
    int live_all;            // with as many as this the operand in tmap_all is taken, unpacked (0: never)
    GemmEpi e;               // of the epilogues other than GM_EPI_PLAIN
    alignas(64) unsigned char tmap_a[128];
    alignas(64) unsigned char tmap_b[128];
    alignas(64) unsigned char tmap_c[128];
    alignas(64) unsigned char tmap_slope[128];
    alignas(64) unsigned char tmap_res[128];
    alignas(64) unsigned char tmap_all[128];
};

// The second product of a GM_EPI_DUAL launch; its tiles come behind the first one's.
struct GemmSecond {
    int M, N, kblocks, tiles_m, tiles_n, a_mn, b_mn, out_f32;
    alignas(64) unsigned char tmap_a[128];
    alignas(64) unsigned char tmap_b[128];
    alignas(64) unsigned char tmap_c[128];
};
// How the first product of a dual launch is cut, in tiles of 256 x 256: the plan for all of its rows, from which that for the rows that
// count follows on the device.
struct GemmCutPlan { int M, tiles_n, kblocks, splits, per_split, second_tiles, second_kblocks, pairs; };
struct GemmCut { int splits, per_split, rows; };   // rows of a partial matrix
// With fewer rows than planned for its few tiles would keep few CTA pairs busy for long: as many parts as make a unit about a third of a
// pair's share of all the work, as far as the scratch goes (the matrices of the planned split, one at least).  171 of 1143 rows,
// 30522 x 768: 67 us for both products in the planned parts, 43 so.
__host__ __device__ inline GemmCut gm_cut(const GemmCutPlan& c, int live) {
    const int all = (c.M - 1) / 256 + 1, some = (live - 1) / 256 + 1;
    if (some >= all) return {c.splits, c.per_split, c.M};
    const int deep = (live - 1) / GM_BK + 1 < c.second_kblocks ? (live - 1) / GM_BK + 1 : c.second_kblocks;
    const long long work = (long long)some * c.tiles_n * c.kblocks + (long long)c.second_tiles * (deep + 8), share = work / c.pairs + 1;
    const long long room = (long long)c.splits * c.M / (some * 256LL);
    long long parts = 3LL * c.kblocks / share;
    if (parts > room) parts = room;
    if (parts > c.kblocks / 4) parts = c.kblocks / 4;
    if (parts > 32) parts = 32;
    if (parts < 2) return {1, c.kblocks, some * 256};
    const int per_split = (int)((c.kblocks + parts - 1) / parts);
    return {(c.kblocks + per_split - 1) / per_split, per_split, some * 256};
}
struct GemmParamsDual : GemmParams { GemmSecond second; GemmCutPlan cut; };
template <int EPI>
using GemmParamsOf = std::conditional_t<EPI == GM_EPI_DUAL, GemmParamsDual, GemmParams>;

struct GemmCtl {
    uint64_t full[8], empty[8], acc_full[2], acc_empty[2];
    uint64_t res_full[16][2];   // GM_EPI_ACT: a warp's residual slabs
    uint32_t tmem_base;
    int abort_flag;
};
static_assert(sizeof(GemmCtl) <= 512, "the barriers have 512 bytes of shared memory");

__device__ __forceinline__ uint64_t gm_desc_mn(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}

// k-blocks [kb0, kb1) of work unit (tile row tm, split sp); at least one block, the same for every warp role.
__device__ __forceinline__ void gm_kb_range(const GemmParams& p, int sp, int tm, int& kb0, int& kb1) {
    kb0 = sp * p.kb_per_split;
    kb1 = kb0 + p.kb_per_split < p.kblocks ? kb0 + p.kb_per_split : p.kblocks;
    if (p.tri == 2) {
        const int lim = (tm * GM_BM + GM_BM + GM_BK - 1) / GM_BK;
        if (lim < kb1) kb1 = lim > kb0 ? lim : kb0 + 1;
    } else if (p.tri == 3) {
        const int lo = (tm * GM_BM) / GM_BK;
        if (lo > kb0) kb0 = lo < kb1 ? lo : kb1 - 1;
    }
}
// With a causal mode the work per tile depends on its row, and a CTA's units (u = blockIdx.x + i * gridDim.x) would keep
// hitting the same rows of every problem.  Rotating the tile index by the problem index gives every CTA a mix of rows.
__device__ __forceinline__ int gm_rotate(const GemmParams& p, int t, int b, int tiles_per_problem) {
    return p.tri ? (t + b) % tiles_per_problem : t;
}
template <int BN>
__device__ __forceinline__ bool gm_tile_skipped(const GemmParams& p, int tm, int tn) {
    return p.tri == 1 && tn * BN > tm * GM_BM + GM_BM - 1;
}

// Packed rows: how many count, at least one (a reduction over none is one over a block of zeros).
__host__ __device__ constexpr bool gm_packs(int epi) { return epi == GM_EPI_ACC || epi == GM_EPI_LSE || epi == GM_EPI_DLOGITS || epi == GM_EPI_DUAL; }
template <int EPI>
__device__ __forceinline__ int gm_live(const GemmParams& p) {
    if constexpr (gm_packs(EPI)) {
        if (p.live) {
            const int n = *(const volatile int*)p.live;
            return n > 1 ? n : 1;
        }
    }
    return 0x7fffffff;
}
template <int EPI>
__device__ __forceinline__ bool gm_unpacked(const GemmParams& p) {
    if constexpr (gm_packs(EPI)) return p.live && p.live_all > 0 && *(const volatile int*)p.live == p.live_all;
    return false;
}

// Work unit u: output tile (tm, tn) of problem b (bi, bo), k-blocks [kb0, kb1), split sp; `second`: of a dual launch's second product.
struct GemmUnit { int sp, bi, bo, tm, tn, kb0, kb1; bool skip, second; };
template <int BN, int CG, int EPI>
__device__ __forceinline__ GemmUnit gm_unit(const GemmParamsOf<EPI>& p, long long u, int tiles_per_problem, int live, const GemmCut& cut) {
    GemmUnit w;
    w.second = false;
    if constexpr (EPI == GM_EPI_DUAL) {
        const long long first = (long long)tiles_per_problem * cut.splits;
        w.second = u >= first;
        w.bi = w.bo = 0;
        w.skip = false;
        if (w.second) {
            const int t = (int)(u - first);
            w.tm = t / p.second.tiles_n;
            w.tn = t - w.tm * p.second.tiles_n;
            w.sp = w.kb0 = 0;
            w.kb1 = p.second.kblocks;
            if ((live - 1) / GM_BK + 1 < w.kb1) w.kb1 = (live - 1) / GM_BK + 1;
        } else {
            const int t = (int)(u / cut.splits);
            w.sp = (int)(u - (long long)t * cut.splits);
            w.tm = t / p.tiles_n;
            w.tn = t - w.tm * p.tiles_n;
            w.kb0 = w.sp * cut.per_split;
            w.kb1 = w.kb0 + cut.per_split < p.kblocks ? w.kb0 + cut.per_split : p.kblocks;
        }
    } else {
        w.sp = (int)(u % p.splits);
        const int tile = (int)(u / p.splits);
        const int b = tile / tiles_per_problem, t = gm_rotate(p, tile - b * tiles_per_problem, b, tiles_per_problem);
        w.tm = t / p.tiles_n;
        w.tn = t - w.tm * p.tiles_n;
        w.bi = b % p.nb_inner;
        w.bo = b / p.nb_inner;
        w.skip = gm_tile_skipped<BN>(p, w.tm, w.tn);
        gm_kb_range(p, w.sp, w.tm, w.kb0, w.kb1);
        if constexpr (gm_packs(EPI)) {
            if (EPI == GM_EPI_ACC && p.live_k) {
                const int blocks = (live - 1) / GM_BK + 1;
                if (blocks < p.kblocks) {
                    const int per_split = (blocks + p.splits - 1) / p.splits;
                    w.kb0 = w.sp * per_split;
                    w.kb1 = w.kb0 + per_split < blocks ? w.kb0 + per_split : blocks;
                    if (w.kb0 >= w.kb1) { w.kb0 = p.kblocks; w.kb1 = w.kb0 + 1; }   // nothing left: a block behind the end, which reads as zeros
                }
            } else {
                w.skip |= (long long)w.tm * (CG * GM_BM) >= live;
            }
        }
    }
    return w;
}

#include "gemm_epilogue.cuh"

template <int BN, int CG, int EPI>
__global__ void __launch_bounds__(gm_threads(EPI), 1) gemm_bf16_kernel(const __grid_constant__ GemmParamsOf<EPI> p) {
    using C = GemmCfg<BN, CG, EPI>;
    constexpr bool kSlope = EPI == GM_EPI_ACT_SLOPE, kAct = EPI == GM_EPI_ACT || kSlope;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* epi_smem = smem + C::STAGES * C::STAGE_BYTES;
    GemmCtl* ctl = reinterpret_cast<GemmCtl*>(epi_smem + C::EPI_BYTES);
    const int tid = threadIdx.x, warp = uniform_warp_index(), lane = tid & 31;
    const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;   // CTA of the pair; CTA 0 issues the MMAs of both

    if (tid == 0) {
        for (int s = 0; s < C::STAGES; s++) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(&ctl->acc_full[a], 1);
            mbar_init(&ctl->acc_empty[a], gm_epi_warps(EPI) * CG);   // the epilogue warps of both CTAs
        }
        if (kAct)
            for (int i = 0; i < 32; i++) mbar_init(&ctl->res_full[i >> 1][i & 1], 1);
        ctl->abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tensormap(p.tmap_a);
        prefetch_tensormap(p.tmap_b);
        if (p.c_tma) prefetch_tensormap(p.tmap_c);
    }
    if (warp == 1) {
        if (CG == 2) {
            tmem_alloc_pair(&ctl->tmem_base, C::TMEM_COLS);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(&ctl->tmem_base, C::TMEM_COLS);
            tmem_relinquish();
        }
        tc_fence_before_sync();
    }
    __syncthreads();
    if (CG == 2) cluster_sync_all();   // the other CTA's barriers and tensor memory are ready
    tc_fence_after_sync();
    pdl_wait();
    if (tid == 0) pdl_launch_dependents();
    const int live = gm_live<EPI>(p);
    const uint32_t tmem_base = ctl->tmem_base;
    volatile int* abort_flag = &ctl->abort_flag;
    int tiles_per_problem = p.tiles_m * p.tiles_n;
    GemmCut cut = {};
    if constexpr (EPI == GM_EPI_DUAL) {
        cut = gm_cut(p.cut, live);
        if (live < p.M) tiles_per_problem = ((live - 1) / (CG * GM_BM) + 1) * p.tiles_n;
    }
    long long units = (long long)p.batch * tiles_per_problem * (EPI == GM_EPI_DUAL ? cut.splits : p.splits);
    if constexpr (EPI == GM_EPI_DUAL) units += p.second.tiles_m * p.second.tiles_n;

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer (the warp as one, see elect_one)
        int s = 0;
        uint32_t ph = 0;
        bool dead = false;
        const bool unpacked = gm_unpacked<EPI>(p);
        for (long long u = blockIdx.x / CG; u < units && !dead; u += gridDim.x / CG) {
            const GemmUnit w = gm_unit<BN, CG, EPI>(p, u, tiles_per_problem, live, cut);
            if (w.skip) continue;
            const int m0 = (w.tm * CG + (int)rank) * GM_BM, nb0 = w.tn * BN + (int)rank * (BN / CG);
            const unsigned char *map_a = p.tmap_a, *map_b = p.tmap_b;
            int a_mn = p.a_mn, b_mn = p.b_mn;
            if constexpr (EPI == GM_EPI_DUAL) {
                if (w.second) { map_a = p.second.tmap_a; map_b = unpacked ? p.tmap_all : p.second.tmap_b; a_mn = p.second.a_mn; b_mn = p.second.b_mn; }
            } else if constexpr (EPI == GM_EPI_ACC) {
                if (unpacked) map_b = p.tmap_all;
            } else if constexpr (gm_packs(EPI)) {
                if (unpacked) map_a = p.tmap_all;
            }
            for (int kb = w.kb0; kb < w.kb1; kb++) {
                if (!mbar_wait_warp(&ctl->empty[s], ph ^ 1u, abort_flag)) {
                    if (!*abort_flag) { ctl->abort_flag = 1; if (p.status) atomicExch(p.status, OB200_ERR_WAIT_EMPTY); }
                    dead = true;
                    break;
                }
                if (elect_one()) {
                    const uint32_t a_dst = smem_u32(smem + s * C::STAGE_BYTES);
                    const uint32_t b_dst = a_dst + GM_A_BYTES;
                    // the leading CTA's barrier counts the bytes of both CTAs
                    if (rank == 0) mbar_arrive_expect_tx(&ctl->full[s], (uint32_t)(CG * C::STAGE_BYTES));
                    const uint32_t bar = CG == 2 ? cluster_addr(smem_u32(&ctl->full[s]), 0) : 0;
                    auto load = [&](uint32_t dst, const void* map, int c0, int c1) {
                        if (CG == 2) tma_load_tile_4d_pair(dst, map, bar, c0, c1, w.bi, w.bo);
                        else tma_load_tile_4d(dst, map, &ctl->full[s], c0, c1, w.bi, w.bo);
                    };
                    if (!a_mn) {
                        load(a_dst, map_a, kb * GM_BK, m0);
                    } else {
#pragma unroll
                        for (int g = 0; g < GM_BM / 64; g++) load(a_dst + g * 8192, map_a, m0 + 64 * g, kb * GM_BK);
                    }
                    if (!b_mn) {
                        load(b_dst, map_b, kb * GM_BK, nb0);
                    } else {
#pragma unroll
                        for (int g = 0; g < BN / CG / 64; g++) load(b_dst + g * 8192, map_b, nb0 + 64 * g, kb * GM_BK);
                    }
                }
                __syncwarp();
                if (++s == C::STAGES) { s = 0; ph ^= 1u; }
            }
        }
        if (rank == 0) ring_settle(ctl->full, C::STAGES, s, ph, C::STAGES);   // the bytes of both CTAs
        // The leading CTA's commits arrive on this CTA's barriers: they must have landed before either CTA leaves.
        for (int i = 0; CG == 2 && i < C::STAGES && !dead; i++) {
            if (!mbar_wait_warp(&ctl->empty[s], ph ^ 1u, abort_flag)) break;
            if (++s == C::STAGES) { s = 0; ph ^= 1u; }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issue (the warp as one)
        if (rank == 0) {
            int s = 0;
            uint32_t ph = 0;
            uint32_t local = 0;
            bool dead = false;
            for (long long u = blockIdx.x / CG; u < units && !dead; u += gridDim.x / CG) {
                const GemmUnit w = gm_unit<BN, CG, EPI>(p, u, tiles_per_problem, live, cut);
                if (w.skip) continue;
                int a_mn = p.a_mn, b_mn = p.b_mn;
                if constexpr (EPI == GM_EPI_DUAL)
                    if (w.second) { a_mn = p.second.a_mn; b_mn = p.second.b_mn; }
                const uint32_t idesc = umma_idesc(1, CG * GM_BM, BN) | (a_mn ? UMMA_IDESC_A_MN : 0u) | (b_mn ? UMMA_IDESC_B_MN : 0u);
                // descriptors above the address; 16 reduction indices further on: 32 bytes along a K-major row, two 8-row atoms of
                // an MN-major tile
                const uint64_t a_bits = a_mn ? gm_desc_mn(0) : umma_desc_sw128(0), b_bits = b_mn ? gm_desc_mn(0) : umma_desc_sw128(0);
                const uint64_t a_step = a_mn ? 2048 >> 4 : 2, b_step = b_mn ? 2048 >> 4 : 2;
                const uint32_t ab = local & 1u, use = local >> 1;
                local++;
                if (!mbar_wait_warp(&ctl->acc_empty[ab], (use & 1u) ^ 1u, abort_flag)) {
                    if (!*abort_flag) { ctl->abort_flag = 1; if (p.status) atomicExch(p.status, OB200_ERR_WAIT_TMEM_EMPTY); }
                    break;
                }
                tc_fence_after_sync();
                const uint32_t d = tmem_base + ab * BN;
                for (int kb = w.kb0; kb < w.kb1; kb++) {
                    if (!mbar_wait_warp(&ctl->full[s], ph, abort_flag)) {
                        if (!*abort_flag) { ctl->abort_flag = 1; if (p.status) atomicExch(p.status, OB200_ERR_WAIT_FULL); }
                        dead = true;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t first = kb > w.kb0 ? 1u : 0u;   // 0: the tile's first product overwrites the accumulator
                    if (elect_one()) {
                        const uint32_t a_base = smem_u32(smem + s * C::STAGE_BYTES);
                        const uint64_t ad = umma_desc_mn(a_bits, a_base), bd = umma_desc_mn(b_bits, a_base + GM_A_BYTES);
#pragma unroll
                        for (int ks = 0; ks < GM_BK / 16; ks++) {
                            if (CG == 2) umma_f16_pair(d, ad + ks * a_step, bd + ks * b_step, idesc, ks > 0 ? 1u : first);
                            else umma_f16(d, ad + ks * a_step, bd + ks * b_step, idesc, ks > 0 ? 1u : first);
                        }
                        if (CG == 2) umma_commit_pair(&ctl->empty[s]);
                        else umma_commit(&ctl->empty[s]);
                        if (kb + 1 == w.kb1) {
                            if (CG == 2) umma_commit_pair(&ctl->acc_full[ab]);
                            else umma_commit(&ctl->acc_full[ab]);
                        }
                    }
                    __syncwarp();
                    if (++s == C::STAGES) { s = 0; ph ^= 1u; }
                }
            }
            ring_settle(ctl->empty, C::STAGES, s, ph, 1);
        }
    } else {
        // ------------------------------------------------------------ epilogue: thread = output row
        const int q = warp & 3;                       // tensor-memory lane group this warp may read
        uint8_t* stage = epi_smem + (warp - 2) * (C::EPI_BYTES / gm_epi_warps(EPI));   // this warp's slabs
        uint32_t local = 0;
        uint32_t slab_i = 0;
        for (long long u = blockIdx.x / CG; u < units; u += gridDim.x / CG) {
            const GemmUnit w = gm_unit<BN, CG, EPI>(p, u, tiles_per_problem, live, cut);
            const int sp = w.sp, tm = w.tm, tn = w.tn, bi = w.bi, bo = w.bo;
            if (w.skip) continue;
            const uint32_t ab = local & 1u, use = local >> 1;
            local++;
            // columns of a tile that a warp takes; a row's maximum and sum are those of 128 columns in one warp
            constexpr int kLeast = EPI == GM_EPI_LSE ? 128 : 32, kCols = BN * 4 / gm_epi_warps(EPI) < kLeast ? kLeast : BN * 4 / gm_epi_warps(EPI);
            const int part = (warp - 2) >> 2;
            const bool idle = part * kCols >= BN;   // a narrow tile has no columns for this warp
            const int m0w = (tm * CG + (int)rank) * GM_BM + q * 32;      // first row of this warp's 32
            bool ahead = false;
            if constexpr (kAct) {
                if (!idle) ahead = gm_residual_ahead<kSlope>(p, m0w, tn * BN + part * kCols, stage, slab_i, ctl->res_full[warp - 2]);
            }
            if (!mbar_wait_warp(&ctl->acc_full[ab], use & 1u, abort_flag)) {
                if (!*abort_flag) { ctl->abort_flag = 1; if (p.status) atomicExch(p.status, OB200_ERR_WAIT_TMEM_FULL); }
                if (ahead) {   // the residual's copy must have landed before the CTA leaves
                    mbar_wait_landed(&ctl->res_full[warp - 2][slab_i & 1], (slab_i >> 1) & 1, clock64());
                }
                break;
            }
            tc_fence_after_sync();
            const int m = m0w + lane;
            const int n0 = tn * BN;
            const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + ab * BN;
            const uint32_t t_part = t_row + part * kCols;
            const int n_part = n0 + part * kCols;
            if (idle) {
            } else if constexpr (kAct || EPI == GM_EPI_ACT_ANY) {
                if (p.splits > 1) gm_epilogue_slab<kCols>(p, t_part, m, n_part, sp, p.M);
                else if constexpr (EPI == GM_EPI_ACT_ANY) gm_epilogue_act_any<kCols>(p, t_part, m, m0w, n_part, lane, stage);
                else if (!gm_epilogue_act<kCols, kSlope>(p, t_part, m, m0w, n_part, lane, stage, slab_i, ctl->res_full[warp - 2], abort_flag)) {
                    if (!*abort_flag) { ctl->abort_flag = 1; if (p.status) atomicExch(p.status, OB200_ERR_WAIT_FULL); }
                    // as above: the slab that it gave up waiting for
                    mbar_wait_landed(&ctl->res_full[warp - 2][slab_i & 1], (slab_i >> 1) & 1, clock64());
                    break;
                }
            } else if constexpr (EPI == GM_EPI_DUAL) {
                if (cut.splits > 1 && !w.second) gm_epilogue_slab<BN>(p, t_row, m, n0, sp, cut.rows);
                else gm_epilogue_dual<BN>(p, w.second, t_row, m, m0w, n0, lane, stage, slab_i);
            } else if constexpr (EPI == GM_EPI_LSE) gm_epilogue_lse<kCols>(p, t_part, m, n_part);
            else if constexpr (EPI == GM_EPI_DLOGITS) gm_epilogue_dlogits<kCols>(p, t_part, m, m0w, n_part, lane, stage, slab_i);
            else {
            const bool to_slab = p.splits > 1;
            const bool row_ok = m < p.M;
            float* srow = to_slab ? p.slabs + (((long long)sp * p.batch + bo * p.nb_inner + bi) * p.M + m) * p.N : nullptr;
            const long long c_off = (long long)bo * p.c_so + (long long)bi * p.c_si + (long long)m * p.ldc;
            const bool by_tma = p.c_tma && !to_slab;
#pragma unroll 1
            for (int c0 = 0; c0 < BN; c0 += 32) {
                if (n0 + c0 >= p.N) break;            // warp-uniform
                uint32_t v[32];
                tmem_ld_32x32(t_row + c0, v);
                tmem_ld_wait();
                const int n = n0 + c0;
                const bool full = n + 32 <= p.N;
                if (to_slab) {
                    if (!row_ok) continue;
                    if (full && (p.N & 3) == 0) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<float4*>(srow + n + j) = make_float4(__uint_as_float(v[j]), __uint_as_float(v[j + 1]),
                                                                                   __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]));
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (n + j < p.N) srow[n + j] = __uint_as_float(v[j]);
                    }
                    continue;
                }
                if (!row_ok && !by_tma) continue;
                float f[32];
#pragma unroll
                for (int j = 0; j < 32; j++) f[j] = __uint_as_float(v[j]) * p.alpha;
                if (p.bias) {
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (full || n + j < p.N) f[j] += __ldg(p.bias + n + j);
                }
                if (p.bias_bf16) {
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (full || n + j < p.N) f[j] += __bfloat162float(p.bias_bf16[n + j]);
                }
                if (p.residual && row_ok) {
                    const __nv_bfloat16* res = p.residual + c_off + n;
                    if (full && p.vec_ok) {
#pragma unroll
                        for (int ch = 0; ch < 4; ch++) {
                            const uint4 rv = __ldg(reinterpret_cast<const uint4*>(res + ch * 8));
                            const __nv_bfloat162* h2 = reinterpret_cast<const __nv_bfloat162*>(&rv);
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                f[ch * 8 + e * 2] += __low2float(h2[e]);
                                f[ch * 8 + e * 2 + 1] += __high2float(h2[e]);
                            }
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (n + j < p.N) f[j] += __bfloat162float(res[j]);
                    }
                }
                if constexpr (EPI == GM_EPI_ACC) {
                    if (p.e.factor) {
                        const float factor = __ldg(p.e.factor);
#pragma unroll
                        for (int j = 0; j < 32; j++) f[j] *= factor;
                    }
                    if (p.e.addend && row_ok) {   // N a multiple of 4: no column of a vector is past the edge alone
                        const float* add = p.e.addend + (long long)m * p.N + n;
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            if (full || n + j < p.N) {
                                const float4 a = *reinterpret_cast<const float4*>(add + j);
                                f[j] += a.x; f[j + 1] += a.y; f[j + 2] += a.z; f[j + 3] += a.w;
                            }
                    }
                }
                if (by_tma) {
                    // Stage the warp's 32 rows x 128 bytes in a swizzled slab (16-byte chunk index XOR row % 8: conflict-free
                    // stores), then one TMA store per slab: 64 bfloat16 or 32 float32 columns.  Two slabs alternate; before a
                    // slab is rewritten the store issued from it two slabs ago must have read it.
                    const int half = p.out_f32 ? 0 : ((c0 >> 5) & 1);
                    uint8_t* slab = stage + (slab_i & 1) * 4096;
                    if (half == 0) {
                        if (lane == 0) bulk_wait_group_read<1>();
                        __syncwarp();
                    }
                    uint8_t* rowp = slab + lane * 128;
                    if (p.out_f32) {
#pragma unroll
                        for (int ch = 0; ch < 8; ch++)
                            *reinterpret_cast<float4*>(rowp + ((ch ^ (lane & 7)) << 4)) = make_float4(f[ch * 4], f[ch * 4 + 1], f[ch * 4 + 2], f[ch * 4 + 3]);
                    } else {
#pragma unroll
                        for (int ch = 0; ch < 4; ch++) {
                            uint4 pk;
                            uint32_t* w = &pk.x;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const __nv_bfloat162 h2 = __floats2bfloat162_rn(f[ch * 8 + e * 2], f[ch * 8 + e * 2 + 1]);
                                w[e] = *reinterpret_cast<const uint32_t*>(&h2);
                            }
                            *reinterpret_cast<uint4*>(rowp + (((half * 4 + ch) ^ (lane & 7)) << 4)) = pk;
                        }
                    }
                    const bool slab_done = p.out_f32 || half == 1 || c0 + 32 >= BN || n + 32 >= p.N;
                    if (slab_done) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {   // a warp whose rows are past the edge commits an empty group: the wait above counts slabs
                            if (m0w < p.M) tma_store_tile_4d(p.tmap_c, smem_u32(slab), n - half * 32, m0w, bi, bo);
                            bulk_commit_group();
                        }
                        slab_i++;
                    }
                    continue;
                }
                if (p.out_f32) {
                    float* out = reinterpret_cast<float*>(p.c) + c_off + n;
                    if (full && p.vec_ok) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(out + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (n + j < p.N) out[j] = f[j];
                    }
                } else {
                    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.c) + c_off + n;
                    if (full && p.vec_ok) {
#pragma unroll
                        for (int ch = 0; ch < 4; ch++) {
                            uint4 pk;
                            uint32_t* w = &pk.x;
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const __nv_bfloat162 h2 = __floats2bfloat162_rn(f[ch * 8 + e * 2], f[ch * 8 + e * 2 + 1]);
                                w[e] = *reinterpret_cast<const uint32_t*>(&h2);
                            }
                            *reinterpret_cast<uint4*>(out + ch * 8) = pk;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (n + j < p.N) out[j] = __float2bfloat16_rn(f[j]);
                    }
                }
            }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2) mbar_arrive_cluster(cluster_addr(smem_u32(&ctl->acc_empty[ab]), 0));
                else mbar_arrive(&ctl->acc_empty[ab]);
            }
        }
        bulk_wait_group<0>();   // the slabs must outlive the stores that read them
    }
    tc_fence_before_sync();
    __syncthreads();
    if (CG == 2) cluster_sync_all();   // nothing of this CTA is used by the other one any more
    if (warp == 1) {
        __syncwarp();
        tc_fence_after_sync();
        if (CG == 2) tmem_dealloc_pair(tmem_base, C::TMEM_COLS);
        else tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

// Sums the split-K partial matrices in split order, applies alpha and the bias, writes C.
__global__ void __launch_bounds__(256) gemm_splitk_finish_kernel(const float* __restrict__ slabs, void* c,
                                                                 const float* __restrict__ bias,
                                                                 const __nv_bfloat16* __restrict__ bias_bf16,
                                                                 const __nv_bfloat16* __restrict__ residual, const float* addend,
                                                                 const float* factor, int splits, int batch, int nb_inner,
                                                                 int M, int N, long long ldc, long long c_si, long long c_so,
                                                                 int out_f32, float alpha) {
    const long long per_split = (long long)batch * M * N;
    if (factor) alpha *= *factor;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < per_split; i += (long long)gridDim.x * blockDim.x) {
        float acc = 0.f;
        for (int s = 0; s < splits; s++) acc += slabs[(long long)s * per_split + i];
        const int n = (int)(i % N);
        const long long bm = i / N;
        const int m = (int)(bm % M), b = (int)(bm / M);
        acc = acc * alpha + (bias ? bias[n] : 0.f) + (bias_bf16 ? __bfloat162float(bias_bf16[n]) : 0.f);
        const long long off = (long long)(b / nb_inner) * c_so + (long long)(b % nb_inner) * c_si + (long long)m * ldc + n;
        if (residual) acc += __bfloat162float(residual[off]);
        if (addend) acc += addend[i];   // may be C itself
        if (out_f32) reinterpret_cast<float*>(c)[off] = acc;
        else reinterpret_cast<__nv_bfloat16*>(c)[off] = __float2bfloat16_rn(acc);
    }
}

// The same four columns at a time, for one problem with rows of a multiple of four columns, all 16-byte aligned (8 bytes for bfloat16):
// same additions in the same order, 13 -> 4 us for 1143 x 768 in five parts.
template <typename T>
__global__ void __launch_bounds__(256) gemm_splitk_finish4_kernel(const float* __restrict__ slabs, T* c, const float* addend, const float* factor, int splits,
                                                                  int M, int N, long long ldc, float alpha, const int* live, GemmCutPlan plan) {
    pdl_wait();
    pdl_launch_dependents();
    if (live) {   // of a dual launch over packed rows: cut on the device
        const GemmCut cut = gm_cut(plan, *live > 1 ? *live : 1);
        if (cut.splits == 1) return;
        splits = cut.splits;
        M = cut.rows;
    }
    const long long per_split = (long long)M * N, quads = per_split / 4;
    const int row = N / 4;
    if (factor) alpha *= *factor;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < quads; i += (long long)gridDim.x * blockDim.x) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < splits; s++) {
            const float4 v = *reinterpret_cast<const float4*>(slabs + s * per_split + i * 4);
            acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
        }
        acc.x *= alpha; acc.y *= alpha; acc.z *= alpha; acc.w *= alpha;
        if (addend) {   // may be C itself
            const float4 v = *reinterpret_cast<const float4*>(addend + i * 4);
            acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
        }
        const long long m = i / row, at = m * ldc + (i - m * row) * 4;
        if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(c + at) = acc;
        else *reinterpret_cast<uint2*>(c + at) = make_uint2(gm_pack(acc.x, acc.y), gm_pack(acc.z, acc.w));
    }
}

// The same for GM_EPI_ACT: bias, activation, dropout and residual behind the sum.  A thread takes eight elements of the flattened
// output, the unit of the dropout's counter; partial matrices lie elems apart, so they are read in vectors where that allows it.
__global__ void __launch_bounds__(256, 6) gemm_splitk_act_kernel(const float* __restrict__ slabs, __nv_bfloat16* __restrict__ c,
                                                              const float* __restrict__ bias, const __nv_bfloat16* __restrict__ bias_bf16,
                                                              const __nv_bfloat16* __restrict__ residual, int splits, int M, int N, GemmEpi e) {
    pdl_wait();
    pdl_launch_dependents();
    const long long elems = (long long)M * N, groups = (elems + 7) / 8;
    const bool vec = elems % 4 == 0;
    DropKey key = {};
    if (e.drop_threshold) key = drop_key(e.rng, e.site);
    for (long long g = (long long)blockIdx.x * blockDim.x + threadIdx.x; g < groups; g += (long long)gridDim.x * blockDim.x) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = 0.f;
        const long long i0 = g * 8;
        const int n = elems - i0 < 8 ? (int)(elems - i0) : 8;
        if (vec && n == 8) {
            for (int s = 0; s < splits; s++) {
                const float4* src = reinterpret_cast<const float4*>(slabs + s * elems + i0);
                const float4 a = src[0], b = src[1];
                f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w;
                f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
            }
        } else {
            for (int s = 0; s < splits; s++)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (j < n) f[j] += slabs[s * elems + i0 + j];
        }
        uint32_t mask = 0;
        if (e.drop_threshold) mask = drop_group_mask(key, (unsigned long long)g, e.drop_threshold);
        long long m = i0 / N;
        int col = (int)(i0 - m * N);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (j < n) {
                float a = f[j];
                if (bias) a += bias[col];
                if (bias_bf16) a += __bfloat162float(bias_bf16[col]);
                if (e.act) {
                    float slope;
                    a = act_slope(a, e.act, slope);
                    if (e.slope) e.slope[m * e.ld_slope + col] = __float2half_rn(slope);
                }
                if (e.drop_threshold) a = mask >> j & 1u ? a * e.drop_scale : 0.f;
                if (residual) a += __bfloat162float(residual[i0 + j]);
                f[j] = a;
            }
            if (++col == N) { col = 0; m++; }
        }
        if (n == 8) {
            uint4 pk;
            pk.x = gm_pack(f[0], f[1]); pk.y = gm_pack(f[2], f[3]); pk.z = gm_pack(f[4], f[5]); pk.w = gm_pack(f[6], f[7]);
            *reinterpret_cast<uint4*>(c + i0) = pk;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (j < n) c[i0 + j] = __float2bfloat16_rn(f[j]);
        }
    }
}

using GmEncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                     const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                     CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static GmEncodeTiledFn gm_encode_fn() {
    static const GmEncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<GmEncodeTiledFn>(f);
    }();
    return fn;
}

// Tensor map of one operand: `inner` contiguous elements per row, `outer` rows `ld` elements apart, two batch levels.
static bool gm_make_map(unsigned char* out, const void* base, long long inner, long long outer, long long ld, int nb_inner,
                        long long s_inner, int nb_outer, long long s_outer, int box_inner, int box_outer) {
    GmEncodeTiledFn enc = gm_encode_fn();
    if (!enc) return false;
    // a batch level of one problem still needs a legal (non-zero, 16-byte multiple) stride
    const long long si = nb_inner > 1 ? s_inner : ld * outer, so = nb_outer > 1 ? s_outer : si * (nb_inner > 1 ? nb_inner : 1);
    cuuint64_t dims[4] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)nb_inner, (cuuint64_t)nb_outer};
    cuuint64_t strides[3] = {(cuuint64_t)ld * 2, (cuuint64_t)si * 2, (cuuint64_t)so * 2};
    cuuint32_t box[4] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1, 1};
    cuuint32_t steps[4] = {1, 1, 1, 1};
    return enc(reinterpret_cast<CUtensorMap*>(out), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, steps,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tensor map of a bfloat16 matrix [M, N] that is copied 32 rows and 32 or 16 columns at a time (64- or 32-byte rows, swizzled).
static bool gm_make_slab_map(unsigned char* out, const void* base, int M, int N, long long ld, int cols) {
    GmEncodeTiledFn enc = gm_encode_fn();
    if (!enc) return false;
    cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)M};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {(cuuint32_t)cols, 32}, steps[2] = {1, 1};
    return enc(reinterpret_cast<CUtensorMap*>(out), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, steps,
               CU_TENSOR_MAP_INTERLEAVE_NONE, cols == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tile width, CTAs per tile and split factor of a problem.
//
// The smallest modelled time in microseconds: rounds of tiles, each as long as its k-blocks or as a tile's way out of tensor
// memory, whichever is longer, the way out of the last one, and for pairs the start of a launch in clusters.  Split-K (few tiles,
// long reduction) adds the second launch and writing and reading the partial matrices at about 6 TB/s.  The constants are a fit
// to 359 shapes (16 - 8192 tokens times the widths of the clients' layers in all three layouts, and batched attention products),
// each measured in every tiling, warm and back to back: the choice is 0.4 % slower than the fastest tiling of the same split on
// average, 7 % at worst.  That fit alone would have put the start of a launch in clusters at 1.8; in the models, where weights come
// from HBM, pairs gain more: BERT request 8 x 384 1466 us at 1.2 and below, 1522 at 1.8.
// A model of k-blocks alone took pairs where the way out bounds (64-deep products 512 x 512 x 256 problems: 54.2 us, 43.3 in single
// CTAs; 3072 x 1024 over 72 tokens 6.9, 6.2) and cut reductions that one round of 128-wide tiles had held (2048 x 768 x 3072: 34.5 us,
// 16.0 now; 3072 x 768 x 8192: 56.3, 33.7): where 128 x 128 tiles fill more than half of the device nothing is cut.
//
// The split is planned for the device's SM count, never for the quota of the call, so the summation order (and the result, bit for
// bit) is the same for every quota.  Tile width and pairing do not touch the order; they are chosen again for a smaller quota, where
// rounds are many and an odd CTA is lost to pairs (three CTAs, 3072 x 2304 x 768: 663 us in two, 348 in three).  With few CTAs at
// work a pair's k-block gains 7 % more on a single CTA's than on the full device (seven CTAs, 8192 x 1024 x 1024: 201 us in six, 212).
// Which splits a call may have.  GM_SPLIT_FILL is the rule above: few tiles are always cut until they fill the device.  GM_SPLIT_PRICED, of the
// epilogues that are not GM_EPI_PLAIN, weighs every number of parts, none among them, with a second launch that costs 4 us: 256 x 4096 x
// 1024 with bias and GELU, 64 tiles, 16.8 us in two parts and 9.3 in one.
enum GemmSplit { GM_SPLIT_NEVER, GM_SPLIT_FILL, GM_SPLIT_PRICED };
static GemmSplit gm_split_rule(int epi) {
    return epi == GM_EPI_LSE || epi == GM_EPI_DLOGITS ? GM_SPLIT_NEVER : epi == GM_EPI_PLAIN ? GM_SPLIT_FILL : GM_SPLIT_PRICED;
}
struct GemmPlan { int bn, cg, splits, grid; };
struct GemmTile { int bn, cg; double kblock_us, tile_us, tail_us, launch_us; };
static GemmPlan gm_plan(int M, int N, int K, long long batch, int tri, int device_sms, int num_ctas, GemmSplit rule = GM_SPLIT_FILL) {
    const bool splittable = rule != GM_SPLIT_NEVER;
    static const GemmTile kNarrow = {64, 1, 0.44, 2.15, 1.0, 0.0};   // outputs of at most 64 columns
    static const GemmTile kTiles[] = {{128, 1, 0.44, 2.15, 1.0, 0.0}, {256, 1, 0.51, 3.0, 2.0, 0.0},
                                      {128, 2, 0.32, 2.15, 1.0, 1.3}, {256, 2, 0.45, 3.0, 2.0, 1.3}};
    const GemmTile* list = N <= 64 && splittable ? &kNarrow : kTiles;
    const int count = N <= 64 && splittable ? 1 : 4;
    const long long kblocks = (K + GM_BK - 1) / GM_BK;
    auto tiles_of = [&](int bn, int cg) { return batch * (((long long)M + cg * GM_BM - 1) / (cg * GM_BM)) * (((long long)N + bn - 1) / bn); };
    auto fits = [&](const GemmTile& t) { return !((t.bn == 256 && N < 256) || (t.cg == 2 && (M <= GM_BM || tri != 0))); };
    auto price = [&](const GemmTile& t, int splits, long long at_once, double pair_relief) {
        const double rounds = (double)((tiles_of(t.bn, t.cg) * splits + at_once - 1) / at_once);
        const double depth = (double)((kblocks + splits - 1) / splits) * t.kblock_us * (t.cg == 2 ? pair_relief : 1.0);
        const double us = t.launch_us + rounds * (depth > t.tile_us ? depth : t.tile_us) + t.tail_us;
        return splits > 1 ? us + (rule == GM_SPLIT_PRICED ? 4.0 : 6.0) + (double)splits * batch * M * N * 8.0 / 6e6 : us;
    };
    const bool may_split = tiles_of(list[0].bn, 1) * 2 <= device_sms && kblocks >= 8 && tri == 0 && splittable;
    GemmPlan pl = {0, 1, 1, 1};
    double best = 0.0;
    for (int i = 0; i < count; i++) {
        const GemmTile& t = list[i];
        const long long at_once = device_sms / t.cg, tiles = tiles_of(t.bn, t.cg);
        if (!fits(t) || at_once < 1) continue;
        long long sp = 1;
        if (may_split && tiles * 2 <= at_once) {
            sp = at_once / tiles;
            if (sp > kblocks / 4) sp = kblocks / 4;
            if (sp > 16) sp = 16;
        }
        for (long long n = rule == GM_SPLIT_PRICED ? 1 : sp; n <= sp; n++) {
            const double us = price(t, (int)n, at_once, 1.0);
            if (pl.bn == 0 || us < best) { best = us; pl.bn = t.bn; pl.cg = t.cg; pl.splits = (int)n; }
        }
    }
    if (num_ctas < device_sms) {
        pl.bn = 0;
        for (int i = 0; i < count; i++) {
            const GemmTile& t = list[i];
            const long long at_once = num_ctas / t.cg;
            if (!fits(t) || at_once < 1) continue;
            const double us = price(t, pl.splits, at_once, 0.93);
            if (pl.bn == 0 || us < best) { best = us; pl.bn = t.bn; pl.cg = t.cg; }
        }
    }
    const long long ctas = tiles_of(pl.bn, pl.cg) * pl.splits * pl.cg, most = num_ctas / pl.cg * pl.cg;   // whole pairs
    pl.grid = (int)(ctas < most ? ctas : most);
    return pl;
}

template <int BN, int CG, int EPI>
static int gm_launch(const GemmParamsOf<EPI>& p, int grid, cudaStream_t stream) {
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 64 && !attr_set[dev]) {
        cudaError_t e = cudaFuncSetAttribute(gemm_bf16_kernel<BN, CG, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, (GemmCfg<BN, CG, EPI>::SMEM));
        if (e != cudaSuccess) return (int)e;
        attr_set[dev] = true;
    }
    OB200_ELASTIC((gemm_bf16_kernel<BN, CG, EPI>), 1);
    // Programmatic dependent launch: the kernel's set-up (barriers, tensor memory, descriptor prefetch) may overlap the tail of
    // the kernel before it in the stream; it reads and writes global memory only behind its griddepcontrol.wait.
    static const bool pdl = [] {   // ORION_PDL=0: plain stream order between consecutive kernels
        const char* e = getenv("ORION_PDL");
        return !(e && e[0] == '0');
    }();
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof cfg);
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(gm_threads(EPI));
    cfg.dynamicSmemBytes = (GemmCfg<BN, CG, EPI>::SMEM);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (CG == 2) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = 2;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    cfg.attrs = attr;
    cfg.numAttrs = (unsigned)n;
    return (int)cudaLaunchKernelEx(&cfg, gemm_bf16_kernel<BN, CG, EPI>, p);
}

}  // namespace ob200

extern "C" int* ob200_status_word_for_current_device(void);
extern "C" float* ob200_stream_slabs(void* stream, size_t* bytes);
extern "C" int ob200_plan_sm_count(void);

// See include/orion_kernels.h.
extern "C" int ob200_plan_gemm_bf16(int M, int N, int K, long long batch, int tri, int num_ctas, int* bn_out, int* ctas_per_tile_out,
                                    int* splits_out, int* grid_out) {
    if (M <= 0 || N <= 0 || K <= 0 || batch <= 0 || tri < 0 || tri > 3 || num_ctas <= 0) return -1;
    const ob200::GemmPlan pl = ob200::gm_plan(M, N, K, batch, tri, ob200_plan_sm_count(), num_ctas);
    if (bn_out) *bn_out = pl.bn;
    if (ctas_per_tile_out) *ctas_per_tile_out = pl.cg;
    if (splits_out) *splits_out = pl.splits;
    if (grid_out) *grid_out = pl.grid;
    return 0;
}

namespace ob200 {

size_t gemm_bf16_slab_bytes(int M, int N, int K, int epi) {
    const int sms = ob200_plan_sm_count();
    const GemmPlan pl = gm_plan(M, N, K, 1, 0, sms, sms, gm_split_rule(epi));
    return pl.splits > 1 ? (size_t)pl.splits * M * N * sizeof(float) : 0;
}

template <int EPI>
static int gm_launch_tile(const GemmParams& p, int bn, int cg, int grid, cudaStream_t st) {
    if (cg == 2) return bn == 256 ? gm_launch<256, 2, EPI>(p, grid, st) : gm_launch<128, 2, EPI>(p, grid, st);
    if (bn == 256) return gm_launch<256, 1, EPI>(p, grid, st);
    if constexpr (EPI != GM_EPI_LSE && EPI != GM_EPI_DLOGITS)
        if (bn == 64) return gm_launch<64, 1, EPI>(p, grid, st);
    return gm_launch<128, 1, EPI>(p, grid, st);
}

static int gm_finish4(const float* slabs, void* c, int out_f32, const float* addend, const float* factor, int splits, int M, int N, long long ldc, float alpha,
                      int num_ctas, cudaStream_t st, const int* live = nullptr, const GemmCutPlan& plan = {}) {
    const long long want = ((long long)M * N / 4 + 255) / 256, most = 8LL * num_ctas;
    const unsigned blocks = (unsigned)(want < most ? want : most);
    if (out_f32) {
        OB200_ELASTIC_HBM(gemm_splitk_finish4_kernel<float>, 8);
        return launch_pdl(gemm_splitk_finish4_kernel<float>, blocks, 256u, st, slabs, (float*)c, addend, factor, splits, M, N, ldc, alpha, live, plan);
    }
    OB200_ELASTIC_HBM(gemm_splitk_finish4_kernel<__nv_bfloat16>, 8);
    return launch_pdl(gemm_splitk_finish4_kernel<__nv_bfloat16>, blocks, 256u, st, slabs, (__nv_bfloat16*)c, addend, factor, splits, M, N, ldc, alpha, live, plan);
}

int gemm_bf16_run(const GemmCall& g) {
    const int M = g.M, N = g.N, K = g.K, a_mn = g.a_mn, b_mn = g.b_mn, batch_inner = g.batch_inner, batch_outer = g.batch_outer;
    const int out_f32 = g.out_f32, tri = g.tri, num_ctas = g.num_ctas;
    int epi = g.epi;
    const long long lda = g.lda, ldb = g.ldb, ldc = g.ldc, c_si = g.c_si, c_so = g.c_so;
    const void *a = g.a, *b = g.b, *residual = g.residual;
    void* c = g.c;
    if (tri < 0 || tri > 3) return -1;
    if (M < 0 || N < 0 || K <= 0 || batch_inner < 0 || batch_outer < 0 || num_ctas <= 0 || lda <= 0 || ldb <= 0 || ldc < N) return -1;
    if (M == 0 || N == 0 || batch_inner == 0 || batch_outer == 0) return 0;
    if (((uintptr_t)a | (uintptr_t)b) % 16 || (lda | ldb) % 8) return -2;
    if ((batch_inner > 1 && ((g.a_si | g.b_si) % 8)) || (batch_outer > 1 && ((g.a_so | g.b_so) % 8))) return -2;
    const long long batch_ll = (long long)batch_inner * batch_outer;
    if (batch_ll > 0x7fffffffLL) return -1;
    GemmParams p;
    memset(&p, 0, sizeof p);
    p.c = c; p.bias = g.bias;
    p.bias_bf16 = reinterpret_cast<const __nv_bfloat16*>(g.bias_bf16);
    p.residual = reinterpret_cast<const __nv_bfloat16*>(residual);
    p.status = ob200_status_word_for_current_device();
    p.M = M; p.N = N; p.K = K;
    p.batch = (int)batch_ll; p.nb_inner = batch_inner;
    p.ldc = ldc; p.c_si = c_si; p.c_so = c_so;
    p.out_f32 = out_f32 ? 1 : 0;
    p.a_mn = a_mn ? 1 : 0; p.b_mn = b_mn ? 1 : 0;
    p.alpha = g.alpha;
    p.tri = tri;
    p.e = g.e;
    const int cal = out_f32 ? 4 : 8;   // elements per 16 bytes of C
    p.vec_ok = ((uintptr_t)c % 16 == 0) && ((uintptr_t)residual % 16 == 0) && (!residual || !out_f32) && (ldc % cal == 0) && (batch_inner == 1 || c_si % cal == 0) && (batch_outer == 1 || c_so % cal == 0);
    const int plan = ob200_plan_sm_count();
    p.kblocks = (K + GM_BK - 1) / GM_BK;
    const GemmPlan pl = gm_plan(M, N, K, batch_ll, tri, plan, num_ctas, gm_split_rule(epi));
    const int bn = pl.bn, cg = pl.cg;
    int splits = pl.splits;
    p.tiles_m = (M + cg * GM_BM - 1) / (cg * GM_BM);
    p.tiles_n = (N + bn - 1) / bn;
    const long long tiles = batch_ll * p.tiles_m * p.tiles_n;
    if (tiles > 0x7fffffffLL) return -1;
    if (splits > 1) {
        size_t slab_bytes = g.slab_bytes;
        float* slabs = g.stream_slabs ? ob200_stream_slabs(g.stream, &slab_bytes) : g.slabs;
        const size_t per_split = (size_t)batch_ll * M * N * sizeof(float);
        if (!slabs || per_split == 0) splits = 1;
        else if ((size_t)splits * per_split > slab_bytes) splits = (int)(slab_bytes / per_split);
        if (splits < 2) splits = 1;
        p.slabs = splits > 1 ? slabs : nullptr;
    }
    p.kb_per_split = (p.kblocks + splits - 1) / splits;
    p.splits = (p.kblocks + p.kb_per_split - 1) / p.kb_per_split;   // every split owns at least one k-block
    if (p.splits <= 1) { p.splits = 1; p.slabs = nullptr; p.kb_per_split = p.kblocks; }
    const bool ok_a = a_mn ? gm_make_map(p.tmap_a, a, M, K, lda, batch_inner, g.a_si, batch_outer, g.a_so, 64, GM_BK)
                           : gm_make_map(p.tmap_a, a, K, M, lda, batch_inner, g.a_si, batch_outer, g.a_so, GM_BK, GM_BM);
    const bool ok_b = b_mn ? gm_make_map(p.tmap_b, b, N, K, ldb, batch_inner, g.b_si, batch_outer, g.b_so, 64, GM_BK)
                           : gm_make_map(p.tmap_b, b, K, N, ldb, batch_inner, g.b_si, batch_outer, g.b_so, GM_BK, bn / cg);
    if (!ok_a || !ok_b) return -4;
    if (g.live) {
        if (!gm_packs(epi) || batch_ll != 1 || tri || (g.live_k && epi != GM_EPI_ACC)) return -1;
        p.live = g.live;
        p.live_k = g.live_k;
        if (g.all) {   // the same boxes as the packed operand's
            p.live_all = g.live_k ? K : M;
            if (g.live_k ? !b_mn : epi == GM_EPI_ACC || a_mn) return -1;
            if (!(g.live_k ? gm_make_map(p.tmap_all, g.all, N, K, g.ld_all, 1, 0, 1, 0, 64, GM_BK)
                           : gm_make_map(p.tmap_all, g.all, K, M, g.ld_all, 1, 0, 1, 0, GM_BK, GM_BM)))
                return -4;
        }
    }
    // C by TMA stores when its rows and batch offsets are 16-byte multiples (always true for the layouts of the clients)
    {
        const int es = out_f32 ? 4 : 2;
        const bool aligned = ((uintptr_t)c % 16 == 0) && (ldc * es) % 16 == 0 && (batch_inner == 1 || (c_si * es) % 16 == 0) &&
                             (batch_outer == 1 || (c_so * es) % 16 == 0);
        static const bool tma_off = [] { const char* e = getenv("ORION_GEMM_TMA_STORE"); return e && e[0] == '0'; }();
        if (epi == GM_EPI_ACT || epi == GM_EPI_DLOGITS) {   // by slabs of 32 rows
            if (epi == GM_EPI_ACT && (!aligned || g.bias || ((uintptr_t)g.bias_bf16 | (uintptr_t)residual) % 16)) epi = GM_EPI_ACT_ANY;
            else if (epi == GM_EPI_ACT && g.e.slope) epi = GM_EPI_ACT_SLOPE;
            const int slab_cols = epi == GM_EPI_ACT_SLOPE ? 16 : 32;
            if (p.splits == 1 && ((epi != GM_EPI_ACT_ANY && !gm_make_slab_map(p.tmap_c, c, M, N, ldc, slab_cols)) ||
                                  (epi != GM_EPI_ACT_ANY && residual && !gm_make_slab_map(p.tmap_res, residual, M, N, N, slab_cols)) ||
                                  (g.e.slope && !gm_make_slab_map(p.tmap_slope, g.e.slope, M, N, g.e.ld_slope, slab_cols))))
                return -4;
        } else if (epi != GM_EPI_LSE && aligned && !tma_off && p.splits == 1) {
            GmEncodeTiledFn enc = gm_encode_fn();
            const long long si = batch_inner > 1 ? c_si : ldc * M, so = batch_outer > 1 ? c_so : si * (batch_inner > 1 ? batch_inner : 1);
            cuuint64_t dims[4] = {(cuuint64_t)N, (cuuint64_t)M, (cuuint64_t)batch_inner, (cuuint64_t)batch_outer};
            cuuint64_t strides[3] = {(cuuint64_t)ldc * es, (cuuint64_t)si * es, (cuuint64_t)so * es};
            cuuint32_t box[4] = {(cuuint32_t)(128 / es), 32, 1, 1};
            cuuint32_t steps[4] = {1, 1, 1, 1};
            if (enc && enc(reinterpret_cast<CUtensorMap*>(p.tmap_c), out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                           c, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS)
                p.c_tma = 1;
        }
    }
    const long long units = tiles * p.splits;
    int grid = units * cg < pl.grid ? (int)(units * cg) : pl.grid;   // fewer where the scratch took fewer splits
    // ORION_GEMM_TILES_PER_CTA=t (t > 0): a CTA retires after about t work units instead of staying for the whole launch, so
    // that the blocks of a higher-priority kernel find a free SM after a few microseconds (the grid is then wider than the
    // quota; the scheduler's cut to the quota, where it applies, still holds).
    static const int tiles_per_cta = [] { const char* e = getenv("ORION_GEMM_TILES_PER_CTA"); return e ? atoi(e) : 0; }();
    if (tiles_per_cta > 0) {
        const long long want = (units + tiles_per_cta - 1) / tiles_per_cta * cg;
        if (want > grid) grid = want > 0x7fffffff ? 0x7fffffff : (int)want;
    }
    {
        const double flop = 2.0 * batch_ll * M * (double)N * K;
        const double bytes = 2.0 * batch_ll * ((double)M * K + (double)N * K) + (out_f32 ? 4.0 : 2.0) * batch_ll * (double)M * N;
        annotate_launch(flop / bytes > ai_threshold(1) ? 1 : 0, flop, bytes);
    }
    cudaStream_t st = (cudaStream_t)g.stream;
    int rc;
    switch (epi) {
        case GM_EPI_ACC: rc = gm_launch_tile<GM_EPI_ACC>(p, bn, cg, grid, st); break;
        case GM_EPI_ACT: rc = gm_launch_tile<GM_EPI_ACT>(p, bn, cg, grid, st); break;
        case GM_EPI_ACT_SLOPE: rc = gm_launch_tile<GM_EPI_ACT_SLOPE>(p, bn, cg, grid, st); break;
        case GM_EPI_ACT_ANY: rc = gm_launch_tile<GM_EPI_ACT_ANY>(p, bn, cg, grid, st); break;
        case GM_EPI_LSE: return gm_launch_tile<GM_EPI_LSE>(p, bn, cg, grid, st);
        case GM_EPI_DLOGITS: return gm_launch_tile<GM_EPI_DLOGITS>(p, bn, cg, grid, st);
        default: rc = gm_launch_tile<GM_EPI_PLAIN>(p, bn, cg, grid, st);
    }
    if (rc != 0 || p.splits == 1) return rc;
    const long long elems = batch_ll * M * N;
    if (epi == GM_EPI_ACT || epi == GM_EPI_ACT_SLOPE || epi == GM_EPI_ACT_ANY) {
        long long blocks = ((elems + 7) / 8 + 255) / 256;
        if (blocks > 6LL * num_ctas) blocks = 6LL * num_ctas;
        OB200_ELASTIC_HBM(gemm_splitk_act_kernel, 6);
        return launch_pdl(gemm_splitk_act_kernel, (unsigned)blocks, 256u, st, (const float*)p.slabs, (__nv_bfloat16*)c, p.bias, p.bias_bf16, p.residual,
                          p.splits, M, N, p.e);
    }
    if (batch_ll == 1 && !g.bias && !p.bias_bf16 && !p.residual && N % 4 == 0 && ldc % 4 == 0 && (uintptr_t)c % 16 == 0)
        return gm_finish4(p.slabs, c, out_f32, epi == GM_EPI_ACC ? p.e.addend : nullptr, epi == GM_EPI_ACC ? p.e.factor : nullptr, p.splits, M, N, ldc,
                          g.alpha, num_ctas, st);
    long long blocks = (elems + 255) / 256;
    if (blocks > 4LL * num_ctas) blocks = 4LL * num_ctas;
    OB200_ELASTIC_HBM(gemm_splitk_finish_kernel, 4);
    gemm_splitk_finish_kernel<<<(int)blocks, 256, 0, st>>>(p.slabs, c, g.bias, p.bias_bf16, p.residual, epi == GM_EPI_ACC ? p.e.addend : nullptr,
                                                           epi == GM_EPI_ACC ? p.e.factor : nullptr, p.splits, p.batch,
                                                           p.nb_inner, M, N, ldc, c_si, c_so, p.out_f32, g.alpha);
    return (int)cudaGetLastError();
}

// Bfloat16 output, or float32 with its addend: 128 bytes x 32 rows a store.
static bool gm_make_c_map(unsigned char* out, const GemmCall& g) {
    GmEncodeTiledFn enc = gm_encode_fn();
    const int es = g.out_f32 ? 4 : 2;
    cuuint64_t dims[2] = {(cuuint64_t)g.N, (cuuint64_t)g.M};
    cuuint64_t strides[1] = {(cuuint64_t)g.ldc * es};
    cuuint32_t box[2] = {(cuuint32_t)(128 / es), 32}, steps[2] = {1, 1};
    return enc && enc(reinterpret_cast<CUtensorMap*>(out), g.out_f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                      g.c, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether two products run as one launch, and the split of the first one's reduction: 0 for no.  The fewest k-blocks of 64 on the CTA pair
// that has most of them, eight added for a tile's way out, and for a split the second launch and its partial matrices at 0.45 us a
// k-block and 6 TB/s.  Planned for the device, so that the order of the sums is the same for every CTA count.
// A first product of at most 128 rows (then the second one's reduction has two blocks at most, and its tiles' way out is all there is) runs
// in single CTAs: 16 x 512 x 512 with GELU, all launches of
// both directions, 18.7 -> 14.4 us, loss over 128 x 32000 x 1024 100 -> 92.  Otherwise pairs:
// outputs of at most 128 columns have narrower tiles in launches of their own; one of 136 is better in one tile of 256 than in two of
// 128 that read the other operand twice (gradient products of 6437 x 13042 x 136: 143 us in two launches, 77 in one).
static int gm_dual_ctas(const GemmCall& a) { return a.M <= GM_BM ? 1 : 2; }
int gemm_bf16_dual_splits(const GemmCall& a, const GemmCall& b) {
    const int cg = gm_dual_ctas(a), pairs = ob200_plan_sm_count() / cg;   // or single CTAs
    if (pairs < 1 || a.N % 8 || b.N % 8) return 0;
    if (cg == 2 && (b.M <= GM_BM || a.N <= 128 || b.N <= 128)) return 0;
    auto tiles = [cg](const GemmCall& g) { return (((long long)g.M - 1) / (cg * GM_BM) + 1) * (((long long)g.N + 255) / 256); };
    const long long ta = tiles(a), tb = tiles(b), ka = (a.K + 63) / 64, kb = (b.K + 63) / 64;
    int best = 1;
    double best_cost = 0.0;
    for (int s = 1; s <= 16 && s <= ka; s++) {
        if (s > 1 && (ta * s > 2 * pairs || ka / s < 4)) break;
        const long long ua = ta * s, ca = (ka + s - 1) / s + 8, cb = kb + 8;
        const long long longest = gemm_longest_share(pairs, ua, ca, tb, cb);
        const double cost = (double)longest + (s > 1 ? (3.0 + (double)s * a.M * a.N * 8.0 / 6e6) / 0.45 : 0.0);
        if (best_cost == 0.0 || cost < best_cost) { best = s; best_cost = cost; }
    }
    return best;
}
size_t gemm_bf16_dual_slab_bytes(const GemmCall& a, const GemmCall& b, bool packed) {
    const int s = gemm_bf16_dual_splits(a, b);
    return s > 1 || (packed && s > 0 && a.M > 256) ? (size_t)s * a.M * a.N * sizeof(float) : 0;
}

int gemm_bf16_run_dual(const GemmCall& a, const GemmCall& b) {
    int splits = gemm_bf16_dual_splits(a, b);
    if (splits < 1) return -1;
    const int kblocks = (a.K + GM_BK - 1) / GM_BK, per_split = (kblocks + splits - 1) / splits;
    splits = (kblocks + per_split - 1) / per_split;   // every split owns at least one k-block
    const bool recut = a.live && a.M > 256;   // fewer rows may be cut into more parts
    if ((splits > 1 || recut) && (!a.slabs || (size_t)splits * a.M * a.N * sizeof(float) > a.slab_bytes)) return -3;
    const int cg = a.num_ctas < 2 ? 1 : gm_dual_ctas(a), tile_m = cg * GM_BM;   // one CTA: tiles of 128 rows, the same sums
    GemmParamsDual p;
    memset(&p, 0, sizeof p);
    p.status = ob200_status_word_for_current_device();
    p.M = a.M; p.N = a.N; p.K = a.K;
    p.batch = p.nb_inner = 1;
    p.splits = splits;
    p.slabs = splits > 1 || recut ? a.slabs : nullptr;
    p.out_f32 = a.out_f32 ? 1 : 0;
    p.a_mn = a.a_mn; p.b_mn = a.b_mn;
    p.alpha = a.alpha;
    p.e = a.e;
    p.kblocks = kblocks;
    p.kb_per_split = per_split;
    p.tiles_m = (a.M - 1) / tile_m + 1;
    p.tiles_n = (a.N + 255) / 256;
    p.second.M = b.M; p.second.N = b.N;
    p.second.out_f32 = b.out_f32 ? 1 : 0;
    p.second.a_mn = b.a_mn; p.second.b_mn = b.b_mn;
    p.second.kblocks = (b.K + GM_BK - 1) / GM_BK;
    p.second.tiles_m = (b.M - 1) / tile_m + 1;
    p.second.tiles_n = (b.N + 255) / 256;
    p.cut = {a.M, p.tiles_n, kblocks, splits, per_split, (int)(((long long)b.M + 255) / 256) * p.second.tiles_n, p.second.kblocks, ob200_plan_sm_count() / 2};
    auto operands = [cg](const GemmCall& g, unsigned char* ta, unsigned char* tb) {
        return (g.a_mn ? gm_make_map(ta, g.a, g.M, g.K, g.lda, 1, 0, 1, 0, 64, GM_BK) : gm_make_map(ta, g.a, g.K, g.M, g.lda, 1, 0, 1, 0, GM_BK, GM_BM)) &&
               (g.b_mn ? gm_make_map(tb, g.b, g.N, g.K, g.ldb, 1, 0, 1, 0, 64, GM_BK) : gm_make_map(tb, g.b, g.K, g.N, g.ldb, 1, 0, 1, 0, GM_BK, 256 / cg));
    };
    if (!operands(a, p.tmap_a, p.tmap_b) || !operands(b, p.second.tmap_a, p.second.tmap_b) || !gm_make_c_map(p.tmap_c, a) ||
        !gm_make_c_map(p.second.tmap_c, b))
        return -4;
    p.c_tma = 1;
    if (a.live) {   // rows of the first product, the reduction of the second
        if (b.live != a.live || a.live_k || !b.live_k || a.M != b.K) return -1;
        p.live = a.live;
        if (b.all) {
            p.live_all = b.K;
            if (!b.b_mn) return -1;
            if (!gm_make_map(p.tmap_all, b.all, b.N, b.K, b.ld_all, 1, 0, 1, 0, 64, GM_BK)) return -4;
        }
    }
    const long long tiles = (long long)p.tiles_m * p.tiles_n * splits + (long long)p.second.tiles_m * p.second.tiles_n;
    if (tiles > 0x3fffffffLL) return -1;
    const long long most = a.num_ctas / cg;
    annotate_launch(1, 2.0 * ((double)a.M * a.N * a.K + (double)b.M * b.N * b.K),
                    2.0 * ((double)a.M * a.K + (double)a.K * a.N + (double)b.M * b.K + (double)b.K * b.N));
    const int grid = (int)(tiles < most ? tiles : most) * cg;
    const int rc = cg == 2 ? gm_launch<256, 2, GM_EPI_DUAL>(p, grid, (cudaStream_t)a.stream) : gm_launch<256, 1, GM_EPI_DUAL>(p, grid, (cudaStream_t)a.stream);
    if (rc || (splits == 1 && !recut)) return rc;
    return gm_finish4(p.slabs, a.c, a.out_f32, a.e.addend, a.e.factor, splits, a.M, a.N, a.ldc, a.alpha, a.num_ctas, (cudaStream_t)a.stream,
                      a.live, p.cut);
}

}  // namespace ob200

// See include/orion_kernels.h.  Returns 0, -1 (unsupported sizes), -2 (misaligned pointers or strides), -4 (no TMA descriptor).
extern "C" int ob200_gemm_bf16_ex(const void* a, const void* b, void* c, const float* bias, const void* bias_bf16, const void* residual,
                                  int M, int N, int K, int a_mn, int b_mn, long long lda, long long ldb, long long ldc, int batch_inner,
                                  int batch_outer, long long a_si, long long a_so, long long b_si, long long b_so, long long c_si,
                                  long long c_so, float alpha, int out_f32, int tri, int num_ctas, void* stream) {
    ob200::GemmCall g;
    g.a = a; g.b = b; g.c = c;
    g.bias = bias; g.bias_bf16 = bias_bf16; g.residual = residual;
    g.M = M; g.N = N; g.K = K; g.a_mn = a_mn; g.b_mn = b_mn;
    g.lda = lda; g.ldb = ldb; g.ldc = ldc;
    g.batch_inner = batch_inner; g.batch_outer = batch_outer;
    g.a_si = a_si; g.a_so = a_so; g.b_si = b_si; g.b_so = b_so; g.c_si = c_si; g.c_so = c_so;
    g.alpha = alpha; g.out_f32 = out_f32; g.tri = tri;
    g.stream_slabs = true;
    g.num_ctas = num_ctas; g.stream = stream;
    return ob200::gemm_bf16_run(g);
}

extern "C" int ob200_gemm_bf16(const void* a, const void* b, void* c, const float* bias, int M, int N, int K, int a_mn, int b_mn,
                               long long lda, long long ldb, long long ldc, int batch_inner, int batch_outer, long long a_si,
                               long long a_so, long long b_si, long long b_so, long long c_si, long long c_so, float alpha, int out_f32,
                               int num_ctas, void* stream) {
    return ob200_gemm_bf16_ex(a, b, c, bias, nullptr, nullptr, M, N, K, a_mn, b_mn, lda, ldb, ldc, batch_inner, batch_outer, a_si, a_so,
                              b_si, b_so, c_si, c_so, alpha, out_f32, 0, num_ctas, stream);
}
