// Products of a few rows (single tokens of a few sequences, a short prompt) with a weight matrix, the epilogues of linear_act and of the
// loss without logits behind them, in one launch:  z[m, n] = sum_k x[m, k] w[n, k].
//
// Bound: reading w once.  Rows of w are the 16-row operand of mma.sync and the tokens its 8 columns, so that nothing is padded to a
// 128-row tensor-memory tile whose way in and out takes longer than the whole product: 4096 x 1024 with bias and GELU, w from HBM,
// launches back to back, 9.7 -> 4.6 us at one token, 9.8 -> 6.4 at sixteen, 11.8 -> 6.8 at 32.  A lane reads 16 bytes of two rows of w
// and of a row of x at the same k and gives the instruction pairs of them as if they lay in its order: the order of a sum's terms is
// free, as long as both operands share it, so wide accesses are all there is.  Warps share a tile's reduction and join their sums
// through shared memory in a fixed order.
// Two kernels: w straight to registers where an SM has a tile or two, and where it has many, through a ring of TMA copies.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "elastic.h"
#include "fast_gelu.cuh"
#include "gemm_call.h"
#include "philox.cuh"
#include "sm100_primitives.cuh"

extern "C" int ob200_plan_sm_count(void);
extern "C" int* ob200_status_word_for_current_device(void);

namespace ob200 {

constexpr int FEW_MAX_ROWS = 32;
constexpr int FEW_CONSUMERS = 16, FEW_GROUPS = 4;                  // warps that multiply, and the groups they form
constexpr int FEW_THREADS = (FEW_CONSUMERS + 1) * 32;              // the last warp issues the copies
constexpr int FEW_BOX = 256, FEW_CHUNK = 2 * FEW_BOX;               // reduction indices of a copy and of a stage
constexpr int FEW_MAX_STAGES = 12, FEW_MAX_CHUNKS = 32;
constexpr int FEW_SMEM = 224 * 1024;

struct FewRowsParams {
    const __nv_bfloat16 *x, *w;
    long long ldx, ldw;
    int M, N, K;
    int tile_rows;         // rows of w in a tile: 16, or 8 (half of the operand's rows idle) where that employs more SMs
    int chunks;            // stages of a tile
    int stages;            // of a group's ring
    int* status;
    const float* bias;
    const __nv_bfloat16 *bias_bf16, *residual;
    __nv_bfloat16* c;
    GemmEpi e;
    alignas(64) unsigned char tmap_x[128], tmap_w[128];   // boxes of 256 columns; zeros past the edges
};

struct FewCtl {
    uint64_t full[FEW_MAX_STAGES], empty[FEW_MAX_STAGES], x_full[FEW_MAX_CHUNKS];
    int abort_flag;
};
constexpr int FEW_CTL = 512;
static_assert(sizeof(FewCtl) <= FEW_CTL, "the barriers lie ahead of the sums");

__device__ __forceinline__ void few_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 few_load(const __nv_bfloat16* p) {   // read once: past the L1 cache
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
template <int NT, int LD>
__device__ __forceinline__ void few_put(float (&red)[16][LD], const float (&acc)[NT][4], int g, int t) {
#pragma unroll
    for (int i = 0; i < NT; i++) {
        red[g][i * 8 + 2 * t] = acc[i][0];
        red[g][i * 8 + 2 * t + 1] = acc[i][1];
        red[g + 8][i * 8 + 2 * t] = acc[i][2];
        red[g + 8][i * 8 + 2 * t + 1] = acc[i][3];
    }
}

// A tile's way out, by WARPS warps, for tokens [first, first + tokens): the sums of the warps that shared the reduction are joined in
// their order, then either the epilogue of linear_act, a thread an output, or, half a warp a token and a lane a row of w, the maximum,
// the sum of exponentials and the label's logit.
template <int WARPS, int LD, bool LSE>
__device__ __forceinline__ void few_way_out(const FewRowsParams& p, const float (*red)[16][LD], int tile, int first, int tokens, int id, int warp, int lane) {
    const int n0 = tile * p.tile_rows;
    if constexpr (LSE) {
        const int r = lane & 15;
        for (int m0 = warp * 2; m0 < tokens; m0 += 2 * WARPS) {
            const int m = m0 + (lane >> 4);
            float v = -INFINITY;
            if (m < tokens && r < p.tile_rows && n0 + r < p.N) {
                v = 0.f;
#pragma unroll
                for (int k = 0; k < WARPS; k++) v += red[k][r][m];
                if (p.e.target[first + m] - n0 == r) p.e.label_logit[first + m] = v;
            }
            float top = v;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            float sum = exp2f((v - (top == -INFINITY ? 0.f : top)) * 1.4426950408889634f);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (r == 0 && m < tokens) p.e.part[(long long)tile * p.M + first + m] = make_float2(top, sum);
        }
    } else {
        for (int i = id; i < p.tile_rows * tokens; i += WARPS * 32) {
            const int r = i % p.tile_rows, m = i / p.tile_rows, n = n0 + r;
            if (n >= p.N) continue;
            const long long index = (long long)(first + m) * p.N + n;
            const float add = p.bias ? p.bias[n] : p.bias_bf16 ? __bfloat162float(p.bias_bf16[n]) : 0.f;
            const float res = p.residual ? __bfloat162float(p.residual[index]) : 0.f;
            float z = 0.f;
#pragma unroll
            for (int k = 0; k < WARPS; k++) z += red[k][r][m];
            z += add;
            if (p.e.act) {
                float slope;
                z = act_slope(z, p.e.act, slope);
                if (p.e.slope) p.e.slope[(first + m) * p.e.ld_slope + n] = __float2half_rn(slope);
            }
            if (p.e.drop_threshold) {
                uint32_t bits[4];
                drop_bits(drop_key(p.e.rng, p.e.site), (unsigned long long)index >> 3, bits);
                const int half = (int)(index & 7);
                const uint32_t word = half < 4 ? (half < 2 ? bits[0] : bits[1]) : (half < 6 ? bits[2] : bits[3]);
                z = (half & 1 ? word : word << 16) > drop_limit(p.e.drop_threshold) ? z * p.e.drop_scale : 0.f;
            }
            p.c[index] = __float2bfloat16_rn(z + res);
        }
    }
}

// ------------------------------------------------------------------ few tiles: straight to registers
// Sixteen warps share a tile's reduction, four k-blocks of 32 (two of them for 32 tokens) under way in each.  There is no ring to fill and
// no copy to wait for, so a launch of one or two tiles an SM is over sooner: 1024 x 4096 at one token 7.6 -> 5.7 us, at sixteen 8.4 -> 6.1.
// More than 32 tokens are groups of 32, each with tiles of its own: w is then read from L2 once a group.
// few_resident: CTAs an SM, what the launch bound, the quota's cut and the grid go by.  One of 9 to 16 tokens has the registers of two
// (110 a thread).
constexpr int few_resident(int nt) { return nt == 2 ? 1 : 2; }
template <int NT, bool LSE>
__global__ void __launch_bounds__(FEW_CONSUMERS * 32, few_resident(NT)) few_tiles_kernel(const __grid_constant__ FewRowsParams p) {
    constexpr int LD = NT * 8 + 1, WARPS = FEW_CONSUMERS, DEPTH = NT == 4 ? 2 : 4;
    __shared__ float red[WARPS][16][LD];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int kblocks = (p.K + 31) / 32, kb0 = kblocks * warp / WARPS, kb1 = kblocks * (warp + 1) / WARPS;
    const int tiles = (p.N + p.tile_rows - 1) / p.tile_rows;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int unit = blockIdx.x; unit < tiles * ((p.M + 31) / 32); unit += gridDim.x) {
        const int tile = unit % tiles, first = unit / tiles * 32, tokens = p.M - first < 32 ? p.M - first : 32;
        const int r0 = tile * p.tile_rows + g, r1 = r0 + 8;
        const bool has0 = r0 < p.N, has1 = p.tile_rows == 16 && r1 < p.N;
        const __nv_bfloat16 *w0 = p.w + (long long)r0 * p.ldw + t * 8, *w1 = w0 + 8 * p.ldw, *x0 = p.x + (long long)(first + g) * p.ldx + t * 8;
        float acc[NT][4];
#pragma unroll
        for (int i = 0; i < NT; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
        for (int kb = kb0; kb < kb1; kb += DEPTH) {
            uint4 a[DEPTH][2], b[DEPTH][NT];
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                const int k = (kb + d) * 32;
                const bool in = kb + d < kb1 && k + t * 8 < p.K;   // K is a multiple of 8
                a[d][0] = in && has0 ? few_load(w0 + k) : zero;
                a[d][1] = in && has1 ? few_load(w1 + k) : zero;
#pragma unroll
                for (int i = 0; i < NT; i++) b[d][i] = in && g + i * 8 < tokens ? __ldg(reinterpret_cast<const uint4*>(x0 + i * 8 * p.ldx + k)) : zero;
            }
#pragma unroll
            for (int d = 0; d < DEPTH; d++)
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    few_mma(acc[i], a[d][0].x, a[d][1].x, a[d][0].y, a[d][1].y, b[d][i].x, b[d][i].y);
                    few_mma(acc[i], a[d][0].z, a[d][1].z, a[d][0].w, a[d][1].w, b[d][i].z, b[d][i].w);
                }
        }
        few_put(red[warp], acc, g, t);
        __syncthreads();
        few_way_out<WARPS, LD, LSE>(p, red, tile, first, tokens, threadIdx.x, warp, lane);
        __syncthreads();
    }
}

// ------------------------------------------------------------------ many tiles: a ring of copies
// Up to 190 KB of w are under way in an SM, in boxes of 256 reduction indices (a bulk copy for each row's piece took about 100 cycles,
// whatever its length).  Four groups of four warps take tiles in turn, so that one on its way out holds up no copies.  A group has its own
// ring and waits on its stages in their order: copies land in any order, and a barrier's parity tells only neighbouring uses apart.
// Every wait is bounded; a warp that gives up goes on meeting the others of its group, and the CTA leaves with no copy under way.
template <int NT, bool LSE>   // NT * 8 >= M columns of tokens
__global__ void __launch_bounds__(FEW_THREADS, 1) few_rows_kernel(const __grid_constant__ FewRowsParams p) {
    constexpr int LD = NT * 8 + 1, GROUPS = FEW_GROUPS, WARPS = FEW_CONSUMERS / GROUPS;
    extern __shared__ __align__(128) uint8_t few_smem[];
    FewCtl* ctl = reinterpret_cast<FewCtl*>(few_smem);
    float(*red)[WARPS][16][LD] = reinterpret_cast<float(*)[WARPS][16][LD]>(few_smem + FEW_CTL);   // [GROUPS]
    uint8_t* xs = few_smem + FEW_CTL + FEW_CONSUMERS * 16 * LD * 4;
    const int x_box = NT * 8 * FEW_BOX * 2, w_box = p.tile_rows * FEW_BOX * 2;
    uint8_t* ring = xs + (p.K + FEW_BOX - 1) / FEW_BOX * x_box;
    const int tid = threadIdx.x, warp = uniform_warp_index(), lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < GROUPS * p.stages; s++) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], WARPS);
        }
        for (int c = 0; c < p.chunks; c++) mbar_init(&ctl->x_full[c], 1);
        ctl->abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == FEW_CONSUMERS && lane == 0) {
        prefetch_tensormap(p.tmap_w);
        prefetch_tensormap(p.tmap_x);
    }
    __syncthreads();
    pdl_wait();
    pdl_launch_dependents();
    const int tiles = (p.N + p.tile_rows - 1) / p.tile_rows;
    volatile int* abort_flag = &ctl->abort_flag;
    auto give_up = [&](int code) {
        if (!*abort_flag) {
            ctl->abort_flag = 1;
            if (p.status) atomicExch(p.status, code);
        }
    };

    if (warp == FEW_CONSUMERS) {
        // ------------------------------------------------------------ copies; the tokens, which stay, with those of the first tile
        int turn = 0, c = 0;
        bool dead = false;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn++) {
            const int group = turn % GROUPS;
            for (c = 0; c < p.chunks; c++) {
                const int step = turn / GROUPS * p.chunks + c, s = group * p.stages + step % p.stages;
                if (!mbar_wait_warp(&ctl->empty[s], ((uint32_t)(step / p.stages) & 1u) ^ 1u, abort_flag)) {
                    give_up(OB200_ERR_WAIT_EMPTY);
                    dead = true;
                    break;
                }
                const int k0 = c * FEW_CHUNK, boxes = p.K - k0 > FEW_BOX ? 2 : 1;
                if (elect_one()) {
                    if (turn == 0) {
                        mbar_arrive_expect_tx(&ctl->x_full[c], (uint32_t)(boxes * x_box));
                        for (int i = 0; i < boxes; i++) tma_load_tile_2d(smem_u32(xs + (2 * c + i) * x_box), p.tmap_x, &ctl->x_full[c], k0 + i * FEW_BOX, 0);
                    }
                    mbar_arrive_expect_tx(&ctl->full[s], (uint32_t)(boxes * w_box));
                    for (int i = 0; i < boxes; i++)
                        tma_load_tile_2d(smem_u32(ring + (2 * s + i) * w_box), p.tmap_w, &ctl->full[s], k0 + i * FEW_BOX, tile * p.tile_rows);
                }
                __syncwarp();
            }
            if (dead) break;
        }
        for (int group = 0; group < GROUPS; group++) {   // copies issued into each ring: of whole tiles, and of the one it gave up on
            const int n = (turn + GROUPS - 1 - group) / GROUPS * p.chunks + (dead && turn % GROUPS == group ? c : 0);
            ring_settle(ctl->full + group * p.stages, p.stages, n % p.stages, (uint32_t)(n / p.stages) & 1u, p.stages);
        }
        const long long t0 = clock64();
        for (int i = 0; i < (turn > 0 ? p.chunks : c); i++) mbar_wait_landed(&ctl->x_full[i], 0, t0);
        __syncwarp();
    } else {
        // ------------------------------------------------------------ products, and a tile's way out
        const int group = warp / WARPS, kw = warp % WARPS, g = lane >> 2, t = lane & 3, id = tid - group * WARPS * 32;
        auto meet = [&] { asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(WARPS * 32) : "memory"); };
        bool ok = true;
        int step = 0;   // stages of the group's ring so far
        int turn = 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn++) {
            if (turn % GROUPS != group) continue;
            float acc[NT][4];
#pragma unroll
            for (int i = 0; i < NT; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
            for (int c = 0; c < p.chunks; c++, step++) {
                const int s = group * p.stages + step % p.stages, left = p.K - c * FEW_CHUNK < FEW_CHUNK ? p.K - c * FEW_CHUNK : FEW_CHUNK;
                if (ok) ok = mbar_wait_warp(&ctl->x_full[c], 0, abort_flag) && mbar_wait_warp(&ctl->full[s], (uint32_t)(step / p.stages) & 1u, abort_flag);
                if (!ok) continue;
                const int kblocks = (left + 31) / 32, kb1 = kblocks * (kw + 1) / WARPS;
                const uint8_t *w0 = ring + 2 * s * w_box + g * (FEW_BOX * 2) + t * 16, *x0 = xs + 2 * c * x_box + g * (FEW_BOX * 2) + t * 16;
#pragma unroll 4
                for (int kb = kblocks * kw / WARPS; kb < kb1; kb++) {
                    const int box = kb >> 3, at = (kb & 7) * 64;
                    const uint8_t* wk = w0 + box * w_box + at;
                    const uint4 a = *reinterpret_cast<const uint4*>(wk);
                    uint4 b = make_uint4(0, 0, 0, 0);
                    if (p.tile_rows == 16) b = *reinterpret_cast<const uint4*>(wk + 8 * FEW_BOX * 2);
#pragma unroll
                    for (int i = 0; i < NT; i++) {
                        const uint4 x = *reinterpret_cast<const uint4*>(x0 + box * x_box + i * 8 * FEW_BOX * 2 + at);
                        few_mma(acc[i], a.x, b.x, a.y, b.y, x.x, x.y);
                        few_mma(acc[i], a.z, b.z, a.w, b.w, x.z, x.w);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl->empty[s]);
            }
            if (!ok) give_up(OB200_ERR_WAIT_FULL);
            meet();   // the sums of the group's tile before have been read
            few_put(red[group][kw], acc, g, t);
            meet();
            if (!ok) continue;
            few_way_out<WARPS, LD, LSE>(p, red[group], tile, 0, p.M, id, kw, lane);
        }
    }
}

// 16 rows of w a tile, or 8 where tiles of 16 would leave SMs without one.
static int few_tile_rows(int M, int N) { return (long long)(N + 15) / 16 * ((M + 31) / 32) >= ob200_plan_sm_count() ? 16 : 8; }

// Whether a launch is of few tiles: two an SM, which are resident at once but for 9 to 16 tokens, whose CTAs take them one after the other
// (4096 x 1024, 256 tiles: 6.4 us in 148 CTAs, 7.0 in 256).  By the sizes and the device, because it sets the order of a sum.
// 32000 x 1024, one token: 25.7 us straight to registers, 14.7 through the ring; 16 tokens 35.9 and 18.1.  4096 x 1024: 4.6 and 4.9; 16
// tokens 6.4 and 5.4.
static bool few_tiles(int M, int N) {
    const int rows = few_tile_rows(M, N);
    return ((long long)N + rows - 1) / rows * ((M + 31) / 32) <= 2 * ob200_plan_sm_count();
}

struct FewPlan { int stages, bytes; };
static FewPlan few_plan(int M, int N, int K) {
    if (K > FEW_CHUNK * FEW_MAX_CHUNKS) return {0, 0};
    const int nt = M <= 8 ? 1 : M <= 16 ? 2 : 4, boxes = (K + FEW_BOX - 1) / FEW_BOX;
    const int fixed = FEW_CTL + FEW_CONSUMERS * 16 * (nt * 8 + 1) * 4 + boxes * nt * 8 * FEW_BOX * 2, stage_bytes = few_tile_rows(M, N) * FEW_CHUNK * 2;
    FewPlan f;
    const int room = FEW_SMEM - fixed, stages = room > 0 ? room / stage_bytes : 0;
    f.stages = (stages < FEW_MAX_STAGES ? stages : FEW_MAX_STAGES) / FEW_GROUPS;
    f.bytes = fixed + FEW_GROUPS * f.stages * stage_bytes;
    return f;
}

using FewEncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// bfloat16 rows of `cols` columns, `ld` apart, in boxes of 256 columns and `box_rows` rows.
static bool few_make_map(unsigned char* out, const void* base, int cols, int rows, long long ld, int box_rows) {
    static const FewEncodeFn enc = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<FewEncodeFn>(f);
    }();
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {FEW_BOX, (cuuint32_t)box_rows}, steps[2] = {1, 1};
    return enc && enc(reinterpret_cast<CUtensorMap*>(out), CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, steps,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool few_rows_fit(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0) return false;
    return few_tiles(M, N) || (M <= FEW_MAX_ROWS && few_plan(M, N, K).stages >= 2);
}
int few_rows_parts(int M, int V) { return (V + few_tile_rows(M, V) - 1) / few_tile_rows(M, V); }

template <int NT, bool LSE>
static int few_launch(const FewRowsParams& p, int num_ctas, cudaStream_t stream) {
    const int tiles = (p.N + p.tile_rows - 1) / p.tile_rows;
    if (few_tiles(p.M, p.N)) {
        const int units = tiles * ((p.M + 31) / 32), most = few_resident(NT) * num_ctas;
        OB200_ELASTIC_HBM((few_tiles_kernel<NT, LSE>), few_resident(NT));
        return launch_pdl(few_tiles_kernel<NT, LSE>, (unsigned)(units < most ? units : most), FEW_CONSUMERS * 32u, stream, p);
    }
    static bool attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 64 && !attr_set[dev]) {
        cudaError_t e = cudaFuncSetAttribute(few_rows_kernel<NT, LSE>, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM);
        if (e != cudaSuccess) return (int)e;
        attr_set[dev] = true;
    }
    OB200_ELASTIC_HBM((few_rows_kernel<NT, LSE>), 1);
    return launch_pdl_smem(few_rows_kernel<NT, LSE>, (unsigned)(tiles < num_ctas ? tiles : num_ctas), (unsigned)FEW_THREADS,
                           (size_t)few_plan(p.M, p.N, p.K).bytes, stream, p);
}

int few_rows_run(const GemmCall& g) {
    if (((uintptr_t)g.a | (uintptr_t)g.b) % 16 || (g.lda | g.ldb) % 8) return -2;
    FewRowsParams p;
    p.x = (const __nv_bfloat16*)g.a; p.w = (const __nv_bfloat16*)g.b;
    p.ldx = g.lda; p.ldw = g.ldb;
    p.M = g.M; p.N = g.N; p.K = g.K;
    p.tile_rows = few_tile_rows(g.M, g.N);
    p.chunks = (g.K + FEW_CHUNK - 1) / FEW_CHUNK;
    p.stages = few_plan(g.M, g.N, g.K).stages;
    p.status = nullptr;
    if (!few_tiles(g.M, g.N)) {   // the other kernel copies by TMA, and waits
        const int box = g.M <= 8 ? 8 : g.M <= 16 ? 16 : 32;
        if (!few_make_map(p.tmap_x, g.a, g.K, g.M, g.lda, box) || !few_make_map(p.tmap_w, g.b, g.K, g.N, g.ldb, p.tile_rows)) return -4;
        p.status = ob200_status_word_for_current_device();
    }
    p.bias = g.bias;
    p.bias_bf16 = (const __nv_bfloat16*)g.bias_bf16;
    p.residual = (const __nv_bfloat16*)g.residual;
    p.c = (__nv_bfloat16*)g.c;
    p.e = g.e;
    cudaStream_t st = (cudaStream_t)g.stream;
    const bool lse = g.epi == GM_EPI_LSE;
    if (g.M <= 8) return lse ? few_launch<1, true>(p, g.num_ctas, st) : few_launch<1, false>(p, g.num_ctas, st);
    if (g.M <= 16) return lse ? few_launch<2, true>(p, g.num_ctas, st) : few_launch<2, false>(p, g.num_ctas, st);
    return lse ? few_launch<4, true>(p, g.num_ctas, st) : few_launch<4, false>(p, g.num_ctas, st);
}

}  // namespace ob200
