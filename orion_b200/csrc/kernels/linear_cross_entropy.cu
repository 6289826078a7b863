// Softmax cross-entropy of logits x . w^T over a large vocabulary, and its gradients, without the logits:
//
//   loss[t] = lse[t] - l[t, target[t]],   l = x . w^T,   lse[t] = log sum_v exp(l[t, v])
//   dl = exp(l - lse) - onehot(target);   dx = c dl . w;   dw = c dl^T . x       c = upstream gradient (/ rows that count)
//
// Forward: one GEMM whose epilogue keeps, of every row and 128 columns, the maximum and the sum of exponentials (gemm_bf16.cu,
// GM_EPI_LSE), and a kernel that joins them: 2 T V H operations and V / 16 bytes a row instead of 2 V.  Backward, in pieces of the
// vocabulary: the logits of a piece are computed again and leave the epilogue as dl in bfloat16 (GM_EPI_DLOGITS), which the two gradient
// products read.  Computing a logit again costs 2 H operations, 1.5 ps on a B200 at H = 1024; keeping it in float32 would cost 4 bytes
// written and 4 read, 1.2 ps, and the memory.  dl is rounded to bfloat16 because the tensor cores take it so: an error of at most
// 2^-9 of each term of dx and dw, as large as that of the rounded result.  dx adds up over the pieces in float32.
// Rows that do not count are left out of every product, by a count that stays on the device (ce_pack_kernel).
// The tensor core bounds it.  8192 x 32000 x 1024: forward 320 us (1.68 PFLOP/s), a third of the logits' gradient 121 (1.49), both gradient
// products of a third 222 (1.63), alone and cold; back to back under the power limit 1.5 - 1.8 ms a step, 1.2 - 1.43 PFLOP/s.  With its
// logits kept (linear_train and cross_entropy) the same step takes 1.41 ms where this takes 1.48, and 1000 MB beside its results, not 343.
// It stands where the reference's clients launch the vocabulary projection's product and the softmax and loss rows behind it
// (reference benchmarking/model_kernels/bert_8_fb1; src/scheduler/utils_sched.cpp:490-501).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "elastic.h"
#include "gemm_call.h"
#include "pdl.cuh"

extern "C" int ob200_plan_sm_count(void);

namespace ob200 {

constexpr int CE_THREADS = 256, CE_PACK_THREADS = 512;
constexpr int CE_IN_PLACE = 128;   // rows of one tile: fewer of them cost the same
constexpr float CE_LOG2E = 1.4426950408889634f;

// lse and loss of every row from its parts.  A CTA has C rows; group g of G = 1024 / C takes parts g, g + G, ..., eight at a time in
// registers (the kernel is a few dependent steps long: their loads are one), then the groups are joined in a fixed tree.  32 rows, or 4
// where rows are few and their parts many.  1024 threads of 64 registers: one CTA an SM.  Packed rows (`order`): row r of the parts is
// row order[r], and those from *live on do not count.
template <int C>
__global__ void __launch_bounds__(1024) ce_rows_kernel(const float2* __restrict__ part, const float* __restrict__ label_logit,
                                                       const long long* __restrict__ target, float* __restrict__ loss, float* __restrict__ lse,
                                                       const int* order, const int* live, int rows, int parts, int V, long long ignore_index) {
    pdl_wait();
    pdl_launch_dependents();
    const int counted = live ? *live : rows;
    constexpr int G = 1024 / C;
    __shared__ float2 sh[G][C + 1];
    const int c = threadIdx.x % C, g = threadIdx.x / C, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // A maximum of minus infinity has a sum of 0, or one that is not a number; it is weighed with 1, so that the latter stays.
    auto weight = [](float top, float now) { return top == -INFINITY ? 1.f : exp2f((top - now) * CE_LOG2E); };
    for (int r0 = blockIdx.x * C; r0 < rows; r0 += gridDim.x * C) {
        const int r = r0 + c;
        float top = -INFINITY, sum = 0.f;
        for (int t0 = g; t0 < parts; t0 += 8 * G) {
            float2 q[8];
#pragma unroll
            for (int i = 0; i < 8; i++) q[i] = r < counted && t0 + G * i < parts ? part[(long long)(t0 + G * i) * rows + r] : make_float2(-INFINITY, 0.f);
            float now = top;
#pragma unroll
            for (int i = 0; i < 8; i++) now = fmaxf(now, q[i].x);
            sum *= weight(top, now);
#pragma unroll
            for (int i = 0; i < 8; i++) sum += q[i].y * weight(q[i].x, now);
            top = now;
        }
        sh[g][c] = make_float2(top, sum);
        __syncthreads();
        if (warp < C && r0 + warp < rows) {   // warp w joins the groups of row r0 + w
            float2 q[G / 32];
            float now = -INFINITY, all = 0.f;
#pragma unroll
            for (int i = 0; i < G / 32; i++) {
                q[i] = sh[i * 32 + lane][warp];
                now = fmaxf(now, q[i].x);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, o));
#pragma unroll
            for (int i = 0; i < G / 32; i++) all += q[i].y * weight(q[i].x, now);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
            if (lane == 0) {
                const int row = r0 + warp, to = order ? order[row] : row;
                // The maximum itself weighs 1 but for roundings.  The loss is taken from the maximum, not from lse, whose rounding would be
                // all that is left of the loss of a row that is sure.
                const float log_sum = logf(all < 1.f && now > -INFINITY ? 1.f : all);
                const long long t = target[to];
                lse[to] = row < counted ? now + log_sum : 0.f;
                loss[to] = t == ignore_index ? 0.f : t >= 0 && t < V ? (now - label_logit[row]) + log_sum : NAN;
            }
        }
        __syncthreads();
    }
}

// Sum or mean of the losses, and the number of rows that count, at least 1: one CTA, in a fixed order.
__global__ void __launch_bounds__(1024) ce_total_kernel(const float* __restrict__ loss, const long long* __restrict__ target,
                                                        float* __restrict__ total, float* __restrict__ count, long long rows,
                                                        long long ignore_index, int mean) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ double sh_sum[32];
    __shared__ long long sh_count[32];
    double s = 0.0;
    long long n = 0;
    for (long long r = threadIdx.x; r < rows; r += 1024) {
        s += loss[r];
        n += target[r] != ignore_index;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        n += __shfl_xor_sync(0xffffffffu, n, o);
    }
    if ((threadIdx.x & 31) == 0) {
        sh_sum[threadIdx.x >> 5] = s;
        sh_count[threadIdx.x >> 5] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        n = 0;
        for (int w = 0; w < 32; w++) {
            s += sh_sum[w];
            n += sh_count[w];
        }
        if (n < 1) n = 1;   // no row counts: the loss is 0
        *total = (float)(mean ? s / (double)n : s);
        *count = (float)n;
    }
}

// Rows that count first, in their order, then the others from the last one down: what the products take instead of x, so that rows
// that do not count (the prompt of an answer, the words that a masked model is not asked for) cost no products, and whatever they hold
// (0 times infinity) reaches none.  A CTA has consecutive rows; it counts those before them and all of them itself, which reads the
// targets once per CTA and saves a launch.  Where every row counts x is not copied: the products take x itself.  Rows that do not
// count become zeros where the last 64-row block of a reduction reads them.  Up to 128 rows, one tile, there is nothing to spare and the
// rows stay in place, which saves the gradients' way back (ce_unpack_kernel; 64 x 1000 x 64 with gradients 91 -> 86 us on the host).
// order: row of every slot, slot: slot of every row, or -1.  For the gradients also per slot the label and (logsumexp, coefficient), and
// the factor of both: an upstream gradient that is one number, and the mean's divisor, multiply the products of the rounded dl; in the
// coefficient they would make every row's largest term, the label's, off by the same rounding.  A label outside the vocabulary makes the
// coefficient, and so the gradients, not a number.
struct CePack {
    const __nv_bfloat16* x;
    const long long* target;
    const float *lse, *grad, *count;   // gradients (lse null: the forward pass)
    __nv_bfloat16* packed;
    long long* label;
    int *order, *slot, *live;          // order or slot may be null
    float2* row;
    float* factor;
    long long ldx, ignore_index;
    int rows, V, H, grad_per_row;
    int in_place;                      // every row keeps its place, those that do not count become zeros
};
__global__ void __launch_bounds__(CE_PACK_THREADS) ce_pack_kernel(const CePack p) {
    pdl_wait();
    pdl_launch_dependents();
    constexpr int W = CE_PACK_THREADS / 32;
    __shared__ int sh_all[W], sh_before[W], sh_slot[CE_PACK_THREADS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long chunk = ((long long)p.rows + gridDim.x - 1) / gridDim.x, r0 = chunk * blockIdx.x, r1 = r0 + chunk < p.rows ? r0 + chunk : p.rows;
    int all = 0, before = 0;
#pragma unroll 8
    for (long long r = tid; r < p.rows; r += CE_PACK_THREADS) {
        const int counts = p.target[r] != p.ignore_index;
        all += counts;
        before += r < r0 ? counts : 0;
    }
    all = __reduce_add_sync(0xffffffffu, all);
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) { sh_all[warp] = all; sh_before[warp] = before; }
    __syncthreads();
    all = before = 0;
    for (int w = 0; w < W; w++) { all += sh_all[w]; before += sh_before[w]; }
    if (blockIdx.x == 0 && tid == 0) {
        *p.live = all;
        if (p.factor) *p.factor = (p.grad_per_row ? 1.f : p.grad[0]) / (p.count ? *p.count : 1.f);
    }
    const int zeros_to = ((all > 1 ? all : 1) + 63) / 64 * 64;
    for (long long base = r0; base < r1; base += CE_PACK_THREADS) {
        const long long r = base + tid;
        const long long t = r < r1 ? p.target[r] : p.ignore_index;
        const bool counts = t != p.ignore_index;
        const uint32_t votes = __ballot_sync(0xffffffffu, counts);
        __syncthreads();   // sh_all and sh_slot of the turn before have been read
        if (lane == 0) sh_all[warp] = __popc(votes);
        __syncthreads();
        int rank = before + __popc(votes & ((1u << lane) - 1));
        int taken = 0;
        for (int w = 0; w < W; w++) {
            if (w < warp) rank += sh_all[w];
            taken += sh_all[w];
        }
        before += taken;
        // a row that does not count is the (r - rank)-th of those
        const int slot = p.in_place ? (int)r : counts ? rank : p.rows - 1 - (int)(r - rank);
        sh_slot[tid] = counts ? slot : r < r1 && (p.in_place || slot < zeros_to) ? ~slot : INT_MIN;
        if (r < r1) {
            p.label[slot] = counts ? t : -1;
            if (p.order) p.order[slot] = (int)r;
            if (p.slot) p.slot[r] = counts ? slot : -1;
            if (p.row) p.row[slot] = make_float2(p.lse[r], !counts ? 0.f : t >= 0 && t < p.V ? (p.grad_per_row ? p.grad[r] : 1.f) : NAN);
        }
        __syncthreads();
        if (all == p.rows && !p.in_place) continue;
        for (int i = warp; i < CE_PACK_THREADS && base + i < r1; i += W) {
            const int to = sh_slot[i];
            if (to == INT_MIN) continue;
            const uint4* src = reinterpret_cast<const uint4*>(p.x + (base + i) * p.ldx);
            uint4* dst = reinterpret_cast<uint4*>(p.packed + (long long)(to < 0 ? ~to : to) * p.H);
#pragma unroll 4
            for (int c = lane; c < p.H / 8; c += 32) dst[c] = to < 0 ? make_uint4(0, 0, 0, 0) : src[c];
        }
    }
}
// dx from its packed rows; zeros for the rows that do not count.  One warp a row.
__global__ void __launch_bounds__(CE_THREADS) ce_unpack_kernel(const __nv_bfloat16* packed, const int* slot, __nv_bfloat16* __restrict__ dx,
                                                               long long rows, int H) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    for (long long r = (long long)blockIdx.x * (CE_THREADS / 32) + (threadIdx.x >> 5); r < rows; r += (long long)gridDim.x * (CE_THREADS / 32)) {
        const int from = slot[r];
        const uint4* src = reinterpret_cast<const uint4*>(packed + (long long)from * H);
        uint4* dst = reinterpret_cast<uint4*>(dx + r * H);
#pragma unroll 4
        for (int c = lane; c < H / 8; c += 32) dst[c] = from < 0 ? make_uint4(0, 0, 0, 0) : src[c];
    }
}
static int ce_pack(const CePack& p, int num_ctas, cudaStream_t st) {
    const long long want = ((long long)p.rows + 15) / 16, cap = (long long)num_ctas * 2;
    OB200_ELASTIC_HBM(ce_pack_kernel, 2);
    return launch_pdl(ce_pack_kernel, (unsigned)(want < cap ? want : cap), (unsigned)CE_PACK_THREADS, st, p);
}

// Columns of the vocabulary a piece of the backward pass has: dl of a piece takes at most 192 MB, or 4 KB a row where that is more (2048
// columns, so that its products are not small: from 49153 rows on), and of the four fewest numbers of pieces the one whose 256 x 256
// tiles fill the last rounds of the CTA pairs best, counted in k-blocks of 64 and eight for a tile's way out.  8192 x 32000 x 1024: three
// pieces of 10752 columns, whose gradient products are 296 tiles for 74 pairs, instead of four of 8192 (256 tiles: 3.46 rounds).  Rows of
// dl start on 128-byte lines: 6437 x 13042 x 136 with gradients 228 us without, 209 with.
static int ce_piece(long long rows, int V, int H, int sms) {
    long long most = (192LL << 20) / (2 * rows) / 256 * 256;
    if (most < 2048) most = 2048;
    const long long all = ((long long)V + 63) / 64 * 64, pairs = sms / 2 > 0 ? sms / 2 : 1, fewest = (V + most - 1) / most;
    if (fewest == 1 && rows <= 128) return (int)all;   // no pairs
    const long long tiles_t = (rows + 255) / 256, tiles_h = (H + 255) / 256;
    long long best = 0, best_cost = 0;
    for (long long n = fewest; n < fewest + 4; n++) {
        const long long v = n == 1 ? all : ((V + n - 1) / n + 255) / 256 * 256;
        long long cost = 0;
        for (long long v0 = 0; v0 < V; v0 += v) {
            const long long nv = V - v0 < v ? V - v0 : v, tiles_v = (nv + 255) / 256;
            const long long work = tiles_t * tiles_h * (nv / 64) + tiles_v * tiles_h * (rows / 64), dw_cost = rows / 64 + 8;
            const long long dx = tiles_t * tiles_h, dw = tiles_v * tiles_h, dx_cost = nv / 64 + 8;
            cost += (tiles_t * tiles_v + pairs - 1) / pairs * (H / 64 + 8) + 16;   // and two launches more
            if (2 * dx <= pairs) {   // few tiles: their reduction is split, and evens the load
                cost += work / pairs + dw_cost / 2 + 16;
                continue;
            }
            cost += gemm_longest_share(pairs, dx, dx_cost, dw, dw_cost);
        }
        if (best == 0 || cost < best_cost) { best = v; best_cost = cost; }
    }
    return (int)best;
}
constexpr int CE_ROW_BLOCK = 65536;   // rows a forward pass has in its workspace at a time
static size_t ce_round(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

struct CeBackwardSpace {
    size_t row, label, slot, packed, dl, acc, dx, slabs, total;
    int piece;
    CeBackwardSpace(long long rows, int V, int H, bool want_dx, bool want_dw) {
        piece = ce_piece(rows, V, H, ob200_plan_sm_count());
        row = ce_round((size_t)rows * sizeof(float2) + 2 * sizeof(float));   // and the factor, and how many rows count
        label = ce_round((size_t)rows * sizeof(long long));
        slot = ce_round((size_t)rows * sizeof(int));
        packed = ce_round((size_t)rows * H * 2);
        dl = ce_round((size_t)rows * piece * 2);
        acc = want_dx && piece < V ? ce_round((size_t)rows * H * sizeof(float)) : 0;
        dx = want_dx && rows > CE_IN_PLACE ? packed : 0;
        slabs = 0;
        const int last = V - (V - 1) / piece * piece;   // columns of the last piece
        for (int v : {piece < V ? piece : V, last}) {
            GemmCall gx, gw;
            gx.M = (int)rows; gx.N = gw.N = H; gx.K = v;
            gw.M = v; gw.K = (int)rows;
            const size_t a = want_dx ? gemm_bf16_slab_bytes((int)rows, H, v, GM_EPI_ACC) : 0, b = want_dw ? gemm_bf16_slab_bytes(v, H, (int)rows, GM_EPI_ACC) : 0;
            const size_t c = want_dx && want_dw ? gemm_bf16_dual_slab_bytes(gx, gw, true) : 0;
            for (size_t n : {a, b, c})
                if (n > slabs) slabs = n;
        }
        slabs = ce_round(slabs);
        total = row + label + slot + packed + dl + acc + dx + slabs;
    }
};

}  // namespace ob200

using namespace ob200;

// Parts of a row that a forward pass writes; the workspace has room for those of either kernel.
static int ce_parts(int rows, int V, int H) { return few_rows_fit(rows, V, H) ? few_rows_parts(rows, V) : (V + 127) / 128; }

// Whether a forward pass packs the rows that count: where it can spare a tile.
static bool ce_packs(int rows, int V, int H) { return rows > CE_IN_PLACE && !few_rows_fit(rows, V, H); }

struct CeForwardSpace {
    size_t part, label_logit, packed, label, order, total;
    CeForwardSpace(long long rows, int V, int H) {
        const size_t block = (size_t)(rows < CE_ROW_BLOCK ? rows : CE_ROW_BLOCK);
        const bool packs = ce_packs((int)rows, V, H);
        part = ce_round(block * ce_parts((int)rows, V, H) * sizeof(float2));
        label_logit = ce_round((block + 1) * sizeof(float));   // and how many rows count
        packed = packs ? ce_round(block * H * 2) : 0;
        label = packs ? ce_round(block * sizeof(long long)) : 0;
        order = packs ? ce_round(block * sizeof(int)) : 0;
        total = part + label_logit + packed + label + order;
    }
};
extern "C" long long ob200_linear_cross_entropy_workspace(int rows, int V, int H) {
    if (rows <= 0 || V <= 0 || H <= 0 || !gm_extents_fit(rows, V, H)) return 0;
    return (long long)CeForwardSpace(rows, V, H).total;
}

// See include/orion_kernels.h.  -1: sizes or arguments, -2: alignment, -3: workspace too small, -4: no TMA descriptor.
extern "C" int ob200_linear_cross_entropy_forward(const void* x, const void* w, const long long* target, float* loss, float* lse, float* total, float* count,
                                                  int rows, int V, int H, long long ldx, long long ldw, long long ignore_index, int mean, void* workspace,
                                                  long long workspace_bytes, int num_ctas, void* stream) {
    if (rows < 0 || V <= 0 || H <= 0 || ldx < H || ldw < H || num_ctas <= 0 || !gm_extents_fit(rows, V, H)) return -1;
    if ((rows > 0 && (!x || !w || !target || !loss || !lse)) || (total && !count)) return -1;
    if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)workspace) % 16 || (ldx | ldw) % 8) return -2;
    if (H % 8) return -2;
    if (workspace_bytes < ob200_linear_cross_entropy_workspace(rows, V, H) || (!workspace && rows > 0)) return -3;
    cudaStream_t st = (cudaStream_t)stream;
    const int block = rows < CE_ROW_BLOCK ? rows : CE_ROW_BLOCK, parts = ce_parts(rows, V, H);
    const bool packs = ce_packs(rows, V, H);
    const CeForwardSpace space(rows, V, H);
    char* at = (char*)workspace;
    float2* part = (float2*)at;
    at += space.part;
    float* label_logit = (float*)at;
    int* live = (int*)(label_logit + block);
    at += space.label_logit;
    __nv_bfloat16* packed = (__nv_bfloat16*)at;
    at += space.packed;
    long long* label = (long long*)at;
    at += space.label;
    int* order = packs ? (int*)at : nullptr;
    for (int r0 = 0; r0 < rows; r0 += CE_ROW_BLOCK) {
        const int n = rows - r0 < CE_ROW_BLOCK ? rows - r0 : CE_ROW_BLOCK;
        const __nv_bfloat16* xb = (const __nv_bfloat16*)x + (long long)r0 * ldx;
        GemmCall g;
        g.a = xb;
        g.b = w;
        g.M = n; g.N = V; g.K = H;
        g.lda = ldx; g.ldb = ldw; g.ldc = V;
        g.epi = GM_EPI_LSE;
        g.e.target = target + r0;
        g.e.part = part;
        g.e.label_logit = label_logit;
        g.num_ctas = num_ctas;
        g.stream = stream;
        int rc;
        if (packs) {
            CePack k = {};
            k.x = xb; k.ldx = ldx;
            k.target = target + r0;
            k.ignore_index = ignore_index;
            k.packed = packed; k.label = label; k.order = order; k.live = live;
            k.rows = n; k.V = V; k.H = H;
            if ((rc = ce_pack(k, num_ctas, st)) != 0) return rc;
            g.a = packed; g.lda = H;
            g.all = xb; g.ld_all = ldx;
            g.live = live;
            g.e.target = label;
        }
        rc = few_rows_fit(rows, V, H) ? few_rows_run(g) : gemm_bf16_run(g);
        if (rc) return rc;
        const int per_cta = n <= 64 ? 4 : 32, want = (n + per_cta - 1) / per_cta;
        const unsigned grid = (unsigned)(want < num_ctas ? want : num_ctas);
        if (per_cta == 4) {
            OB200_ELASTIC_HBM(ce_rows_kernel<4>, 1);
            rc = launch_pdl(ce_rows_kernel<4>, grid, 1024u, st, (const float2*)part, (const float*)label_logit, target + r0, loss + r0, lse + r0, (const int*)order,
                            (const int*)(packs ? live : nullptr), n, parts, V,
                            ignore_index);
        } else {
            OB200_ELASTIC_HBM(ce_rows_kernel<32>, 1);
            rc = launch_pdl(ce_rows_kernel<32>, grid, 1024u, st, (const float2*)part, (const float*)label_logit, target + r0, loss + r0, lse + r0, (const int*)order,
                            (const int*)(packs ? live : nullptr), n, parts, V,
                            ignore_index);
        }
        if (rc) return rc;
    }
    if (!total) return 0;
    OB200_HBM_BOUND();
    return launch_pdl(ce_total_kernel, 1u, 1024u, st, (const float*)loss, target, total, count, (long long)rows, ignore_index, mean);
}

extern "C" long long ob200_linear_cross_entropy_backward_workspace(int rows, int V, int H, int want_dx, int want_dw) {
    if (rows <= 0 || V <= 0 || H <= 0 || !gm_extents_fit(rows, V, H)) return 0;
    return (long long)CeBackwardSpace(rows, V, H, want_dx, want_dw).total;
}

extern "C" int ob200_linear_cross_entropy_backward(const void* x, const void* w, const long long* target, const float* lse, const float* grad,
                                                   int grad_per_row, const float* count, void* dx, void* dw, int rows, int V, int H, long long ldx,
                                                   long long ldw, long long ignore_index, void* workspace, long long workspace_bytes, int num_ctas,
                                                   void* stream) {
    if (rows < 0 || V <= 0 || H <= 0 || ldx < H || ldw < H || num_ctas <= 0 || !gm_extents_fit(rows, V, H)) return -1;
    if (rows == 0) return dw ? (int)cudaMemsetAsync(dw, 0, (size_t)V * H * 2, (cudaStream_t)stream) : 0;
    if (!x || !w || !target || !lse || !grad) return -1;
    if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)workspace) % 16 || (ldx | ldw) % 8 || H % 8) return -2;
    if (!dx && !dw) return 0;
    const CeBackwardSpace space(rows, V, H, dx != nullptr, dw != nullptr);
    if (workspace_bytes < (long long)space.total || !workspace) return -3;
    cudaStream_t st = (cudaStream_t)stream;
    char* at = (char*)workspace;
    float2* row = (float2*)at;
    float* factor = (float*)(row + rows);
    int* live = (int*)(factor + 1);
    at += space.row;
    long long* label = (long long*)at;
    at += space.label;
    int* slot = (int*)at;
    at += space.slot;
    __nv_bfloat16* packed = (__nv_bfloat16*)at;
    at += space.packed;
    __nv_bfloat16* dl = (__nv_bfloat16*)at;
    at += space.dl;
    float* acc = (float*)at;
    at += space.acc;
    __nv_bfloat16* packed_dx = (__nv_bfloat16*)at;
    at += space.dx;
    CePack k = {};
    k.x = (const __nv_bfloat16*)x; k.ldx = ldx;
    k.target = target;
    k.ignore_index = ignore_index;
    k.lse = lse; k.grad = grad; k.grad_per_row = grad_per_row; k.count = count;
    k.packed = packed; k.label = label; k.slot = slot; k.live = live; k.row = row; k.factor = factor;
    k.rows = rows; k.V = V; k.H = H;
    const bool packs = rows > CE_IN_PLACE;
    k.in_place = !packs;
    int rc = ce_pack(k, num_ctas, st);
    if (rc) return rc;
    for (long long v0 = 0; v0 < V; v0 += space.piece) {
        const int nv = V - v0 < space.piece ? (int)(V - v0) : space.piece;
        const bool first = v0 == 0, last = v0 + nv == V;
        const __nv_bfloat16* wp = (const __nv_bfloat16*)w + v0 * ldw;
        GemmCall g;
        g.num_ctas = num_ctas;
        g.stream = stream;
        g.a = packed; g.b = wp; g.c = dl;
        g.M = rows; g.N = nv; g.K = H;
        g.lda = H; g.ldb = ldw; g.ldc = space.piece;
        g.live = packs ? live : nullptr;
        g.all = packs ? x : nullptr;
        g.ld_all = ldx;
        g.epi = GM_EPI_DLOGITS;
        g.e.target = label;
        g.e.col0 = v0;
        g.e.row = row;
        if ((rc = gemm_bf16_run(g)) != 0) return rc;
        g.slabs = (float*)at;
        g.slab_bytes = space.slabs;
        g.a = dl; g.lda = space.piece;
        g.b_mn = 1;
        g.N = H;
        g.ldc = H;
        GemmCall gx = g, gw = g;
        // dx[t, h] += sum_v dl[t, v] w[v, h]
        gx.b = wp; gx.ldb = ldw;
        gx.M = rows; gx.K = nv;
        gx.epi = GM_EPI_ACC;
        gx.e.addend = first ? nullptr : acc;
        gx.e.factor = factor;
        gx.out_f32 = last ? 0 : 1;
        gx.all = nullptr;
        gx.c = !last ? (void*)acc : packs ? (void*)packed_dx : dx;
        // dw[v, h] = sum_t dl[t, v] x[t, h]
        gw.a_mn = 1;
        gw.live_k = packs;
        gw.b = packed; gw.ldb = H;
        gw.M = nv; gw.K = rows;
        gw.epi = GM_EPI_ACC;
        gw.e.factor = factor;
        gw.c = (__nv_bfloat16*)dw + v0 * H;
        if (dx && dw && gemm_bf16_dual_splits(gx, gw) > 0) {
            rc = gemm_bf16_run_dual(gx, gw);
        } else {
            if (dx) rc = gemm_bf16_run(gx);
            if (dw && !rc) rc = gemm_bf16_run(gw);
        }
        if (rc) return rc;
    }
    if (!dx || !packs) return 0;
    const long long want = ((long long)rows + CE_THREADS / 32 - 1) / (CE_THREADS / 32), cap = (long long)num_ctas * 8;
    OB200_ELASTIC_HBM(ce_unpack_kernel, 8);
    return launch_pdl(ce_unpack_kernel, (unsigned)(want < cap ? want : cap), (unsigned)CE_THREADS, st, (const __nv_bfloat16*)packed_dx, (const int*)slot,
                      (__nv_bfloat16*)dx, (long long)rows, H);
}
