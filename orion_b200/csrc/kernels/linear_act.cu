// The linear layer of the transformer clients with everything behind it in one launch, its backward pass, and dropout alone:
//
//   y = residual + D(act(z)),   z = x . w^T + bias,   D(a) = a / (1 - p) where the element is kept, else 0
//   dz = D(dy) * act'(z);   dbias = column sums of dz;   dx = dz . w;   dw = dz^T . x;   dresidual = dy
//
// The products are gemm_bf16.cu's with the GM_EPI_ACT epilogue; here are the elementwise kernels.  No mask is stored: it is a function
// of the element's index (philox.cuh) and drawn again in the backward pass.  The reference's clients launch these steps as the bias,
// GELU, add and dropout rows of benchmarking/model_kernels/bert_8_fb1 behind its cudaLaunchKernel trap
// (reference src/cuda_capture/intercept_temp.cpp:418-458).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "elastic.h"
#include "fast_gelu.cuh"
#include "gemm_call.h"
#include "pdl.cuh"
#include "philox.cuh"

namespace ob200 {

constexpr int LA_THREADS = 256;
constexpr int LA_COLS = 256;    // columns of a work item of the backward pass: 32 lanes x 8
constexpr int LA_ROWS = 8;      // rows that a CTA has under way at a time, one per warp

template <typename T>
struct Pack8;
template <>
struct Pack8<float> {
    __device__ static void load(const float* p, float (&v)[8]) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    __device__ static void store(float* p, const float (&v)[8]) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    __device__ static float get(float x) { return x; }
    __device__ static float put(float x) { return x; }
};
template <>
struct Pack8<__nv_bfloat16> {
    __device__ static void load(const __nv_bfloat16* p, float (&v)[8]) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __bfloat1622float2(h[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
    __device__ static void store(__nv_bfloat16* p, const float (&v)[8]) {
        uint4 q;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&q);
#pragma unroll
        for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4*>(p) = q;
    }
    __device__ static float get(__nv_bfloat16 x) { return __bfloat162float(x); }
    __device__ static __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};

__device__ __forceinline__ void load_half8(const __half* p, float (&v)[8]) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&q);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// ------------------------------------------------------------------ dropout (+ residual)
// A thread takes eight consecutive elements, one draw of the generator.  VEC: all pointers are 16-byte aligned.
template <typename T, bool VEC>
__global__ void __launch_bounds__(LA_THREADS, 6) dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ y, long long n,
                                                             const long long* __restrict__ rng, uint32_t site, uint32_t threshold, float scale) {
    pdl_wait();
    pdl_launch_dependents();
    DropKey key = {};
    if (threshold) key = drop_key_warp(rng, site);
    const uint32_t limit = drop_limit(threshold);
    const long long groups = (n + 7) / 8;
    for (long long g = (long long)blockIdx.x * blockDim.x + threadIdx.x; g < groups; g += (long long)gridDim.x * blockDim.x) {
        const long long i = g * 8;
        const int left = n - i < 8 ? (int)(n - i) : 8;
        float v[8], r[8];
        if (VEC && left == 8) {
            Pack8<T>::load(x + i, v);
            if (residual) Pack8<T>::load(residual + i, r);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < left) {
                    v[e] = Pack8<T>::get(x[i + e]);
                    if (residual) r[e] = Pack8<T>::get(residual[i + e]);
                }
        }
        uint32_t c[4] = {0, 0, 0, 0};
        if (threshold) drop_bits(key, (unsigned long long)g, c);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            v[e] = threshold == 0 || drop_keeps(c, e, limit) ? v[e] * scale : 0.f;
            if (residual) v[e] += r[e];
        }
        if (VEC && left == 8) {
            Pack8<T>::store(y + i, v);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < left) y[i + e] = Pack8<T>::put(v[e]);
        }
    }
}

// ------------------------------------------------------------------ backward of bias, activation and dropout
// dz = D(dy) * slope without dropout's factor, which the products and the column sums take instead, so that dz is rounded only where a
// slope made it inexact (where nothing is behind the product dz is dy itself), and the column sums of dz per range of rows.  A work
// item is 256 columns of one range of rows; the ranges follow from the sizes alone, so the sums do not depend on the CTA count.
// Where there is one range its sums are the bias's gradient (dbias), otherwise they go to `partial` and are added by the next kernel.
// VEC: rows of dy are 16-byte multiples (an even width); rows of slope and dz always are.
template <bool VEC>
__global__ void __launch_bounds__(LA_THREADS, 4) act_backward_kernel(const __nv_bfloat16* __restrict__ dy, const __half* __restrict__ slope,
                                                                  long long ld_slope, __nv_bfloat16* __restrict__ dz, long long ld_dz,
                                                                  float* __restrict__ partial, void* dbias, int bias_f32, float scale, long long rows,
                                                                  int N, int ranges,
                                                                  const long long* __restrict__ rng, uint32_t site, uint32_t threshold) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float sh[LA_ROWS][LA_COLS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col_tiles = (N + LA_COLS - 1) / LA_COLS;
    DropKey key = {};
    if (threshold) key = drop_key_warp(rng, site);
    const uint32_t limit = drop_limit(threshold);
    for (int item = blockIdx.x; item < col_tiles * ranges; item += gridDim.x) {
        const int ct = item % col_tiles, range = item / col_tiles;
        const int col = ct * LA_COLS + lane * 8;
        const long long r0 = rows * range / ranges, r1 = rows * (range + 1) / ranges;
        float acc[8];
#pragma unroll
        for (int e = 0; e < 8; e++) acc[e] = 0.f;
        if (col < N) {
            // two rows under way at a time
            for (long long row = r0 + warp; row < r1; row += 2 * LA_ROWS) {
                float d[2][8], z[2][8];
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const long long r = row + u * LA_ROWS < r1 ? row + u * LA_ROWS : row;
                    if (VEC) {
                        Pack8<__nv_bfloat16>::load(dy + r * N + col, d[u]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++) d[u][e] = col + e < N ? __bfloat162float(dy[r * N + col + e]) : 0.f;
                    }
                    if (slope) load_half8(slope + r * ld_slope + col, z[u]);
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const long long r = row + u * LA_ROWS;
                    if (r >= r1) break;
                    if (threshold) {
                        if (VEC) {
                            uint32_t c[4];
                            drop_bits(key, ((unsigned long long)r * N + col) >> 3, c);
#pragma unroll
                            for (int e = 0; e < 8; e++) d[u][e] = drop_keeps(c, e, limit) ? d[u][e] : 0.f;
                        } else {
                            const uint32_t mask = drop_mask<8>(key, (unsigned long long)r * N + col, threshold);
#pragma unroll
                            for (int e = 0; e < 8; e++) d[u][e] = mask >> e & 1u ? d[u][e] : 0.f;
                        }
                    }
                    if (slope) {
#pragma unroll
                        for (int e = 0; e < 8; e++) d[u][e] *= z[u][e];
                    }
                    if (dz) Pack8<__nv_bfloat16>::store(dz + r * ld_dz + col, d[u]);
#pragma unroll
                    for (int e = 0; e < 8; e++) acc[e] += d[u][e];
                }
            }
        }
        if (partial || dbias) {
#pragma unroll
            for (int e = 0; e < 8; e += 4) *reinterpret_cast<float4*>(&sh[warp][lane * 8 + e]) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
            __syncthreads();
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < LA_ROWS; w++) s += sh[w][threadIdx.x];
            const int n = ct * LA_COLS + threadIdx.x;
            if (n < N) {
                if (!dbias) partial[(long long)range * N + n] = s;
                else if (bias_f32) ((float*)dbias)[n] = s * scale;
                else ((__nv_bfloat16*)dbias)[n] = __float2bfloat16_rn(s * scale);
            }
            __syncthreads();
        }
    }
}

// out[col] = sum over the ranges, in their order: thread (g, c) of 256 takes ranges g, g + 8, ..., then the eight sums are added.
template <typename T>
__global__ void __launch_bounds__(LA_THREADS) act_colsum_kernel(const float* __restrict__ partial, int ranges, int N, float scale, T* __restrict__ out) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ float sh[8][32];
    const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
    for (int c0 = blockIdx.x * 32; c0 < N; c0 += gridDim.x * 32) {
        float s = 0.f;
        if (c0 + c < N) {
#pragma unroll 8
            for (int r = g; r < ranges; r += 8) s += partial[(long long)r * N + c0 + c];
        }
        sh[g][c] = s;
        __syncthreads();
        if (g == 0 && c0 + c < N) {
            float t = 0.f;
#pragma unroll
            for (int k = 0; k < 8; k++) t += sh[k][c];
            out[c0 + c] = Pack8<T>::put(t * scale);
        }
        __syncthreads();
    }
}

// Ranges of rows of the backward pass: one round of items for four CTAs an SM where that is possible, at least 32 rows each; one range, and
// a launch less, up to 128 rows (77 x 768 x 768 with GELU and gradients: 80 -> 77 us on the host, 25.6 -> 26.4 on the device).
static int la_ranges(long long rows, int N, int sms) {
    if (rows <= 128) return 1;
    const long long col_tiles = (N + LA_COLS - 1) / LA_COLS;
    long long n = 4LL * sms / col_tiles, most = (rows + 31) / 32;
    if (n > most) n = most;
    return (int)(n < 1 ? 1 : n);
}
static size_t la_round(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

}  // namespace ob200

using namespace ob200;

extern "C" int ob200_plan_sm_count(void);

// See include/orion_kernels.h.  -1: sizes or arguments, -2: alignment, -3: workspace too small, -4: no TMA descriptor.
extern "C" int ob200_dropout(const void* x, const void* residual, void* y, long long n, float p, const long long* rng, int site, int dtype,
                             int num_ctas, void* stream) {
    if (n < 0 || (dtype != 0 && dtype != 1) || !(p >= 0.f && p <= 1.f) || (p > 0.f && !rng) || num_ctas <= 0) return -1;
    if (n == 0) return 0;
    if (!x || !y) return -1;
    const DropRate rate = drop_rate(p);
    long long want = ((n + 7) / 8 + LA_THREADS - 1) / LA_THREADS, cap = (long long)num_ctas * 6 * grid_oversubscription();
    const unsigned grid = (unsigned)(want < cap ? want : cap);
    const bool vec = (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) % 16) == 0;
#define OB200_DROP(T, VEC)                                                                                                                     \
    do {                                                                                                                                       \
        OB200_ELASTIC_HBM((dropout_kernel<T, VEC>), 6);                                                                                        \
        return launch_pdl(dropout_kernel<T, VEC>, grid, (unsigned)LA_THREADS, (cudaStream_t)stream, (const T*)x, (const T*)residual, (T*)y, n, \
                          rng, (uint32_t)site, rate.threshold, rate.scale);                                                                    \
    } while (0)
    if (dtype == 0) {
        if (vec) OB200_DROP(float, true); else OB200_DROP(float, false);
    }
    if (vec) OB200_DROP(__nv_bfloat16, true); else OB200_DROP(__nv_bfloat16, false);
#undef OB200_DROP
}

extern "C" long long ob200_linear_act_workspace(int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || !gm_extents_fit(M, N, K) || few_rows_fit(M, N, K)) return 0;
    return (long long)gemm_bf16_slab_bytes(M, N, K, GM_EPI_ACT);
}

extern "C" int ob200_linear_act_bf16(const void* x, const void* w, void* y, void* slope, const void* bias, int bias_f32, const void* residual, int act,
                                     float p, const long long* rng, int site, int M, int N, int K, long long ldx, long long ldw, long long ld_slope,
                                     void* workspace, long long workspace_bytes, int num_ctas, void* stream) {
    if (M < 0 || N < 0 || K <= 0 || act < 0 || act > 2 || !(p >= 0.f && p <= 1.f) || (p > 0.f && !rng) || num_ctas <= 0 || ldx < K || ldw < K ||
        !gm_extents_fit(M, N, K))
        return -1;
    if (M == 0 || N == 0) return 0;
    if (!x || !w || !y || (slope && (ld_slope < N || ld_slope % 8 || !act))) return -1;
    if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)y | (uintptr_t)slope | (uintptr_t)workspace) % 16 || (K | ldx | ldw) % 8) return -2;
    if (workspace_bytes < ob200_linear_act_workspace(M, N, K) || (!workspace && workspace_bytes > 0)) return -3;
    const DropRate rate = drop_rate(p);
    GemmCall g;
    g.a = x; g.b = w; g.c = y;
    if (bias_f32) g.bias = (const float*)bias;
    else g.bias_bf16 = bias;
    g.residual = residual;
    g.M = M; g.N = N; g.K = K;
    g.lda = ldx; g.ldb = ldw; g.ldc = N;
    g.epi = GM_EPI_ACT;
    g.e.act = act;
    g.e.drop_threshold = rate.threshold;
    g.e.drop_scale = rate.scale;
    g.e.rng = rng;
    g.e.site = (uint32_t)site;
    g.e.slope = (__half*)slope;
    g.e.ld_slope = ld_slope;
    g.slabs = (float*)workspace;
    g.slab_bytes = (size_t)workspace_bytes;
    g.num_ctas = num_ctas;
    g.stream = stream;
    return few_rows_fit(M, N, K) ? few_rows_run(g) : gemm_bf16_run(g);
}

namespace {
struct LinearBackwardSpace {
    size_t dz, partial, slabs, total;
    LinearBackwardSpace(long long M, int N, int K, int act, uint32_t threshold, bool want_dx, bool want_dw, bool want_db) {
        const long long ld = (N + 7) / 8 * 8;
        dz = act || threshold || N % 8 ? la_round((size_t)M * ld * 2) : 0;
        const int ranges = la_ranges(M, N, ob200_plan_sm_count());
        partial = want_db && ranges > 1 ? la_round((size_t)ranges * N * sizeof(float)) : 0;
        const size_t a = want_dx ? gemm_bf16_slab_bytes((int)M, K, N, GM_EPI_ACC) : 0, b = want_dw ? gemm_bf16_slab_bytes(N, K, (int)M, GM_EPI_ACC) : 0;
        GemmCall gx, gw;
        gx.M = (int)M; gx.N = gw.N = K; gx.K = N;
        gw.M = N; gw.K = (int)M;
        const size_t both = want_dx && want_dw ? gemm_bf16_dual_slab_bytes(gx, gw) : 0;
        slabs = a > b ? a : b;
        slabs = la_round(both > slabs ? both : slabs);
        total = dz + partial + slabs;
    }
};
}  // namespace

extern "C" long long ob200_linear_act_backward_workspace(int M, int N, int K, int act, float p, int want_dx, int want_dw, int want_dbias) {
    if (M <= 0 || N <= 0 || K <= 0 || !gm_extents_fit(M, N, K) || !(p >= 0.f && p <= 1.f)) return 0;
    return (long long)LinearBackwardSpace(M, N, K, act, drop_rate(p).threshold, want_dx, want_dw, want_dbias).total;
}

extern "C" int ob200_linear_act_backward_bf16(const void* dy, const void* slope, const void* x, const void* w, void* dx, void* dw, void* dbias,
                                              int bias_f32, int act, float p, const long long* rng, int site, int M, int N, int K, long long ldx,
                                              long long ldw, long long ld_slope, void* workspace, long long workspace_bytes, int num_ctas, void* stream) {
    if (M < 0 || N < 0 || K <= 0 || act < 0 || act > 2 || !(p >= 0.f && p <= 1.f) || (p > 0.f && !rng) || num_ctas <= 0 || ldx < K || ldw < K ||
        !gm_extents_fit(M, N, K))
        return -1;
    if (M == 0 || N == 0) {   // sums over nothing
        cudaError_t e = cudaSuccess;
        if (dx && M > 0) e = cudaMemsetAsync(dx, 0, (size_t)M * K * 2, (cudaStream_t)stream);
        if (dw && N > 0 && e == cudaSuccess) e = cudaMemsetAsync(dw, 0, (size_t)N * K * 2, (cudaStream_t)stream);
        if (dbias && N > 0 && e == cudaSuccess) e = cudaMemsetAsync(dbias, 0, (size_t)N * (bias_f32 ? 4 : 2), (cudaStream_t)stream);
        return (int)e;
    }
    if (!dy || (act && !slope) || (slope && (ld_slope < N || ld_slope % 8 || !act)) || (dx && !w) || (dw && !x)) return -1;
    if (((uintptr_t)dy | (uintptr_t)slope | (uintptr_t)x | (uintptr_t)w | (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)workspace) % 16 ||
        (K | ldx | ldw) % 8)
        return -2;
    const DropRate rate = drop_rate(p);
    const LinearBackwardSpace space(M, N, K, act, rate.threshold, dx != nullptr, dw != nullptr, dbias != nullptr);
    if (workspace_bytes < (long long)space.total || (!workspace && space.total > 0)) return -3;
    cudaStream_t st = (cudaStream_t)stream;
    char* at = (char*)workspace;
    const long long ld_dz = (N + 7) / 8 * 8;
    __nv_bfloat16* dz = space.dz ? (__nv_bfloat16*)at : nullptr;
    at += space.dz;
    float* partial = space.partial ? (float*)at : nullptr;
    at += space.partial;
    const void* gz = dz ? (const void*)dz : dy;
    const float factor = rate.threshold ? rate.scale : 1.f;
    if ((dz && (dx || dw)) || dbias) {
        const int ranges = la_ranges(M, N, ob200_plan_sm_count());
        const long long items = (long long)ranges * ((N + LA_COLS - 1) / LA_COLS), cap = (long long)num_ctas * 4 * grid_oversubscription();
        const unsigned grid = (unsigned)(items < cap ? items : cap);
        __nv_bfloat16* out = dx || dw ? dz : nullptr;
        int rc;
        if (N % 8 == 0) {
            OB200_ELASTIC_HBM(act_backward_kernel<true>, 4);
            rc = launch_pdl(act_backward_kernel<true>, grid, (unsigned)LA_THREADS, st, (const __nv_bfloat16*)dy, (const __half*)slope, ld_slope, out, ld_dz,
                            partial, partial ? nullptr : dbias, bias_f32, factor, (long long)M, N, ranges, rng, (uint32_t)site, rate.threshold);
        } else {
            OB200_ELASTIC_HBM(act_backward_kernel<false>, 4);
            rc = launch_pdl(act_backward_kernel<false>, grid, (unsigned)LA_THREADS, st, (const __nv_bfloat16*)dy, (const __half*)slope, ld_slope, out,
                            ld_dz, partial, partial ? nullptr : dbias, bias_f32, factor, (long long)M, N, ranges, rng, (uint32_t)site, rate.threshold);
        }
        if (rc) return rc;
        if (partial) {
            const long long want = (N + 31) / 32, most = (long long)num_ctas * 8;
            const unsigned blocks = (unsigned)(want < most ? want : most);
            if (bias_f32) {
                OB200_ELASTIC_HBM(act_colsum_kernel<float>, 8);
                rc = launch_pdl(act_colsum_kernel<float>, blocks, (unsigned)LA_THREADS, st, (const float*)partial, ranges, N, factor, (float*)dbias);
            } else {
                OB200_ELASTIC_HBM(act_colsum_kernel<__nv_bfloat16>, 8);
                rc = launch_pdl(act_colsum_kernel<__nv_bfloat16>, blocks, (unsigned)LA_THREADS, st, (const float*)partial, ranges, N, factor,
                                (__nv_bfloat16*)dbias);
            }
            if (rc) return rc;
        }
    }
    GemmCall g;
    g.slabs = (float*)at;
    g.slab_bytes = space.slabs;
    g.num_ctas = num_ctas;
    g.stream = stream;
    g.a = gz;
    g.lda = dz ? ld_dz : N;
    g.b_mn = 1;
    g.ldc = K;
    g.alpha = factor;
    g.epi = GM_EPI_ACC;
    GemmCall gx = g, gw = g;
    // dx[m, k] = sum_n dz[m, n] w[n, k]: w is [reduction, columns] as it lies
    gx.b = w; gx.ldb = ldw; gx.c = dx;
    gx.M = M; gx.N = K; gx.K = N;
    // dw[n, k] = sum_m dz[m, n] x[m, k]: both operands are [reduction, ...] as they lie
    gw.a_mn = 1;
    gw.b = x; gw.ldb = ldx; gw.c = dw;
    gw.M = N; gw.N = K; gw.K = M;
    if (dx && dw && gemm_bf16_dual_splits(gx, gw) > 0) return gemm_bf16_run_dual(gx, gw);
    if (dx) {
        const int rc = gemm_bf16_run(gx);
        if (rc) return rc;
    }
    if (dw) return gemm_bf16_run(gw);
    return 0;
}
