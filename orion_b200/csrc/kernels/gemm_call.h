// The bfloat16 GEMM (gemm_bf16.cu) as the other kernels of the library call it: one problem with one of several epilogues.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ob200 {

// Largest row count, width and reduction of the fused operators: positions are ints, and loops over blocks (65536 rows at most) and tiles
// step past the last one before they stop.
constexpr int GM_MOST_EXTENT = 0x7fffffff - 65535;
inline bool gm_extents_fit(int M, int N, int K) { return M <= GM_MOST_EXTENT && N <= GM_MOST_EXTENT && K <= GM_MOST_EXTENT; }

enum : int {
    GM_EPI_PLAIN = 0,    // C = alpha * A.B^T (+ bias) (+ bfloat16 residual)
    GM_EPI_ACC = 1,      // the same with a factor from device memory and a float32 addend (which may be C itself)
    GM_EPI_ACT = 2,      // C = residual + dropout(act(A.B^T + bias)), optionally the activation's slope beside it
    GM_EPI_ACT_ANY = 3,  // GM_EPI_ACT for widths, types and alignments that its vector accesses do not take (chosen by the launcher)
    GM_EPI_ACT_SLOPE = 7,// GM_EPI_ACT with the slope (chosen by the launcher)
    GM_EPI_LSE = 4,      // no C: per row and 128 columns the maximum and the sum of exponentials, and the label's column
    GM_EPI_DLOGITS = 5,  // C = (exp(A.B^T - lse) - onehot(label)) * coefficient
    GM_EPI_DUAL = 6,     // two products of one launch, each plain (the first one with GM_EPI_ACC's addend)
};

struct GemmEpi {
    // GM_EPI_ACC, GM_EPI_DUAL
    const float* addend;            // [M, N], rows N apart, or null
    const float* factor;            // optional: what the products are multiplied by, in device memory
    // GM_EPI_ACT
    int act;                        // 0 none, 1 ReLU, 2 GELU
    uint32_t drop_threshold;        // 0: no dropout
    float drop_scale;
    const long long* rng;           // (seed, step), in device memory
    uint32_t site;
    __half* slope;                  // optional, with an activation: act'(A.B^T + bias), rows ld_slope apart (a multiple of 8)
    long long ld_slope;
    // GM_EPI_LSE, GM_EPI_DLOGITS
    const long long* target;        // label of every row
    long long col0;                 // column of the vocabulary that column 0 of this product is
    float2* part;                   // GM_EPI_LSE: [ceil(N / 128)][M] (maximum, sum of exp(x - maximum)) of 128 columns
    float* label_logit;             // GM_EPI_LSE: [M], written where the label is one of the columns
    const float2* row;              // GM_EPI_DLOGITS: [M] (logsumexp, coefficient); a coefficient of zero gives zeros whatever else the row holds
};

struct GemmCall {
    const void* a = nullptr;
    const void* b = nullptr;
    void* c = nullptr;
    const float* bias = nullptr;
    const void* bias_bf16 = nullptr;
    const void* residual = nullptr;
    int M = 0, N = 0, K = 0, a_mn = 0, b_mn = 0;
    long long lda = 0, ldb = 0, ldc = 0;
    int batch_inner = 1, batch_outer = 1;
    long long a_si = 0, a_so = 0, b_si = 0, b_so = 0, c_si = 0, c_so = 0;
    float alpha = 1.0f;
    int out_f32 = 0, tri = 0;
    int epi = GM_EPI_PLAIN;
    GemmEpi e = {};
    bool stream_slabs = false;      // split-K partial matrices in the stream's own scratch; otherwise in `slabs` (none: no split)
    float* slabs = nullptr;
    size_t slab_bytes = 0;
    // Packed rows (GM_EPI_ACC, GM_EPI_LSE, GM_EPI_DLOGITS and both products of a dual launch): only the first *live rows of A count, or with
    // live_k the first *live indices of the reduction.  Tiles and k-blocks behind them are left out (their outputs unwritten); *live may be
    // 0.  `all`: what stands for the packed operand (A of the losses, B of a product with live_k) where *live is everything, M or K.
    const int* live = nullptr;
    int live_k = 0;
    const void* all = nullptr;
    long long ld_all = 0;
    int num_ctas = 0;
    void* stream = nullptr;
};

// 0, a cudaError_t, -1 (sizes), -2 (alignment), -4 (no TMA descriptor).
int gemm_bf16_run(const GemmCall& call);
// Work of the CTA pair that has most of it: a pair takes every pairs-th unit, `a` of cost ca first, then `b` of cost cb.  What a pair gets
// changes with its number at two places only.
inline long long gemm_longest_share(long long pairs, long long a, long long ca, long long b, long long cb) {
    long long longest = 0;
    for (const long long p : {0LL, a % pairs, (a + b) % pairs}) {
        const long long na = a > p ? (a - p - 1) / pairs + 1 : 0, n = a + b > p ? (a + b - p - 1) / pairs + 1 : 0, cost = na * ca + (n - na) * cb;
        if (cost > longest) longest = cost;
    }
    return longest;
}

// Two products in one launch of CTA pairs, 256 x 256 tiles (of single CTAs, 128 x 256, where the first one has at most 128 rows), so that
// the last round of tiles is one and not two: no batch, bias or residual, one alpha, epilogue GM_EPI_ACC (the addend is the first one's),
// rows of C 16-byte multiples.  `splits`: into how many parts the first one's reduction is cut for that, 0 where the products are too
// narrow.  `packed`: with `live`, whose rows may be cut into more parts.
int gemm_bf16_dual_splits(const GemmCall& first, const GemmCall& second);
size_t gemm_bf16_dual_slab_bytes(const GemmCall& first, const GemmCall& second, bool packed = false);
int gemm_bf16_run_dual(const GemmCall& first, const GemmCall& second);
// Bytes of partial matrices that the split of a product with this epilogue wants; 0 where it is not split.
size_t gemm_bf16_slab_bytes(int M, int N, int K, int epi);

// The same for few rows (few_rows.cu; up to 32, more where all tiles are resident at once): GM_EPI_ACT, and GM_EPI_LSE with
// `few_rows_parts` parts a row instead of N / 128.
bool few_rows_fit(int M, int N, int K);
int few_rows_parts(int M, int V);
int few_rows_run(const GemmCall& call);

}  // namespace ob200
