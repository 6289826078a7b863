// Gaussian CDF for GELU without the library erff: Abramowitz & Stegun 7.1.26,
//   erf(x) = 1 - (a1 t + a2 t^2 + a3 t^3 + a4 t^4 + a5 t^5) exp(-x^2),  t = 1 / (1 + 0.3275911 x),  x >= 0,
// absolute error below 1.5e-7 (plus ~1e-6 relative from the fast exponential): two orders of magnitude inside the float32
// tolerance of the model outputs (1e-4) and far below bfloat16 resolution.  `e` = exp(-a^2 / 2) is passed in because the
// backward pass needs the same exponential for the density.
// About 18 instructions, two of them on the special-function unit (16 results per clock and SM): the arithmetic of 32 Mi elements
// takes about as long as their bfloat16 traffic.  The library's correctly rounded reciprocal took a dozen instructions more and
// bound the row kernels: bias + GELU of 8192 x 4096 50 -> 40 us, 3072 x 3072
// 16.6 -> 12.5 us.  The Newton step below gives the same bits for every float from
// 1 to 64, so the results did not change.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ob200 {

// 1 / x for x >= 1: the special-function unit's approximation and one Newton step.  For x = infinity the step would be
// infinity * 0; the approximation, zero, stands.
__device__ __forceinline__ float reciprocal_from_1(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    const float e = fmaf(-x, r, 1.0f);
    return x < 1e30f ? fmaf(r, e, r) : r;
}
__device__ __forceinline__ float gauss_exp(float a) { return __expf(-0.5f * a * a); }
__device__ __forceinline__ float gauss_cdf_with_exp(float a, float e) {
    const float ax = fabsf(a) * 0.70710678118654752f;
    const float t = reciprocal_from_1(fmaf(0.3275911f, ax, 1.0f));
    float poly = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);   // halved: 0.5 * (1 - erf(|a| / sqrt 2))
    poly = fmaf(poly, t, 0.5f * 1.421413741f);
    poly = fmaf(poly, t, 0.5f * -0.284496736f);
    poly = fmaf(poly, t, 0.5f * 0.254829592f);
    const float half_tail = poly * t * e;
    return a >= 0.f ? 1.0f - half_tail : half_tail;
}
__device__ __forceinline__ float gauss_cdf(float a) { return gauss_cdf_with_exp(a, gauss_exp(a)); }

// Two float32 operations an instruction (sm_100).
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void split_f32x2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// GELU for two values at a time, where the tensor core's epilogue and not HBM is what waits for it:
//   1 - Phi(x) = P(x) exp(-x^2 / 2) for 0 <= x <= 5.6, P of degree 11
// fitted here (linear programming) for both errors of the product: 1.1e-7 absolute and 0.15 % relative, evaluated in float32 (the formula
// above: 1.5e-7, and 0.25 % at 5.5), so that the tail of a * Phi(a), small as it is, stays within bfloat16's rounding too.  A fit of degree
// 10 for the absolute error alone was 23 % off at 5 and three times too large at 5.5; the one degree costs 0.5 us of 54 (8192 x 4096 x
// 1024, bias and GELU).  Beyond 5.6 both P and the factor x stay and the exponential goes on falling: x P(x) tends to a constant, and is
// 2.4 % off at most (of values below 6e-8).  One special-function result a value instead of two, because 16 of them a clock and SM is
// what the epilogue of a 128 x 256 tile then took (4100 of 7000 cycles at K = 512), and eleven instructions.  a * Phi(a) = max(a, 0) -
// x (1 - Phi(x)) needs no select; infinities come out as their limits.
// Returns 1 - Phi(x) and exp(-a^2 / 2); nx = -min(|a|, 5.6).
__device__ __forceinline__ uint64_t gauss_tail_pair(uint64_t a, uint64_t nx, uint64_t& e) {
    constexpr float c[12] = {0.4999999403953552f, 0.3989368975162506f, 0.24992355704307556f, 0.1325579285621643f, 0.061295535415410995f,
                             0.024564430117607117f, 0.008206812664866447f, 0.002151405205950141f, 0.000412277557188645f,
                             5.309922562446445e-05f, 4.049104518344393e-06f, 1.368912023735902e-07f};   // of powers of -x
    constexpr float kExp = -0.72134752044448170f;                               // -log2(e) / 2
    float x0, x1;
    split_f32x2(mul_f32x2(mul_f32x2(a, f32x2(kExp, kExp)), a), x0, x1);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x0) : "f"(x0));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(x1) : "f"(x1));
    e = f32x2(x0, x1);
    uint64_t poly = f32x2(c[11], c[11]);
#pragma unroll
    for (int i = 10; i >= 0; i--) poly = fma_f32x2(poly, nx, f32x2(c[i], c[i]));
    return mul_f32x2(poly, e);
}
__device__ __forceinline__ uint64_t gauss_clamp_pair(float a0, float a1) { return f32x2(fmaxf(-fabsf(a0), -5.6f), fmaxf(-fabsf(a1), -5.6f)); }
__device__ __forceinline__ void gelu_pair(float& a0, float& a1) {
    const uint64_t nx = gauss_clamp_pair(a0, a1);
    uint64_t e;
    const uint64_t tail = gauss_tail_pair(f32x2(a0, a1), nx, e);
    split_f32x2(fma_f32x2(nx, tail, f32x2(fmaxf(a0, 0.f), fmaxf(a1, 0.f))), a0, a1);
}
// The same with the slopes Phi(a) + a * density(a), from the exponential that is there.
__device__ __forceinline__ void gelu_slope_pair(float& a0, float& a1, float& s0, float& s1) {
    const uint64_t a = f32x2(a0, a1), nx = gauss_clamp_pair(a0, a1);
    constexpr float kDensity = 0.3989422804014327f;
    uint64_t e;
    const uint64_t tail = gauss_tail_pair(a, nx, e);
    float t0, t1;
    split_f32x2(tail, t0, t1);
    const uint64_t cdf = f32x2(a0 >= 0.f ? 1.0f - t0 : t0, a1 >= 0.f ? 1.0f - t1 : t1);
    split_f32x2(fma_f32x2(mul_f32x2(a, f32x2(kDensity, kDensity)), e, cdf), s0, s1);
    split_f32x2(fma_f32x2(nx, tail, f32x2(fmaxf(a0, 0.f), fmaxf(a1, 0.f))), a0, a1);
}
// max(a, 0) and its slope.  What is not a number stays one in both, as behind GELU: fmaxf would give 0, and a step that has diverged
// would look healthy behind the layer.
__device__ __forceinline__ float relu(float a) {
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(a));
    return r;
}
__device__ __forceinline__ float relu_slope(float a) { return a > 0.f ? 1.f : a <= 0.f ? 0.f : a; }
// One value: act(a) and its slope; 0 none, 1 ReLU, 2 GELU.
__device__ __forceinline__ float act_slope(float a, int act, float& slope) {
    if (act == 2) {
        float b = 0.f, unused;
        gelu_slope_pair(a, b, slope, unused);
        return a;
    }
    slope = act == 1 ? relu_slope(a) : 1.f;
    return act == 1 ? relu(a) : a;
}

}  // namespace ob200
