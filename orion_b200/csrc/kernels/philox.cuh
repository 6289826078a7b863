// Counter-based random bits for dropout: Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
// 1, 2, 3", SC'11), so that a mask is a function of (seed, step, site, element) and is drawn again where it is needed instead of
// being stored.
//
// Element i of a tensor (index into its contiguous layout) takes 16 of the 128 bits at counter
//   (low word of i / 8, bits 32..47 of i / 8 | bits 32..47 of step << 16, low word of step, site)      under the key seed,
// half i % 8 of the four words, low halves first.  It is kept where those 16 bits are at least the threshold round(65536 p): the
// probability moves in steps of 2^-16, and the factor 65536 / (65536 - threshold) makes the mean exact for the one that is used.
// Sixteen bits an element and not 32, because the ten rounds (20 wide multiplications) are what dropout computes: eight elements a
// call instead of four keep the arithmetic of the elementwise kernel below its HBM time.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ob200 {

struct DropKey {
    uint32_t k0, k1;         // seed
    uint32_t step, step_hi;  // low word; bits 32..47 in the upper half
    uint32_t site;
};

__device__ __forceinline__ DropKey drop_key(const long long* rng, uint32_t site) {
    const unsigned long long seed = (unsigned long long)rng[0], step = (unsigned long long)rng[1];
    return {(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)step, (uint32_t)(step >> 32) << 16, site};
}
// The same for a converged warp: taken by shuffle the key is known to be the same in all lanes, and its rounds cost a warp's
// arithmetic nothing.
__device__ __forceinline__ DropKey drop_key_warp(const long long* rng, uint32_t site) {
    DropKey k = drop_key(rng, site);
    k.k0 = __shfl_sync(0xffffffffu, k.k0, 0);
    k.k1 = __shfl_sync(0xffffffffu, k.k1, 0);
    k.step = __shfl_sync(0xffffffffu, k.step, 0);
    k.step_hi = __shfl_sync(0xffffffffu, k.step_hi, 0);
    return k;
}

// The 128 bits of elements 8 * group .. 8 * group + 7.
__device__ __forceinline__ void drop_bits(const DropKey& key, unsigned long long group, uint32_t (&c)[4]) {
    c[0] = (uint32_t)group;
    c[1] = ((uint32_t)(group >> 32) & 0xFFFFu) | key.step_hi;
    c[2] = key.step;
    c[3] = key.site;
    uint32_t k0 = key.k0, k1 = key.k1;
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const unsigned long long a = (unsigned long long)c[0] * 0xD2511F53u, b = (unsigned long long)c[2] * 0xCD9E8D57u;
        c[0] = (uint32_t)(b >> 32) ^ c[1] ^ k0;
        c[1] = (uint32_t)b;
        c[2] = (uint32_t)(a >> 32) ^ c[3] ^ k1;
        c[3] = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

// Half e of a group is kept.  The halves are compared in the upper half of a word with limit = 65536 * threshold - 1 (threshold > 0; for
// 65536, where nothing is kept, that is the largest word), so that the high one needs no shift.
__device__ __forceinline__ uint32_t drop_limit(uint32_t threshold) { return (threshold << 16) - 1u; }
__device__ __forceinline__ bool drop_keeps(const uint32_t (&c)[4], int e, uint32_t limit) { return ((e & 1) ? c[e >> 1] : c[e >> 1] << 16) > limit; }
// The same as a mask, bit e for half e.
__device__ __forceinline__ uint32_t drop_group_mask(const DropKey& key, unsigned long long group, uint32_t threshold) {
    uint32_t c[4], mask = 0;
    drop_bits(key, group, c);
    const uint32_t limit = drop_limit(threshold);
#pragma unroll
    for (int e = 0; e < 8; e++) mask |= drop_keeps(c, e, limit) ? 1u << e : 0u;
    return mask;
}

// The mask of COUNT (8 to 32, a multiple of 8) consecutive elements from `index` on: bit j for element index + j.  An index that
// is no multiple of 8 (rows of an odd width) costs one group more.
template <int COUNT>
__device__ __forceinline__ uint32_t drop_mask(const DropKey& key, unsigned long long index, uint32_t threshold) {
    const unsigned long long g = index >> 3;
    const int off = (int)(index & 7);
    unsigned long long bits = 0;
#pragma unroll
    for (int i = 0; i < COUNT / 8; i++) bits |= (unsigned long long)drop_group_mask(key, g + i, threshold) << (8 * i);
    if (off) bits |= (unsigned long long)drop_group_mask(key, g + COUNT / 8, threshold) << COUNT;
    return (uint32_t)(bits >> off);
}

// f[j] = kept ? f[j] * scale : 0 for the W elements from group `group` on: draws side by side, which share the keys.
template <int W>
__device__ __forceinline__ void drop_apply(const DropKey& key, unsigned long long group, uint32_t threshold, float scale, float (&f)[W]) {
    uint32_t c[W / 8][4];
#pragma unroll
    for (int i = 0; i < W / 8; i++) drop_bits(key, group + i, c[i]);
    const uint32_t limit = drop_limit(threshold);
#pragma unroll
    for (int j = 0; j < W; j++) f[j] = drop_keeps(c[j >> 3], j & 7, limit) ? f[j] * scale : 0.f;
}

// A probability as the kernels use it.
struct DropRate { uint32_t threshold; float scale; };
inline DropRate drop_rate(float p) {
    const double t = (double)p * 65536.0 + 0.5;
    DropRate r;
    r.threshold = t >= 65536.0 ? 65536u : (uint32_t)t;
    r.scale = r.threshold < 65536u ? (float)(65536.0 / (65536.0 - r.threshold)) : 0.f;
    return r;
}

}  // namespace ob200
