// Epilogues of the bfloat16 GEMM (included by gemm_bf16.cu, inside its namespace): what a warp does with its 32 rows of a finished
// tile in tensor memory, thread = row, 32 columns at a time.  Arithmetic is float32; an output is rounded to bfloat16 once, staged in
// a swizzled slab of 32 rows x 64 bytes and written by a TMA store.  A warp's turns alternate between two slabs.

__device__ __forceinline__ uint32_t gm_pack(float a, float b) {
    const __nv_bfloat162 h2 = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h2);
}

// Slopes are kept in float16: they lie between -0.13 and 1.13, and three more bits than bfloat16's keep what multiplies the gradient an
// eighth as far off as the rounding of the product.  Below 2^-14 (behind GELU, arguments below -4.5) they have an absolute error of
// 2^-25; keeping the argument in bfloat16 instead would move them by up to 7 % there.
__device__ __forceinline__ uint32_t gm_pack_half(float a, float b) {
    const __half2 h2 = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h2);
}

// Byte of 16-byte chunk `ch` of this thread's row in a slab of 32 rows x W columns, in the swizzle of its tensor map (64 or 32 bytes
// wide: eight consecutive rows of one chunk fall into eight different bank groups).
template <int W>
__device__ __forceinline__ int gm_slab_chunk(int lane, int ch) {
    return W == 32 ? lane * 64 + ((ch ^ ((lane >> 1) & 3)) << 4) : lane * 32 + ((ch ^ ((lane >> 2) & 1)) << 4);
}
// W bfloat16 values of this thread's row into a slab.
template <int W>
__device__ __forceinline__ void gm_stage(uint8_t* slab, int lane, const float (&f)[W]) {
#pragma unroll
    for (int ch = 0; ch < W / 8; ch++)
        *reinterpret_cast<uint4*>(slab + gm_slab_chunk<W>(lane, ch)) =
            make_uint4(gm_pack(f[ch * 8], f[ch * 8 + 1]), gm_pack(f[ch * 8 + 2], f[ch * 8 + 3]), gm_pack(f[ch * 8 + 4], f[ch * 8 + 5]),
                       gm_pack(f[ch * 8 + 6], f[ch * 8 + 7]));
}

// f += eight bfloat16 values (the upper halves of float32 ones).
__device__ __forceinline__ void gm_add8(float* f, uint4 v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; e++)
        split_f32x2(add_f32x2(f32x2(f[e * 2], f[e * 2 + 1]), f32x2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xFFFF0000u))), f[e * 2],
                    f[e * 2 + 1]);
}

// (Never issued ahead of its wait: the compiler takes the registers for filled and may move them.)
__device__ __forceinline__ void gm_load(uint32_t t_addr, float (&f)[32]) {
    uint32_t v[32];
    tmem_ld_32x32(t_addr, v);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 32; j++) f[j] = __uint_as_float(v[j]);
}
__device__ __forceinline__ void gm_load(uint32_t t_addr, float (&f)[16]) {
    uint32_t v[16];
    tmem_ld_32x16(t_addr, v);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; j++) f[j] = __uint_as_float(v[j]);
}

// The activation of W values, and its slopes into a slab.
template <int W>
__device__ __forceinline__ void gm_act_slope(float (&f)[W], int act, uint8_t* slab, int lane) {
#pragma unroll
    for (int ch = 0; ch < W / 8; ch++) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float &a0 = f[ch * 8 + e * 2], &a1 = f[ch * 8 + e * 2 + 1];
            float s0, s1;
            if (act == 2) {
                gelu_slope_pair(a0, a1, s0, s1);
            } else {
                s0 = relu_slope(a0);
                s1 = relu_slope(a1);
                a0 = relu(a0);
                a1 = relu(a1);
            }
            w[e] = gm_pack_half(s0, s1);
        }
        *reinterpret_cast<uint4*>(slab + gm_slab_chunk<W>(lane, ch)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Partial matrices of a product with split-K, as they are: the rest is a second kernel's.
template <int COLS>
__device__ __forceinline__ void gm_epilogue_slab(const GemmParams& p, uint32_t t_row, int m, int n0, int sp, int rows) {
#pragma unroll 1
    for (int c0 = 0; c0 < COLS; c0 += 32) {
        const int n = n0 + c0;
        if (n >= p.N) break;            // warp-uniform
        uint32_t v[32];
        tmem_ld_32x32(t_row + c0, v);
        tmem_ld_wait();
        if (m >= rows) continue;
        float* srow = p.slabs + ((long long)sp * rows + m) * p.N + n;
        if (n + 32 <= p.N && (p.N & 3) == 0) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) *reinterpret_cast<uint4*>(srow + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (n + j < p.N) srow[j] = __uint_as_float(v[j]);
        }
    }
}

// C = residual + dropout(act(A.B^T + bias)): N a multiple of 8, all pointers 16-byte aligned, the bias bfloat16.
//
// What bounds it is latency (a warp's turn is a chain: tensor memory, arithmetic, slab, fence, store), so a turn has little in it beside
// the arithmetic: no path for ragged widths, and the residual
// brought into the slab that the output will leave from by a TMA load one turn ahead (read by the threads, each a row, it took 25 us of
// 8192 x 4096; so 13).  The residual of the first turn is asked for before the accumulator is waited for (gm_residual_ahead).
// With the slope a turn has 16 columns instead of 32, so that a warp's 4 KB still are two turns of slabs and the registers suffice.
template <bool SLOPE>
constexpr int kActCols = SLOPE ? 16 : 32;
template <bool SLOPE>
__device__ __forceinline__ bool gm_residual_ahead(const GemmParams& p, int m0w, int n0, uint8_t* stage, uint32_t turn, uint64_t* bars) {
    if (!p.residual || p.splits > 1 || n0 >= p.N) return false;
    if (elect_one()) {
        bulk_wait_group_read<1>();
        mbar_arrive_expect_tx(&bars[turn & 1], kActCols<SLOPE> * 64);
        tma_load_tile_2d(smem_u32(stage + (turn & 1) * 2048), p.tmap_res, &bars[turn & 1], n0, m0w);
    }
    __syncwarp();
    return true;
}
template <int COLS, bool SLOPE>
__device__ __forceinline__ bool gm_epilogue_act(const GemmParams& p, uint32_t t_row, int m, int m0w, int n0, int lane, uint8_t* stage, uint32_t& turn,
                                                uint64_t* bars, volatile int* abort_flag) {
    constexpr int W = kActCols<SLOPE>;
    if (n0 >= p.N) return true;
    const bool has_res = p.residual != nullptr;
    const int cols = p.N - n0 < COLS ? p.N - n0 : COLS, act = p.e.act;
    const uint32_t threshold = p.e.drop_threshold;
    DropKey key = {};
    if (threshold) key = drop_key_warp(p.e.rng, p.e.site);
    unsigned long long group = ((unsigned long long)m * p.N + n0) >> 3;
    const __nv_bfloat16* bias = p.bias_bf16 ? p.bias_bf16 + n0 : nullptr;
#pragma unroll 1
    for (int c0 = 0; c0 < cols; c0 += W, turn++) {
        uint4 b[W / 8];
        if (bias) {
#pragma unroll
            for (int ch = 0; ch < W / 8; ch++)
                if (c0 + ch * 8 < cols) b[ch] = __ldg(reinterpret_cast<const uint4*>(bias + c0 + ch * 8));
        }
        float f[W];
        gm_load(t_row + c0, f);
        if (bias) {
#pragma unroll
            for (int ch = 0; ch < W / 8; ch++) gm_add8(f + ch * 8, b[ch]);
        }
        uint8_t* slab = stage + (turn & 1) * 2048;
        if (SLOPE) {
            if (!has_res) {
                if (elect_one()) bulk_wait_group_read<1>();   // the stores of two turns ago have read their slabs
                __syncwarp();
            }
            gm_act_slope<W>(f, act, slab + 1024, lane);
        } else if (act == 2) {
#pragma unroll
            for (int j = 0; j < W; j += 2) gelu_pair(f[j], f[j + 1]);
        } else if (act == 1) {
#pragma unroll
            for (int j = 0; j < W; j++) f[j] = relu(f[j]);
        }
        if (threshold) {
            drop_apply<W>(key, group, threshold, p.e.drop_scale, f);
            group += W / 8;
        }
        if (has_res) {
            if (!mbar_wait_warp(&bars[turn & 1], (turn >> 1) & 1, abort_flag)) return false;
#pragma unroll
            for (int ch = 0; ch < W / 8; ch++) gm_add8(f + ch * 8, *reinterpret_cast<const uint4*>(slab + gm_slab_chunk<W>(lane, ch)));
        } else if (!SLOPE) {
            if (elect_one()) bulk_wait_group_read<1>();
            __syncwarp();
        }
        gm_stage<W>(slab, lane, f);
        fence_proxy_async_smem();
        __syncwarp();
        if (elect_one()) {
            if (m0w < p.M) {
                tma_store_tile_2d(p.tmap_c, smem_u32(slab), n0 + c0, m0w);
                if (SLOPE) tma_store_tile_2d(p.tmap_slope, smem_u32(slab + 1024), n0 + c0, m0w);
            }
            bulk_commit_group();
        }
        __syncwarp();
        if (c0 + W < cols) gm_residual_ahead<SLOPE>(p, m0w, n0 + c0 + W, stage, turn + 1, bars);
    }
    return true;
}

// The same for any width, alignment and type of the bias, which costs: 8192 x 4095 x 1024 takes 86 us with a bias (8192 x 4096 x 1024: 52),
// 100 with GELU (58), 181 with a residual (58), 216 with GELU, dropout and residual (79).  A thread reads its row's residual element by
// element, 32 rows apart, and a turn waits for the stores of the one before.
template <int COLS>
__device__ __forceinline__ void gm_epilogue_act_any(const GemmParams& p, uint32_t t_row, int m, int m0w, int n0, int lane, uint8_t* stage) {
    const bool row_ok = m < p.M;
    DropKey key = {};
    if (p.e.drop_threshold) key = drop_key_warp(p.e.rng, p.e.site);
#pragma unroll 1
    for (int c0 = 0; c0 < COLS; c0 += 32) {
        const int n = n0 + c0;
        if (n >= p.N) break;            // warp-uniform
        float f[32];
        gm_load(t_row + c0, f);
        const long long index = (long long)m * p.N + n;
        if (p.bias || p.bias_bf16) {
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (n + j < p.N) f[j] += p.bias ? __ldg(p.bias + n + j) : __bfloat162float(p.bias_bf16[n + j]);
        }
        if (elect_one()) bulk_wait_group_read<0>();   // the slopes of the turn before have left
        __syncwarp();
        if (p.e.slope) {
            gm_act_slope<32>(f, p.e.act, stage + 2048, lane);
        } else if (p.e.act == 2) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) gelu_pair(f[j], f[j + 1]);
        } else if (p.e.act == 1) {
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] = relu(f[j]);
        }
        if (p.e.drop_threshold) {
            const uint32_t mask = drop_mask<32>(key, (unsigned long long)index, p.e.drop_threshold);
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] = mask >> j & 1u ? f[j] * p.e.drop_scale : 0.f;
        }
        if (p.residual && row_ok) {
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (n + j < p.N) f[j] += __bfloat162float(p.residual[index + j]);
        }
        gm_stage<32>(stage, lane, f);
        fence_proxy_async_smem();
        __syncwarp();
        if (elect_one()) {
            if (m0w < p.M && p.e.slope) tma_store_tile_2d(p.tmap_slope, smem_u32(stage + 2048), n, m0w);
            bulk_commit_group();
        }
        // lane = column, one row after the other, so that a store covers 64 consecutive bytes
        __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.c) + (long long)m0w * p.ldc + n + lane;
        const int rows = p.M - m0w < 32 ? p.M - m0w : 32;
#pragma unroll 4
        for (int r = 0; r < rows; r++)
            if (n + lane < p.N)
                out[r * p.ldc] = *reinterpret_cast<const __nv_bfloat16*>(stage + gm_slab_chunk<32>(r, lane >> 3) + (lane & 7) * 2);
        __syncwarp();
    }
}

// 2^(ref - x log2(e)) for ref = x log2(e) as float32 rounds it; the multiply-add takes the difference exactly.
__device__ __forceinline__ float gm_ref_error(float x, float ref) { return exp2f(-fmaf(x, 1.4426950408889634f, -ref)); }

// Of every row and 128 columns the maximum and the sum of exponentials relative to it, and the logit of the row's label.
//
// Exponents are one multiply-add against a reference rounded to float32, 2^(x log2(e) - ref), and so off by what the rounding took from it,
// up to 2^-24 of the maximum's exponent.  That is one factor for all columns: gm_ref_error, once a row, takes it out of the sum.
template <int COLS>
__device__ __forceinline__ void gm_epilogue_lse(const GemmParams& p, uint32_t t_row, int m, int n0) {
    constexpr float kLog2e = 1.4426950408889634f;
    const bool row_ok = m < p.M;
    const long long at = row_ok ? p.e.target[m] - p.e.col0 - n0 : -1;
    const int label = at >= 0 && at < COLS ? (int)at : -1;   // the label's column of this warp's
    float top = -INFINITY, sum = 0.f, ref = 0.f;
#pragma unroll 1
    for (int c0 = 0; c0 < COLS; c0 += 32) {
        const int n = n0 + c0;
        if (n >= p.N) break;            // warp-uniform
        float f[32];
        gm_load(t_row + c0, f);
        if (n + 32 > p.N) {
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (n + j >= p.N) f[j] = -INFINITY;
        }
        if (__any_sync(0xffffffffu, label >= c0 && label < c0 + 32)) {
#pragma unroll
            for (int j = 0; j < 32; j++)
                if (label == c0 + j) p.e.label_logit[m] = f[j];
        }
        float mx[4] = {f[0], f[1], f[2], f[3]};
#pragma unroll
        for (int j = 4; j < 32; j++) mx[j & 3] = fmaxf(mx[j & 3], f[j]);
        const float now = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), top);
        const float was = ref;
        ref = now == -INFINITY ? 0.f : __fmul_rn(now, kLog2e);   // columns of minus infinity alone weigh nothing
        // nothing above minus infinity so far: a sum of 0, or not a number
        uint64_t part[2] = {f32x2(top == -INFINITY ? sum : sum * exp2f(was - ref), 0.f), f32x2(0.f, 0.f)};
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            float e0, e1;
            split_f32x2(fma_f32x2(f32x2(f[j], f[j + 1]), f32x2(kLog2e, kLog2e), f32x2(-ref, -ref)), e0, e1);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(e0));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(e1));
            part[j >> 1 & 1] = add_f32x2(part[j >> 1 & 1], f32x2(e0, e1));
        }
        float s0, s1, s2, s3;
        split_f32x2(part[0], s0, s1);
        split_f32x2(part[1], s2, s3);
        sum = (s0 + s1) + (s2 + s3);
        top = now;
        if (((c0 + 32) & 127) == 0 || n + 32 >= p.N) {
            if (row_ok) p.e.part[(long long)(n >> 7) * p.M + m] = make_float2(top, top == -INFINITY ? sum : sum * gm_ref_error(top, ref));
            top = -INFINITY;
            sum = 0.f;
        }
    }
}

// C = (softmax - onehot(label)) * coefficient, the probabilities from this product's logits and the row's logsumexp (see gm_ref_error).
template <int COLS>
__device__ __forceinline__ void gm_epilogue_dlogits(const GemmParams& p, uint32_t t_row, int m, int m0w, int n0, int lane, uint8_t* stage,
                                                    uint32_t& turn) {
    constexpr float kLog2e = 1.4426950408889634f;
    const bool row_ok = m < p.M;
    const float2 row = row_ok ? p.e.row[m] : make_float2(0.f, 0.f);
    const float ref = __fmul_rn(row.x, kLog2e), scale = row.y * gm_ref_error(row.x, ref);
    const long long at = row_ok ? p.e.target[m] - p.e.col0 - n0 : -1;
    const int label = at >= 0 && at < COLS ? (int)at : -1;
#pragma unroll 1
    for (int c0 = 0; c0 < COLS; c0 += 32) {
        const int n = n0 + c0;
        if (n >= p.N) break;            // warp-uniform
        float f[32];
        gm_load(t_row + c0, f);
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            float e0, e1;
            split_f32x2(fma_f32x2(f32x2(f[j], f[j + 1]), f32x2(kLog2e, kLog2e), f32x2(-ref, -ref)), e0, e1);
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(e0));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(e1));
            split_f32x2(mul_f32x2(f32x2(e0, e1), f32x2(scale, scale)), f[j], f[j + 1]);
        }
        if (__any_sync(0xffffffffu, label >= c0 && label < c0 + 32)) {
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] -= label == c0 + j ? row.y : 0.f;
        }
        if (__any_sync(0xffffffffu, row.y == 0.f)) {
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] = row.y == 0.f ? 0.f : f[j];
        }
        uint8_t* slab = stage + (turn++ & 1) * 2048;
        if (elect_one()) bulk_wait_group_read<1>();
        __syncwarp();
        gm_stage<32>(slab, lane, f);
        __syncwarp();
        fence_proxy_async_smem();
        __syncwarp();
        if (elect_one()) {
            if (m0w < p.M) tma_store_tile_2d(p.tmap_c, smem_u32(slab), n, m0w);
            bulk_commit_group();
        }
        __syncwarp();
    }
}

// A dual launch's tiles: float32 accumulators times the factor, plus the first product's addend (which may be its output), rounded to the output's type.
template <int BN>
__device__ __forceinline__ void gm_epilogue_dual(const GemmParamsDual& p, bool second, uint32_t t_row, int m, int m0w, int n0, int lane, uint8_t* stage,
                                                 uint32_t& turn) {
    const int M = second ? p.second.M : p.M, N = second ? p.second.N : p.N;
    const bool out_f32 = second ? p.second.out_f32 : p.out_f32;
    const unsigned char* map = second ? p.second.tmap_c : p.tmap_c;
    const float* addend = second || m >= M || !p.e.addend ? nullptr : p.e.addend + (long long)m * N;
    const float factor = p.e.factor ? p.alpha * __ldg(p.e.factor) : p.alpha;
#pragma unroll 1
    for (int c0 = 0; c0 < BN; c0 += 32) {
        const int n = n0 + c0;
        if (n >= N) break;              // warp-uniform
        float f[32];
        gm_load(t_row + c0, f);
#pragma unroll
        for (int j = 0; j < 32; j++) f[j] *= factor;
        if (addend) {                   // N is a multiple of 8
#pragma unroll
            for (int j = 0; j < 32; j += 4)
                if (n + j < N) {
                    const float4 a = *reinterpret_cast<const float4*>(addend + n + j);
                    f[j] += a.x; f[j + 1] += a.y; f[j + 2] += a.z; f[j + 3] += a.w;
                }
        }
        // 64 bfloat16 or 32 float32 columns a slab of 128-byte rows
        const int half = out_f32 ? 0 : (c0 >> 5) & 1;
        uint8_t* slab = stage + (turn & 1) * 4096;
        if (half == 0) {
            if (elect_one()) bulk_wait_group_read<1>();
            __syncwarp();
        }
        uint8_t* row = slab + lane * 128;
        if (out_f32) {
#pragma unroll
            for (int ch = 0; ch < 8; ch++)
                *reinterpret_cast<float4*>(row + ((ch ^ (lane & 7)) << 4)) = make_float4(f[ch * 4], f[ch * 4 + 1], f[ch * 4 + 2], f[ch * 4 + 3]);
        } else {
#pragma unroll
            for (int ch = 0; ch < 4; ch++)
                *reinterpret_cast<uint4*>(row + (((half * 4 + ch) ^ (lane & 7)) << 4)) =
                    make_uint4(gm_pack(f[ch * 8], f[ch * 8 + 1]), gm_pack(f[ch * 8 + 2], f[ch * 8 + 3]), gm_pack(f[ch * 8 + 4], f[ch * 8 + 5]),
                               gm_pack(f[ch * 8 + 6], f[ch * 8 + 7]));
        }
        if (out_f32 || half == 1 || c0 + 32 >= BN || n + 32 >= N) {
            fence_proxy_async_smem();
            __syncwarp();
            if (elect_one()) {
                if (m0w < M) tma_store_tile_2d(map, smem_u32(slab), n - half * 32, m0w);
                bulk_commit_group();
            }
            __syncwarp();
            turn++;
        }
    }
}
