// Epilogues of the bfloat16 GEMM (included by gemm_bf16.cu, inside its namespace): what a warp does with its 32 rows of a finished
// tile in tensor memory, thread = row, 32 columns at a time.  Arithmetic is float32; an output is rounded to bfloat16 once, staged in
// a swizzled slab of 32 rows x 64 bytes and written by a TMA store.  A warp has 8 KB of shared memory: two turns of two slabs (the
// output, and the pre-activation beside it), so that a slab is filled while the stores of the turn before read theirs.

__device__ __forceinline__ uint32_t gm_pack(float a, float b) {
    const __nv_bfloat162 h2 = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h2);
}
__device__ __forceinline__ float gm_activate(float a, int act) { return act == 2 ? a * gauss_cdf(a) : act == 1 ? fmaxf(a, 0.f) : a; }

// 32 bfloat16 values of this thread's row into a slab of 64-byte rows, 64-byte swizzle (16-byte chunk index XOR (row / 2) % 4: eight
// consecutive rows of one chunk fall into eight different bank groups).
__device__ __forceinline__ void gm_stage32(uint8_t* slab, int lane, const float (&f)[32]) {
#pragma unroll
    for (int ch = 0; ch < 4; ch++) {
        uint4 pk;
        pk.x = gm_pack(f[ch * 8], f[ch * 8 + 1]);
        pk.y = gm_pack(f[ch * 8 + 2], f[ch * 8 + 3]);
        pk.z = gm_pack(f[ch * 8 + 4], f[ch * 8 + 5]);
        pk.w = gm_pack(f[ch * 8 + 6], f[ch * 8 + 7]);
        *reinterpret_cast<uint4*>(slab + lane * 64 + ((ch ^ ((lane >> 1) & 3)) << 4)) = pk;
    }
}

__device__ __forceinline__ void gm_load32(uint32_t t_addr, float (&f)[32]) {
    uint32_t v[32];
    tmem_ld_32x32(t_addr, v);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 32; j++) f[j] = __uint_as_float(v[j]);
}

// C = residual + dropout(act(A.B^T + bias)); the split-K partial matrices of such a product are written as they are.
template <int BN>
__device__ __forceinline__ void gm_epilogue_act(const GemmParams& p, uint32_t t_row, int m, int m0w, int n0, int sp, int lane, uint8_t* stage,
                                                uint32_t& turn) {
    const bool row_ok = m < p.M;
    const bool aligned = p.c_tma;   // rows of C are 16-byte multiples: N is a multiple of 8
    DropKey key = {};
    if (p.e.drop_threshold && p.splits == 1) key = drop_key(p.e.rng, p.e.site);
#pragma unroll 1
    for (int c0 = 0; c0 < BN; c0 += 32) {
        const int n = n0 + c0;
        if (n >= p.N) break;            // warp-uniform
        float f[32];
        gm_load32(t_row + c0, f);
        const bool full = n + 32 <= p.N;
        if (p.splits > 1) {
            if (row_ok) {
                float* srow = p.slabs + ((long long)sp * p.M + m) * p.N + n;
                if (full && (p.N & 3) == 0) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(srow + j) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        if (n + j < p.N) srow[j] = f[j];
                }
            }
            continue;
        }
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
        uint8_t* slab = stage + (turn & 1) * 4096;
        if (lane == 0) bulk_wait_group_read<1>();   // the stores of two turns ago have read their slabs
        __syncwarp();
        turn++;
        if (p.e.pre) gm_stage32(slab + 2048, lane, f);
        if (p.e.act == 2) {
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] *= gauss_cdf(f[j]);
        } else if (p.e.act == 1) {
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] = fmaxf(f[j], 0.f);
        }
        if (p.e.drop_threshold) {
            const unsigned long long index = (unsigned long long)m * p.N + n;
            const uint32_t mask = drop_mask<32>(key, index, p.e.drop_threshold);
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] = mask >> j & 1u ? f[j] * p.e.drop_scale : 0.f;
        }
        if (p.residual && row_ok) {
            const __nv_bfloat16* res = p.residual + (long long)m * p.N + n;
            if (p.vec_ok) {             // N a multiple of 8
#pragma unroll
                for (int ch = 0; ch < 4; ch++)
                    if (full || n + ch * 8 < p.N) {
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
        gm_stage32(slab, lane, f);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            if (m0w < p.M) {
                if (p.e.pre) tma_store_tile_2d(p.tmap_pre, smem_u32(slab + 2048), n, m0w);
                if (aligned) tma_store_tile_2d(p.tmap_c, smem_u32(slab), n, m0w);
            }
            bulk_commit_group();
        }
        if (!aligned) {
            // rows of an odd width: lane = column, one row after the other, so that a store covers 64 consecutive bytes
            __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.c) + (long long)m0w * p.ldc + n + lane;
            const int rows = p.M - m0w < 32 ? p.M - m0w : 32;
            for (int r = 0; r < rows; r++)
                if (n + lane < p.N)
                    out[r * p.ldc] = *reinterpret_cast<const __nv_bfloat16*>(slab + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2);
            __syncwarp();
        }
    }
}

// Of every row and 128 columns the maximum and the sum of exponentials relative to it, and the logit of the row's label.
template <int BN>
__device__ __forceinline__ void gm_epilogue_lse(const GemmParams& p, uint32_t t_row, int m, int n0) {
    constexpr float kLog2e = 1.4426950408889634f;
    const bool row_ok = m < p.M;
    const long long at = row_ok ? p.e.target[m] - p.e.col0 - n0 : -1;
    const int label = at >= 0 && at < BN ? (int)at : -1;   // the label's column of this tile
    float top = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int c0 = 0; c0 < BN; c0 += 32) {
        const int n = n0 + c0;
        if (n >= p.N) break;            // warp-uniform
        float f[32];
        gm_load32(t_row + c0, f);
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
        const float ref = now == -INFINITY ? 0.f : now * kLog2e;   // columns of minus infinity alone weigh nothing
        // nothing above minus infinity so far: a sum of 0, or not a number
        float part[4] = {top == -INFINITY ? sum : sum * exp2f(top * kLog2e - ref), 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 32; j++) {
            float e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(f[j], kLog2e, -ref)));
            part[j & 3] += e;
        }
        sum = (part[0] + part[1]) + (part[2] + part[3]);
        top = now;
        if (((c0 + 32) & 127) == 0 || n + 32 >= p.N) {
            if (row_ok) p.e.part[(long long)(n >> 7) * p.M + m] = make_float2(top, sum);
            top = -INFINITY;
            sum = 0.f;
        }
    }
}

// C = (softmax - onehot(label)) * coefficient, the probabilities from this product's logits and the row's logsumexp.
template <int BN>
__device__ __forceinline__ void gm_epilogue_dlogits(const GemmParams& p, uint32_t t_row, int m, int m0w, int n0, int lane, uint8_t* stage,
                                                    uint32_t& turn) {
    constexpr float kLog2e = 1.4426950408889634f;
    const bool row_ok = m < p.M;
    const float2 row = row_ok ? p.e.row[m] : make_float2(0.f, 0.f);
    const long long at = row_ok ? p.e.target[m] - p.e.col0 - n0 : -1;
    const int label = at >= 0 && at < BN ? (int)at : -1;
#pragma unroll 1
    for (int c0 = 0; c0 < BN; c0 += 32) {
        const int n = n0 + c0;
        if (n >= p.N) break;            // warp-uniform
        float f[32];
        gm_load32(t_row + c0, f);
#pragma unroll
        for (int j = 0; j < 32; j++) {
            float e;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(f[j], kLog2e, -row.x)));
            f[j] = e;
        }
        if (__any_sync(0xffffffffu, label >= c0 && label < c0 + 32)) {
#pragma unroll
            for (int j = 0; j < 32; j++) f[j] -= label == c0 + j ? 1.f : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 32; j++) f[j] = row.y == 0.f ? 0.f : f[j] * row.y;
        uint8_t* slab = stage + (turn & 1) * 4096;
        if (lane == 0) bulk_wait_group_read<1>();
        __syncwarp();
        turn++;
        gm_stage32(slab, lane, f);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
            if (m0w < p.M) tma_store_tile_2d(p.tmap_c, smem_u32(slab), n, m0w);
            bulk_commit_group();
        }
    }
}
