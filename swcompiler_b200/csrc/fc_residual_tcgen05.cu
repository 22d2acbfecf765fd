// Matrix product with bias, activation and residual in its epilogue, on the 5th-generation tensor cores:
//     C[m,n] = R[m,n] + scale * act( A[m,k] . Wp[n,k]^T + bias[n] )       A, Wp bf16 (K-major), fp32 accumulate
//
// Both kernels compute the TRANSPOSED product, D = Wp . A^T: the weight's rows are the lanes of tensor memory, the rows of A
// (tokens) its columns.  Two reasons.
//   * Few tokens: the instruction's M is 128 whatever happens, its N can be 16.  With tokens on the N side a single token costs
//     an eighth of the operand traffic and of the tensor time that a 128-row tile of tokens would.
//   * The epilogue: a thread holds one output column for 32 tokens, so for each token a warp reads 32 neighbouring residual
//     values and writes 32 neighbouring outputs -- whole sectors, at any alignment of C and R -- and one bias value per tile.
//
// fc_res_split_kernel: one 128 x BN tile per cluster, the k range divided over the cluster's CTAs (up to 8), partial sums joined
//   through distributed shared memory in rank order, no workspace, the same result on every run.  For calls whose tiles alone
//   would leave SMs idle; with few tokens it is bound by reading Wp once.
// fc_res_pair_kernel: persistent CTA pairs (cta_group::2), 256 x BN tiles, two accumulators so that the epilogue of a tile runs
//   beside the main loop of the next.  For everything else; bound by the tensor pipe.
#include "tc_common.cuh"

namespace {

using namespace tc;

constexpr int BM = 128;  // weight rows per CTA
constexpr int BK = 64;   // one 128-byte swizzle row of bf16
constexpr int UMMA_K = 16;
constexpr int W_BYTES = BM * BK * 2;

struct FcrParams {
    int m, n, k;
    int bn;                // tokens per tile
    int tiles_n, tiles_m;  // weight tiles, token tiles
    int band;              // weight tiles per band of the tile order
    int stages, splits;    // split kernel
    const float *bias;
    int act;
    float scale;
    const void *residual;
    int r16;
    size_t ldr;
    void *c;
    int c16;
    size_t ldc;
    int *status;
};

template <int kAct>
__device__ __forceinline__ float activate(float v) {
    if (kAct == SWCB200_ACT_RELU) return v > 0.f ? v : 0.f;
    if (kAct == SWCB200_ACT_TANH) return tanhf(v);
    // v * Phi(v) with Phi(v) = erfc(-v / sqrt 2) / 2: the form without cancellation for negative v
    if (kAct == SWCB200_ACT_GELU) return 0.5f * v * erfcf(-0.70710678118654752f * v);
    // (1 + tanh u) / 2 = 1 / (1 + exp(-2u)), which does not cancel for negative u either
    if (kAct == SWCB200_ACT_GELU_TANH) return __fdividef(v, 1.f + __expf(-1.5957691216057308f * fmaf(0.044715f * v * v, v, v)));
    if (kAct == SWCB200_ACT_SILU) return __fdividef(v, 1.f + __expf(-v));
    return v;
}

__device__ __forceinline__ float load_elem(const void *p, bool is16, size_t i) {
    return is16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]) : reinterpret_cast<const float *>(p)[i];
}

// kTok tokens of one output column: acc[j] belongs to token t0 + j
template <int kAct, int kTok>
__device__ __forceinline__ void finish_act(const FcrParams &p, const float (&acc)[kTok], int t0, int tokens, int col, float bias) {
    float r[kTok];
    if (p.residual) {
        if (p.r16) {
            const __nv_bfloat16 *src = reinterpret_cast<const __nv_bfloat16 *>(p.residual) + (size_t)t0 * p.ldr + col;
#pragma unroll
            for (int j = 0; j < kTok; j++) r[j] = j < tokens ? __bfloat162float(src[j * p.ldr]) : 0.f;
        } else {
            const float *src = reinterpret_cast<const float *>(p.residual) + (size_t)t0 * p.ldr + col;
#pragma unroll
            for (int j = 0; j < kTok; j++) r[j] = j < tokens ? src[j * p.ldr] : 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kTok; j++) r[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < kTok; j++) r[j] = fmaf(p.scale, activate<kAct>(acc[j] + bias), r[j]);
    if (p.c16) {
        __nv_bfloat16 *dst = reinterpret_cast<__nv_bfloat16 *>(p.c) + (size_t)t0 * p.ldc + col;
#pragma unroll
        for (int j = 0; j < kTok; j++)
            if (j < tokens) dst[j * p.ldc] = __float2bfloat16_rn(r[j]);
    } else {
        float *dst = reinterpret_cast<float *>(p.c) + (size_t)t0 * p.ldc + col;
#pragma unroll
        for (int j = 0; j < kTok; j++)
            if (j < tokens) dst[j * p.ldc] = r[j];
    }
}

template <int kTok>
__device__ __forceinline__ void finish(const FcrParams &p, const float (&acc)[kTok], int t0, int col, float bias) {
    const int tokens = min(kTok, p.m - t0);
    if (tokens <= 0 || col >= p.n) return;
    switch (p.act) {
        case SWCB200_ACT_RELU: return finish_act<SWCB200_ACT_RELU, kTok>(p, acc, t0, tokens, col, bias);
        case SWCB200_ACT_TANH: return finish_act<SWCB200_ACT_TANH, kTok>(p, acc, t0, tokens, col, bias);
        case SWCB200_ACT_GELU: return finish_act<SWCB200_ACT_GELU, kTok>(p, acc, t0, tokens, col, bias);
        case SWCB200_ACT_GELU_TANH: return finish_act<SWCB200_ACT_GELU_TANH, kTok>(p, acc, t0, tokens, col, bias);
        case SWCB200_ACT_SILU: return finish_act<SWCB200_ACT_SILU, kTok>(p, acc, t0, tokens, col, bias);
        default: return finish_act<SWCB200_ACT_NONE, kTok>(p, acc, t0, tokens, col, bias);
    }
}

__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// A wait that gave up leaves copies possibly still in flight towards this CTA's shared memory: give them a bounded time to land
// before anyone tears down (the clean path needs none: every load was consumed).
__device__ __forceinline__ void drain_after_failure() {
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000ll) {
    }
}

// tokens t .. t + kTok - 1 of this CTA's `own`: their partial sums added in rank order
template <int kTok>
__device__ __forceinline__ void finish_joined(const FcrParams &p, const float *slots, int own, int t, int row, int token, int col,
                                              float bias) {
    float v[kTok];
#pragma unroll
    for (int j = 0; j < kTok; j++) v[j] = 0.f;
    for (int s = 0; s < p.splits; s++)
#pragma unroll
        for (int j = 0; j < kTok; j++) v[j] += slots[(s * own + t + j) * BM + row];
    finish<kTok>(p, v, token, col, bias);
}

constexpr int kSplitThreads = 192;  // TMA warp, MMA warp, 4 epilogue warps

// shared memory: `stages` x (weight tile, token tile), then the join's slots [splits][BN / splits][128] fp32, then barriers
__global__ void __launch_bounds__(kSplitThreads) fc_res_split_kernel(const __grid_constant__ CUtensorMap tmW,
                                                                     const __grid_constant__ CUtensorMap tmA, const FcrParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t stage_bytes = W_BYTES + (uint32_t)p.bn * BK * 2;
    float *slots = reinterpret_cast<float *>(smem + (size_t)p.stages * stage_bytes);
    uint64_t *full = reinterpret_cast<uint64_t *>(slots + (p.splits > 1 ? p.bn * BM : 0));
    uint64_t *empty = full + p.stages;
    uint64_t *done = empty + p.stages;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(done + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t tmem_cols = p.bn < 32 ? 32u : (uint32_t)p.bn;
    const uint32_t rank = p.splits > 1 ? cluster_ctarank() : 0;
    const int tile = blockIdx.x / p.splits;
    const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
    const int kblocks = (p.k + BK - 1) / BK;
    const int kb0 = (int)((long long)kblocks * rank / p.splits), kb1 = (int)((long long)kblocks * (rank + 1) / p.splits);

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmA);
        for (int s = 0; s < p.stages; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(done, 1);
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 1) {
        tmem_alloc(tmem_holder, tmem_cols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    if (p.splits > 1) cluster_sync();  // every CTA of the cluster runs before its shared memory is written from another
    tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;
    bool failed = false;

    if (warp == 0) {
        if (lane == 0) {
            int st = 0;
            uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!mbar_wait(&empty[st], ph ^ 1, p.status, kWaitEmpty)) {
                    failed = true;
                    break;
                }
                mbar_expect_tx(&full[st], stage_bytes);
                uint8_t *sw = smem + (size_t)st * stage_bytes;
                tma_load_2d(sw, &tmW, &full[st], kb * BK, tn * BM);
                tma_load_2d(sw + W_BYTES, &tmA, &full[st], kb * BK, tm * p.bn);
                if (++st == p.stages) {
                    st = 0;
                    ph ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = idesc_bf16_f32(BM, p.bn);
            int st = 0;
            uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!mbar_wait(&full[st], ph, p.status, kWaitFull)) {
                    failed = true;
                    break;
                }
                tc_fence_after();
                const uint32_t sw = smem_u32(smem + (size_t)st * stage_bytes);
                const uint64_t dw = smem_desc_sw128(sw), da = smem_desc_sw128(sw + W_BYTES);
#pragma unroll
                for (int j = 0; j < BK / UMMA_K; j++)
                    umma_bf16(tmem_base, dw + 2 * j, da + 2 * j, idesc, (uint32_t)(kb != kb0 || j != 0));
                umma_commit(&empty[st]);
                if (++st == p.stages) {
                    st = 0;
                    ph ^= 1;
                }
            }
            if (!failed) umma_commit(done);
        }
    } else {
        bool ok = true;
        if (lane == 0) ok = mbar_wait(done, 0, p.status, kWaitTmemFull);
        failed = !__shfl_sync(0xffffffffu, ok, 0);
        tc_fence_after();
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const int col = tn * BM + row;
        if (!failed) {
            if (p.splits == 1) {
                const float bias = p.bias && col < p.n ? __ldg(p.bias + col) : 0.f;
                for (int c0 = 0; c0 < p.bn; c0 += 16) {
                    if (tm * p.bn + c0 >= p.m) break;
                    uint32_t r[16];
                    float acc[16];
                    tmem_ld_32x16(taddr + c0, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; j++) acc[j] = __uint_as_float(r[j]);
                    finish<16>(p, acc, tm * p.bn + c0, col, bias);
                    __syncwarp();
                }
            } else {
                // this CTA's partial sums go to the CTAs that own the tokens, slot `rank`
                const int own = p.bn / p.splits;  // a power of two, at least 2
                const int own_log2 = 31 - __clz(own);
                const uint32_t mine = smem_u32(slots + (int)rank * own * BM + row);
                for (int c0 = 0; c0 < p.bn; c0 += 16) {
                    if (tm * p.bn + c0 >= p.m) break;
                    uint32_t r[16];
                    tmem_ld_32x16(taddr + c0, r);
                    tmem_ld_wait();
                    // 16 columns lie in one owner's part (own >= 16) or cover 16 / own owners
#pragma unroll
                    for (int j = 0; j < 16; j += 2) {
                        const int q = (c0 + j) >> own_log2, t = (c0 + j) & (own - 1);
                        const uint32_t dst = map_to_cta(mine + (uint32_t)t * (BM * 4), (uint32_t)q);
                        st_cluster(dst, __uint_as_float(r[j]));
                        st_cluster(dst + BM * 4, __uint_as_float(r[j + 1]));
                    }
                }
            }
        }
    }
    if (failed) drain_after_failure();
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (p.splits > 1) {
        cluster_sync();  // all partial sums have arrived
        if (warp >= 2) {
            const int row = (warp & 3) * 32 + lane, col = tn * BM + row;
            const float bias = p.bias && col < p.n ? __ldg(p.bias + col) : 0.f;
            const int own = p.bn / p.splits;
            const int token0 = tm * p.bn + (int)rank * own;
            if (own < 8) {
                for (int t = 0; t < own; t += 2) finish_joined<2>(p, slots, own, t, row, token0 + t, col, bias);
            } else {
                for (int t = 0; t < own; t += 8) finish_joined<8>(p, slots, own, t, row, token0 + t, col, bias);
            }
        }
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, tmem_cols);
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
constexpr int BN_MAX = 256;
constexpr int A_BYTES = (BN_MAX / 2) * BK * 2;  // this CTA's half of the token tile
constexpr int kPairStages = 6;
constexpr int kPairStageBytes = W_BYTES + A_BYTES;
constexpr int kPairEpiWarps = 8;  // two per lane quarter of tensor memory, each half of a tile's tokens
constexpr int kPairThreads = 64 + 32 * kPairEpiWarps;
constexpr size_t kPairSmem = (size_t)kPairStages * kPairStageBytes + 1024 + 256;
constexpr int kTmemCols = 512;  // two accumulators of 256 columns

// Tiles are taken band by band: a band is `band` weight tiles wide and is walked token panel by token panel, weight tiles fastest,
// so that the pairs running together share a few token panels and at most `band` weight tiles, which keeps both in L2.
__device__ __forceinline__ void tile_coords(const FcrParams &p, int t, int &tm, int &tn) {
    const int per_band = p.band * p.tiles_m;
    const int b = t / per_band, i = t - b * per_band;
    const int n0 = b * p.band;
    const int gw = min(p.band, p.tiles_n - n0);
    tm = i / gw;
    tn = n0 + (i - tm * gw);
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
fc_res_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA, const FcrParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + (size_t)kPairStages * kPairStageBytes);
    uint64_t *empty = full + kPairStages;
    uint64_t *tmem_full = empty + kPairStages;
    uint64_t *tmem_empty = tmem_full + 2;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(tmem_empty + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int num_tiles = p.tiles_m * p.tiles_n;
    const int kblocks = (p.k + BK - 1) / BK;
    const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
    const int half_bn = p.bn >> 1;

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmA);
        for (int s = 0; s < kPairStages; s++) {
            mbar_init(&full[s], 1);   // leader: counts the bytes of both CTAs' loads
            mbar_init(&empty[s], 1);  // signalled in both CTAs by one commit
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&tmem_full[b], 1);
            mbar_init(&tmem_empty[b], 2 * kPairEpiWarps);  // leader: the epilogue warps of both CTAs
        }
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_holder, kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peer's barriers exist before anything is signalled across the pair
    tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;
    bool failed = false;

    if (warp == 0) {
        if (lane == 0) {
            const uint32_t tx_bytes = 2u * (uint32_t)(W_BYTES + half_bn * BK * 2);
            int st = 0;
            uint32_t ph = 0;
            for (int t = cluster_id; t < num_tiles && !failed; t += num_clusters) {
                int tm, tn;
                tile_coords(p, t, tm, tn);
                const int row_w = tn * (2 * BM) + (int)rank * BM, row_a = tm * p.bn + (int)rank * half_bn;
                for (int kb = 0; kb < kblocks; kb++) {
                    if (!mbar_wait(&empty[st], ph ^ 1, p.status, kWaitEmpty)) {
                        failed = true;
                        break;
                    }
                    const uint32_t full_leader = map_to_cta(smem_u32(&full[st]), 0);
                    if (leader) mbar_expect_tx(&full[st], tx_bytes);
                    uint8_t *sw = smem + (size_t)st * kPairStageBytes;
                    tma_load_2d_pair(sw, &tmW, full_leader, kb * BK, row_w);
                    tma_load_2d_pair(sw + W_BYTES, &tmA, full_leader, kb * BK, row_a);
                    if (++st == kPairStages) {
                        st = 0;
                        ph ^= 1;
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (leader && lane == 0) {
            const uint32_t idesc = idesc_bf16_f32(2 * BM, p.bn);
            const uint64_t dw0 = smem_desc_sw128(smem_u32(smem)), da0 = smem_desc_sw128(smem_u32(smem + W_BYTES));
            int st = 0;
            uint32_t ph = 0, it = 0;
            for (int t = cluster_id; t < num_tiles && !failed; t += num_clusters, it++) {
                const uint32_t buf = it & 1, aph = (it >> 1) & 1;
                if (!mbar_wait(&tmem_empty[buf], aph ^ 1, p.status, kWaitTmemEmpty)) {
                    failed = true;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + buf * BN_MAX;
                for (int kb = 0; kb < kblocks; kb++) {
                    if (!mbar_wait(&full[st], ph, p.status, kWaitFull)) {
                        failed = true;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t off = (uint64_t)st * (kPairStageBytes >> 4);
                    const uint64_t dw = dw0 + off, da = da0 + off;
                    umma_bf16_pair(d_tmem, dw, da, idesc, (uint32_t)(kb != 0));
                    umma_bf16_pair(d_tmem, dw + 2, da + 2, idesc, 1u);
                    umma_bf16_pair(d_tmem, dw + 4, da + 4, idesc, 1u);
                    umma_bf16_pair(d_tmem, dw + 6, da + 6, idesc, 1u);
                    umma_commit_pair(&empty[st], 3);
                    if (++st == kPairStages) {
                        st = 0;
                        ph ^= 1;
                    }
                }
                if (!failed) umma_commit_pair(&tmem_full[buf], 3);
            }
        }
    } else {
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        uint32_t it = 0;
        for (int t = cluster_id; t < num_tiles; t += num_clusters, it++) {
            const uint32_t buf = it & 1, aph = (it >> 1) & 1;
            int tm, tn;
            tile_coords(p, t, tm, tn);
            bool ok = true;
            if (lane == 0) ok = mbar_wait(&tmem_full[buf], aph, p.status, kWaitTmemFull);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) {
                failed = true;
                break;
            }
            tc_fence_after();
            const int col = tn * (2 * BM) + (int)rank * BM + quarter * 32 + lane;
            const float bias = p.bias && col < p.n ? __ldg(p.bias + col) : 0.f;
            for (int c0 = half * half_bn; c0 < (half + 1) * half_bn; c0 += 32) {
                if (tm * p.bn + c0 >= p.m) break;
                uint32_t r[32];
                float acc[32];
                __syncwarp();
                tmem_ld_32x32(tmem_base + ((uint32_t)(quarter * 32) << 16) + buf * BN_MAX + c0, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; j++) acc[j] = __uint_as_float(r[j]);
                finish<32>(p, acc, tm * p.bn + c0, col, bias);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&tmem_empty[buf]), 0));
        }
    }
    if (failed) drain_after_failure();
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // neither CTA leaves while the other's MMAs may read its shared memory or signal its barriers
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

// row-major [rows, cols] bf16 with leading dimension ld; box = box_rows x 64
int tmap_rows(swcb200_ctx *ctx, const void *base, int rows, int cols, int ld, int box_rows, CUtensorMap *out) {
    const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows}, strides[2] = {2, (uint64_t)ld * 2};
    const uint32_t box[2] = {(uint32_t)BK, (uint32_t)box_rows};
    return make_tmap_bf16(ctx, out, base, 2, dims, strides, box);
}

size_t split_smem(const FcrParams &p) {
    return (size_t)p.stages * (W_BYTES + p.bn * BK * 2) + (p.splits > 1 ? (size_t)p.bn * BM * 4 : 0) + 1024 + 256;
}

}  // namespace

SWC_EXPORT int swcb200_fc_bf16_residual(swcb200_ctx *ctx, int m, int n, int k, const void *a_bf16, int lda, const void *wp_bf16,
                                        int ldw, const swcb200_fc_epilogue *ep, void *c, int c_dtype, int ldc) {
    SWC_CTX(ctx);
    SWC_REQUIRE(ctx, ep != nullptr, SWCB200_ERR_BAD_ARG, "fc_bf16_residual: null epilogue");
    SWC_REQUIRE(ctx, m >= 0 && n >= 0 && k > 0, SWCB200_ERR_BAD_ARG, "fc_bf16_residual: bad shape %d x %d x %d", m, n, k);
    SWC_REQUIRE(ctx, ep->act >= SWCB200_ACT_NONE && ep->act <= SWCB200_ACT_SILU, SWCB200_ERR_BAD_ARG,
                "fc_bf16_residual: unknown activation %d", ep->act);
    SWC_REQUIRE(ctx, (c_dtype == SWCB200_F32 || c_dtype == SWCB200_BF16) &&
                (!ep->residual || ep->residual_dtype == SWCB200_F32 || ep->residual_dtype == SWCB200_BF16),
                SWCB200_ERR_BAD_ARG, "fc_bf16_residual: C and the residual are fp32 or bf16");
    if (m == 0 || n == 0) return SWCB200_OK;
    SWC_REQUIRE(ctx, a_bf16 && wp_bf16 && c, SWCB200_ERR_BAD_ARG, "fc_bf16_residual: null tensor");
    SWC_REQUIRE(ctx, swc_aligned16(a_bf16) && swc_aligned16(wp_bf16) && lda % 8 == 0 && ldw % 8 == 0, SWCB200_ERR_MISALIGNED,
                "fc_bf16_residual: A and Wp start on 16 bytes, lda (%d) and ldw (%d) are multiples of 8 elements", lda, ldw);
    SWC_REQUIRE(ctx, lda >= k && ldw >= k && ldc >= n && (!ep->residual || ep->ld_residual >= n), SWCB200_ERR_BAD_SHAPE,
                "fc_bf16_residual: leading dimension too small");
    const size_t ce = c_dtype == SWCB200_BF16 ? 2 : 4, re = ep->residual_dtype == SWCB200_BF16 ? 2 : 4;
    SWC_REQUIRE(ctx, !ep->residual || (ep->residual == c && ce == re && (m == 1 || ep->ld_residual == ldc)) ||
                !swc_rows_overlap(c, ldc * ce, n * ce, ep->residual, ep->ld_residual * re, n * re, (size_t)m),
                SWCB200_ERR_BAD_ARG, "fc_bf16_residual: C overlaps the residual without being the same tensor");
    FcrParams p = {};
    p.m = m, p.n = n, p.k = k;
    p.bias = ep->bias, p.act = ep->act, p.scale = ep->scale;
    p.residual = ep->residual, p.r16 = re == 2, p.ldr = (size_t)ep->ld_residual;
    p.c = c, p.c16 = ce == 2, p.ldc = (size_t)ldc;
    p.status = ctx->dev_status;
    const int sms = swc_tc_sms(ctx);
    CUtensorMap tmW, tmA;

    const long long pairs = sms / 2;
    const long long tiles256 = (long long)((n + 255) / 256) * ((m + 255) / 256);
    if (tiles256 >= pairs && pairs > 0) {
        p.bn = BN_MAX;
        p.tiles_n = (n + 2 * BM - 1) / (2 * BM);
        p.tiles_m = (m + p.bn - 1) / p.bn;
        SWC_REQUIRE(ctx, (long long)p.tiles_n * p.tiles_m < 0x7fffffff, SWCB200_ERR_TOO_LARGE, "fc_bf16_residual: too many tiles");
        p.band = ((size_t)n * k * 2 <= ((size_t)48 << 20) || p.tiles_n <= 8) ? p.tiles_n : 8;
        int rc = tmap_rows(ctx, wp_bf16, n, k, ldw, BM, &tmW);
        if (!rc) rc = tmap_rows(ctx, a_bf16, m, k, lda, p.bn / 2, &tmA);
        if (rc) return rc;
        SWC_CUDA(ctx, cudaFuncSetAttribute(fc_res_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPairSmem));
        const long long tiles = (long long)p.tiles_n * p.tiles_m;
        const unsigned grid = 2u * (unsigned)(tiles < pairs ? tiles : pairs);
        fc_res_pair_kernel<<<grid, kPairThreads, kPairSmem, ctx->stream>>>(tmW, tmA, p);
        return swc_check_launch(ctx, "fc_bf16_residual");
    }
    p.bn = 16;
    while (p.bn < m && p.bn < 128) p.bn *= 2;
    p.tiles_n = (n + BM - 1) / BM;
    p.tiles_m = (m + p.bn - 1) / p.bn;
    SWC_REQUIRE(ctx, (long long)p.tiles_n * p.tiles_m < 0x7fffffff / 8, SWCB200_ERR_TOO_LARGE, "fc_bf16_residual: too many tiles");
    const long long tiles = (long long)p.tiles_n * p.tiles_m;
    const int kblocks = (k + BK - 1) / BK;
    p.splits = 1;
    while (p.splits < 8 && tiles * p.splits * 2 <= 2 * sms && kblocks >= p.splits * 2 * 4) p.splits *= 2;
    p.stages = p.bn <= 32 ? 5 : 4;
    int rc = tmap_rows(ctx, wp_bf16, n, k, ldw, BM, &tmW);
    if (!rc) rc = tmap_rows(ctx, a_bf16, m, k, lda, p.bn, &tmA);
    if (rc) return rc;
    const size_t smem = split_smem(p);
    SWC_CUDA(ctx, cudaFuncSetAttribute(fc_res_split_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * p.splits));
    cfg.blockDim = dim3(kSplitThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)p.splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    SWC_CUDA(ctx, cudaLaunchKernelEx(&cfg, fc_res_split_kernel, tmW, tmA, p));
    return swc_check_launch(ctx, "fc_bf16_residual");
}
