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
//   beside the main loop of the next.  For everything else; bound by the tensor pipe: 16384 x 4096 x 4096 with bias, tanh-GELU and a
//   bf16 residual 381 us in a burst, 1442 TFLOP/s, 0.90 of the burst rate of a library product measured here, and 441 us in calls that
//   go on for seconds (1.28 GHz under the power limit), 0.93 of the sustained one.
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

__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// A wait that gave up leaves copies possibly still in flight towards this CTA's shared memory: give them a bounded time to land
// before anyone tears down (the clean path needs none: every load was consumed).
__device__ __forceinline__ void drain_after_failure() {
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000ll) {
    }
}

// kTok tokens of one column: the partial sums of all slots added in rank order
template <int kTok>
__device__ __forceinline__ void finish_joined(const FcrParams &p, const float *mine, int slot, int token, int col, float bias) {
    float v[kTok];
#pragma unroll
    for (int j = 0; j < kTok; j++) v[j] = 0.f;
    for (int s = 0; s < p.splits; s++)
#pragma unroll
        for (int j = 0; j < kTok; j++) v[j] += mine[s * slot + j * BM];
    finish<kTok>(p, v, token, col, bias);
}

constexpr int kSplitThreads = 320;  // TMA warp, MMA warp, 8 epilogue warps: two per lane quarter of tensor memory

// shared memory: `stages` x (weight tile, token tile), then barriers; once every CTA of the cluster has multiplied its last stage
// the ring becomes the join's slots, [splits][own][128 rows] fp32 with own = BN / splits tokens: a warp's store to another CTA is
// 128 contiguous bytes (16-byte pieces at the pitch of a row took 2 us longer per join)
// kSub: 64-deep blocks per stage of the ring.  Two of them halve the waits and commits, which at few tokens cost the issuing
// threads more than the blocks do (64 tokens, 4096 x 4096, k undivided: 22.1 -> 17.7 us); at 256 tokens a stage of one keeps the
// ring four deep.
template <int kSub>
__global__ void __launch_bounds__(kSplitThreads) fc_res_split_kernel(const __grid_constant__ CUtensorMap tmW,
                                                                     const __grid_constant__ CUtensorMap tmA, const FcrParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t block_bytes = W_BYTES + (uint32_t)p.bn * BK * 2, stage_bytes = kSub * block_bytes;
    float *slots = reinterpret_cast<float *>(smem);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + (size_t)p.stages * stage_bytes);
    uint64_t *empty = full + p.stages;
    uint64_t *done = empty + p.stages;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(done + 1);

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;  // warp: known to be uniform
    const uint32_t tmem_cols = p.bn < 32 ? 32u : (uint32_t)p.bn;
    const uint32_t rank = p.splits > 1 ? cluster_ctarank() : 0;
    const int tile = blockIdx.x / p.splits;
    const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
    const int kblocks = (p.k + kSub * BK - 1) / (kSub * BK);
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
    swc_let_next_start();
    swc_after_previous();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_holder, 0);
    bool failed = false;
    // epilogue warps: a row of the tile (an output column) per thread, in the lane quarter that the warp may read
    const int row = (warp & 3) * 32 + lane, col = tn * BM + row, half = (warp - 2) >> 2;
    const int own = p.bn / p.splits;  // tokens that this CTA joins: a power of two, at least 2
    const uint32_t taddr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);

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
#pragma unroll
                for (int b = 0; b < kSub; b++) {
                    tma_load_2d(sw + b * block_bytes, &tmW, &full[st], (kb * kSub + b) * BK, tn * BM);
                    tma_load_2d(sw + b * block_bytes + W_BYTES, &tmA, &full[st], (kb * kSub + b) * BK, tm * p.bn);
                }
                if (++st == p.stages) {
                    st = 0;
                    ph ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        const uint32_t idesc = idesc_bf16_f32(BM, p.bn);
        const uint32_t dw0 = desc_low(smem_u32(smem), 16), da0 = desc_low(smem_u32(smem + W_BYTES), 16);
        int st = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; kb++) {
            if (!warp_wait(&full[st], ph, p.status, kWaitFull)) {
                failed = true;
                break;
            }
            tc_fence_after();
            const uint32_t off = (uint32_t)st * (stage_bytes >> 4);
            if (elect_one()) {
#pragma unroll
                for (int b = 0; b < kSub; b++)
#pragma unroll
                    for (int j = 0; j < BK / UMMA_K; j++)
                        umma_bf16_words(tmem_base, dw0 + off + b * (block_bytes >> 4) + 2 * j, da0 + off + b * (block_bytes >> 4) + 2 * j, idesc,
                                        kb != kb0 || b + j != 0);
                umma_commit(&empty[st]);
                if (kb + 1 == kb1) umma_commit(done);
            }
            __syncwarp();
            if (++st == p.stages) {
                st = 0;
                ph ^= 1;
            }
        }
    } else {
        // the residual's rows are brought as near as L2 while the products run
        if (p.residual && col - lane < p.n) {
            const int first = p.splits > 1 ? (int)rank * own : 0, count = min(p.splits > 1 ? own : p.bn, p.m - tm * p.bn - first);
            const size_t e = p.r16 ? 2 : 4;
            for (int t = half * 32 + lane; t < count; t += 64) {
                const char *at = reinterpret_cast<const char *>(p.residual) + ((size_t)(tm * p.bn + first + t) * p.ldr + col - lane) * e;
                asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
                asm volatile("prefetch.global.L2 [%0];" ::"l"(at + (min(31, p.n - 1 - (col - lane))) * e));
            }
        }
        bool ok = true;
        if (lane == 0) ok = mbar_wait(done, 0, p.status, kWaitTmemFull);
        failed = !__shfl_sync(0xffffffffu, ok, 0);
        tc_fence_after();
        if (!failed && p.splits == 1) {
            const float bias = p.bias && col < p.n ? p.bias[col] : 0.f;
            for (int c0 = half * 16; c0 < p.bn; c0 += 32) {
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
        }
    }
    if (failed) drain_after_failure();
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (p.splits > 1) {
        cluster_sync();  // every CTA has read its last stage: the rings may be overwritten
        const int own_log2 = 31 - __clz(own);
        if (warp >= 2) {
            // this CTA's partial sums go to the CTAs that own the tokens, slot `rank`
            tc_fence_after();
            const uint32_t mine = smem_u32(slots + (int)rank * own * BM + row);
            for (int c0 = half * 16; c0 < p.bn; c0 += 32) {
                if (tm * p.bn + c0 >= p.m) break;
                uint32_t r[16];
                tmem_ld_32x16(taddr + c0, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const int q = (c0 + j) >> own_log2, t = (c0 + j) & (own - 1);
                    const uint32_t dst = map_to_cta(mine + (uint32_t)t * (BM * 4), (uint32_t)q);
                    st_cluster(dst, r[j]);
                    st_cluster(dst + BM * 4, r[j + 1]);
                }
            }
        }
        cluster_sync();  // all partial sums have arrived
        if (warp >= 2) {
            const float bias = p.bias && col < p.n ? p.bias[col] : 0.f;
            // the CTA's tokens, half of them for each of the two warps of a quarter
            const int count = own > 2 ? own / 2 : half == 0 ? own : 0, first = count * half, slot = own * BM;
            const float *mine = slots + first * BM + row;
            const int token0 = tm * p.bn + (int)rank * own + first;
            if (count == 2)
                finish_joined<2>(p, mine, slot, token0, col, bias);
            else if (count < 16)
                for (int t = 0; t < count; t += 4) finish_joined<4>(p, mine + t * BM, slot, token0 + t, col, bias);
            else if (count < 32)
                finish_joined<16>(p, mine, slot, token0, col, bias);
            else
                for (int t = 0; t < count; t += 32) finish_joined<32>(p, mine + t * BM, slot, token0 + t, col, bias);
        }
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, tmem_cols);
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
// One or two tokens.  Reading the weights is all there is to it (a multiply-add per weight and token), and at these sizes a call is
// a few microseconds, of which a tensor-core kernel's set-up and drain would be half: here every thread requests its whole share of
// 8 (two tokens: 4) weight rows at once, multiplies on the FP32 pipe, and the CTA adds up.  4096 x 4096: 7.5 and 9 us, 0.69 of
// the bytes' rate at one token (a tensor-core tile 10 us); 8192 x 8192 at one token 23.6 us, 0.87.  From three tokens on the
// registers that hold them cost more loads in flight than the tensor cores' set-up (four tokens: 11.1 us against 9.9).
constexpr int kFewThreads = 256;
__host__ __device__ constexpr int few_rows(int tokens) { return tokens > 1 ? 4 : 8; }

// sums of kV values over the 32 lanes: lane l ends up with the sum of value l % kV
template <int kV> __device__ __forceinline__ float lanes_sum(float (&v)[kV], int lane) {
#pragma unroll
    for (int n = kV / 2; n >= 1; n /= 2) {  // halve the values: keep the half that this lane's bit names, send the other
        const bool upper = lane & n;
#pragma unroll
        for (int i = 0; i < n; i++) {
            const float keep = upper ? v[i + n] : v[i], give = upper ? v[i] : v[i + n];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, n);
        }
    }
#pragma unroll
    for (int o = kV; o < 32; o *= 2) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    return v[0];
}

// the last `count` < 8 elements of a row, zeros behind them
__device__ __noinline__ uint4 load_end(const __nv_bfloat16 *p, int count) {
    uint32_t r[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 7; e++)
        if (e < count) r[e / 2] |= (uint32_t)__bfloat16_as_ushort(p[e]) << (e & 1) * 16;
    return make_uint4(r[0], r[1], r[2], r[3]);
}

template <int kTokens>
__global__ void __launch_bounds__(kFewThreads, kTokens == 1 ? 4 : 1) fc_res_few_kernel(const __nv_bfloat16 *a, size_t lda,
                                                                 const __nv_bfloat16 *w, size_t ldw, const FcrParams p) {
    constexpr int kFewRows = few_rows(kTokens), kV = kFewRows * kTokens;
    __shared__ float part[kFewThreads / 32][kV];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n0 = blockIdx.x * kFewRows;
    float acc[kV];
#pragma unroll
    for (int i = 0; i < kV; i++) acc[i] = 0.f;
    swc_let_next_start();
    swc_after_previous();
    // k in steps of 8 elements per thread
#pragma unroll 2
    for (int k = threadIdx.x * 8; k < p.k; k += kFewThreads * 8) {
        uint4 wv[kFewRows], av[kTokens];
        if (k + 8 <= p.k) {
#pragma unroll
            for (int r = 0; r < kFewRows; r++) {
                const __nv_bfloat16 *src = w + (size_t)min(n0 + r, p.n - 1) * ldw + k;
                asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(wv[r].x), "=r"(wv[r].y), "=r"(wv[r].z), "=r"(wv[r].w)
                             : "l"(src));
            }
#pragma unroll
            for (int t = 0; t < kTokens; t++) av[t] = *reinterpret_cast<const uint4 *>(a + (size_t)min(t, p.m - 1) * lda + k);
        } else {  // the end of the rows: nothing behind it is read
#pragma unroll
            for (int r = 0; r < kFewRows; r++) wv[r] = load_end(w + (size_t)min(n0 + r, p.n - 1) * ldw + k, p.k - k);
#pragma unroll
            for (int t = 0; t < kTokens; t++) av[t] = load_end(a + (size_t)min(t, p.m - 1) * lda + k, p.k - k);
        }
#pragma unroll
        for (int t = 0; t < kTokens; t++) {
            const uint32_t x[4] = {av[t].x, av[t].y, av[t].z, av[t].w};
#pragma unroll
            for (int r = 0; r < kFewRows; r++) {
                const uint32_t y[4] = {wv[r].x, wv[r].y, wv[r].z, wv[r].w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    acc[t * kFewRows + r] = fmaf(__uint_as_float(x[e] << 16), __uint_as_float(y[e] << 16), acc[t * kFewRows + r]);
                    acc[t * kFewRows + r] = fmaf(__uint_as_float(x[e] & 0xffff0000u), __uint_as_float(y[e] & 0xffff0000u), acc[t * kFewRows + r]);
                }
            }
        }
    }
    const float sum = lanes_sum<kV>(acc, lane);
    if (lane < kV) part[warp][lane] = sum;
    __syncthreads();
    if (threadIdx.x < kV) {
        const int t = threadIdx.x / kFewRows, col = n0 + threadIdx.x % kFewRows;
        float v[1] = {0.f};
#pragma unroll
        for (int i = 0; i < kFewThreads / 32; i++) v[0] += part[i][threadIdx.x];
        if (col < p.n) finish<1>(p, v, t, col, p.bias ? p.bias[col] : 0.f);
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

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;  // warp: known to be uniform
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
    swc_let_next_start();
    swc_after_previous();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_holder, 0);
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
        if (leader) {
            const uint32_t idesc = idesc_bf16_f32(2 * BM, p.bn);
            const uint32_t dw0 = desc_low(smem_u32(smem), 16), da0 = desc_low(smem_u32(smem + W_BYTES), 16);
            int st = 0;
            uint32_t ph = 0, it = 0;
            for (int t = cluster_id; t < num_tiles && !failed; t += num_clusters, it++) {
                const uint32_t buf = it & 1, aph = (it >> 1) & 1;
                if (!warp_wait(&tmem_empty[buf], aph ^ 1, p.status, kWaitTmemEmpty)) {
                    failed = true;
                    break;
                }
                const uint32_t d_tmem = tmem_base + buf * BN_MAX;
                for (int kb = 0; kb < kblocks; kb++) {
                    if (!warp_wait(&full[st], ph, p.status, kWaitFull)) {
                        failed = true;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t off = (uint32_t)st * (kPairStageBytes >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int j = 0; j < BK / UMMA_K; j++)
                            umma_bf16_pair_words(d_tmem, dw0 + off + 2 * j, da0 + off + 2 * j, idesc, kb != 0 || j != 0);
                        umma_commit_pair(&empty[st], 3);
                        if (kb + 1 == kblocks) umma_commit_pair(&tmem_full[buf], 3);
                    }
                    __syncwarp();
                    if (++st == kPairStages) {
                        st = 0;
                        ph ^= 1;
                    }
                }
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
            const float bias = p.bias && col < p.n ? p.bias[col] : 0.f;
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

constexpr int kSplitSmem = 226 * 1024;

struct Choice {
    bool pair;
    int bn, splits;
};

// The form with the least time by a model of it: waves over the SMs, times what a CTA spends on its k blocks and beside them.
// Measured at k = 4096, in us: a 64-deep block takes 0.11 / 0.12 / 0.155 / 0.19 / 0.28 at 16 / 32 / 64 / 128 / 256 tokens (the
// issuing threads, then loads), 0.30 in the pair form (the tensor pipe at 256 x 256); launch, first loads, epilogue 6.5 + 0.016 per
// token; the join over 2 / 4 / 8 CTAs 0.8 / 2 / 3.5.  Forms compared in one run, (m, n) = (777, 1000): chosen 128 tokens over 2
// CTAs 14.7 us; 4 CTAs (two waves) 21.6; undivided 19.9; 256 tokens over 4 18.1; pairs 26.1.  (64, 4096): 64 over 4 11.1; over 8
// 12.4; undivided 17.7.  Different weights in every call, from HBM, and a bf16 residual, at n = k = 4096: 3 tokens 10.4 us, 16 10.6,
// 64 13.3, 256 17.3; the bytes alone 5.2 to 6.1, and no weight is requested before the stream's previous kernel has ended.
// limited: no more than `sms` CTAs at all, as each holds an SM of its own.  Only the pairs walk over tiles, so a split form is open
// to calls of one wave; a limit of one SM gets a pair all the same.
Choice choose(int m, int n, int kblocks, int sms, bool limited) {
    Choice best = {true, BN_MAX, 1};
    const auto up = [](long long a, long long b) { return (a + b - 1) / b; };
    double least = sms < 2 ? 1e30 : (double)up(up(n, 2 * BM) * up(m, BN_MAX), sms / 2) * kblocks * 0.30 + 6.5;
    const double step[5] = {0.11, 0.12, 0.155, 0.19, 0.28}, join[4] = {0, 0.8, 2.0, 3.5};
    for (int i = 0; i < 5; i++)
        for (int j = 0; j < 4; j++) {
            const int bn = 16 << i, s = 1 << j;
            if ((j > 0 && s * 2 > kblocks) || (i > 0 && bn >= 2 * m)) continue;
            const long long waves = up(up(n, BM) * up(m, bn) * s, sms);
            if (limited && waves > 1) continue;
            const double t = (double)waves * ((double)up(kblocks, s) * step[i] + 6.5 + 0.016 * bn + join[j]);
            if (t < least) least = t, best = {false, bn, s};
        }
    return best;
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
    SWC_REQUIRE(ctx, m <= 1 << 30 && n <= 1 << 30 && k <= 1 << 30, SWCB200_ERR_TOO_LARGE, "fc_bf16_residual: more than 2^30 rows or columns");
    SWC_REQUIRE(ctx, lda >= k && ldw >= k && ldc >= n && (!ep->residual || ep->ld_residual >= n), SWCB200_ERR_BAD_SHAPE,
                "fc_bf16_residual: leading dimension too small");
    const size_t ce = c_dtype == SWCB200_BF16 ? 2 : 4, re = ep->residual_dtype == SWCB200_BF16 ? 2 : 4;
    SWC_REQUIRE(ctx, !ep->residual || (ep->residual == c && ce == re && (m == 1 || ep->ld_residual == ldc)) ||
                !swc_rows_overlap(c, ldc * ce, n * ce, ep->residual, ep->ld_residual * re, n * re, (size_t)m),
                SWCB200_ERR_BAD_ARG, "fc_bf16_residual: C overlaps the residual without being the same tensor");
    // other CTAs still read A, Wp and the bias when one stores its tile
    const auto end = [](const void *q, int rows, size_t pitch, size_t width) { return (const char *)q + (size_t)(rows - 1) * pitch + width; };
    const char *c0 = (const char *)c, *c1 = end(c, m, ldc * ce, n * ce), *w0 = (const char *)wp_bf16;
    SWC_REQUIRE(ctx, !swc_rows_overlap(c, ldc * ce, n * ce, a_bf16, (size_t)lda * 2, (size_t)k * 2, (size_t)m) &&
                (c1 <= w0 || end(w0, n, (size_t)ldw * 2, (size_t)k * 2) <= c0) &&
                (!ep->bias || c1 <= (const char *)ep->bias || (const char *)(ep->bias + n) <= c0),
                SWCB200_ERR_BAD_ARG, "fc_bf16_residual: C overlaps A, Wp or the bias");
    FcrParams p = {};
    p.m = m, p.n = n, p.k = k;
    p.bias = ep->bias, p.act = ep->act, p.scale = ep->scale;
    p.residual = ep->residual, p.r16 = re == 2, p.ldr = (size_t)ep->ld_residual;
    p.c = c, p.c16 = ce == 2, p.ldc = (size_t)ldc;
    p.status = ctx->dev_status;
    const int sms = swc_tc_sms(ctx);
    CUtensorMap tmW, tmA;

    if (m <= 2) {
        const auto kernel = m == 1 ? fc_res_few_kernel<1> : fc_res_few_kernel<2>;
        SWC_CUDA(ctx, swc_launch_early(kernel, (unsigned)((n + few_rows(m) - 1) / few_rows(m)), kFewThreads, 0, ctx->stream, 1,
                                       (const __nv_bfloat16 *)a_bf16, (size_t)lda, (const __nv_bfloat16 *)wp_bf16, (size_t)ldw, p));
        return swc_check_launch(ctx, "fc_bf16_residual");
    }
    const int kblocks = (k + BK - 1) / BK;
    const Choice best = choose(m, n, kblocks, sms, sms < ctx->sm_count);
    p.bn = best.bn;
    p.splits = best.splits;
    p.tiles_m = (m + p.bn - 1) / p.bn;
    if (best.pair) {
        p.tiles_n = (n + 2 * BM - 1) / (2 * BM);
        SWC_REQUIRE(ctx, (long long)p.tiles_n * p.tiles_m < 0x7fffffff, SWCB200_ERR_TOO_LARGE, "fc_bf16_residual: too many tiles");
        p.band = ((size_t)n * k * 2 <= ((size_t)48 << 20) || p.tiles_n <= 8) ? p.tiles_n : 8;
        int rc = tmap_rows(ctx, wp_bf16, n, k, ldw, BM, &tmW);
        if (!rc) rc = tmap_rows(ctx, a_bf16, m, k, lda, p.bn / 2, &tmA);
        if (rc) return rc;
        SWC_CUDA(ctx, cudaFuncSetAttribute(fc_res_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPairSmem));
        const long long tiles = (long long)p.tiles_n * p.tiles_m, pairs = sms > 1 ? sms / 2 : 1;
        SWC_CUDA(ctx, swc_launch_early(fc_res_pair_kernel, 2u * (unsigned)(tiles < pairs ? tiles : pairs), kPairThreads, kPairSmem,
                                       ctx->stream, 1, tmW, tmA, p));
        return swc_check_launch(ctx, "fc_bf16_residual");
    }
    p.tiles_n = (n + BM - 1) / BM;
    SWC_REQUIRE(ctx, (long long)p.tiles_n * p.tiles_m < 0x7fffffff / 8, SWCB200_ERR_TOO_LARGE, "fc_bf16_residual: too many tiles");
    // the ring: as deep as the CTA's k range and shared memory allow, and never smaller than the join's slots
    const int sub = p.bn > 128 ? 1 : 2;
    const int stage = sub * (W_BYTES + p.bn * BK * 2);
    const int most = (kblocks + sub * p.splits - 1) / (sub * p.splits), fit = (kSplitSmem - 1280) / stage;
    p.stages = most < fit ? most : fit;
    const int slots = p.splits > 1 ? BM * p.bn * 4 : 0;
    if (p.stages * stage < slots) p.stages = (slots + stage - 1) / stage;
    int rc = tmap_rows(ctx, wp_bf16, n, k, ldw, BM, &tmW);
    if (!rc) rc = tmap_rows(ctx, a_bf16, m, k, lda, p.bn, &tmA);
    if (rc) return rc;
    const size_t smem = (size_t)p.stages * stage + 1280;
    const auto kernel = sub == 1 ? fc_res_split_kernel<1> : fc_res_split_kernel<2>;
    SWC_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSplitSmem));
    SWC_CUDA(ctx, swc_launch_early(kernel, (unsigned)((long long)p.tiles_n * p.tiles_m * p.splits), kSplitThreads, smem, ctx->stream,
                                   (unsigned)p.splits, tmW, tmA, p));
    return swc_check_launch(ctx, "fc_bf16_residual");
}
