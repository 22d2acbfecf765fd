// Attention of whole prompts on the 5th-generation tensor cores, one pass over the keys with the running maximum and sum of the
// softmax:
//     s_ij = scale * q_i . k_j;   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)
//
// A CTA holds two tiles of 128 query rows and walks the keys in blocks of 128.  Rows of a tile are (token, head) pairs of `pack`
// heads that read the same key head, so one block of keys serves the whole group.
//   * warps 0-3 and 4-7: softmax of tile 0 and 1, a thread per row (a lane of tensor memory).  Scores come from tensor memory
//     into registers, go back as bf16 weights over the same columns, and are the A operand of the second product there; scores
//     and weights never pass through shared memory.  The output's rescaling to a new maximum is done by the same threads and
//     only when the maximum has grown by more than 2^kSlack.
//   * warp 8: issues the products.  The order QK0 QK1 | PV0 QK0' | PV1 QK1' | ... keeps the pipe on one tile while the other
//     tile's softmax runs.
//   * warp 9: TMA loads: both query tiles once, then K and V blocks into a ring.
// Tensor memory: scores 2 x 128 columns, outputs 2 x 128 columns, all 512.  Head widths up to 64 use one 128-byte chunk per row,
// up to 128 two; TMA fills the rest with zeros.
// What bounds it: at width 128 a block of a tile costs 1024 cycles of tensor pipe and as many of the exponential unit (16 per
// cycle); at width 64 the exponentials alone take twice the pipe's time.
#include "attention_common.cuh"

namespace {

using namespace tc;
using namespace attn;

constexpr int kKeys = 128;   // keys per block
constexpr int kRows = 128;   // rows per tile
constexpr int kThreads = 384;
constexpr int kChunk = kKeys * 128;  // bytes of one 64-wide chunk of a block or tile

template <int CH> struct Shape {
    static constexpr int kStages = CH == 2 ? 5 : 8;
    static constexpr int kBlock = CH * kChunk;  // bytes of a K or V block, and of a query tile
    static constexpr size_t kSmem = 2 * kBlock + (size_t)kStages * kBlock + 1024 + 256;
};

// 32 lanes x 32 columns from registers
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
        "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D (+)= A[tmem] . B[smem]: the weights are the A operand in tensor memory
__device__ __forceinline__ void umma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        :
        : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// V as the B operand: columns of the product (d) are contiguous, keys are rows of 128 bytes, 8 keys 1024 bytes apart (stride
// offset), the second chunk of 64 columns kChunk bytes further (leading offset)
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFF) >> 4) | ((uint64_t)(kChunk >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

// a whole warp waits, and gives up together
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, int *status, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code));
}

template <int CH>
__global__ void __launch_bounds__(kThreads, 1)
attention_prompt_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const Params p, int tiles, int parts) {
    using Sh = Shape<CH>;
    constexpr int kStages = Sh::kStages, kBlock = Sh::kBlock;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = smem + 2 * kBlock;
    uint64_t *full = reinterpret_cast<uint64_t *>(ring + kStages * kBlock);
    uint64_t *empty = full + kStages;
    uint64_t *q_full = empty + kStages;
    uint64_t *s_full = q_full + 1;  // [2] scores of a tile are in tensor memory
    uint64_t *p_full = s_full + 2;  // [2] its weights are
    uint64_t *o_full = p_full + 2;  // [2] the tile's last product with V is complete
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(o_full + 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // blocks of the grid: heads fastest, the last tiles (causal: the longest) first
    const int unit = blockIdx.x % p.units;
    const int part = (blockIdx.x / p.units) % parts;
    Seq seq;
    int tile;
    const int per_cta = 2 * p.tokens;
    if (!find_seq(p, tiles - 1 - (int)(blockIdx.x / (p.units * parts)), [&](const Seq &s) { return (s.nq + per_cta - 1) / per_cta; }, seq,
                  tile))
        return;
    // key blocks of each tile, and of this part
    const int t0 = tile * per_cta;
    int blocks[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int first = t0 + h * p.tokens, last = min(first + p.tokens, seq.nq) - 1;
        blocks[h] = first < seq.nq ? (visible(p, seq, last) + kKeys - 1) / kKeys : 0;
    }
    const int most = max(blocks[0], blocks[1]);
    const int j0 = (int)((long long)most * part / parts), j1 = (int)((long long)most * (part + 1) / parts);
    const int n0 = max(min(blocks[0], j1) - j0, 0), n1 = max(min(blocks[1], j1) - j0, 0);
    const int n_all = max(n0, n1);

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        for (int s = 0; s < kStages; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(q_full, 1);
        for (int h = 0; h < 2; h++) {
            mbar_init(&s_full[h], 1);
            mbar_init(&p_full[h], 4);
            mbar_init(&o_full[h], 1);
        }
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 8) {
        tmem_alloc(tmem_holder, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;
    bool failed = false;

    // registers: 384 x 168 at launch = 256 x 216 for the softmax + 128 x 72
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 9) {
            // ------------------------------------------------------------ loads
            if (lane == 0 && n_all > 0) {
                const int head_k = unit * p.pack / p.group;
                const int tile_bytes = p.tokens * p.pack * 128;  // bytes of a chunk's box
                mbar_expect_tx(q_full, (uint32_t)((n0 > 0) + (n1 > 0)) * CH * tile_bytes);
                for (int h = 0; h < 2; h++)
                    if ((h ? n1 : n0) > 0)
                        for (int c = 0; c < CH; c++)
                            tma_load_3d(smem + h * kBlock + c * kChunk, &tmQ, q_full, c * 64, unit * p.pack, seq.q0 + t0 + h * p.tokens);
                int st = 0;
                uint32_t ph = 0;
                bool ok = true;
                for (int i = 0; i < 2 * n_all && ok; i++) {  // K and V blocks in turn
                    ok = mbar_wait(&empty[st], ph ^ 1, p.status, kWaitEmpty);
                    if (!ok) break;
                    mbar_expect_tx(&full[st], kBlock);
                    for (int c = 0; c < CH; c++)
                        tma_load_3d(ring + st * kBlock + c * kChunk, i & 1 ? &tmV : &tmK, &full[st], c * 64, head_k,
                                    seq.k0 + (j0 + (i >> 1)) * kKeys);
                    if (++st == kStages) {
                        st = 0;
                        ph ^= 1;
                    }
                }
                failed = !ok;
            }
        } else if (warp == 8) {
            // ------------------------------------------------------------ products
            const int dk = (p.d + 15) / 16;
            const uint32_t idesc_s = idesc_bf16_f32(kRows, kKeys);
            const uint32_t idesc_o = idesc_bf16_f32(kRows, dk * 16) | (1u << 16);  // B: columns contiguous
            const uint64_t dq[2] = {smem_desc_sw128(smem_u32(smem)), smem_desc_sw128(smem_u32(smem + kBlock))};
            bool ok = n_all > 0;
            if (ok) ok = warp_wait(q_full, 0, p.status, kWaitFull);
            int st = 0;
            uint32_t ph = 0;
            const auto next = [&] {
                if (++st == kStages) {
                    st = 0;
                    ph ^= 1;
                }
            };
            const auto scores = [&](int h, int stage) {
                const uint64_t dkey = smem_desc_sw128(smem_u32(ring + stage * kBlock));
                for (int s = 0; s < dk; s++) {
                    const uint64_t off = (uint64_t)((s >> 2) * (kChunk >> 4) + (s & 3) * 2);
                    umma_bf16(tmem + h * kKeys, dq[h] + off, dkey + off, idesc_s, (uint32_t)(s != 0));
                }
                umma_commit(&s_full[h]);
            };
            if (ok) ok = warp_wait(&full[st], ph, p.status, kWaitFull);
            if (ok) {
                tc_fence_after();
                if (lane == 0) {
                    if (n0 > 0) scores(0, st);
                    if (n1 > 0) scores(1, st);
                    umma_commit(&empty[st]);
                }
                next();
            }
            for (int j = 0; j < n_all && ok; j++) {
                ok = warp_wait(&full[st], ph, p.status, kWaitFull);  // V of block j
                if (!ok) break;
                const int stage_v = st;
                next();
                const int stage_k = st;
                if (j + 1 < n_all) {
                    ok = warp_wait(&full[st], ph, p.status, kWaitFull);  // K of block j + 1
                    if (!ok) break;
                    next();
                }
                // The second product runs over whole groups of 16 keys.  Keys of the last group past the sequence have weight 0, but
                // V there is another sequence's or nobody's, and 0 times infinity or NaN is not 0: those rows are cleared.
                const int keys = min(seq.nk - (j0 + j) * kKeys, kKeys), steps = (keys + 15) / 16;
                if (keys & 15) {
                    uint4 *v = reinterpret_cast<uint4 *>(ring + stage_v * kBlock);
                    const int count = (steps * 16 - keys) * 8;
                    for (int c = 0; c < CH; c++)
                        for (int i = lane; i < count; i += 32) v[c * (kChunk / 16) + keys * 8 + i] = make_uint4(0, 0, 0, 0);
                    fence_proxy_async();
                    __syncwarp();
                }
                for (int h = 0; h < 2 && ok; h++) {
                    const int n = h ? n1 : n0;
                    if (j >= n) continue;
                    ok = warp_wait(&p_full[h], j & 1, p.status, kWaitTmemEmpty);
                    if (!ok) break;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint64_t dv = desc_v(smem_u32(ring + stage_v * kBlock));
                        for (int s = 0; s < steps; s++)
                            umma_bf16_ts(tmem + 256 + h * 128, tmem + h * kKeys + s * 8, dv + s * (16 * 128 >> 4), idesc_o,
                                         (uint32_t)(j != 0 || s != 0));
                        if (j + 1 < n)
                            scores(h, stage_k);
                        else
                            umma_commit(&o_full[h]);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (lane == 0) {
                    umma_commit(&empty[stage_v]);
                    if (j + 1 < n_all) umma_commit(&empty[stage_k]);
                }
            }
            failed = n_all > 0 && !ok;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ------------------------------------------------------------ softmax, a row per thread
        const int h = warp >> 2, n = h ? n1 : n0;
        const int row = threadIdx.x & 127;
        const int tok = row / p.pack, head = unit * p.pack + (row - tok * p.pack);
        const int t = t0 + h * p.tokens + tok;  // token inside the sequence
        const bool valid = tok < p.tokens && t < seq.nq;
        const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t t_s = lane_base + h * kKeys, t_o = lane_base + 256 + h * 128;
        const int sees = visible(p, seq, min(t, seq.nq - 1)) - j0 * kKeys;  // keys of this part that the row sees
        const int all_see = visible(p, seq, t0 + h * p.tokens) - j0 * kKeys;
        float m = -INFINITY, l = 0.f;  // the maximum that the weights are relative to (raw scores), and their sum
        bool ok = true;
        for (int j = 0; j < n; j++) {
            ok = warp_wait(&s_full[h], j & 1, p.status, kWaitTmemFull);
            if (!ok) break;
            tc_fence_after();
            float s[kKeys];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld_32x32(t_s + c * 32, reinterpret_cast<uint32_t(&)[32]>(s[c * 32]));
            tmem_ld_wait();
            if ((j + 1) * kKeys > all_see) {
#pragma unroll
                for (int c = 0; c < kKeys; c++) s[c] = j * kKeys + c < sees ? s[c] : -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int c = 1; c < kKeys; c++) mx = fmaxf(mx, s[c]);
            float factor = 1.f;
            if ((mx - m) * p.scale_log2 > kSlack) {  // also where m is -inf; not where mx is (NaN compares false)
                factor = exp2_fast((m - mx) * p.scale_log2);
                m = mx;
            }
            if (__any_sync(0xffffffffu, factor != 1.f)) {
                l *= factor;
                if (j > 0) {
                    // the product that wrote the output last was issued before these scores' and is complete with them
                    for (int c = 0; c < p.d; c += 32) {
                        uint32_t r[32];
                        tmem_ld_32x32(t_o + c, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; i++) r[i] = __float_as_uint(__uint_as_float(r[i]) * factor);
                        tmem_st_32x32(t_o + c, r);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.f : m * p.scale_log2;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t w[32];
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    const float a = exp2_fast(fmaf(s[c * 64 + 2 * i], p.scale_log2, -base));
                    const float b = exp2_fast(fmaf(s[c * 64 + 2 * i + 1], p.scale_log2, -base));
                    sum += a + b;
                    w[i] = pack_bf16(a, b);
                }
                tmem_st_32x32(t_s + c * 32, w);
            }
            l += sum;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[h]);
        }
        if (ok && n > 0) {
            ok = warp_wait(&o_full[h], 0, p.status, kWaitTmemFull);
            tc_fence_after();
        }
        if (ok) {
            const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // a NaN stays one
            const bool empty_row = !(l != 0.f);
            const size_t at = (size_t)(seq.q0 + t);
            if (parts > 1) {
                const size_t slot = ((size_t)part * p.total_q + at) * p.heads_q + head;
                float *dst = p.part_o + slot * p.d;
                for (int c = 0; c < p.d; c += 32) {
                    uint32_t r[32] = {};
                    if (n > 0) {
                        tmem_ld_32x32(t_o + c, r);
                        tmem_ld_wait();
                    }
                    if (valid) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            if (c + i < p.d)
                                *reinterpret_cast<float4 *>(dst + c + i) =
                                    empty_row ? make_float4(0, 0, 0, 0)
                                              : make_float4(__uint_as_float(r[i]) * inv, __uint_as_float(r[i + 1]) * inv,
                                                            __uint_as_float(r[i + 2]) * inv, __uint_as_float(r[i + 3]) * inv);
                    }
                }
                if (valid) p.part_lse[slot] = empty_row ? -INFINITY : fmaf(m, p.scale_log2, __log2f(l));
            } else {
                __nv_bfloat16 *dst = p.o + at * p.o_row + (size_t)head * p.o_head;
                for (int c = 0; c < p.d; c += 32) {
                    uint32_t r[32] = {};
                    if (n > 0) {
                        tmem_ld_32x32(t_o + c, r);
                        tmem_ld_wait();
                    }
                    if (valid) {
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            if (c + i >= p.d) break;
                            uint4 w = make_uint4(0, 0, 0, 0);
                            if (!empty_row) {
                                w.x = pack_bf16(__uint_as_float(r[i]) * inv, __uint_as_float(r[i + 1]) * inv);
                                w.y = pack_bf16(__uint_as_float(r[i + 2]) * inv, __uint_as_float(r[i + 3]) * inv);
                                w.z = pack_bf16(__uint_as_float(r[i + 4]) * inv, __uint_as_float(r[i + 5]) * inv);
                                w.w = pack_bf16(__uint_as_float(r[i + 6]) * inv, __uint_as_float(r[i + 7]) * inv);
                            }
                            *reinterpret_cast<uint4 *>(dst + c + i) = w;
                        }
                    }
                }
                if (valid && p.lse)
                    p.lse[at * p.heads_q + head] = empty_row ? -INFINITY : 0.69314718055994531f * fmaf(m, p.scale_log2, log2f(l));
            }
        }
        failed = !ok;
    }
    // A wait that gave up leaves copies possibly still in flight towards this CTA's shared memory: give them a bounded time to
    // land (the clean path needs none: every load was consumed).
    if (failed) {
        const long long since = clock64();
        while (clock64() - since < 4000000ll) {
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int CH>
int launch(swcb200_ctx *ctx, const Params &p, const CUtensorMap &tmQ, const CUtensorMap &tmK, const CUtensorMap &tmV, int tiles,
           int parts) {
    SWC_CUDA(ctx, cudaFuncSetAttribute(attention_prompt_kernel<CH>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<CH>::kSmem));
    attention_prompt_kernel<CH><<<(unsigned)tiles * p.units * parts, kThreads, Shape<CH>::kSmem, ctx->stream>>>(tmQ, tmK, tmV, p, tiles, parts);
    return swc_check_launch(ctx, "attention_bf16");
}

}  // namespace

int swc_attention_prompt(swcb200_ctx *ctx, Params &p, const CUtensorMap &tmQ, const CUtensorMap &tmK, const CUtensorMap &tmV, int tiles,
                         int parts) {
    return p.d > 64 ? launch<2>(ctx, p, tmQ, tmK, tmV, tiles, parts) : launch<1>(ctx, p, tmQ, tmK, tmV, tiles, parts);
}
