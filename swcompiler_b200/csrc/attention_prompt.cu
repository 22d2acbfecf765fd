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
//   * warps 8-11: finished outputs, divided by their sums and stored, while the softmax goes on with the next item.
//   * warp 12: issues the products.  The order QK0 QK1 | PV0 QK0' | PV1 QK1' | ... keeps the pipe on one tile while the other
//     tile's softmax runs; it goes on across work items, so the first scores of the next item are there when one ends.
//   * warp 13: TMA loads: query tiles when their last products have been issued, K and V blocks into a ring.
//   * warp 14: work items.  The grid has one block per item; a resident CTA takes over blocks that have not started yet (cluster
//     launch control), finds their sequence and hands the item to the other warps ahead of time.  Under an SM limit there is one
//     CTA for each SM, and they take the blocks by stride.
// Tensor memory: scores 2 x 128 columns, outputs 2 x 128 columns, all 512.  Head widths up to 64 use one 128-byte chunk per row,
// up to 128 two; TMA fills the rest with zeros.
// What bounds it: a block of a tile costs 1024 cycles of tensor pipe at width 128 (512 at 64) and 1024 of the exponential unit (16
// per cycle), but the two tiles together take some 3200 cycles per block: a tile's softmax (1900) and the products between two
// of them (1030) are a chain, as there is room for one block of scores per tile.  At width 128 and long prompts that is also
// where the power limit sets the clock: 16 heads, 4 key heads, 16384 keys, causal: 857 us in a burst, 1283 TFLOP/s, 0.80 of the burst
// bf16 rate measured here, and 982 us in calls that go on for seconds (1.63 GHz), 0.84 of the sustained one; width 64: 764 us.
// Prompts of a few hundred tokens spend as long at the items' ends as in between: 64 sequences of 197, 16 heads of 64: 46 to 56 us
// from one process to the next, 0.28 to 0.35 of the bytes' rate.  There the softmax runs its first and
// masked blocks, whose code the warps do not have at hand (a fifth of their time went to waiting for instructions; a block took 2600
// to 5200 cycles instead of 1900), while the output warps turn the item before around.  So what nobody needs is left out (tiles
// without rows, warps whose rows are nobody's, the last quarter of a block that is seen half: 64 sequences of 128 keys of width 64,
// 38 -> 31 us), and there is less code: the output warps' loop over the two tiles is rolled, and in the form for short prompts
// (kShort) also that of the issuing warp, and an item's first block goes through the loop of the others (-> 29 us).
// Weights are rounded to bf16 for the second product, as their tensor's type has to be that of V: about as much as the bf16 result is
// rounded itself (1.9e-3 to 2.3e-3 of the result, root mean square, against 64 bits; 1.5e-3 to 1.7e-3 with weights of 32 bits).  Two
// bf16 terms would cost half as many products again.
// Measured and not kept: scores of blocks of 64 keys two ahead (the instructions around twice as many blocks cost what the chain
// does), an issuing warp per tile (the tiles fall into step: 1088 us).
#include "attention_common.cuh"

namespace {

using namespace tc;
using namespace attn;

constexpr int kKeys = 128;   // keys per block
constexpr int kRows = 128;   // rows per tile
constexpr int kThreads = 512;
constexpr int kChunk = kKeys * 128;  // bytes of one 64-wide chunk of a block or tile

constexpr int kPatch = 32 * 128;       // an output warp's rows of 128 bytes on their way out

template <int CH> struct Shape {
    static constexpr int kStages = CH == 2 ? 4 : 8;
    static constexpr int kBlock = CH * kChunk;  // bytes of a K or V block, and of a query tile
    static constexpr size_t kSmem = 2 * kBlock + (size_t)kStages * kBlock + 4 * kPatch + 1024 + 512;
};

// 32 lanes x 16 columns from registers
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D (+)= A[tmem] . B[smem]: the weights are the A operand in tensor memory; V is the B operand with its columns (d) contiguous, keys
// as rows of 128 bytes, and the second chunk of 64 columns kChunk bytes behind the first (the leading offset of its descriptor)
__device__ __forceinline__ void umma_output(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(kDescHigh), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

// Two fp32 at a time (one instruction for both)
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// maximum of three, NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The weights of 32 keys of a row: powers of two of s * scale - base, as bf16 pairs into tensor memory; their sum is added to l.
// (The exponential unit gives 16 values per cycle and SM; a part of them on the FMA pipe, by a polynomial of degree 3, was measured
// and is slower at every share: 905 us without against 941 with a quarter of them, 16384 keys of width 128.)
__device__ __forceinline__ void weights(const float *s, uint64_t scale, uint64_t minus_base, uint32_t t_p, uint64_t &l) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        float2 e = unpair(fma2(pair(s[2 * i], s[2 * i + 1]), scale, minus_base));
        e = make_float2(exp2_fast(e.x), exp2_fast(e.y));
        l = add2(l, pair(e.x, e.y));
        w[i] = pack_bf16(e.x, e.y);
    }
    tmem_st_32x16(t_p, w);
}

// the largest of kCount scores, NaN if one is
template <int kCount> __device__ __forceinline__ float largest(const float *s) {
    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
    for (int c = 4; c + 8 <= kCount; c += 8)
#pragma unroll
        for (int i = 0; i < 4; i++) mx[i] = max3(mx[i], s[c + i], s[c + 4 + i]);
    const float a = max3(mx[0], s[kCount - 4], s[kCount - 3]), b = max3(mx[1], s[kCount - 2], s[kCount - 1]);
    return max3(max3(a, b, mx[2]), mx[3], mx[3]);
}

// What a row's weights are relative to: a weight is 2^(s * scale - base).  base is m * scale for the maximum m, rounded; `off` is what
// the rounding left, so a score of m has the weight 2^off.  For products of 2^30 and more that alone would leave the range of fp32;
// there a smaller scale keeps the product at 2^30, where scores one step of fp32 apart still have weights 2^64 apart.  (A
// difference s - m per score is as good, and took 2 % longer; this takes 0.7 %: 16384 keys 850 -> 857 us.)
struct Reference {
    float scale, base, off;
};
__device__ __forceinline__ Reference relative_to(float m, float scale) {
    if (m == -INFINITY) return {scale, 0.f, 0.f};
    float top;  // 2^30 / |m|
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(top) : "f"(fabsf(m) * 0x1p-30f));
    scale = fminf(scale, top);
    const float base = m * scale;
    return {scale, base, fmaf(m, scale, -base)};
}

// Takes over a block of the grid that has not started: 16 bytes of answer land at `result`, counted on `bar`.
__device__ __forceinline__ void steal_block(uint4 *result, uint64_t *bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(result)),
                 "r"(smem_u32(bar))
                 : "memory");
}
// the block's number, or -1: none is left
__device__ __forceinline__ int stolen_block(const uint4 *result) {
    uint32_t ok, x;
    asm volatile(
        "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t.reg .b64 lo, hi;\n\t"
        "ld.shared.v2.b64 {lo, hi}, [%2];\n\t"
        "mov.b128 h, {lo, hi};\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
        : "=r"(ok), "=r"(x)
        : "r"(smem_u32(result))
        : "memory");
    return ok ? (int)x : -1;
}

// One work item: two tiles of rows against a range of key blocks.
struct Item {
    Seq seq;
    int t0;      // first token of tile 0
    int unit, part;
    int j0;      // first key block
    int n0, n1;  // key blocks of each tile
    int sees0, sees1;  // keys, from block j0 on, that a row of each tile sees at most
    int valid;   // 0: no more items
    __device__ __forceinline__ int n(int h) const { return h ? n1 : n0; }
    __device__ __forceinline__ int sees(int h) const { return h ? sees1 : sees0; }
    __device__ __forceinline__ int most() const { return max(n0, n1); }
};
constexpr int kSlots = 2;
constexpr int kItemReaders = 14;  // warps: softmax 8, output 4, products, loads

__device__ __forceinline__ bool make_item(const Params &p, int block, int parts, Item &it) {
    // blocks of the grid: heads fastest, sequences in turn, of each the last tiles (causal: the longest) first
    it.unit = block % p.units;
    it.part = (block / p.units) % parts;
    int tile;
    const int per_cta = 2 * p.tokens;
    if (!find_seq(p, block / (p.units * parts), [&](const Seq &s) { return (s.nq + per_cta - 1) / per_cta; }, it.seq, tile))
        return false;
    it.t0 = ((it.seq.nq + per_cta - 1) / per_cta - 1 - tile) * per_cta;
    const auto last_sees = [&](int first) {  // the last row of a tile sees the most
        return first < it.seq.nq ? visible(p, it.seq, min(first + p.tokens, it.seq.nq) - 1) : 0;
    };
    const int v0 = last_sees(it.t0), v1 = last_sees(it.t0 + p.tokens);
    const int b0 = (v0 + kKeys - 1) / kKeys, b1 = (v1 + kKeys - 1) / kKeys, most = max(b0, b1);
    it.j0 = (int)((long long)most * it.part / parts);
    const int j1 = (int)((long long)most * (it.part + 1) / parts);
    it.n0 = max(min(b0, j1) - it.j0, 0);
    it.n1 = max(min(b1, j1) - it.j0, 0);
    it.sees0 = v0 - it.j0 * kKeys;
    it.sees1 = v1 - it.j0 * kKeys;
    it.valid = 1;
    return true;
}

// kStrided: for a grid of fewer CTAs than blocks.  (Compiled apart: a branch in the others cost them 1 %.)
template <int CH, bool kShort, bool kStrided>
__global__ void __launch_bounds__(kThreads, 1)
attention_prompt_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const Params p, int parts, int blocks) {
    using Sh = Shape<CH>;
    constexpr int kStages = Sh::kStages, kBlock = Sh::kBlock;
    constexpr int kTileUnroll = kShort ? 1 : 2;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Item s_items[kSlots];
    __shared__ alignas(16) uint4 s_stolen;
    __shared__ float2 s_stat[2][kRows];  // of a finished row: sum of its weights, and the maximum they are relative to
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = smem + 2 * kBlock;
    uint8_t *patches = ring + kStages * kBlock;
    uint64_t *full = reinterpret_cast<uint64_t *>(patches + 4 * kPatch);
    uint64_t *empty = full + kStages;
    uint64_t *q_full = empty + kStages;   // [2] a query tile has landed
    uint64_t *q_empty = q_full + 2;       // [2] its last products have read it
    uint64_t *s_full = q_empty + 2;       // [2] scores of a tile are in tensor memory
    uint64_t *p_half = s_full + 2;        // [2] the weights of its first 64 keys are
    uint64_t *p_full = p_half + 2;        // [2] all weights are
    uint64_t *o_full = p_full + 2;        // [2] the tile's last product with V is complete
    uint64_t *o_empty = o_full + 2;       // [2] its output has been read
    uint64_t *stat_full = o_empty + 2;    // [2] s_stat of a tile is written
    uint64_t *stat_empty = stat_full + 2; // [2] and read
    uint64_t *item_full = stat_empty + 2; // [kSlots]
    uint64_t *item_empty = item_full + kSlots;
    uint64_t *stolen = item_empty + kSlots;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(stolen + 1);

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;  // warp: known to be uniform
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        for (int s = 0; s < kStages; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int h = 0; h < 2; h++) {
            mbar_init(&q_full[h], 1);
            mbar_init(&q_empty[h], 1);
            mbar_init(&s_full[h], 1);
            mbar_init(&p_half[h], 4);
            mbar_init(&p_full[h], 4);
            mbar_init(&o_full[h], 1);
            mbar_init(&o_empty[h], 4);
            mbar_init(&stat_full[h], 4);
            mbar_init(&stat_empty[h], 4);
        }
        for (int s = 0; s < kSlots; s++) {
            mbar_init(&item_full[s], 1);
            mbar_init(&item_empty[s], kItemReaders);
        }
        mbar_init(stolen, 1);
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 12) {
        tmem_alloc(tmem_holder, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    // A block that gave up on a wait has recorded it: blocks that start after that do not wait in their turn.
    const bool given_up = __syncthreads_or(*reinterpret_cast<const volatile int *>(p.status) != 0);
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_holder, 0);
    bool failed = false;
    if (given_up) {
        if (warp == 12) tmem_dealloc(tmem, 512);
        return;
    }

    // The items in turn, for every reader alike: slot and phase follow from the count.
    uint32_t items = 0;
    const auto next_item = [&](Item &it) {  // false: no more, or a wait ran out (`failed`)
        const uint32_t slot = items % kSlots, phase = (items / kSlots) & 1;
        items++;
        if (!warp_wait(&item_full[slot], phase, p.status, kWaitFull)) {
            failed = true;
            return false;
        }
        it = s_items[slot];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[slot]);
        return it.valid != 0;
    };

    // registers: 512 x 128 at launch = 256 x 192 for the softmax + 128 x 72 for the output + 128 x 56
    if (warp >= 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 14) {
            // ------------------------------------------------------------ work items
            int block = blockIdx.x;
            uint32_t count = 0, asked = 0;
            while (!failed) {
                if (lane == 0 && !kStrided) {  // ask for the block after this one
                    fence_proxy_async();
                    mbar_expect_tx(stolen, 16);
                    steal_block(&s_stolen, stolen);
                }
                Item it;
                if (make_item(p, block, parts, it)) {  // (the grid is an upper bound of the tiles there are)
                    const uint32_t slot = count % kSlots, phase = (count / kSlots) & 1;
                    count++;
                    if (!warp_wait(&item_empty[slot], phase ^ 1, p.status, kWaitEmpty)) failed = true;
                    if (lane == 0 && !failed) {
                        s_items[slot] = it;
                        mbar_arrive(&item_full[slot]);
                    }
                    __syncwarp();
                }
                if constexpr (kStrided) {
                    if (blocks - block <= (int)gridDim.x) break;
                    block += gridDim.x;
                    continue;
                }
                if (!warp_wait(stolen, asked++ & 1, p.status, kWaitFull)) failed = true;
                block = stolen_block(&s_stolen);
                __syncwarp();
                if (block < 0) break;
            }
            if (!failed) {
                const uint32_t slot = count % kSlots, phase = (count / kSlots) & 1;
                if (!warp_wait(&item_empty[slot], phase ^ 1, p.status, kWaitEmpty)) failed = true;
                if (lane == 0 && !failed) {
                    s_items[slot].valid = 0;
                    mbar_arrive(&item_full[slot]);
                }
            }
        } else if (warp == 13) {
            // ------------------------------------------------------------ loads
            const int tile_bytes = p.tokens * p.pack * 128;  // bytes of a chunk's box
            int st = 0;
            uint32_t ph = 0, tiles_done[2] = {0, 0};
            Item it;
            while (!failed && next_item(it)) {
                const int head_k = it.unit * p.pack / p.group, n_all = it.most();
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (it.n(h) == 0 || failed) continue;
                    if (!warp_wait(&q_empty[h], (tiles_done[h]++ & 1) ^ 1, p.status, kWaitEmpty)) failed = true;
                    if (lane == 0 && !failed) {
                        mbar_expect_tx(&q_full[h], CH * tile_bytes);
                        for (int c = 0; c < CH; c++)
                            tma_load_3d(smem + h * kBlock + c * kChunk, &tmQ, &q_full[h], c * 64, it.unit * p.pack,
                                        it.seq.q0 + it.t0 + h * p.tokens);
                    }
                }
                for (int i = 0; i < 2 * n_all && !failed; i++) {  // K and V blocks in turn
                    if (!warp_wait(&empty[st], ph ^ 1, p.status, kWaitEmpty)) failed = true;
                    if (lane == 0 && !failed) {
                        mbar_expect_tx(&full[st], kBlock);
                        for (int c = 0; c < CH; c++)
                            tma_load_3d(ring + st * kBlock + c * kChunk, i & 1 ? &tmV : &tmK, &full[st], c * 64, head_k,
                                        it.seq.k0 + (it.j0 + (i >> 1)) * kKeys);
                    }
                    __syncwarp();
                    if (++st == kStages) {
                        st = 0;
                        ph ^= 1;
                    }
                }
            }
        } else if (warp == 12) {
            // ------------------------------------------------------------ products
            // This warp shares its scheduler with two softmax warps, and what it executes beside the products idles the tensor pipe:
            // whole blocks in the middle of an item take a path without conditions.  The operands of an instruction have to be the
            // same in all lanes, and known to be by the compiler (what comes from shared memory is spread from lane 0): otherwise
            // each took 110 to 160 cycles to issue.
            const int dk = (p.d + 15) / 16;
            const uint32_t idesc_o = idesc_bf16_f32(kRows, dk * 16) | (1u << 16);  // B: columns contiguous
            const uint32_t q_lo = desc_low(smem_u32(smem), 16), ring_k = desc_low(smem_u32(ring), 16), ring_v = desc_low(smem_u32(ring), kChunk);
            struct Work {
                int n0, n1, sees0, sees1, keys;  // key blocks of each tile, keys it sees, keys there are
                __device__ __forceinline__ int n(int h) const { return h ? n1 : n0; }
                __device__ __forceinline__ int sees(int h) const { return h ? sees1 : sees0; }
                __device__ __forceinline__ int most() const { return max(n0, n1); }
            };
            const auto next_work = [&](Work &w) {
                Item it;
                bool any;
                do any = next_item(it);
                while (any && it.most() == 0);
                w.n0 = __shfl_sync(0xffffffffu, it.n0, 0);
                w.n1 = __shfl_sync(0xffffffffu, it.n1, 0);
                w.sees0 = __shfl_sync(0xffffffffu, it.sees0, 0);
                w.sees1 = __shfl_sync(0xffffffffu, it.sees1, 0);
                w.keys = __shfl_sync(0xffffffffu, it.seq.nk - it.j0 * kKeys, 0);
                return any;
            };
            int st = 0;
            uint32_t ph = 0, blocks_done = 0, tiles_q = 0, tiles_o = 0;  // phases, a bit per tile
            const auto wait = [&](uint64_t *bar, uint32_t parity, int code) {
                if (!failed && !warp_wait(bar, parity, p.status, code)) failed = true;
            };
            const auto take_stage = [&] {  // the next K or V block of the ring
                wait(&full[st], ph, kWaitFull);
                const int s = st;
                if (++st == kStages) {
                    st = 0;
                    ph ^= 1;
                }
                return s;
            };
            // scores of tile h for block j of an item
            const auto scores = [&](const Work &w, int h, int j, int stage) {
                if (j >= w.n(h)) return;
                if (j == 0) {
                    wait(&q_full[h], tiles_q >> h & 1, kWaitFull);
                    tiles_q ^= 1u << h;
                }
                tc_fence_after();
                const uint32_t idesc_s = idesc_bf16_f32(kRows, min((w.sees(h) - j * kKeys + 15) & ~15, kKeys));  // keys that are seen
                if (!failed && elect_one()) {
                    const uint32_t dq = q_lo + h * (kBlock >> 4), dkey = ring_k + stage * (kBlock >> 4);
#pragma unroll
                    for (int s = 0; s < CH * 4; s++) {
                        const uint32_t off = (s >> 2) * (kChunk >> 4) + (s & 3) * 2;
                        if (s < dk) umma_bf16_words(tmem + h * kKeys, dq + off, dkey + off, idesc_s, s != 0);
                    }
                    umma_commit(&s_full[h]);
                    if (j + 1 == w.n(h)) umma_commit(&q_empty[h]);
                }
                __syncwarp();
            };
            Work now, after;
            bool more = next_work(now);
            if (more) {
                const int stage = take_stage();
                scores(now, 0, 0, stage);
                scores(now, 1, 0, stage);
                if (!failed && elect_one()) umma_commit(&empty[stage]);
                __syncwarp();
            }
            int j = 0;
            while (more && !failed) {
                // what comes next: the item's next block, or the first one of the next item that has any
                const bool last = j + 1 == now.most();
                const int j_next = last ? 0 : j + 1;
                after = now;
                if (last) more = next_work(after);
                const int stage_v = take_stage();
                int stage_k = -1;  // taken when it is needed: behind the first tile's weights
                // The second product runs over whole groups of 16 keys, as far as some row of the tile sees.  Keys of the last group
                // past the sequence have weight 0, but V there is another sequence's or nobody's, and 0 times infinity or NaN is
                // not 0: those rows are cleared.
                const int keys = min(now.keys - j * kKeys, kKeys);
                if (keys & 15) {
                    uint4 *v = reinterpret_cast<uint4 *>(ring + stage_v * kBlock);
                    const int count = (16 - (keys & 15)) * 8;
                    for (int c = 0; c < CH; c++)
                        for (int i = lane; i < count; i += 32) v[c * (kChunk / 16) + keys * 8 + i] = make_uint4(0, 0, 0, 0);
                    fence_proxy_async();
                    __syncwarp();
                }
                const uint32_t dv = ring_v + stage_v * (kBlock >> 4);
#pragma unroll kTileUnroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t t_s = tmem + h * kKeys, t_o = tmem + 256 + h * 128;
                    const uint32_t parity = blocks_done >> h & 1;
                    if (j + 1 < now.n(h) && dk == CH * 4) {
                        blocks_done ^= 1u << h;
                        if (j == 0) {
                            wait(&o_empty[h], tiles_o >> h & 1 ^ 1, kWaitTmemEmpty);
                            tiles_o ^= 1u << h;
                        }
                        wait(&p_half[h], parity, kWaitTmemEmpty);
                        tc_fence_after();
                        if (!failed && elect_one()) {
#pragma unroll
                            for (int s = 0; s < kKeys / 32; s++)
                                umma_output(t_o, t_s + s * 8, dv + s * (16 * 128 >> 4), idesc_o, s != 0 || j != 0);
                        }
                        __syncwarp();
                        if (stage_k < 0) stage_k = take_stage();
                        const uint32_t dkey = ring_k + stage_k * (kBlock >> 4);
                        wait(&p_full[h], parity, kWaitTmemEmpty);
                        tc_fence_after();
                        if (!failed && elect_one()) {
#pragma unroll
                            for (int s = kKeys / 32; s < kKeys / 16; s++)
                                umma_output(t_o, t_s + s * 8, dv + s * (16 * 128 >> 4), idesc_o, true);
#pragma unroll
                            for (int s = 0; s < CH * 4; s++) {
                                const uint32_t off = (s >> 2) * (kChunk >> 4) + (s & 3) * 2;
                                umma_bf16_words(t_s, q_lo + h * (kBlock >> 4) + off, dkey + off, idesc_bf16_f32(kRows, kKeys), s != 0);
                            }
                            umma_commit(&s_full[h]);
                            if (j + 2 == now.n(h)) umma_commit(&q_empty[h]);
                        }
                        __syncwarp();
                        continue;
                    }
                    if (j < now.n(h)) {
                        const int steps = (min(now.sees(h) - j * kKeys, kKeys) + 15) / 16;
                        blocks_done ^= 1u << h;
                        if (j == 0) {
                            wait(&o_empty[h], tiles_o >> h & 1 ^ 1, kWaitTmemEmpty);
                            tiles_o ^= 1u << h;
                        }
                        wait(&p_half[h], parity, kWaitTmemEmpty);
                        tc_fence_after();
                        if (!failed && elect_one()) {
#pragma unroll
                            for (int s = 0; s < kKeys / 32; s++)
                                if (s < steps) umma_output(t_o, t_s + s * 8, dv + s * (16 * 128 >> 4), idesc_o, s != 0 || j != 0);
                        }
                        __syncwarp();
                        wait(&p_full[h], parity, kWaitTmemEmpty);
                        tc_fence_after();
                        if (!failed && elect_one()) {
#pragma unroll
                            for (int s = kKeys / 32; s < kKeys / 16; s++)
                                if (s < steps) umma_output(t_o, t_s + s * 8, dv + s * (16 * 128 >> 4), idesc_o, true);
                            if (j + 1 == now.n(h)) umma_commit(&o_full[h]);
                        }
                        __syncwarp();
                    }
                    if (more) {
                        if (stage_k < 0) stage_k = take_stage();
                        scores(after, h, j_next, stage_k);
                    }
                }
                if (!failed && elect_one()) {
                    umma_commit(&empty[stage_v]);
                    if (stage_k >= 0) umma_commit(&empty[stage_k]);
                }
                __syncwarp();
                now = after;
                j = j_next;
            }
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // ------------------------------------------------------------ output, a row per thread and then a row per 8 lanes
        const int quarter = warp & 3, row = quarter * 32 + lane;
        const int tok = row * p.pack_inv >> 16, head_in = row - tok * p.pack;
        uint8_t *patch = patches + quarter * kPatch;
        uint32_t tiles_done = 0, items_done = 0;  // tiles_done: a bit per tile
        Item it;
        while (!failed && next_item(it)) {
#pragma unroll 1
            for (int h = 0; h < 2; h++) {
                const int n = it.n(h), first = it.t0 + h * p.tokens;
                const uint32_t t_o = tmem + ((uint32_t)(quarter * 32) << 16) + 256 + h * 128;
                if (!failed && !warp_wait(&stat_full[h], items_done & 1, p.status, kWaitTmemFull)) failed = true;
                const float2 stat = s_stat[h][row];
                __syncwarp();
                if (lane == 0) mbar_arrive(&stat_empty[h]);
                if (first >= it.seq.nq) continue;  // no rows, and n is 0
                if (!failed && n > 0 && !warp_wait(&o_full[h], tiles_done >> h & 1, p.status, kWaitTmemFull)) failed = true;
                if (failed) break;
                if (n > 0) tiles_done ^= 1u << h;
                tc_fence_after();
                const bool empty_row = stat.x == 0.f;  // nothing seen
                const float inv = 1.f / stat.x;
                // Rows leave through shared memory: a thread holds a row, and 32 rows in one store instruction are 32 lines of which
                // each gets 16 bytes; turned around, a row's 128 bytes come from 8 neighbouring lanes.  16-byte pieces, xor-ed with
                // the row against bank conflicts.
                const int columns = parts > 1 ? 32 : 64;  // of 4 and 2 bytes
                for (int c = 0; c < p.d; c += columns) {
#pragma unroll 1
                    for (int half = 0; half < columns; half += 16) {
                        uint32_t r[16] = {};
                        if (n > 0) {
                            tmem_ld_32x16(t_o + c + half, r);
                            tmem_ld_wait();
                        }
#pragma unroll
                        for (int i = 0; i < 16; i++) r[i] = empty_row ? 0u : __float_as_uint(__uint_as_float(r[i]) * inv);
                        const float *f = reinterpret_cast<const float *>(r);
                        if (parts > 1) {
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                *reinterpret_cast<uint4 *>(patch + lane * 128 + (((i + half / 4) ^ (lane & 7)) << 4)) =
                                    make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 2; i++)
                                *reinterpret_cast<uint4 *>(patch + lane * 128 + (((i + half / 8) ^ (lane & 7)) << 4)) =
                                    make_uint4(pack_bf16(f[8 * i], f[8 * i + 1]), pack_bf16(f[8 * i + 2], f[8 * i + 3]),
                                               pack_bf16(f[8 * i + 4], f[8 * i + 5]), pack_bf16(f[8 * i + 6], f[8 * i + 7]));
                        }
                    }
                    if (n > 0 && c + columns >= p.d) {  // the last of it: the next item's products may overwrite the output
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&o_empty[h]);
                    }
                    __syncwarp();
                    const int piece = lane & 7, column = c + piece * (columns / 8);
#pragma unroll 2
                    for (int i = 0; i < 8; i++) {
                        const int r = i * 4 + (lane >> 3), in_tile = quarter * 32 + r;
                        const int r_tok = in_tile * p.pack_inv >> 16, r_head = it.unit * p.pack + in_tile - r_tok * p.pack;
                        const uint4 v = *reinterpret_cast<const uint4 *>(patch + r * 128 + ((piece ^ (r & 7)) << 4));
                        if (r_tok >= p.tokens || first + r_tok >= it.seq.nq || column >= p.d) continue;
                        const size_t token = (size_t)(it.seq.q0 + first + r_tok);
                        if (parts > 1)
                            *reinterpret_cast<uint4 *>(p.part_o + (((size_t)it.part * p.total_q + token) * p.heads_q + r_head) * p.d + column) = v;
                        else
                            *reinterpret_cast<uint4 *>(p.o + token * p.o_row + (size_t)r_head * p.o_head + column) = v;
                    }
                    __syncwarp();
                }
                if ((parts > 1 || p.lse) && tok < p.tokens && first + tok < it.seq.nq) {
                    const float sum_log2 = empty_row ? -INFINITY : fmaf(stat.y, p.scale_log2, log2f(stat.x) - relative_to(stat.y, p.scale_log2).off);
                    const size_t token = (size_t)(it.seq.q0 + first + tok), head = (size_t)it.unit * p.pack + head_in;
                    if (parts > 1)
                        p.part_lse[((size_t)it.part * p.total_q + token) * p.heads_q + head] = sum_log2;
                    else
                        p.lse[token * p.heads_q + head] = 0.69314718055994531f * sum_log2;
                }
            }
            items_done++;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        // ------------------------------------------------------------ softmax, a row per thread
        const int h = warp >> 2;
        const int row = threadIdx.x & 127;
        const int tok = row * p.pack_inv >> 16;
        const uint32_t t_s = tmem + ((uint32_t)((warp & 3) * 32) << 16) + h * kKeys, t_o = t_s - h * kKeys + 256 + h * 128;
        uint32_t blocks_done = 0, tiles_done = 0;
        Item it;
        while (!failed && next_item(it)) {
            const int n = it.n(h);
            const int first = it.t0 + h * p.tokens, t = first + tok;  // token inside the sequence
            const int sees = visible(p, it.seq, min(t, it.seq.nq - 1)) - it.j0 * kKeys;  // keys of this part that the row sees,
            const int all_see = visible(p, it.seq, first) - it.j0 * kKeys;              // that every row of the tile sees,
            const int one_sees = it.sees(h);                                            // that some row of it sees
            const bool idle = !__any_sync(0xffffffffu, tok < p.tokens && t < it.seq.nq);  // no row of this warp is anybody's
            float m = -INFINITY;                                // the maximum that the weights are relative to (raw scores)
            Reference ref = relative_to(m, p.scale_log2);
            uint64_t l = pair(0.f, 0.f);    // the weights' sum
            for (int j = 0; j < n; j++) {
                if (!warp_wait(&s_full[h], blocks_done++ & 1, p.status, kWaitTmemFull)) {
                    failed = true;
                    break;
                }
                tc_fence_after();
                const int keys = one_sees - j * kKeys, mine = sees - j * kKeys;
                const bool whole = all_see - j * kKeys >= kKeys;
                float s[kKeys];
                const auto publish = [&](uint64_t *bar) {
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar);
                };
                if (idle) {
                    publish(&p_half[h]);
                    publish(&p_full[h]);
                    continue;
                }
                // a maximum that has grown: sums and output are brought to it
                const auto grow = [&](float top) {
                    float factor = 1.f;
                    if (!((top - m) * p.scale_log2 <= kSlack) && top != -INFINITY) {  // also where m is -inf, and where top is NaN: so is the row
                        const float off = ref.off;
                        ref = relative_to(top, p.scale_log2);
                        factor = exp2_fast(fmaf(m - top, ref.scale, ref.off - off));
                        m = top;
                    }
                    l = fma2(l, pair(factor, factor), pair(0.f, 0.f));
                    if (j == 0 || !__any_sync(0xffffffffu, factor != 1.f)) return;
                    // the product that wrote the output last was issued before these scores' and is complete with them
#pragma unroll 1
                    for (int c = 0; c < p.d; c += 16) {
                        uint32_t r[16];
                        tmem_ld_32x16(t_o + c, r);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) r[i] = __float_as_uint(__uint_as_float(r[i]) * factor);
                        tmem_st_32x16(t_o + c, r);
                    }
                };
                const auto scale = [&] { return pair(ref.scale, ref.scale); };
                const auto base = [&] { return pair(-ref.base, -ref.base); };
#pragma unroll
                for (int c = 0; c < 4; c++) tmem_ld_32x32(t_s + c * 32, reinterpret_cast<uint32_t(&)[32]>(s[c * 32]));
                tmem_ld_wait();
                if (!whole) {
#pragma unroll
                    for (int c0 = 0; c0 < kKeys; c0 += 32) {
                        const int left = mine - c0;
                        const uint32_t seen = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1 : 0u;
#pragma unroll
                        for (int c = 0; c < 32; c++) s[c0 + c] = seen & (1u << c) ? s[c0 + c] : -INFINITY;
                    }
                }
                if (!kShort && j == 0) grow(largest<kKeys>(s));
                // (kShort: an item's first block has no maximum yet and goes around twice, the first time for that alone.)
                // The first half's weights are taken relative to the maximum so far, while this block's is looked for: that is off the
                // path between the products, and rarely are they to be done again.
                uint64_t l_half;
#pragma unroll 1
                for (int pass = 0;; pass++) {
                    l_half = l;
                    const uint64_t b = base();
                    if (!kShort || j > 0 || pass > 0) weights(s, scale(), b, t_s, l_half);
                    const float top = largest<kKeys>(s);
                    if (!kShort || j > 0 || pass > 0) weights(s + 32, scale(), b, t_s + 16, l_half);
                    const bool stays = (!kShort || j > 0) && ((top - m) * p.scale_log2 <= kSlack || top == -INFINITY);
                    if (pass == 1 || __all_sync(0xffffffffu, stays)) break;
                    grow(top);
                }
                l = l_half;
                publish(&p_half[h]);
                if (keys > 64) {  // (weights of keys that no row of the tile sees are not multiplied either)
                    const uint64_t b = base();
                    weights(s + 64, scale(), b, t_s + 32, l);
                    if (keys > 96) weights(s + 96, scale(), b, t_s + 48, l);
                }
                publish(&p_full[h]);
            }
            if (failed || !warp_wait(&stat_empty[h], (tiles_done++ & 1) ^ 1, p.status, kWaitTmemEmpty)) {
                failed = true;
                break;
            }
            const float2 halves = unpair(l);
            s_stat[h][row] = make_float2(halves.x + halves.y, m);
            __syncwarp();
            if (lane == 0) mbar_arrive(&stat_full[h]);
        }
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
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int CH, bool kShort, bool kStrided = false>
int launch_form(swcb200_ctx *ctx, const Params &p, const CUtensorMap &tmQ, const CUtensorMap &tmK, const CUtensorMap &tmV, int parts,
                int blocks, int grid) {
    const auto kernel = attention_prompt_kernel<CH, kShort, kStrided>;
    SWC_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<CH>::kSmem));
    kernel<<<(unsigned)grid, kThreads, Shape<CH>::kSmem, ctx->stream>>>(tmQ, tmK, tmV, p, parts, blocks);
    return swc_check_launch(ctx, "attention_bf16");
}

template <int CH>
int launch(swcb200_ctx *ctx, const Params &p, const CUtensorMap &tmQ, const CUtensorMap &tmK, const CUtensorMap &tmV, int tiles,
           int parts) {
    // The form with less code up to 1024 keys per sequence: on average, as the lengths are on the device, and rows of a cache that are
    // not filled count as keys.  Short against long form, 16384 tokens in sequences of one length, 32
    // heads, 8 key heads of 128, causal: 256 keys 111 / 115 us, 512 136 / 153, 1024 185 / 198, 2048 297 / 289; 16384 keys, 16 heads,
    // 885 / 855.  Width 64, 16 heads, all keys: 64 sequences of 197 46 / 52 us, 32 of 1024 202 / 207 (all of these before the row's
    // Reference, which adds up to 1 %).  Under an SM limit the short one, whatever the length.
    const int blocks = tiles * p.units * parts, sms = swc_tc_sms(ctx);
    if (sms < ctx->sm_count && sms < blocks) return launch_form<CH, true, true>(ctx, p, tmQ, tmK, tmV, parts, blocks, sms);
    return p.total_k / p.batch <= 1024 ? launch_form<CH, true>(ctx, p, tmQ, tmK, tmV, parts, blocks, blocks)
                                       : launch_form<CH, false>(ctx, p, tmQ, tmK, tmV, parts, blocks, blocks);
}

}  // namespace

int swc_attention_prompt(swcb200_ctx *ctx, Params &p, const CUtensorMap &tmQ, const CUtensorMap &tmK, const CUtensorMap &tmV, int tiles,
                         int parts) {
    return p.d > 64 ? launch<2>(ctx, p, tmQ, tmK, tmV, tiles, parts) : launch<1>(ctx, p, tmQ, tmK, tmV, tiles, parts);
}
