// Attention of a few new tokens per sequence over long caches.  What bounds it is reading the keys and values once.
//
// Rows of a tile are (token, head) pairs of the heads that read one key head, 16, 32 or 64 of them, so the cache is read once
// for the whole group.  Work items are pieces of `part` keys of one sequence and key head (sequences of very different lengths
// make items of the same size); persistent CTAs take them in turn.  One warp finds the items and brings their query rows into
// shared memory, another one loads their keys and values; both run ahead of the products, so the ring of 64-key blocks does not
// drain between items.  Partial results of a sequence with several items go to the workspace and are joined
// by a second kernel, in a fixed order; a sequence of one item is written directly.
//
// With 16 rows the tensor cores are a side matter (a 128-row tcgen05 tile would be seven eighths padding), so each warp runs
// mma.sync m16n8k16 on 16 of a block's 64 keys with a softmax of its own in registers -- no barrier between warps until the end
// of an item, where the four key groups are merged.
//
// Weights go into the second product as bf16: its A operand has the type of B, the values.  That rounding (half a step is 2^-8 of a
// weight, and the sum is of the unrounded ones) is about as large as the one of the bf16 result: 2.3e-3 of the result, root mean
// square, against 64 bits, where weights of 32 bits would leave 1.7e-3.
//
// 32 heads, 8 key heads of 128, one token each: 64 caches of 4096 keys 171 us, 0.96 of the copy rate measured here; 64 ragged ones of up
// to 4096 keys 64 us, 0.72 (items are dealt out by stride, and CTAs end apart); one cache of 65536 keys 50 us with its join, 0.82.
// Slow by comparison: a sequence with more rows than fit the tile, which the AVERAGE number of rows sizes, has a CTA per row tile walk
// all of its keys (16 new tokens behind 65536 keys beside 63 single ones: 777 us, 44 would do for the bytes); 64 rows per tile of
// width 128 spill registers (64 caches of 2048 keys with 8 new tokens of 8 heads: 387 us, 85); thousands of sequences, as a search for
// an item passes over all sequences before it (4096 caches of 256 keys: 4.5 ms, 0.67; 1024 of 512: 433 us, 332).
#include "attention_common.cuh"

namespace {

using namespace tc;
using namespace attn;

constexpr int kKeys = 64;             // keys per block
constexpr int kChunk = kKeys * 128;   // bytes of a 64-wide chunk of a block

template <int CH, int RG> struct Shape {
    static constexpr int kStage = 2 * CH * kChunk;  // K and V of a block
    static constexpr int kCtas = RG == 1 ? 2 : 1;   // per SM
    static constexpr int kStages = RG == 1 ? (CH == 1 ? 4 : 2) : CH == 1 ? 8 : RG < 4 ? 5 : 3;
    static constexpr int kPitch = CH * 64 + 8;      // of a row that is being merged: 16-byte rows, spread over the banks
    static constexpr int kQPitch = CH * 128 + 16;   // bytes of a query row: likewise
    static constexpr int kQTile = RG * 16 * kQPitch;
    static constexpr size_t kSmem = (size_t)kStages * kStage + 1024 + 512 + (size_t)RG * 2 * 16 * kPitch * 4 + 2 * kQTile;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A barrier of `nthreads` threads that also says whether `ok` held for all of them.
__device__ __forceinline__ bool barrier_all(int id, int nthreads, bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %1, 0;\n\t"
        "bar.red.and.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"((uint32_t)ok), "r"(id), "r"(nthreads)
        : "memory");
    return all != 0;
}

// items of a sequence for one unit of heads: pieces of its keys where its rows fit one tile, else its row tiles
__device__ __forceinline__ int row_tiles(const Params &p, const Seq &s) { return (s.nq + p.tokens - 1) / p.tokens; }
__device__ __forceinline__ int items_of(const Params &p, const Seq &s) {
    const int rt = row_tiles(p, s);
    return rt == 1 ? max((s.nk + p.part - 1) / p.part, 1) : rt;
}

struct Item {
    Seq seq;
    int index;     // over all sequences
    int t0;        // first token of the rows
    int k0, k1;    // keys
    int unit;
    bool partial;  // one of several pieces of its rows
};

// The first 32 sequences, one per lane, looked up once: with no more than that an item is found without a memory access.
struct Known {
    Seq seq;
    int upto;  // items of this lane's sequence and of those before it
};
__device__ __forceinline__ Known look_up(const Params &p) {
    const int lane = threadIdx.x & 31;
    Known k = {{0, 0, 0, 0}, 0};
    if (lane < p.batch) {
        k.seq = load_seq(p, lane);
        k.upto = items_of(p, k.seq);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, k.upto, o);
        if (lane >= o) k.upto += t;
    }
    return k;
}

__device__ __forceinline__ bool find_item(const Params &p, const Known &known, int work, Item &it) {
    int i;
    it.index = work / p.units;
    it.unit = work - it.index * p.units;
    if (it.index >= p.max_items) return false;
    const unsigned hit = __ballot_sync(0xffffffffu, it.index < known.upto);
    if (hit) {
        const int src = __ffs(hit) - 1;
        it.seq.q0 = __shfl_sync(0xffffffffu, known.seq.q0, src);
        it.seq.nq = __shfl_sync(0xffffffffu, known.seq.nq, src);
        it.seq.k0 = __shfl_sync(0xffffffffu, known.seq.k0, src);
        it.seq.nk = __shfl_sync(0xffffffffu, known.seq.nk, src);
        const int before = __shfl_sync(0xffffffffu, known.upto, max(src - 1, 0));
        i = it.index - (src > 0 ? before : 0);
    } else if (p.batch <= 32 || !find_seq(p, it.index, [&](const Seq &s) { return items_of(p, s); }, it.seq, i)) {
        return false;
    }
    int part = 0;
    if (row_tiles(p, it.seq) == 1) {
        it.t0 = 0;
        it.partial = it.seq.nk > p.part;
        // pieces of one size, so that the CTAs' shares differ little: n of them cover the keys in whole blocks, none above p.part
        const int n = (it.seq.nk + p.part - 1) / p.part;
        part = it.partial ? ((it.seq.nk + n - 1) / n + kKeys - 1) / kKeys * kKeys : p.part;
        it.k0 = i * part;
    } else {
        it.t0 = i * p.tokens;
        it.k0 = 0;
        it.partial = false;
    }
    const int sees = visible(p, it.seq, min(it.t0 + p.tokens, it.seq.nq) - 1);  // the last row sees the most
    it.k1 = it.partial ? min(it.k0 + part, sees) : sees;
    return true;
}

// RG groups of 16 rows x 4 groups of 16 keys of each block, a warp each; a warp that loads keys and values; a warp for items
template <int CH, int RG>
__global__ void __launch_bounds__(RG * 128 + 64, Shape<CH, RG>::kCtas)
attention_token_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const Params p) {
    using Sh = Shape<CH, RG>;
    constexpr int kStages = Sh::kStages, kStage = Sh::kStage, kPitch = Sh::kPitch, kWarps = RG * 4, kD = CH * 64;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Item s_items[2];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + kStages * kStage);
    uint64_t *empty = full + kStages;
    uint64_t *item_known = empty + kStages;  // [2] an item's description is there
    uint64_t *item_full = item_known + 2;    // [2] its query rows as well
    uint64_t *item_empty = item_full + 2;
    uint8_t *q_tiles = smem + kStages * kStage + 512;
    // merging: two slots per row group, 16 rows of kD outputs, then the maximum and the sum
    float *merge = reinterpret_cast<float *>(q_tiles + 2 * Sh::kQTile);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        for (int s = 0; s < kStages; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kWarps);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(&item_known[s], 1);
            mbar_init(&item_full[s], 1);
            mbar_init(&item_empty[s], kWarps + 1);
        }
        fence_barrier_init();
        fence_proxy_async();
    }
    __syncthreads();
    swc_let_next_start();
    swc_after_previous();

    int st = 0;
    uint32_t ph = 0, items = 0;
    const auto next = [&] {
        if (++st == kStages) {
            st = 0;
            ph ^= 1;
        }
    };
    bool ok = true;
    Item it;
    const auto next_item = [&](uint64_t *there) {  // false: no more, or a wait ran out
        ok = warp_wait(&there[items & 1], (items >> 1) & 1, p.status, kWaitFull);
        if (ok) it = s_items[items & 1];
        return ok && it.unit >= 0;
    };
    if (warp == kWarps + 1) {
        // ------------------------------------------------------------ items
        const Known known = look_up(p);
        for (int work = blockIdx.x; ok; work += gridDim.x, items++) {
            const bool any = find_item(p, known, work, it);
            if (!any) it.unit = -1;
            ok = warp_wait(&item_empty[items & 1], ((items >> 1) & 1) ^ 1, p.status, kWaitEmpty);
            if (!ok) break;
            if (lane == 0) {
                s_items[items & 1] = it;
                mbar_arrive(&item_known[items & 1]);
            }
            if (any) {
                // query rows, 16 bytes at a time; rows of nobody and columns past the width are zeros
                uint8_t *tile = q_tiles + (items & 1) * Sh::kQTile;
                constexpr int kPieces = RG * 16 * CH * 8;
#pragma unroll 8
                for (int i = lane; i < kPieces; i += 32) {
                    const int row = i / (CH * 8), c = i % (CH * 8) * 8, tok = row * p.pack_inv >> 16, t = it.t0 + tok;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (tok < p.tokens && t < it.seq.nq && c < p.d)
                        v = *reinterpret_cast<const uint4 *>(p.q + (size_t)(it.seq.q0 + t) * p.q_row +
                                                             (size_t)(it.unit * p.pack + row - tok * p.pack) * p.q_head + c);
                    *reinterpret_cast<uint4 *>(tile + row * Sh::kQPitch + c * 2) = v;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_full[items & 1]);
            if (!any) break;
        }
    } else if (warp == kWarps) {
        // ------------------------------------------------------------ loads
        for (; ok && next_item(item_known); items++) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[items & 1]);
            const int head_k = it.unit * p.pack / p.group;
            for (int k = it.k0; k < it.k1 && ok; k += kKeys) {
                ok = warp_wait(&empty[st], ph ^ 1, p.status, kWaitEmpty);
                if (!ok) break;
                if (elect_one()) {
                    uint8_t *dst = smem + st * kStage;
                    mbar_expect_tx(&full[st], kStage);
                    for (int c = 0; c < CH; c++) tma_load_3d(dst + c * kChunk, &tmK, &full[st], c * 64, head_k, it.seq.k0 + k);
                    for (int c = 0; c < CH; c++) tma_load_3d(dst + (CH + c) * kChunk, &tmV, &full[st], c * 64, head_k, it.seq.k0 + k);
                }
                __syncwarp();
                next();
            }
        }
    } else {
        const int rg = warp >> 2, kg = warp & 3;
        const int g = lane >> 2, c2 = (lane & 3) * 2;  // row (and row + 8) and first column of this lane in mma fragments
        // ldmatrix addresses inside a chunk: keys kg*16 + (0..15); the 16-byte piece is xor-ed with the row by the swizzle
        const int k_row = kg * 16 + (lane & 7) + ((lane >> 4) << 3), k_piece = (lane >> 3) & 1;   // K: (keys 0-7: d 0-7, 8-15), (keys 8-15: ..)
        const int v_row = kg * 16 + (lane & 15), v_piece = lane >> 4;                            // V: (keys 0-7, 8-15: d 0-7), (.. d 8-15)
        const int q_row = rg * 16 + (lane & 15), q_piece = lane >> 4;                            // Q: (rows 0-7, 8-15: d 0-7), (.. d 8-15)
        // The four warps of a row group leave together.  One whose wait has run out still comes to the item's first merge barrier,
        // which tells the others, as they may have got what it waited for; no wait lies between that barrier and the next item.
        for (;; items++) {
            if (!next_item(item_full)) {
                __syncwarp();
                barrier_all(1 + rg, 128, ok);
                break;
            }
            // query fragments, rows g and g + 8 of this row group
            uint32_t qf[kD / 16][4];
            const uint32_t sq = smem_u32(q_tiles + (items & 1) * Sh::kQTile) + q_row * Sh::kQPitch + q_piece * 16;
#pragma unroll
            for (int s = 0; s < kD / 16; s++) ldmatrix4(qf[s], sq + s * 32);
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[items & 1]);
            int sees[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int row = rg * 16 + g + h * 8, tok = row * p.pack_inv >> 16, t = it.t0 + tok;
                sees[h] = tok < p.tokens && t < it.seq.nq ? visible(p, it.seq, t) : 0;
            }
            float o[kD / 8][4];
#pragma unroll
            for (int i = 0; i < kD / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
            float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

            for (int k = it.k0; k < it.k1; k += kKeys) {
                ok = warp_wait(&full[st], ph, p.status, kWaitFull);
                if (!ok) break;
                const uint32_t sk = smem_u32(smem + st * kStage), sv = sk + CH * kChunk;
                const int first = k + kg * 16;  // this warp's first key
                if (first < it.k1) {
                    float s[2][4] = {};
#pragma unroll
                    for (int i = 0; i < kD / 16; i++) {
                        uint32_t b[4];
                        const int piece = (i & 3) * 2 + k_piece;
                        ldmatrix4(b, sk + (i >> 2) * kChunk + k_row * 128 + ((piece ^ (k_row & 7)) << 4));
                        mma_16x8x16(s[0], qf[i][0], qf[i][1], qf[i][2], qf[i][3], b[0], b[1]);
                        mma_16x8x16(s[1], qf[i][0], qf[i][1], qf[i][2], qf[i][3], b[2], b[3]);
                    }
                    uint32_t w[4];  // the weights as the A operand of the second product
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float x[4] = {s[0][2 * h], s[0][2 * h + 1], s[1][2 * h], s[1][2 * h + 1]};
                        const int lim = min(sees[h], it.k1) - first - c2;
                        x[0] = lim > 0 ? x[0] : -INFINITY;
                        x[1] = lim > 1 ? x[1] : -INFINITY;
                        x[2] = lim > 8 ? x[2] : -INFINITY;
                        x[3] = lim > 9 ? x[3] : -INFINITY;
                        float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        float factor = 1.f;
                        if ((mx - m[h]) * p.scale_log2 > kSlack) {  // also where m is -inf; not where mx is (NaN compares false)
                            factor = exp2_fast((m[h] - mx) * p.scale_log2);
                            m[h] = mx;
                        }
                        if (__any_sync(0xffffffffu, factor != 1.f)) {
                            l[h] *= factor;
#pragma unroll
                            for (int i = 0; i < kD / 8; i++) {
                                o[i][2 * h] *= factor;
                                o[i][2 * h + 1] *= factor;
                            }
                        }
                        // (the difference first: x * scale - m * scale is off by the rounding of a product that has no bound)
                        const float base = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
                        for (int i = 0; i < 4; i++) x[i] = exp2_fast((x[i] - base) * p.scale_log2);
                        l[h] += (x[0] + x[1]) + (x[2] + x[3]);
                        w[h] = pack_bf16(x[0], x[1]);
                        w[h + 2] = pack_bf16(x[2], x[3]);
                    }
                    // Keys past the item's last one have weight 0, but their V belongs to somebody else (or to nobody), and 0 times
                    // infinity or NaN is not 0: those rows of V count as 0.
                    const int lim = it.k1 - first - c2;
                    const uint32_t keep0 = lim > 1 ? 0xffffffffu : lim > 0 ? 0x0000ffffu : 0u;
                    const uint32_t keep1 = lim > 9 ? 0xffffffffu : lim > 8 ? 0x0000ffffu : 0u;
                    const bool whole = first + 16 <= it.k1;
#pragma unroll
                    for (int i = 0; i < kD / 16; i++) {
                        uint32_t b[4];
                        const int piece = (i & 3) * 2 + v_piece;
                        ldmatrix4_trans(b, sv + (i >> 2) * kChunk + v_row * 128 + ((piece ^ (v_row & 7)) << 4));
                        if (!whole) {
                            b[0] &= keep0;
                            b[1] &= keep1;
                            b[2] &= keep0;
                            b[3] &= keep1;
                        }
                        mma_16x8x16(o[2 * i], w[0], w[1], w[2], w[3], b[0], b[1]);
                        mma_16x8x16(o[2 * i + 1], w[0], w[1], w[2], w[3], b[2], b[3]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[st]);
                next();
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            }
            // merge the four key groups: 2 and 3 into 0 and 1, then 1 into 0
#pragma unroll
            for (int step = 2; step >= 1; step >>= 1) {
                if (kg >= step && kg < 2 * step) {
                    float *dst = merge + (rg * 2 + kg - step) * 16 * kPitch;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float *r = dst + (g + 8 * h) * kPitch;
#pragma unroll
                        for (int i = 0; i < kD / 8; i++) *reinterpret_cast<float2 *>(r + i * 8 + c2) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
                        if (c2 == 0) *reinterpret_cast<float2 *>(r + kD) = make_float2(m[h], l[h]);
                    }
                }
                if (step == 2) {
                    __syncwarp();
                    ok = barrier_all(1 + rg, 128, ok);
                    if (!ok) break;
                } else {
                    named_barrier(1 + rg, 128);
                }
                if (kg < step) {
                    const float *src = merge + (rg * 2 + kg) * 16 * kPitch;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float *r = src + (g + 8 * h) * kPitch;
                        const float2 ml = *reinterpret_cast<const float2 *>(r + kD);
                        const float top = fmaxf(m[h], ml.x);
                        const float a = m[h] == -INFINITY ? 0.f : exp2_fast((m[h] - top) * p.scale_log2);
                        const float b = ml.x == -INFINITY ? 0.f : exp2_fast((ml.x - top) * p.scale_log2);
                        // (a group without keys has l = 0 and o = 0, or NaN where its scores were NaN: kept by the plain sums below)
                        l[h] = l[h] * (m[h] == -INFINITY ? 1.f : a) + ml.y * (ml.x == -INFINITY ? 1.f : b);
#pragma unroll
                        for (int i = 0; i < kD / 8; i++) {
                            const float2 v = *reinterpret_cast<const float2 *>(r + i * 8 + c2);
                            o[i][2 * h] = o[i][2 * h] * a + v.x * b;
                            o[i][2 * h + 1] = o[i][2 * h + 1] * a + v.y * b;
                        }
                        m[h] = top;
                    }
                }
                named_barrier(1 + rg, 128);
            }
            if (!ok) break;
            if (kg == 0) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int row = rg * 16 + g + h * 8, tok = row * p.pack_inv >> 16, t = it.t0 + tok;
                    if (tok >= p.tokens || t >= it.seq.nq) continue;
                    const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];
                    const int head = it.unit * p.pack + row - tok * p.pack;
                    if (it.partial) {
                        const size_t slot = ((size_t)it.index * p.units + it.unit) * (RG * 16) + row;
                        float *dst = p.part_o + slot * p.d;
#pragma unroll
                        for (int i = 0; i < kD / 8; i++)
                            if (i * 8 < p.d) *reinterpret_cast<float2 *>(dst + i * 8 + c2) = make_float2(o[i][2 * h] * inv, o[i][2 * h + 1] * inv);
                        if (c2 == 0) p.part_lse[slot] = l[h] == 0.f ? -INFINITY : fmaf(m[h], p.scale_log2, log2f(l[h]));
                    } else {
                        const size_t at = (size_t)(it.seq.q0 + t);
                        __nv_bfloat16 *dst = p.o + at * p.o_row + (size_t)head * p.o_head;
#pragma unroll
                        for (int i = 0; i < kD / 8; i++)
                            if (i * 8 < p.d) *reinterpret_cast<uint32_t *>(dst + i * 8 + c2) = pack_bf16(o[i][2 * h] * inv, o[i][2 * h + 1] * inv);
                        if (c2 == 0 && p.lse)
                            p.lse[at * p.heads_q + head] =
                                l[h] == 0.f ? -INFINITY : 0.69314718055994531f * fmaf(m[h], p.scale_log2, log2f(l[h]));
                    }
                }
            }
        }
    }
    // a wait that gave up leaves copies possibly still in flight towards this CTA's shared memory: a bounded time to land
    if (!ok) {
        const long long since = clock64();
        while (clock64() - since < 4000000ll) {
        }
    }
    __syncwarp();
}

// Joins the parts of a row (token, head): kWarps warps take them in turn, then a fixed-order sum over the warps.  Eight where a row
// has many parts, one (eight rows per CTA) where it has few.
// kItems: parts are the items of the token kernel (slot = item), else `parts` of every token of the prompt kernel.
constexpr int kJoinThreads = 256;
template <bool kItems, int kWarps>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(const Params p, int rows, int parts) {
    constexpr int kRowsPerCta = kJoinThreads / 32 / kWarps;
    __shared__ float s_o[kWarps > 1 ? kWarps : 1][128], s_l[kWarps], s_m[kWarps];
    const int warp = kWarps > 1 ? threadIdx.x >> 5 : 0, lane = threadIdx.x & 31;
    const long long which = (long long)blockIdx.x * kRowsPerCta + (kWarps > 1 ? 0 : threadIdx.x >> 5);
    swc_let_next_start();
    swc_after_previous();
    if (which >= (long long)p.total_q * p.heads_q) return;
    const int token = (int)(which / p.heads_q), head = (int)(which - (long long)token * p.heads_q);
    size_t slot, step;
    int n;
    if (kItems) {
        // the sequence that holds the token, and the items before it
        int before = 0, found = -1;
        Seq seq = {0, 0, 0, 0};
        for (int base = 0; base < p.batch && found < 0; base += 32) {
            Seq s = {0, 0, 0, 0};
            int count = 0;
            if (base + lane < p.batch) {
                s = load_seq(p, base + lane);
                count = min(items_of(p, s), p.max_items);
            }
            const unsigned hit = __ballot_sync(0xffffffffu, token >= s.q0 && token < s.q0 + s.nq);
            const int src = hit ? __ffs(hit) - 1 : 32;
            int add = lane < src ? count : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) add += __shfl_xor_sync(0xffffffffu, add, o);
            before = min(before + add, p.max_items);  // (sequences that overlap may number more than there is room for)
            if (hit) {
                found = base + src;
                seq.q0 = __shfl_sync(0xffffffffu, s.q0, src);
                seq.nq = __shfl_sync(0xffffffffu, s.nq, src);
                seq.nk = __shfl_sync(0xffffffffu, s.nk, src);
            }
        }
        if (found < 0 || row_tiles(p, seq) != 1 || seq.nk <= p.part) return;  // no sequence's row, or written already
        n = min(items_of(p, seq), p.max_items - before);
        const int unit = head / p.pack;
        slot = ((size_t)before * p.units + unit) * rows + (token - seq.q0) * p.pack + (head - unit * p.pack);
        step = (size_t)p.units * rows;
    } else {
        bool mine = false;  // rows of no sequence stay as they were
        for (int b = lane; b < p.batch; b += 32) {
            const Seq s = load_seq(p, b);
            mine = mine || (token >= s.q0 && token < s.q0 + s.nq);
        }
        if (!__any_sync(0xffffffffu, mine)) return;
        n = parts;
        slot = (size_t)token * p.heads_q + head;
        step = (size_t)p.total_q * p.heads_q;
    }
    // This warp's parts are warp, warp + kWarps, ...: several at once, their sums (a part per lane) and outputs requested together,
    // with a running maximum.
    float m = -INFINITY, acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
    const int c = lane * 4;
    constexpr int kAtOnce = kWarps > 1 ? 16 : 8;
    for (int first = warp; first < n; first += kWarps * kAtOnce) {
        const int mine = first + lane * kWarps;
        const float lse = lane < kAtOnce && mine < n ? p.part_lse[slot + mine * step] : -INFINITY;
        float4 v[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) {
            const int i = first + k * kWarps;
            v[k] = i < n && c < p.d ? *reinterpret_cast<const float4 *>(p.part_o + (slot + i * step) * p.d + c) : make_float4(0, 0, 0, 0);
        }
        float top = lse;
#pragma unroll
        for (int o = kAtOnce / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(m, __shfl_sync(0xffffffffu, top, 0));
        const float base = top == -INFINITY ? 0.f : top, factor = exp2_fast(m - base), w_mine = exp2_fast(lse - base);
        m = top;
        l *= factor;
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] *= factor;
#pragma unroll
        for (int k = 0; k < kAtOnce; k++) {
            const float w = __shfl_sync(0xffffffffu, w_mine, k);
            l += w;
            acc[0] = fmaf(w, v[k].x, acc[0]);
            acc[1] = fmaf(w, v[k].y, acc[1]);
            acc[2] = fmaf(w, v[k].z, acc[2]);
            acc[3] = fmaf(w, v[k].w, acc[3]);
        }
    }
    if (kWarps > 1) {
        *reinterpret_cast<float4 *>(&s_o[warp][c]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (lane == 0) {
            s_l[warp] = l;
            s_m[warp] = m;
        }
        __syncthreads();
        if (warp != 0) return;
        l = 0.f;
        acc[0] = acc[1] = acc[2] = acc[3] = 0.f;
        m = s_m[0];
#pragma unroll
        for (int w = 1; w < kWarps; w++) m = fmaxf(m, s_m[w]);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float4 v = *reinterpret_cast<const float4 *>(&s_o[w][c]);
            const float f = exp2_fast(s_m[w] - (m == -INFINITY ? 0.f : m));
            l = fmaf(s_l[w], f, l);
            acc[0] = fmaf(v.x, f, acc[0]), acc[1] = fmaf(v.y, f, acc[1]), acc[2] = fmaf(v.z, f, acc[2]), acc[3] = fmaf(v.w, f, acc[3]);
        }
    }
    if (c < p.d) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint2 w;
        w.x = pack_bf16(acc[0] * inv, acc[1] * inv);
        w.y = pack_bf16(acc[2] * inv, acc[3] * inv);
        *reinterpret_cast<uint2 *>(p.o + (size_t)token * p.o_row + (size_t)head * p.o_head + c) = w;
    }
    if (lane == 0 && p.lse) p.lse[(size_t)token * p.heads_q + head] = l == 0.f ? -INFINITY : 0.69314718055994531f * (m + log2f(l));
}

template <bool kItems, int kWarps> int join(swcb200_ctx *ctx, const Params &p, int rows, int parts) {
    constexpr int kRowsPerCta = kJoinThreads / 32 / kWarps;
    const long long all = (long long)p.total_q * p.heads_q;
    SWC_CUDA(ctx, swc_launch_early(attention_join_kernel<kItems, kWarps>, (unsigned)((all + kRowsPerCta - 1) / kRowsPerCta), kJoinThreads, 0,
                                   ctx->stream, 1, p, rows, parts));
    return swc_check_launch(ctx, "attention_bf16");
}

template <int CH, int RG>
int launch(swcb200_ctx *ctx, const Params &p, const CUtensorMap &tmK, const CUtensorMap &tmV, int max_items) {
    const size_t smem = Shape<CH, RG>::kSmem;
    SWC_CUDA(ctx, cudaFuncSetAttribute(attention_token_kernel<CH, RG>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    const long long work = (long long)max_items * p.units;
    // (under a limit one CTA for each SM: two would not share one, but take an SM each)
    const int sms = swc_tc_sms(ctx);
    const long long slots = sms < ctx->sm_count ? sms : (long long)sms * Shape<CH, RG>::kCtas;
    const unsigned grid = (unsigned)(work < slots ? work : slots);
    SWC_CUDA(ctx, swc_launch_early(attention_token_kernel<CH, RG>, grid, RG * 128 + 64, smem, ctx->stream, 1, tmK, tmV, p));
    return swc_check_launch(ctx, "attention_bf16");
}

}  // namespace

int swc_attention_token(swcb200_ctx *ctx, Params &p, const CUtensorMap &tmK, const CUtensorMap &tmV, int rows, int max_items) {
    int rc;
    if (p.d > 64)
        rc = rows == 16 ? launch<2, 1>(ctx, p, tmK, tmV, max_items) : rows == 32 ? launch<2, 2>(ctx, p, tmK, tmV, max_items) : launch<2, 4>(ctx, p, tmK, tmV, max_items);
    else
        rc = rows == 16 ? launch<1, 1>(ctx, p, tmK, tmV, max_items) : rows == 32 ? launch<1, 2>(ctx, p, tmK, tmV, max_items) : launch<1, 4>(ctx, p, tmK, tmV, max_items);
    if (rc || p.part >= p.total_k) return rc;  // no sequence has more than one part
    return p.total_k / p.batch > 16ll * p.part ? join<true, 8>(ctx, p, rows, 0) : join<true, 1>(ctx, p, rows, 0);
}

int swc_attention_join_parts(swcb200_ctx *ctx, Params &p, int parts) { return join<false, 1>(ctx, p, 0, parts); }
