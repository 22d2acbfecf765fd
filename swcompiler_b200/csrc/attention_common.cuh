// What the attention kernels share: the call's parameters, the sequences' bounds, and the search for the sequence that a piece
// of work belongs to.
#pragma once
#include "tc_common.cuh"

namespace attn {

struct Params {
    const __nv_bfloat16 *q;
    __nv_bfloat16 *o;
    float *lse;
    size_t q_row, q_head, o_row, o_head;  // elements
    const int *q_off, *k_off, *k_lens;    // device; q_off and k_off [batch + 1]
    int batch, total_q, total_k;
    int heads_q, group, d;  // group: query heads per key head
    int pack;               // query heads in one tile (a divisor of group): tile rows are (token, head), head fastest
    unsigned pack_inv;      // (2^16 + pack - 1) / pack: x / pack = x * pack_inv >> 16 for the rows x of a tile, 0 .. 127
    int units;              // heads_q / pack
    int tokens;             // tokens per tile
    float scale_log2;       // scale * log2(e): the softmax runs on powers of two
    int causal;
    // work split over the keys: keys per part (token kernel) or parts per tile (prompt kernel), and where parts go
    int part;
    float *part_o, *part_lse;
    int max_items;  // token kernel: items that part_o has room for
    int *status;
};

struct Seq {
    int q0, nq, k0, nk;
};

// The offsets live in device memory, so nobody has checked them: they are clamped to the tensors, and whatever they hold
// nothing outside q, k, v, o is touched.
__device__ __forceinline__ Seq load_seq(const Params &p, int b) {
    Seq s;
    s.q0 = min(max(p.q_off[b], 0), p.total_q);
    s.nq = max(min(p.q_off[b + 1], p.total_q), s.q0) - s.q0;  // (the lower bound first: no offset overflows)
    s.k0 = min(max(p.k_off[b], 0), p.total_k);
    s.nk = max(min(p.k_off[b + 1], p.total_k), s.k0) - s.k0;
    if (p.k_lens) s.nk = min(max(p.k_lens[b], 0), s.nk);
    return s;
}

// The sequence that item `want` falls into when sequence b has count(seq) items; a whole warp calls it.  `item` becomes the
// number inside the sequence; false: there are fewer items.
template <class Count>
__device__ __forceinline__ bool find_seq(const Params &p, int want, Count count, Seq &seq, int &item) {
    const int lane = threadIdx.x & 31;
    int before = 0;
    for (int base = 0; base < p.batch; base += 32) {
        Seq s = {0, 0, 0, 0};
        int n = 0;
        if (base + lane < p.batch) {
            s = load_seq(p, base + lane);
            n = count(s);
        }
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, want < before + upto);
        if (hit) {
            const int src = __ffs(hit) - 1;
            seq.q0 = __shfl_sync(0xffffffffu, s.q0, src);
            seq.nq = __shfl_sync(0xffffffffu, s.nq, src);
            seq.k0 = __shfl_sync(0xffffffffu, s.k0, src);
            seq.nk = __shfl_sync(0xffffffffu, s.nk, src);
            item = want - before - __shfl_sync(0xffffffffu, upto - n, src);
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// keys that token t of a sequence sees, counted from the first
__device__ __forceinline__ int visible(const Params &p, const Seq &s, int t) {
    return p.causal ? max(min(s.nk, t + 1 + s.nk - s.nq), 0) : s.nk;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t *>(&h);
}

// A row's maximum may lie this far (in powers of two) under the true one before sums and output are rescaled: the weights then
// reach 2^8 instead of 1, which neither fp32 sums nor bf16 weights (relative rounding) mind, and rescaling becomes rare.
constexpr float kSlack = 8.f;

}  // namespace attn

int swc_attention_token(swcb200_ctx *ctx, attn::Params &p, const CUtensorMap &tmK, const CUtensorMap &tmV, int rows, int max_items);
int swc_attention_prompt(swcb200_ctx *ctx, attn::Params &p, const CUtensorMap &tmQ, const CUtensorMap &tmK, const CUtensorMap &tmV,
                         int tiles, int parts);
int swc_attention_join_parts(swcb200_ctx *ctx, attn::Params &p, int parts);
