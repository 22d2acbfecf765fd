// Attention entry points: argument checks, and which kernel takes a call.
#include <float.h>

#include "attention_common.cuh"

using namespace attn;

namespace {

struct Plan {
    bool token;
    int pack, units, tokens;
    int rows, max_items, part;  // token kernel
    int tiles, parts;           // prompt kernel
    size_t lse_at, bytes;       // workspace: partial outputs, then at lse_at what they weigh
};

// the largest divisor of n up to top that fills the rows of a tile to 7/8 (1 always does)
int heads_per_tile(int n, int top, int rows) {
    for (int v = n < top ? n : top; v > 1; v--)
        if (n % v == 0 && rows / v * v * 8 >= rows * 7) return v;
    return 1;
}

int make_plan(swcb200_ctx *ctx, const swcb200_attention *a, Plan &pl) {
    pl = {};
    const int group = a->heads_q / a->heads_kv;
    const long long average = ((long long)a->total_q + a->batch - 1) / a->batch;  // the lengths themselves are on the device
    long long work, slots = 0;
    // Up to 64 (token, head) rows per sequence and key head a call is bound by reading the cache: the token kernel.  Above, the
    // products weigh in and its mma.sync would set the pace: the prompt kernel.
    pl.pack = group <= 64 ? group : heads_per_tile(group, 64, 64);
    pl.token = pl.pack * average <= 64;
    if (pl.token) {
        pl.rows = 16;
        while (pl.rows < pl.pack * average) pl.rows *= 2;
        pl.tokens = pl.rows / pl.pack;
        pl.units = a->heads_q / pl.pack;
        // Keys per item.  One item for each of two CTAs per SM while that is no more than 2048 keys: one wave, and the fewest parts
        // to join (one sequence of 65536 keys: 59 -> 52 us).  Else 512, which evens out lengths that differ (256 KiB of cache at
        // width 128, about 6 us of an SM's share of HBM), and more only where items would number beyond 32 per SM.
        const long long keys = (long long)a->total_k * pl.units;
        long long part = keys / (2ll * ctx->sm_count);
        if (part > 2048) part = 512;
        part = part > keys / (32ll * ctx->sm_count) ? part : keys / (32ll * ctx->sm_count);
        part = part < a->total_k ? part : a->total_k;
        pl.part = (int)((part + 63) / 64 * 64);
        if (pl.part < 64) pl.part = 64;
        const long long items = a->total_k / pl.part + a->total_q / pl.tokens + a->batch;  // each sequence rounds up once
        work = items * pl.units;
        // (sums over 32 sequences of up to as many items each have to fit 31 bits)
        SWC_REQUIRE(ctx, work < 0x7fffffff && items < 1 << 25, SWCB200_ERR_TOO_LARGE, "attention_bf16: too many work items");
        pl.max_items = (int)items;
        if (pl.part < a->total_k) slots = work * pl.rows;
    } else {
        pl.pack = heads_per_tile(group, 128, 128);
        pl.tokens = 128 / pl.pack;
        pl.units = a->heads_q / pl.pack;
        const long long tiles = a->total_q / (2 * pl.tokens) + a->batch;  // each sequence rounds up once
        work = tiles * pl.units;
        // Too few tiles for the SMs, as with a short chunk behind a long cache: the keys are divided, in parts of 512 at least.
        pl.parts = 1;
        while (pl.parts < 16 && work * pl.parts * 2 <= ctx->sm_count && (long long)a->total_k / a->batch >= pl.parts * 2ll * 512) pl.parts *= 2;
        SWC_REQUIRE(ctx, work * pl.parts < 0x7fffffff && tiles < 1 << 25, SWCB200_ERR_TOO_LARGE, "attention_bf16: too many tiles");
        pl.tiles = (int)tiles;
        if (pl.parts > 1) slots = (long long)pl.parts * a->total_q * a->heads_q;
    }
    SWC_REQUIRE(ctx, (long long)a->total_q * a->heads_q < 0x7fffffff, SWCB200_ERR_TOO_LARGE, "attention_bf16: too many rows");
    pl.lse_at = ((size_t)slots * a->head_dim * 4 + 255) & ~(size_t)255;
    pl.bytes = slots ? pl.lse_at + (size_t)slots * 4 : 0;
    return SWCB200_OK;
}

// the fields that the workspace's size follows from
int check(swcb200_ctx *ctx, const swcb200_attention *a) {
    SWC_REQUIRE(ctx, a != nullptr, SWCB200_ERR_BAD_ARG, "attention_bf16: null description");
    SWC_REQUIRE(ctx, a->batch >= 0 && a->total_q >= 0 && a->total_k >= 0 && a->heads_q >= 1 && a->heads_kv >= 1 && a->head_dim >= 1,
                SWCB200_ERR_BAD_ARG, "attention_bf16: bad shape");
    SWC_REQUIRE(ctx, a->total_q <= 1 << 30 && a->total_k <= 1 << 30 && a->batch <= 1 << 30, SWCB200_ERR_TOO_LARGE,
                "attention_bf16: more than 2^30 rows or sequences");
    SWC_REQUIRE(ctx, a->heads_q % a->heads_kv == 0, SWCB200_ERR_BAD_SHAPE,
                "attention_bf16: %d query heads are no multiple of %d key heads", a->heads_q, a->heads_kv);
    SWC_REQUIRE(ctx, a->head_dim % 8 == 0 && a->head_dim <= 128, SWCB200_ERR_UNSUPPORTED,
                "attention_bf16: head width %d (multiples of 8 up to 128)", a->head_dim);
    return SWCB200_OK;
}

// one tensor [rows, heads, head_dim]
struct Rows {
    const void *p;
    size_t row, head;
    int rows, heads;
    const char *name;
};

int check_rows(swcb200_ctx *ctx, const Rows &t, int d) {
    SWC_REQUIRE(ctx, swc_aligned16(t.p) && (t.rows == 1 || t.row % 8 == 0) && (t.heads == 1 || t.head % 8 == 0), SWCB200_ERR_MISALIGNED,
                "attention_bf16: %s starts on 16 bytes, its strides are multiples of 8 elements", t.name);
    SWC_REQUIRE(ctx, (t.rows == 1 || t.row >= (size_t)d) && (t.heads == 1 || t.head >= (size_t)d), SWCB200_ERR_BAD_SHAPE,
                "attention_bf16: a stride of %s is smaller than the head width", t.name);
    SWC_REQUIRE(ctx, t.row < ((size_t)1 << 38) && t.head < ((size_t)1 << 38), SWCB200_ERR_TOO_LARGE,
                "attention_bf16: a stride of %s is too large", t.name);
    return SWCB200_OK;
}

bool ranges_meet(const Rows &a, const Rows &b, int d) {
    const auto end = [&](const Rows &t) { return (const char *)t.p + ((size_t)(t.rows - 1) * t.row + (size_t)(t.heads - 1) * t.head + d) * 2; };
    return (const char *)a.p < end(b) && (const char *)b.p < end(a);
}

// [rows, heads, head_dim] in boxes of 64 columns x heads x rows
int tmap_heads(swcb200_ctx *ctx, const Rows &t, int d, int box_heads, int box_rows, CUtensorMap *out) {
    const uint64_t dims[3] = {(uint64_t)d, (uint64_t)t.heads, (uint64_t)t.rows};
    // a dimension of one element has no stride of its own
    const uint64_t strides[3] = {2, t.heads > 1 ? (uint64_t)t.head * 2 : 256, t.rows > 1 ? (uint64_t)t.row * 2 : 256};
    const uint32_t box[3] = {64, (uint32_t)box_heads, (uint32_t)box_rows};
    return tc::make_tmap_bf16(ctx, out, t.p, 3, dims, strides, box);
}

}  // namespace

SWC_EXPORT int swcb200_attention_workspace(swcb200_ctx *ctx, const swcb200_attention *a, size_t *bytes) {
    SWC_CTX(ctx);
    SWC_REQUIRE(ctx, bytes != nullptr, SWCB200_ERR_BAD_ARG, "attention_workspace: null result");
    *bytes = 0;
    int rc = check(ctx, a);
    if (rc || a->batch == 0 || a->total_q == 0) return rc;
    Plan pl;
    rc = make_plan(ctx, a, pl);
    if (!rc) *bytes = pl.bytes;
    return rc;
}

SWC_EXPORT int swcb200_attention_bf16(swcb200_ctx *ctx, const swcb200_attention *a) {
    SWC_CTX(ctx);
    int rc = check(ctx, a);
    if (rc) return rc;
    const float scale_log2 = a->scale * 1.4426950408889634f;  // finite, too
    SWC_REQUIRE(ctx, a->scale > 0.f && scale_log2 <= FLT_MAX, SWCB200_ERR_BAD_ARG, "attention_bf16: the scale must be positive and at most 2e38");
    if (a->batch == 0 || a->total_q == 0) return SWCB200_OK;
    SWC_REQUIRE(ctx, a->q && a->o && (a->total_k == 0 || (a->k && a->v)) && a->q_offsets && a->k_offsets, SWCB200_ERR_BAD_ARG,
                "attention_bf16: null tensor");
    // (with no keys at all every row is empty: q stands in for the tensors that nothing is read from)
    const Rows q = {a->q, a->q_row, a->q_head, a->total_q, a->heads_q, "q"}, o = {a->o, a->o_row, a->o_head, a->total_q, a->heads_q, "o"};
    const Rows k = a->total_k ? Rows{a->k, a->k_row, a->k_head, a->total_k, a->heads_kv, "k"} : q;
    const Rows v = a->total_k ? Rows{a->v, a->v_row, a->v_head, a->total_k, a->heads_kv, "v"} : q;
    for (const Rows *t : {&q, &k, &v, &o})
        if ((rc = check_rows(ctx, *t, a->head_dim))) return rc;
    // (several CTAs write o: one of its strides steps over all that the other one reaches)
    SWC_REQUIRE(ctx, o.rows == 1 || o.heads == 1 || o.row >= (size_t)(o.heads - 1) * o.head + a->head_dim ||
                o.head >= (size_t)(o.rows - 1) * o.row + a->head_dim, SWCB200_ERR_BAD_SHAPE, "attention_bf16: rows and heads of o overlap");
    for (const Rows *t : {&q, &k, &v})
        SWC_REQUIRE(ctx, !ranges_meet(*t, o, a->head_dim), SWCB200_ERR_BAD_ARG, "attention_bf16: o overlaps %s", t->name);
    Plan pl;
    if ((rc = make_plan(ctx, a, pl))) return rc;
    SWC_REQUIRE(ctx, pl.bytes == 0 || (a->workspace && a->workspace_bytes >= pl.bytes), SWCB200_ERR_BAD_ARG,
                "attention_bf16: the workspace has %zu bytes, the call needs %zu", a->workspace ? a->workspace_bytes : (size_t)0, pl.bytes);
    SWC_REQUIRE(ctx, pl.bytes == 0 || swc_aligned16(a->workspace), SWCB200_ERR_MISALIGNED, "attention_bf16: the workspace starts on 16 bytes");
    Params p = {};
    p.q = (const __nv_bfloat16 *)a->q, p.q_row = a->q_row, p.q_head = a->q_head;
    p.o = (__nv_bfloat16 *)a->o, p.o_row = a->o_row, p.o_head = a->o_head;
    p.lse = a->lse;
    p.q_off = a->q_offsets, p.k_off = a->k_offsets, p.k_lens = a->k_lens;
    p.batch = a->batch, p.total_q = a->total_q, p.total_k = a->total_k;
    p.heads_q = a->heads_q, p.group = a->heads_q / a->heads_kv, p.d = a->head_dim;
    p.pack = pl.pack, p.pack_inv = (65536u + pl.pack - 1) / pl.pack, p.units = pl.units, p.tokens = pl.tokens;
    p.scale_log2 = scale_log2;
    p.causal = a->causal != 0;
    p.part = pl.part, p.max_items = pl.max_items;
    p.part_o = (float *)a->workspace;
    p.part_lse = (float *)((char *)a->workspace + pl.lse_at);
    p.status = ctx->dev_status;
    CUtensorMap tmQ, tmK, tmV;
    const int keys = pl.token ? 64 : 128;  // of a block
    if ((rc = tmap_heads(ctx, k, a->head_dim, 1, keys, &tmK)) || (rc = tmap_heads(ctx, v, a->head_dim, 1, keys, &tmV))) return rc;
    if (pl.token) return swc_attention_token(ctx, p, tmK, tmV, pl.rows, pl.max_items);
    if ((rc = tmap_heads(ctx, q, a->head_dim, pl.pack, pl.tokens, &tmQ))) return rc;
    rc = swc_attention_prompt(ctx, p, tmQ, tmK, tmV, pl.tiles, pl.parts);
    if (rc || pl.parts == 1) return rc;
    return swc_attention_join_parts(ctx, p, pl.parts);
}
