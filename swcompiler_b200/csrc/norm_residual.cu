// The rows between two blocks of a transformer, in one pass:
//     t = residual + scale * gate * post(x)        sum <- t
//     y = pre(t)
// post and pre are RMS norms (x * w / sqrt(mean(x^2) + eps)), layer norms ((x - mean) / sqrt(var + eps) * w + b, biased
// variance) or absent.
//
// What bounds it: the bytes of x, residual, sum and y; about ten operations per element.  So a row is read once, held in
// registers as fp32 through up to four row sums, and written once.  The layer norm's variance is the mean of
// (t - mean)^2 over the registers (no E[t^2] - mean^2, which cancels).  pre() reads t before it is rounded to sum's type:
// the value is there, and rounding it first would only add an error to y.
//
// 65536 rows of 4096, gate, fp32 stream, layer norm: 570 us, 0.87 of the copy rate measured here (629 us, 0.79, once calls have gone on
// long enough for the power limit to take the clock to 1.76 GHz).  8192 rows with RMS norms on both
// sides, all bf16: 61 us, 0.67: two row sums one behind the other, warps wait for loads and shared memory half of the time, and 61 % of
// the issue slots are taken; requesting
// whole rows ahead through shared memory (bulk copies, persistent CTAs) took 77 us and more.  Rows of odd width, read one element per
// access, keep the issue slots busy instead (76 %): bf16, 20000 rows of 1003 63 us, 0.39; 50000 of 333 71 us, 0.29; 10000 of 4097, where
// a thread's 17 elements take the form for 32, which spills, 239 us, 0.21.
//
// Layout: a row belongs to `tpr` threads.  Up to 32 of them (rows of at most 512 elements, 256 read singly) are a part of one
// warp and the sums are shuffles; above that the row is a CTA of its own.  A thread holds at most 32 elements of a row.  Rows whose
// tensors are all aligned move in chunks of 8 elements (16 bytes of bf16, one 32-byte access of fp32); other rows one
// element per access, neighbouring threads at neighbouring elements.
#include <cuda_bf16.h>

#include "common.cuh"

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kMaxThreads = 512;  // 128 registers each: 64 hold the row and its residual
constexpr int kMaxCols = kMaxThreads * 32;

struct NormParams {
    const float *w, *b;
    float eps;
    int kind;
};

struct RowParams {
    const void *x, *residual, *gate;
    void *sum, *y;
    size_t ldx, ldr, ldg, lds, ldy;  // elements
    int x_how, r_how, g_how;         // how they are read
    int s16, y16;                    // 1: bf16, 0: fp32
    long long rows, gate_rows;
    int cols, tpr;
    float scale, inv_cols;
    NormParams post, pre;
};

// How a tensor is read: not at all, as bf16, as fp32.
enum : int { kSkip = 0, kBf16 = 1, kF32 = 2 };

template <int kVec, int kType> __device__ __forceinline__ void load_chunk(const void *p, size_t i, bool in, uint32_t (&r)[kVec]) {
    if constexpr (kVec == 8 && kType == kBf16)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\t@p ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
                     : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3])
                     : "l"(reinterpret_cast<const __nv_bfloat16 *>(p) + i), "r"((uint32_t)in));
    else if constexpr (kVec == 8)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %9, 0;\n\t"
            "@p ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t}"
            : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
            : "l"(reinterpret_cast<const float *>(p) + i), "r"((uint32_t)in));
    else if constexpr (kType == kBf16)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.global.u16 %0, [%1];\n\t}"
                     : "+r"(r[0])
                     : "l"(reinterpret_cast<const __nv_bfloat16 *>(p) + i), "r"((uint32_t)in));
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}"
                     : "+r"(r[0])
                     : "l"(reinterpret_cast<const float *>(p) + i), "r"((uint32_t)in));
}
// All chunks of a thread, as they are: requested one behind the other, and none converted before the last is requested.  kType: the
// type where the kernel is compiled for it (selecting it per element took a third of the instructions), 0 for either.  (One
// statement with two predicated loads into a register, one of them never executed, waits for the first all the same: 20000 rows
// of 1003 took 150 us that way.)
template <int kVec, int kN, int kType>
__device__ __forceinline__ void load_chunks(const void *p, size_t at, int how, int tpr, int cols, int tid, uint32_t (&r)[kN][kVec]) {
#pragma unroll
    for (int i = 0; i < kN; i++)
#pragma unroll
        for (int e = 0; e < kVec; e++) r[i][e] = 0u;
    if (kType != kF32 && how == kBf16) {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int c = (i * tpr + tid) * kVec;
            load_chunk<kVec, kBf16>(p, at + c, c < cols, r[i]);
        }
    } else if (kType != kBf16 && how == kF32) {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int c = (i * tpr + tid) * kVec;
            load_chunk<kVec, kF32>(p, at + c, c < cols, r[i]);
        }
    }
}
template <int kVec, int kType> __device__ __forceinline__ float element(const uint32_t (&r)[kVec], int e, int how) {
    const bool is16 = (kType ? kType : how) == kBf16;
    if (kVec == 1) return __uint_as_float(is16 ? r[0] << 16 : r[0]);
    const uint32_t h = e & 1 ? r[e / 2] & 0xffff0000u : r[e / 2] << 16;
    return __uint_as_float(is16 ? h : r[e]);
}

__device__ __forceinline__ void store8(void *p, size_t i, bool is16, const float (&v)[8]) {
    if (is16) {
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            r[j] = *reinterpret_cast<uint32_t *>(&h);
        }
        asm volatile("st.global.L1::no_allocate.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(reinterpret_cast<__nv_bfloat16 *>(p) + i),
                     "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
                     : "memory");
    } else {
        asm volatile("st.global.L1::no_allocate.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(
                         reinterpret_cast<float *>(p) + i),
                     "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                     : "memory");
    }
}

// the per-channel vectors: every row reads them, so they stay in L1
__device__ __forceinline__ void vector8(const float *p, int i, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p + i), b = *reinterpret_cast<const float4 *>(p + i + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// (cols: 0 for a row past the last one, whose gate row may not exist)
template <int kVec, int kN>
__device__ __forceinline__ void vector_chunks(const float *v, const RowParams &p, int cols, int tid, float (&out)[kN * kVec]) {
#pragma unroll
    for (int i = 0; i < kN; i++) {
        const int c = (i * p.tpr + tid) * kVec;
        if constexpr (kVec == 8) {
            float x[8] = {};
            if (c < cols) vector8(v, c, x);
#pragma unroll
            for (int e = 0; e < 8; e++) out[i * 8 + e] = x[e];
        } else {
            out[i] = c < cols ? v[c] : 0.f;
        }
    }
}

// sum over the row's threads; every thread gets it
template <bool kCta>
__device__ __forceinline__ float row_sum(float v, int tpr, float *red) {
    if (!kCta) {
        for (int o = tpr >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
        return v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;  // (the other sums of a few warps: reads of one address are cheaper than another round of shuffles)
#pragma unroll
    for (int i = 0; i < kMaxThreads / 32; i += 4)
        if (i < warps) {
            const float4 q = *reinterpret_cast<const float4 *>(red + i);
            v += (q.x + (i + 1 < warps ? q.y : 0.f)) + ((i + 2 < warps ? q.z : 0.f) + (i + 3 < warps ? q.w : 0.f));
        }
    return v;
}

// t <- norm(t) over the kN * kVec elements of this thread; element e of chunk i is column (i * tpr + tid) * kVec + e
template <int kVec, int kN, bool kCta>
__device__ __forceinline__ void norm_row(const NormParams &n, const RowParams &p, float (&t)[kN * kVec], int tid, float *red) {
    if (n.kind == SWCB200_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < kN * kVec; j++) s += t[j];  // elements past the row are 0
        const float mean = row_sum<kCta>(s, p.tpr, red) * p.inv_cols;
#pragma unroll
        for (int i = 0; i < kN; i++)
#pragma unroll
            for (int e = 0; e < kVec; e++)
                t[i * kVec + e] = (i * p.tpr + tid) * kVec + e < p.cols ? t[i * kVec + e] - mean : 0.f;
    }
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < kN * kVec; j++) q = fmaf(t[j], t[j], q);
    // the vectors come from L1: all of a thread's chunks at once, behind the sum
    float w[kN * kVec], b[kN * kVec];
    if (n.w) vector_chunks<kVec, kN>(n.w, p, p.cols, tid, w);
    if (n.b) vector_chunks<kVec, kN>(n.b, p, p.cols, tid, b);
    const float rstd = 1.0f / sqrtf(row_sum<kCta>(q, p.tpr, red + 32) * p.inv_cols + n.eps);
#pragma unroll
    for (int j = 0; j < kN * kVec; j++) {
        t[j] *= n.w ? rstd * w[j] : rstd;
        if (n.b) t[j] += b[j];
    }
}

__device__ __forceinline__ void store1(void *p, size_t i, bool is16, float v) {
    if (is16)
        reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else
        reinterpret_cast<float *>(p)[i] = v;
}

template <int kVec, int kN, bool kCta, int kX, int kR>
// (up to 16 elements a thread come with 256 threads at most, and four such CTAs keep an SM busier than three)
__global__ void __launch_bounds__(!kCta ? 128 : kN * kVec <= 16 ? 256 : kMaxThreads, kCta && kVec == 8 && kN <= 2 ? 4 : 1)
norm_residual_kernel(const RowParams p) {
    swc_let_next_start();
    swc_after_previous();
    __shared__ alignas(16) float red[128];  // one part for each of the four row sums: no barrier between reading one and writing the next
    const int tid = kCta ? threadIdx.x : threadIdx.x & (p.tpr - 1);
    const int rows_per_cta = kCta ? 1 : blockDim.x / p.tpr;
    const long long row = (long long)blockIdx.x * rows_per_cta + (kCta ? 0 : threadIdx.x / p.tpr);
    // threads of a row past the last one keep their lanes in the shuffles and touch no memory
    const int cols = row < p.rows ? p.cols : 0;
    float t[kN * kVec];
    uint32_t x[kN][kVec], r[kN][kVec];
    load_chunks<kVec, kN, kX>(p.x, (size_t)row * p.ldx, p.x_how, p.tpr, cols, tid, x);
    load_chunks<kVec, kN, kR>(p.residual, (size_t)row * p.ldr, p.r_how, p.tpr, cols, tid, r);
#pragma unroll
    for (int j = 0; j < kN * kVec; j++) t[j] = element<kVec, kX>(x[j / kVec], j % kVec, p.x_how);
    if (p.post.kind) norm_row<kVec, kN, kCta>(p.post, p, t, tid, red);
#pragma unroll
    for (int j = 0; j < kN * kVec; j++) t[j] *= p.scale;
    if (p.gate) {  // one row of it serves many: through L1
        const size_t base = p.gate_rows ? (size_t)(row / p.gate_rows) * p.ldg : 0;
        float g[kN * kVec];
        if (p.g_how == kF32) {
            vector_chunks<kVec, kN>(reinterpret_cast<const float *>(p.gate) + base, p, cols, tid, g);
        } else {
#pragma unroll
            for (int i = 0; i < kN; i++) {
                const int c = (i * p.tpr + tid) * kVec;
                const __nv_bfloat16 *src = reinterpret_cast<const __nv_bfloat16 *>(p.gate) + base + c;
                uint32_t v[4] = {0u, 0u, 0u, 0u};
                if (kVec == 8 && c < cols) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(src);
                if (kVec == 1 && c < cols) v[0] = (uint32_t)__bfloat16_as_ushort(*src);
#pragma unroll
                for (int e = 0; e < kVec; e++) g[i * kVec + e] = __uint_as_float(e & 1 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16);
            }
        }
#pragma unroll
        for (int j = 0; j < kN * kVec; j++) t[j] *= g[j];
    }
    if (p.residual) {
#pragma unroll
        for (int j = 0; j < kN * kVec; j++) t[j] += element<kVec, kR>(r[j / kVec], j % kVec, p.r_how);
    }
    if (p.sum) {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int c = (i * p.tpr + tid) * kVec;
            if (c >= cols) continue;
            if constexpr (kVec == 8) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = t[i * 8 + e];
                store8(p.sum, (size_t)row * p.lds + c, p.s16, v);
            } else {
                store1(p.sum, (size_t)row * p.lds + c, p.s16, t[i]);
            }
        }
    }
    if (p.pre.kind) {
        norm_row<kVec, kN, kCta>(p.pre, p, t, tid, red + 64);
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int c = (i * p.tpr + tid) * kVec;
            if (c >= cols) continue;
            if constexpr (kVec == 8) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = t[i * 8 + e];
                store8(p.y, (size_t)row * p.ldy + c, p.y16, v);
            } else {
                store1(p.y, (size_t)row * p.ldy + c, p.y16, t[i]);
            }
        }
    }
}

template <int kVec, bool kCta, int kX, int kR> cudaError_t launch_types(int n, unsigned grid, int threads, cudaStream_t s, const RowParams &p) {
    constexpr int k = kVec == 8 ? 1 : 8;  // chunks of one element come in eights
    auto kernel = norm_residual_kernel<kVec, k, kCta, kX, kR>;
    // (rows inside a warp have no more than two chunks of 8, or eight of one element, a thread)
    if constexpr (kCta || kVec == 8)
        if (n > k) kernel = norm_residual_kernel<kVec, 2 * k, kCta, kX, kR>;
    if constexpr (kCta)
        if (n > 2 * k) kernel = norm_residual_kernel<kVec, 4 * k, kCta, kX, kR>;
    return swc_launch_early(kernel, grid, (unsigned)threads, 0, s, 1, p);
}
template <bool kCta> cudaError_t launch(bool vec, int n, unsigned grid, int threads, cudaStream_t s, const RowParams &p) {
    if (!vec) return launch_types<1, kCta, 0, 0>(n, grid, threads, s, p);
    if (p.x_how == kBf16)
        return p.r_how == kF32 ? launch_types<8, kCta, kBf16, kF32>(n, grid, threads, s, p) : launch_types<8, kCta, kBf16, kBf16>(n, grid, threads, s, p);
    return p.r_how == kF32 ? launch_types<8, kCta, kF32, kF32>(n, grid, threads, s, p) : launch_types<8, kCta, kF32, kBf16>(n, grid, threads, s, p);
}

bool known_dtype(int d) { return d == SWCB200_F32 || d == SWCB200_BF16; }

}  // namespace

bool swc_rows_overlap(const void *a, size_t a_pitch, size_t a_width, const void *b, size_t b_pitch, size_t b_width, size_t rows) {
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
    const uintptr_t a1 = a0 + (rows - 1) * a_pitch + a_width, b1 = b0 + (rows - 1) * b_pitch + b_width;
    if (a1 <= b0 || b1 <= a0) return false;
    if (rows == 1 || a_pitch != b_pitch) return true;  // ranges meet: taken as an overlap
    const size_t d = b0 >= a0 ? (b0 - a0) % a_pitch : (a_pitch - (a0 - b0) % a_pitch) % a_pitch;
    return d < a_width || d + b_width > a_pitch;  // else columns of one tensor side by side
}

SWC_EXPORT int swcb200_norm_residual(swcb200_ctx *ctx, size_t rows, int cols, const swcb200_norm_block *d) {
    SWC_CTX(ctx);
    SWC_REQUIRE(ctx, d != nullptr, SWCB200_ERR_BAD_ARG, "norm_residual: null description");
    SWC_REQUIRE(ctx, cols >= 1, SWCB200_ERR_BAD_ARG, "norm_residual: bad column count %d", cols);
    SWC_REQUIRE(ctx, cols <= kMaxCols && rows <= 0x7fffffffu, SWCB200_ERR_TOO_LARGE,
                "norm_residual: at most %d columns and 2^31 - 1 rows", kMaxCols);
    const swcb200_norm *norms[2] = {&d->post, &d->pre};
    for (const swcb200_norm *n : norms) {
        SWC_REQUIRE(ctx, n->kind >= SWCB200_NORM_NONE && n->kind <= SWCB200_NORM_LAYER, SWCB200_ERR_BAD_ARG,
                    "norm_residual: unknown norm %d", n->kind);
        SWC_REQUIRE(ctx, n->kind == SWCB200_NORM_NONE || n->eps >= 0.f, SWCB200_ERR_BAD_ARG, "norm_residual: negative eps");
    }
    SWC_REQUIRE(ctx, known_dtype(d->x_dtype) && (!d->residual || known_dtype(d->residual_dtype)) &&
                (!d->gate || known_dtype(d->gate_dtype)) && (!d->sum || known_dtype(d->sum_dtype)) &&
                (!d->y || known_dtype(d->y_dtype)), SWCB200_ERR_BAD_ARG, "norm_residual: tensors are fp32 or bf16");
    SWC_REQUIRE(ctx, d->gate_rows >= 0, SWCB200_ERR_BAD_ARG, "norm_residual: negative gate_rows");
    if (rows == 0) return SWCB200_OK;
    SWC_REQUIRE(ctx, (d->y != nullptr) == (d->pre.kind != SWCB200_NORM_NONE), SWCB200_ERR_BAD_ARG,
                "norm_residual: y and the norm that writes it go together");
    SWC_REQUIRE(ctx, d->x && (d->sum || d->y), SWCB200_ERR_BAD_ARG, "norm_residual: null tensor");
    const size_t c = (size_t)cols;
    SWC_REQUIRE(ctx, rows == 1 || (d->ldx >= c && (!d->residual || d->ld_residual >= c) && (!d->sum || d->ld_sum >= c) &&
                                   (!d->y || d->ldy >= c) && (!d->gate || !d->gate_rows || d->ld_gate >= c)),
                SWCB200_ERR_BAD_SHAPE, "norm_residual: leading dimension too small");
    // an output may be one of the inputs in place (a thread reads what it overwrites before it writes); nothing else may overlap
    struct Tensor {
        const void *p;
        size_t ld, size, rows;
    };
    const auto size = [](int dt) { return dt == SWCB200_BF16 ? (size_t)2 : (size_t)4; };
    const Tensor in[3] = {{d->x, d->ldx, size(d->x_dtype), rows},
                          {d->residual, d->ld_residual, size(d->residual_dtype), rows},
                          {d->gate, d->ld_gate, size(d->gate_dtype), d->gate_rows ? (rows - 1) / (size_t)d->gate_rows + 1 : 1}};
    const Tensor out[2] = {{d->sum, d->ld_sum, size(d->sum_dtype), rows}, {d->y, d->ldy, size(d->y_dtype), rows}};
    const auto meet = [&](const Tensor &a, const Tensor &b) {
        if (!a.p || !b.p) return false;
        if (a.rows == b.rows)
            return swc_rows_overlap(a.p, a.ld * a.size, c * a.size, b.p, b.ld * b.size, c * b.size, a.rows);
        const char *a0 = (const char *)a.p, *b0 = (const char *)b.p;
        return a0 < b0 + ((b.rows - 1) * b.ld + c) * b.size && b0 < a0 + ((a.rows - 1) * a.ld + c) * a.size;
    };
    for (const Tensor &o : out) {
        for (const swcb200_norm *n : norms)
            for (const float *v : {n->weight, n->bias})
                SWC_REQUIRE(ctx, !o.p || !v || n->kind == SWCB200_NORM_NONE || (const char *)o.p + ((rows - 1) * o.ld + c) * o.size <= (const char *)v ||
                            v + c <= o.p, SWCB200_ERR_BAD_ARG, "norm_residual: an output overlaps a norm's vector");
        for (int i = 0; i < 3; i++) {
            const bool in_place = i < 2 && o.p == in[i].p && o.size == in[i].size && (rows == 1 || o.ld == in[i].ld);
            SWC_REQUIRE(ctx, in_place || !meet(o, in[i]), SWCB200_ERR_BAD_ARG,
                        "norm_residual: an output overlaps an input without being the same tensor");
        }
    }
    SWC_REQUIRE(ctx, !meet(out[0], out[1]), SWCB200_ERR_BAD_ARG, "norm_residual: the two outputs overlap");

    RowParams p = {};
    const auto how = [](const void *t, int dt) { return !t ? kSkip : dt == SWCB200_BF16 ? kBf16 : kF32; };
    p.x = d->x, p.ldx = d->ldx, p.x_how = how(d->x, d->x_dtype);
    p.residual = d->residual, p.ldr = d->ld_residual, p.r_how = how(d->residual, d->residual_dtype);
    p.gate = d->gate, p.ldg = d->ld_gate, p.g_how = how(d->gate, d->gate_dtype);
    p.sum = d->sum, p.lds = d->ld_sum, p.s16 = d->sum_dtype == SWCB200_BF16;
    p.y = d->y, p.ldy = d->ldy, p.y16 = d->y_dtype == SWCB200_BF16;
    p.rows = (long long)rows, p.gate_rows = d->gate_rows;
    p.cols = cols, p.scale = d->scale, p.inv_cols = 1.0f / (float)cols;
    p.post = {d->post.weight, d->post.bias, d->post.eps, d->post.kind};
    p.pre = {d->pre.weight, d->pre.bias, d->pre.eps, d->pre.kind};

    // chunks of 8: every row of every tensor starts on 16 bytes (bf16) or 32 (fp32), every vector on 16
    bool vec = cols % 8 == 0;
    const auto rows_ok = [&](const void *q, size_t ld, bool is16, bool many) {
        if (q) vec = vec && ((uintptr_t)q & (is16 ? 15u : 31u)) == 0 && (!many || ld % 8 == 0);
    };
    rows_ok(p.x, p.ldx, p.x_how == kBf16, rows > 1);
    rows_ok(p.residual, p.ldr, p.r_how == kBf16, rows > 1);
    rows_ok(p.sum, p.lds, p.s16, rows > 1);
    rows_ok(p.y, p.ldy, p.y16, rows > 1);
    rows_ok(p.gate, p.ldg, p.g_how == kBf16, p.gate_rows != 0);
    for (const float *v : {p.post.w, p.post.b, p.pre.w, p.pre.b}) vec = vec && swc_aligned16(v);
    const int chunks = vec ? cols / 8 : cols;
    const int most = vec ? 4 : 32;  // chunks per thread: 32 elements
    if (chunks <= (vec ? 64 : 256)) {  // rows inside a warp
        p.tpr = 1;
        while (p.tpr < 32 && p.tpr * (vec ? 1 : 8) < chunks) p.tpr *= 2;
        const int per_cta = 128 / p.tpr;
        const unsigned grid = (unsigned)((rows + per_cta - 1) / per_cta);
        const int n = (chunks + p.tpr - 1) / p.tpr;
        SWC_CUDA(ctx, launch<false>(vec, n, grid, 128, ctx->stream, p));
    } else {
        // 256 threads where a thread can hold its share (8192 rows of 4096 with both norms: 60 us, 62 with 128 and 88 with 512 threads);
        // where there are rows for every SM, 16 elements a thread at least, 8 read singly: fewer warps to add up (16384 rows of 2048
        // with both norms 69 -> 56 us)
        int per = (chunks + 255) / 256, least = rows >= 2 * (size_t)ctx->sm_count ? (vec ? 2 : 8) : 1;
        per = per < least ? least : per;
        per = per < most ? per : most;
        int threads = (chunks + per - 1) / per;
        threads = (threads + 31) / 32 * 32;
        p.tpr = threads;
        const int n = (chunks + threads - 1) / threads;
        SWC_CUDA(ctx, launch<true>(vec, n, (unsigned)rows, threads, ctx->stream, p));
    }
    return swc_check_launch(ctx, "norm_residual");
}
