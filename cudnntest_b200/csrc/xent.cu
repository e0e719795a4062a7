// Linear softmax cross entropy with its gradient: driver and row kernels (the products are in xent_gemm.cu).
//
// The logits z = x W^T exist one tile at a time.  Two ways, by size:
//   * kept: where rows or classes are few the logits product is split along the features until the GPU is full; its
//     float parts in the scratch become lse, loss and dz in row kernels.  Unsplit, floats are kept as well where that is
//     cheaper than a fourth product (below);
//   * as exponentials: BF16 without a bias whose dz fits the scratch.  The logits product leaves a maximum and a sum per
//     row and 128 classes and exp(z - maximum) as BF16 in the place of dz; one pass over it makes dz.  Three products
//     (2 n v d flops each) either way;
//   * recomputed: the logits product leaves only the statistics; the gradient then walks the vocabulary in pieces, computes
//     a piece's logits again, turns them into dz in the epilogue, and multiplies dz into dx and dW before the next piece:
//     four products, scratch bounded by desc.scratch_limit.
// dz is held as BF16 (one part; the rounding is that of every BF16 operand, and halves what the two gradient products
// read) or as three BF16 parts (FP32X3).  dbias sums the unrounded dz.  Statistics, lse and losses are FP32, the sum over
// rows FP64.
#include <cmath>

#include "xent.cuh"

namespace wino {

namespace {

constexpr long long XE_DEFAULT_LIMIT = 1ll << 30;
constexpr int XE_ROWS_PER_PART = 32;           // rows per partial column sum of dz

struct RowRule {                               // which rows count
    int v, has_ignore;
    long long ignore_index;
};
__host__ __device__ inline bool row_ignored(const RowRule& r, long long t) { return r.has_ignore && t == r.ignore_index; }
__host__ __device__ inline bool row_counts(const RowRule& r, long long t) { return !row_ignored(r, t) && t >= 0 && t < r.v; }

// ---- operand packing ---------------------------------------------------------------------------------------
// src (rows x cols, pitch ld) -> PLANES x rows x pitch BF16; rows that do not count become zero where target is given
template <typename T, int PLANES>
__global__ void __launch_bounds__(256) xe_pack_kernel(const T* __restrict__ src, long long ld, __nv_bfloat16* __restrict__ dst, long long rows,
                                                      int cols, int pitch, const long long* __restrict__ target, const RowRule rule) {
    const int quads = pitch / 4;
    const long long total = rows * quads;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / quads;
        const int c = (int)(i - r * quads) * 4;
        const bool live = !target || row_counts(rule, target[r]);
        __nv_bfloat16 part[PLANES][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const T v = live && c + e < cols ? src[r * ld + c + e] : from_float<T>(0.f);
            if constexpr (PLANES == 3) xe_split3(to_float<T>(v), part[0][e], part[1][e], part[2][e]);
            else part[0][e] = __float2bfloat16_rn(to_float<T>(v));
        }
#pragma unroll
        for (int q = 0; q < PLANES; ++q)
            *reinterpret_cast<uint2*>(dst + (q * rows + r) * pitch + c) = *reinterpret_cast<const uint2*>(part[q]);
    }
}

// ---- rows --------------------------------------------------------------------------------------------------
struct RowArgs {
    RowRule rule;
    long long n;
    const long long* target;
    float smooth;               // s
    float inv_v;                // 1 / v
    float* lse;                 // scratch
    float* lse_out;             // caller's, or NULL
    float* rowloss;
    int* status;
};

__device__ __forceinline__ void finish_row(const RowArgs& a, long long row, float m, float s, float zsum, float zt) {
    const long long t = a.target[row];
    const bool counts = row_counts(a.rule, t);
    const float lse = m + logf(s);
    float loss = (1.f - a.smooth) * (lse - zt);
    if (a.smooth > 0.f) loss += a.smooth * (lse - zsum * a.inv_v);
    if (!counts) {
        loss = row_ignored(a.rule, t) ? 0.f : __int_as_float(0x7fffffff);
        if (loss != 0.f) atomicCAS(a.status, 0, XE_STATUS_TARGET);
    }
    a.lse[row] = lse;
    a.rowloss[row] = loss;
    if (a.lse_out) a.lse_out[row] = counts ? lse : 0.f;
}

// joins (maximum, sum) pairs
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float mm = fmaxf(m, m2), ref = mm == -INFINITY ? 0.f : mm;
    s = s * xe_ex2((m - ref) * XE_LOG2E) + s2 * xe_ex2((m2 - ref) * XE_LOG2E);
    m = mm;
}

// 32 rows x 8 threads per row over the column tiles' statistics
__global__ void __launch_bounds__(256) xe_rows_from_stats_kernel(const float2* __restrict__ stats, const float* __restrict__ zsum,
                                                                 const float* __restrict__ zt, int tiles, const RowArgs a) {
    __shared__ float2 red[8][32];
    __shared__ float redz[8][32];
    const int l = threadIdx.x % 32, g = threadIdx.x / 32;
    const long long row = (long long)blockIdx.x * 32 + l;
    float m = -INFINITY, s = 0.f, z = 0.f;
    if (row < a.n) {
        for (int i = g; i < tiles; i += 8) {
            const float2 v = stats[(long long)i * a.n + row];
            join(m, s, v.x, v.y);
            if (zsum) z += zsum[(long long)i * a.n + row];
        }
    }
    red[g][l] = make_float2(m, s);
    redz[g][l] = z;
    __syncthreads();
    if (g == 0 && row < a.n) {
        for (int i = 1; i < 8; ++i) {
            join(m, s, red[i][l].x, red[i][l].y);
            z += redz[i][l];
        }
        finish_row(a, row, m, s, z, row_counts(a.rule, a.target[row]) ? zt[row] : 0.f);
    }
}

// one block per row over `splits` partial logits: their sum (with the bias) replaces the first part
__global__ void __launch_bounds__(128) xe_rows_from_logits_kernel(float* __restrict__ z, int splits, int v, int pitch, const float* __restrict__ bias,
                                                                  const RowArgs a) {
    __shared__ float red[3][4];
    __shared__ float zt_s;
    const long long row = blockIdx.x;
    const long long t = a.target[row];
    float* zr = z + row * pitch;
    const long long plane = a.n * pitch;
    float m = -INFINITY, s = 0.f, zsum = 0.f;
    if (threadIdx.x == 0) zt_s = 0.f;
    __syncthreads();
    for (int c = threadIdx.x * 4; c < v; c += 512) {
        float4 q = *reinterpret_cast<const float4*>(zr + c);
        for (int i = 1; i < splits; ++i) {
            const float4 o = *reinterpret_cast<const float4*>(zr + i * plane + c);
            q.x += o.x; q.y += o.y; q.z += o.z; q.w += o.w;
        }
        float e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = c + i < v;
            if (bias && in) e[i] += bias[c + i];
            if (in) zsum += e[i];
            if (c + i == t) zt_s = e[i];
            if (!in) e[i] = -INFINITY;
        }
        *reinterpret_cast<float4*>(zr + c) = make_float4(e[0], e[1], e[2], e[3]);
        const float cm = fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), m2 = fmaxf(m, cm), ref = m2 == -INFINITY ? 0.f : m2;
        s = s * xe_ex2((m - ref) * XE_LOG2E) + ((xe_ex2((e[0] - ref) * XE_LOG2E) + xe_ex2((e[1] - ref) * XE_LOG2E)) +
                                                (xe_ex2((e[2] - ref) * XE_LOG2E) + xe_ex2((e[3] - ref) * XE_LOG2E)));
        m = m2;
    }
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, w), s2 = __shfl_xor_sync(0xffffffffu, s, w);
        join(m, s, m2, s2);
        zsum += __shfl_xor_sync(0xffffffffu, zsum, w);
    }
    if (threadIdx.x % 32 == 0) {
        red[0][threadIdx.x / 32] = m;
        red[1][threadIdx.x / 32] = s;
        red[2][threadIdx.x / 32] = zsum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 4; ++i) {
            join(m, s, red[0][i], red[1][i]);
            zsum += red[2][i];
        }
        finish_row(a, row, m, s, zsum, zt_s);
    }
}

// one block: loss over the rows; every row's own weight in the gradient (rowg) and the factor they share (scale), to which
// dz_factor (XeDzRule's f) belongs
__global__ void __launch_bounds__(1024) xe_loss_kernel(const RowArgs a, int reduction, const float* __restrict__ dloss, float dz_factor,
                                                       float* __restrict__ loss, float* __restrict__ rowg, float* __restrict__ scale) {
    __shared__ double rs[32];
    __shared__ long long rc[32];
    double sum = 0;
    long long count = 0;
    for (long long i = threadIdx.x; i < a.n; i += 1024) {
        const float l = a.rowloss[i];
        sum += l;
        count += row_counts(a.rule, a.target[i]);
        if (reduction == WINO_NONE) loss[i] = l;
    }
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, w);
        count += __shfl_xor_sync(0xffffffffu, count, w);
    }
    if (threadIdx.x % 32 == 0) { rs[threadIdx.x / 32] = sum; rc[threadIdx.x / 32] = count; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 32; ++i) { sum += rs[i]; count += rc[i]; }
        const double inv = reduction == WINO_MEAN ? 1.0 / (double)(count > 0 ? count : 1) : 1.0;
        if (reduction != WINO_NONE) loss[0] = (float)(sum * inv);
        if (rowg) scale[0] = (float)(inv * dz_factor * (dloss && reduction != WINO_NONE ? (double)dloss[0] : 1.0));
    }
    if (!rowg) return;
    for (long long i = threadIdx.x; i < a.n; i += 1024) {
        const float own = dloss && reduction == WINO_NONE ? dloss[i] : 1.f;
        rowg[i] = row_counts(a.rule, a.target[i]) ? own : 0.f;
    }
}

// dz of kept logits: two classes per thread, 32 rows per block, and the block's column sums
template <int PLANES>
__global__ void __launch_bounds__(128) xe_dz_from_logits_kernel(const float* __restrict__ z, int v, int zpitch, long long n, const float* __restrict__ lse,
                                                                const float* __restrict__ rowg, const long long* __restrict__ target, const XeDzRule rule,
                                                                __nv_bfloat16* __restrict__ dz, int dpitch, float* __restrict__ db_part) {
    const unsigned cblocks = (unsigned)(v + 255) / 256, part = blockIdx.x / cblocks;
    const int c = (int)((blockIdx.x % cblocks) * 128 + threadIdx.x) * 2;
    if (c >= v) return;
    const long long r0 = (long long)part * XE_ROWS_PER_PART;
    const long long r1 = r0 + XE_ROWS_PER_PART < n ? r0 + XE_ROWS_PER_PART : n;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll 4
    for (long long r = r0; r < r1; ++r) {
        const float2 q = *reinterpret_cast<const float2*>(z + r * zpitch + c);
        const float l = lse[r], g = rowg[r];
        const long long t = target[r];
        float a = xe_ex2((q.x - l) * XE_LOG2E) * rule.pf - rule.smooth_all, b = xe_ex2((q.y - l) * XE_LOG2E) * rule.pf - rule.smooth_all;
        if (t == c) a -= rule.smooth_t;
        if (t == c + 1) b -= rule.smooth_t;
        a = g == 0.f ? 0.f : a * g;                       // a row that does not count: exactly 0, whatever its logits
        b = g == 0.f || c + 1 >= v ? 0.f : b * g;
        s0 += a;
        s1 += b;
#pragma unroll
        for (int p = 0; p < PLANES; ++p) {
            const __nv_bfloat162 o = __floats2bfloat162_rn(a, b);
            *reinterpret_cast<__nv_bfloat162*>(dz + (p * n + r) * dpitch + c) = o;
            a -= __low2float(o);
            b -= __high2float(o);
        }
    }
    if (db_part) *reinterpret_cast<float2*>(db_part + (long long)part * dpitch + c) = make_float2(s0, s1);
}

// exponentials (kept in the place of dz) -> dz, eight classes per thread.  The target's probability comes from its logit in
// FP32, the others' from the rounded exponential: off by one more BF16 rounding.
__global__ void __launch_bounds__(256) xe_dz_from_exp_kernel(__nv_bfloat16* __restrict__ dz, int pitch, long long n, const float2* __restrict__ stats,
                                                             const float* __restrict__ zt, const float* __restrict__ lse, const float* __restrict__ rowg,
                                                             const long long* __restrict__ target, const XeDzRule rule) {
    const int octs = pitch / 8;
    const long long total = n * octs;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / octs;
        const int c = (int)(i - r * octs) * 8;
        uint4* at = reinterpret_cast<uint4*>(dz + r * pitch + c);
        const float g = rowg[r];
        uint4 q = make_uint4(0, 0, 0, 0);
        if (g != 0.f) {
            q = *at;
            const float l = lse[r], f = xe_ex2((stats[c / XE_STAT_COLS * n + r].x - l) * XE_LOG2E) * rule.pf;
            const long long t = target[r] - c;
            uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float a = __uint_as_float(w[e] << 16) * f - rule.smooth_all, b = __uint_as_float(w[e] & 0xffff0000u) * f - rule.smooth_all;
                if (t >> 1 == e) {
                    const float pt = xe_ex2((zt[r] - l) * XE_LOG2E) * rule.pf - rule.smooth_all - rule.smooth_t;
                    if (t & 1) b = pt; else a = pt;
                }
                const __nv_bfloat162 o = __floats2bfloat162_rn(a * g, b * g);
                w[e] = *reinterpret_cast<const uint32_t*>(&o);
            }
            q = make_uint4(w[0], w[1], w[2], w[3]);
        }
        *at = q;
    }
}

__global__ void __launch_bounds__(256) xe_db_kernel(const float* __restrict__ part, int parts, int pitch, int cols, const float* __restrict__ scale,
                                                    float* __restrict__ db) {
    __shared__ float red[8][32];
    const int l = threadIdx.x % 32, g = threadIdx.x / 32, c = blockIdx.x * 32 + l;
    float s = 0.f;
    if (c < cols)
        for (int i = g; i < parts; i += 8) s += part[(long long)i * pitch + c];
    red[g][l] = s;
    __syncthreads();
    if (g == 0 && c < cols) {
        for (int i = 1; i < 8; ++i) s += red[i][l];
        db[c] = s * *scale;
    }
}

// out (rows x cols, pitch ld) = sum of `splits` float buffers (pitch `pitch`)
template <typename T>
__global__ void __launch_bounds__(256) xe_finish_kernel(const float* __restrict__ part, int splits, long long rows, int cols, int pitch, T* __restrict__ out,
                                                        long long ld) {
    const int quads = (cols + 3) / 4;
    const long long total = rows * quads, plane = rows * pitch;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / quads;
        const int c = (int)(i - r * quads) * 4;
        float4 q = *reinterpret_cast<const float4*>(part + r * pitch + c);
        for (int s = 1; s < splits; ++s) {
            const float4 o = *reinterpret_cast<const float4*>(part + s * plane + r * pitch + c);
            q.x += o.x; q.y += o.y; q.z += o.z; q.w += o.w;
        }
        const float e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c + k < cols) out[r * ld + c + k] = from_float<T>(e[k]);
    }
}

unsigned loop_blocks(long long items) {
    const long long b = (items + 255) / 256, most = 16ll * sm_count();
    return (unsigned)(b < 1 ? 1 : b < most ? b : most);
}

// ---- plan ----------------------------------------------------------------------------------------------------
struct Plan {
    int planes, es, dp;
    long long ldx, ldw, lddx, lddw;
    bool pack_x, pack_w;
    bool kept, exps;                     // floats of all logits, BF16 exponentials of all logits (else recomputed by piece)
    int splits_z, splits_dx, splits_dw;
    int zpitch, piece, pieces, dzpitch;
    bool dx_direct, dw_direct;           // the product's epilogue stores the caller's matrix
    int dpitch;                          // of float dx / dw buffers in the scratch
    size_t off_x, off_w, off_z, off_zsum, off_zt, off_lse, off_rowloss, off_rowg, off_scale, off_dz, off_db, off_dx, off_dw, total;
};

// parts of the contraction so that tiles * parts fills the CTA pairs, each with at least four ring slots of work
int split_count(long long tiles, long long chunks, int partial_products) {
    const long long pairs = sm_count() / 2;
    if (tiles >= pairs || tiles == 0) return 1;
    long long s = pairs / tiles;
    if (s > chunks * partial_products / 4) s = chunks * partial_products / 4;
    if (s > chunks) s = chunks;
    return (int)(s < 1 ? 1 : s);
}

long long tiles_of(long long rows, long long cols) { return ((rows + XE_BM - 1) / XE_BM) * ((cols + XE_BN - 1) / XE_BN); }

int make_plan(const wino_xent_desc* d, bool grad, Plan* out) {
    if (!d) return fail(WINO_E_BADARG, "xent: NULL descriptor");
    if (d->n < 0 || d->d <= 0 || d->v <= 0) return fail(WINO_E_BADARG, "xent: n must be at least 0, d and v positive");
    if (d->d > (1 << 30) || d->v > (1 << 30) || d->n > (1 << 30)) return fail(WINO_E_UNSUPPORTED, "xent: extents above 2^30");
    if (d->dtype != WINO_BF16 && d->dtype != WINO_FP32X3) return fail(WINO_E_UNSUPPORTED, "xent: dtype must be WINO_BF16 or WINO_FP32X3");
    if (d->has_bias != 0 && d->has_bias != 1) return fail(WINO_E_BADARG, "xent: has_bias must be 0 or 1");
    if (d->has_ignore != 0 && d->has_ignore != 1) return fail(WINO_E_BADARG, "xent: has_ignore must be 0 or 1");
    if (d->reduction != WINO_MEAN && d->reduction != WINO_SUM && d->reduction != WINO_NONE) return fail(WINO_E_BADARG, "xent: bad reduction %d", d->reduction);
    if (!(d->label_smoothing >= 0.f && d->label_smoothing <= 1.f)) return fail(WINO_E_BADARG, "xent: label_smoothing must lie in [0, 1]");
    if (d->scratch_limit < 0) return fail(WINO_E_BADARG, "xent: negative scratch_limit");
    Plan p = {};
    const bool bf16 = d->dtype == WINO_BF16;
    p.planes = bf16 ? 1 : 3;
    p.es = bf16 ? 2 : 4;
    const int products = bf16 ? 1 : 6;
    const long long lds[4] = {d->ldx, d->ldw, d->lddx, d->lddw};
    long long* dst[4] = {&p.ldx, &p.ldw, &p.lddx, &p.lddw};
    for (int i = 0; i < 4; ++i) {
        if (lds[i] != 0 && (lds[i] < d->d || lds[i] > (1ll << 36))) return fail(WINO_E_BADARG, "xent: pitch %lld of a row of %d elements", lds[i], d->d);
        *dst[i] = lds[i] ? lds[i] : d->d;
    }
    const long long n = d->n, v = d->v, limit = d->scratch_limit ? d->scratch_limit : XE_DEFAULT_LIMIT;
    p.dp = round_up(d->d, 8);
    // TMA wants rows that start on 16-byte boundaries; rows that do not count must not reach dW, whatever they hold
    p.pack_x = !bf16 || p.ldx % 8 != 0 || (grad && d->has_ignore);
    p.pack_w = !bf16 || p.ldw % 8 != 0;
    const long long kd = (d->d + XE_BK - 1) / XE_BK;
    p.splits_z = split_count(tiles_of(n, v), kd, products);
    p.zpitch = round_up(d->v, 4);
    const long long dz_bytes = n * round_up(d->v, 8) * 2ll * p.planes, z_bytes = n * p.zpitch * 4ll * p.splits_z;
    // Kept floats cost 14 bytes a logit (18 in three parts) against 2 d flops (12 d) for another product: at the measured
    // 6.5 TB/s and 1.4 PFLOP/s the product is the dearer one from d = 1000 (200) on.
    if (p.splits_z > 1) p.kept = true;
    else if (grad && bf16 && !d->has_bias && dz_bytes <= limit) p.exps = true;
    else p.kept = grad && z_bytes + dz_bytes <= limit && d->d >= (bf16 ? 1024 : 256);
    if (!p.kept) p.splits_z = 1;
    p.piece = d->v;
    p.pieces = 1;
    if (grad && !p.kept && !p.exps) {
        long long most = limit / (n > 0 ? n * 2 * p.planes : 1) / XE_BN * XE_BN;
        if (most < XE_BN) most = XE_BN;
        if (most < v) {
            p.pieces = (int)((v + most - 1) / most);
            p.piece = (int)round_up_ll((v + p.pieces - 1) / p.pieces, XE_BN);
            p.pieces = (int)((v + p.piece - 1) / p.piece);
        }
    }
    p.dzpitch = round_up(p.piece, 8);
    p.dpitch = round_up(d->d, 4);
    p.splits_dx = split_count(tiles_of(n, d->d), (p.piece + XE_BK - 1) / XE_BK, products);
    p.splits_dw = split_count(tiles_of(p.piece, d->d), (n + XE_BK - 1) / XE_BK, products);
    p.dx_direct = p.splits_dx == 1 && (p.pieces == 1 || !bf16) && (p.lddx * p.es) % 16 == 0;
    p.dw_direct = p.splits_dw == 1 && (p.lddw * p.es) % 16 == 0;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off += (bytes + 255) / 256 * 256;
        return at;
    };
    const size_t un = (size_t)n;
    p.off_lse = take(un * 4);
    p.off_rowloss = take(un * 4);
    p.off_rowg = take(un * 4);
    p.off_zt = take(un * 4);
    p.off_scale = take(4);
    const size_t vtiles = (size_t)((v + XE_STAT_COLS - 1) / XE_STAT_COLS);
    p.off_zsum = take(p.kept || d->label_smoothing <= 0.f ? 0 : vtiles * un * 4);
    p.off_z = take(p.kept ? un * p.zpitch * 4 * p.splits_z : vtiles * un * 8);
    p.off_x = take(p.pack_x ? un * p.dp * 2 * p.planes : 0);
    p.off_w = take(p.pack_w ? (size_t)v * p.dp * 2 * p.planes : 0);
    if (grad) {
        p.off_dz = take(un * p.dzpitch * 2 * p.planes);
        p.off_db = take(d->has_bias ? (size_t)((n + XE_ROWS_PER_PART - 1) / XE_ROWS_PER_PART) * p.dzpitch * 4 : 0);
        p.off_dx = take(p.dx_direct ? 0 : un * p.dpitch * 4 * p.splits_dx);
        p.off_dw = take(p.dw_direct ? 0 : (size_t)p.piece * p.dpitch * 4 * p.splits_dw);
    }
    p.total = off + 256;
    *out = p;
    return WINO_OK;
}

int pack(const wino_xent_desc& d, const Plan& p, const void* src, long long ld, long long rows, void* dst, const long long* target, const RowRule& rule,
         cudaStream_t st) {
    const unsigned blocks = loop_blocks(rows * (p.dp / 4));
    count_launch();
    if (d.dtype == WINO_BF16)
        xe_pack_kernel<__nv_bfloat16, 1><<<blocks, 256, 0, st>>>((const __nv_bfloat16*)src, ld, (__nv_bfloat16*)dst, rows, d.d, p.dp, target, rule);
    else
        xe_pack_kernel<float, 3><<<blocks, 256, 0, st>>>((const float*)src, ld, (__nv_bfloat16*)dst, rows, d.d, p.dp, target, rule);
    WINO_CUDA_CHECK(cudaGetLastError());
    return WINO_OK;
}

// one gradient product: into the caller's matrix where its epilogue can store it, else through float buffers
int grad_product(const Plan& p, const wino_xent_desc& d, const XeOperand& a, const XeOperand& b, long long rows, long long k, bool direct, int splits,
                 bool first, bool last, void* out, long long ld, float* buf, const float* scale, cudaStream_t st) {
    XeOutput o;
    int rc;
    o.add = !first;
    o.scale = scale;
    if (direct) {
        o.ptr = out;
        o.pitch = ld;
        return xe_gemm(d.dtype == WINO_BF16 ? XE_BF16 : XE_F32, a, b, rows, d.d, k, o, st);
    }
    o.ptr = buf;
    o.pitch = p.dpitch;
    const long long chunks = (k + XE_BK - 1) / XE_BK;          // a short last piece adds to fewer of the parts
    o.splits = chunks < splits ? (int)chunks : splits;
    if ((rc = xe_gemm(XE_F32, a, b, rows, d.d, k, o, st))) return rc;
    if (!last) return WINO_OK;
    const unsigned blocks = loop_blocks(rows * ((d.d + 3) / 4));
    count_launch();
    if (d.dtype == WINO_BF16) xe_finish_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(buf, splits, rows, d.d, p.dpitch, (__nv_bfloat16*)out, ld);
    else xe_finish_kernel<float><<<blocks, 256, 0, st>>>(buf, splits, rows, d.d, p.dpitch, (float*)out, ld);
    WINO_CUDA_CHECK(cudaGetLastError());
    return WINO_OK;
}

int xent(const wino_xent_desc* dd, bool grad, const void* x, const void* w, const float* bias, const long long* target, const float* dloss, float* loss,
         float* lse, void* dx, void* dw, float* db, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    Plan p;
    int rc = make_plan(dd, grad, &p);
    if (rc) return rc;
    const wino_xent_desc& d = *dd;
    const bool rows = d.n > 0;
    if ((rows && (!x || !target)) || !w || (!loss && (rows || d.reduction != WINO_NONE))) return fail(WINO_E_BADARG, "xent: NULL pointer");
    if (d.has_bias && !bias) return fail(WINO_E_BADARG, "xent: the descriptor has a bias, the call has none");
    if (db && !d.has_bias) return fail(WINO_E_BADARG, "xent: gradient of a bias the descriptor does not have");
    if (((uintptr_t)x | (uintptr_t)w | (uintptr_t)bias | (uintptr_t)dx | (uintptr_t)dw | (uintptr_t)workspace) & 15)
        return fail(WINO_E_BADARG, "xent: matrices, bias and workspace must be 16-byte aligned");
    if (((uintptr_t)target & 7) || (((uintptr_t)loss | (uintptr_t)lse | (uintptr_t)dloss | (uintptr_t)db) & 3)) return fail(WINO_E_BADARG, "xent: misaligned pointer");
    if (!workspace || workspace_bytes < p.total) return fail(WINO_E_WORKSPACE, "xent: workspace of %zu bytes, %zu needed", workspace_bytes, p.total);
    if ((rc = check_device())) return rc;
    const long long n = d.n, v = d.v;
    if (!rows) {        // no rows: loss 0, gradients of W and bias 0
        if (d.reduction != WINO_NONE) WINO_CUDA_CHECK(cudaMemsetAsync(loss, 0, 4, st));
        if (dw) WINO_CUDA_CHECK(cudaMemset2DAsync(dw, (size_t)p.lddw * p.es, 0, (size_t)d.d * p.es, (size_t)v, st));
        if (db) WINO_CUDA_CHECK(cudaMemsetAsync(db, 0, (size_t)v * 4, st));
        return WINO_OK;
    }
    char* ws = static_cast<char*>(workspace);
    auto f = [&](size_t off) { return reinterpret_cast<float*>(ws + off); };

    const RowRule rule = {d.v, d.has_ignore, d.ignore_index};
    XeOperand ox = {x, n, d.d, p.ldx, n * p.ldx, 1, false}, ow = {w, v, d.d, p.ldw, v * p.ldw, 1, false};
    if (p.pack_x) {
        if ((rc = pack(d, p, x, p.ldx, n, ws + p.off_x, grad && d.has_ignore ? target : nullptr, rule, st))) return rc;
        ox = {ws + p.off_x, n, d.d, p.dp, n * p.dp, p.planes, false};
    }
    if (p.pack_w) {
        if ((rc = pack(d, p, w, p.ldw, v, ws + p.off_w, nullptr, rule, st))) return rc;
        ow = {ws + p.off_w, v, d.d, p.dp, v * p.dp, p.planes, false};
    }

    RowArgs ra;
    ra.rule = rule; ra.n = n; ra.target = target;
    ra.smooth = d.label_smoothing; ra.inv_v = (float)(1.0 / (double)v);
    ra.lse = f(p.off_lse); ra.lse_out = lse; ra.rowloss = f(p.off_rowloss);
    if ((rc = status_word(&ra.status))) return rc;
    const float* b = d.has_bias ? bias : nullptr;
    XeOutput oz;
    if (p.kept) {
        oz.ptr = ws + p.off_z;
        oz.pitch = p.zpitch;
        oz.splits = p.splits_z;
        if ((rc = xe_gemm(XE_F32, ox, ow, n, v, d.d, oz, st))) return rc;
        count_launch();
        xe_rows_from_logits_kernel<<<(unsigned)n, 128, 0, st>>>(f(p.off_z), p.splits_z, d.v, p.zpitch, b, ra);
    } else {
        oz.bias = b;
        oz.target = target;
        oz.stats = reinterpret_cast<float2*>(ws + p.off_z);
        oz.zsum = d.label_smoothing > 0.f ? f(p.off_zsum) : nullptr;
        oz.zt = f(p.off_zt);
        if (p.exps) {
            oz.ptr = ws + p.off_dz;
            oz.pitch = p.dzpitch;
        }
        if ((rc = xe_gemm(p.exps ? XE_STATS_E : XE_STATS, ox, ow, n, v, d.d, oz, st))) return rc;
        count_launch();
        xe_rows_from_stats_kernel<<<(unsigned)((n + 31) / 32), 256, 0, st>>>(oz.stats, oz.zsum, oz.zt, (int)((v + XE_STAT_COLS - 1) / XE_STAT_COLS), ra);
    }
    WINO_CUDA_CHECK(cudaGetLastError());
    XeDzRule dzr;
    const float s = d.label_smoothing, dz_factor = s <= 0.5f ? 1.f - s : 1.f;
    dzr.pf = 1.f / dz_factor;
    dzr.smooth_t = s <= 0.5f ? 1.f : 1.f - s;
    dzr.smooth_all = (float)((double)s / (double)v / (double)dz_factor);
    count_launch();
    xe_loss_kernel<<<1, 1024, 0, st>>>(ra, d.reduction, dloss, dz_factor, loss, grad ? f(p.off_rowg) : nullptr, f(p.off_scale));
    WINO_CUDA_CHECK(cudaGetLastError());
    if (!grad || (!dx && !dw && !db)) return WINO_OK;

    const int parts = (int)((n + XE_ROWS_PER_PART - 1) / XE_ROWS_PER_PART);
    __nv_bfloat16* dz = reinterpret_cast<__nv_bfloat16*>(ws + p.off_dz);
    float* db_part = db ? f(p.off_db) : nullptr;
    for (int i = 0; i < p.pieces; ++i) {
        const int v0 = i * p.piece, vc = d.v - v0 < p.piece ? d.v - v0 : p.piece;
        XeOperand wp = ow;                 // the piece's rows of W
        wp.ptr = static_cast<const char*>(ow.ptr) + (size_t)v0 * ow.pitch * 2;
        wp.rows = vc;
        if (p.kept) {
            const unsigned grid = (unsigned)((vc + 255) / 256) * (unsigned)parts;
            count_launch();
            if (p.planes == 1)
                xe_dz_from_logits_kernel<1><<<grid, 128, 0, st>>>(f(p.off_z), vc, p.zpitch, n, ra.lse, f(p.off_rowg), target, dzr, dz, p.dzpitch, db_part);
            else
                xe_dz_from_logits_kernel<3><<<grid, 128, 0, st>>>(f(p.off_z), vc, p.zpitch, n, ra.lse, f(p.off_rowg), target, dzr, dz, p.dzpitch, db_part);
            WINO_CUDA_CHECK(cudaGetLastError());
        } else if (p.exps) {
            count_launch();
            xe_dz_from_exp_kernel<<<loop_blocks(n * (p.dzpitch / 8)), 256, 0, st>>>(dz, p.dzpitch, n, oz.stats, oz.zt, ra.lse, f(p.off_rowg), target, dzr);
            WINO_CUDA_CHECK(cudaGetLastError());
        } else {
            XeOutput o;
            o.ptr = dz; o.pitch = p.dzpitch;
            o.bias = b ? b + v0 : nullptr;
            o.target = target; o.col_base = v0;
            o.lse = ra.lse; o.rowg = f(p.off_rowg); o.rule = dzr;
            o.db_part = db_part; o.db_pitch = p.dzpitch;
            if ((rc = xe_gemm(XE_DZ, ox, wp, n, vc, d.d, o, st))) return rc;
        }
        if (db) {
            count_launch();
            xe_db_kernel<<<(unsigned)((vc + 31) / 32), 256, 0, st>>>(db_part, parts, p.dzpitch, vc, f(p.off_scale), db + v0);
            WINO_CUDA_CHECK(cudaGetLastError());
        }
        XeOperand odz = {dz, n, vc, p.dzpitch, n * p.dzpitch, p.planes, false};
        if (dx) {
            XeOperand wr = wp;
            wr.along_rows = true;
            if ((rc = grad_product(p, d, odz, wr, n, vc, p.dx_direct, p.splits_dx, i == 0, i == p.pieces - 1, dx, p.lddx, f(p.off_dx), f(p.off_scale), st))) return rc;
        }
        if (dw) {
            XeOperand zr = odz, xr = ox;
            zr.along_rows = xr.along_rows = true;
            if ((rc = grad_product(p, d, zr, xr, vc, n, p.dw_direct, p.splits_dw, true, true, static_cast<char*>(dw) + (size_t)v0 * p.lddw * p.es, p.lddw,
                                   f(p.off_dw), f(p.off_scale), st)))
                return rc;
        }
    }
    return WINO_OK;
}

}  // namespace

}  // namespace wino

extern "C" {

size_t wino_xent_workspace_bytes(const wino_xent_desc* d, int grad) {
    wino::Plan p;
    return wino::make_plan(d, grad != 0, &p) == WINO_OK ? p.total : 0;
}

int wino_xent_forward(const wino_xent_desc* d, const void* x, const void* w, const float* bias, const long long* target, float* loss, float* lse,
                      void* workspace, size_t workspace_bytes, wino_stream_t stream) {
    return wino::xent(d, false, x, w, bias, target, nullptr, loss, lse, nullptr, nullptr, nullptr, workspace, workspace_bytes, (cudaStream_t)stream);
}

int wino_xent_grad(const wino_xent_desc* d, const void* x, const void* w, const float* bias, const long long* target, const float* dloss, float* loss,
                   float* lse, void* dx, void* dw, float* dbias, void* workspace, size_t workspace_bytes, wino_stream_t stream) {
    return wino::xent(d, true, x, w, bias, target, dloss, loss, lse, dx, dw, dbias, workspace, workspace_bytes, (cudaStream_t)stream);
}

}  // extern "C"
