// Linear softmax cross entropy with its gradient: driver and row kernels (the products are in xent_gemm.cu and xent_thin.cu).
//
// The logits z = x W^T exist in the workspace at most, as far as desc.scratch_limit allows.  Ways, by size (build_plan):
//   * few products, few rows, few classes: FP32 kernels on the caller's matrices (xe_tiny_kernel, xe_small_*, xe_few_*);
//   * kept: where rows or classes are few the logits product is split along the features until the GPU is full; its
//     float parts in the scratch become lse, loss and dz in row kernels.  Unsplit, floats are kept as well where that is
//     cheaper than a fourth product.  FP32X3 with up to 128 rows or classes: the longer matrix is split into BF16 parts
//     inside its products (xent_thin.cu), the others beforehand;
//   * as exponentials: BF16 without a bias whose dz fits the scratch.  The logits product leaves a maximum and a sum per
//     row and 128 classes and exp(z - maximum) in 16 bits in the place of dz; one pass over it makes dz.  Three products
//     (2 n v d flops each) in all these ways;
//   * recomputed: the logits product leaves only the statistics; the gradient then walks the vocabulary in pieces, computes
//     a piece's logits again, turns them into dz in the epilogue, and multiplies dz into dx and dW before the next piece:
//     four products, scratch bounded by desc.scratch_limit.
// dz is held as BF16 (one part; the rounding is that of every BF16 operand, and halves what the two gradient products
// read) or as three BF16 parts (FP32X3).  dbias sums the unrounded dz.  Statistics, lse and losses are FP32, the sum over
// rows FP64.
#include <cmath>
#include <cstring>
#include <type_traits>

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
struct PackJob {
    const void* src;
    long long ld, rows;
    __nv_bfloat16* dst;
    const long long* target;            // rows that do not count become zero where target is given
};
// four neighbouring elements, `left` of which exist, by the widest loads that the address allows
template <typename T> using Wide = std::conditional_t<sizeof(T) == 4, float4, uint2>;
template <typename T> using Pair = std::conditional_t<sizeof(T) == 4, float2, uint32_t>;
template <typename T>
__device__ __forceinline__ void load4(T (&v)[4], const T* p, int left) {
    const unsigned at = (unsigned)(uintptr_t)p;
    if (left < 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < left ? p[e] : from_float<T>(0.f);
    } else if (at % (4 * sizeof(T)) == 0) {
        const Wide<T> q = *reinterpret_cast<const Wide<T>*>(p);
        memcpy(v, &q, sizeof(q));
    } else if (at % (2 * sizeof(T)) == 0) {
        const Pair<T> q[2] = {reinterpret_cast<const Pair<T>*>(p)[0], reinterpret_cast<const Pair<T>*>(p)[1]};
        memcpy(v, q, sizeof(q));
    } else {
        v[0] = p[0];
        const Pair<T> q = *reinterpret_cast<const Pair<T>*>(p + 1);
        memcpy(v + 1, &q, sizeof(q));
        v[3] = p[3];
    }
}
template <typename T>
__device__ __forceinline__ void load4_aligned(float (&v)[4], const T* p) {
    const Wide<T> q = *reinterpret_cast<const Wide<T>*>(p);
    T t[4];
    memcpy(t, &q, sizeof(q));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = to_float<T>(t[e]);
}
template <typename T>
__device__ __forceinline__ void load4f(float (&v)[4], const T* p, int left) {
    T t[4];
    load4(t, p, left);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = to_float<T>(t[e]);
}

// The same for BF16 rows that start anywhere: a warp copies 256 columns of a row, neighbouring lanes neighbouring elements (PAIRS:
// pairs of them, where every row starts on 4 bytes), so that both sides are whole lines whatever the pitch
template <bool PAIRS>
__global__ void __launch_bounds__(256) xe_pack_rows_kernel(const PackJob j0, const PackJob j1, int cols, int pitch, const RowRule rule) {
    pdl_wait();
    const int lane = threadIdx.x % 32;
    const unsigned chunks = (unsigned)(pitch + 255) / 256;
    const long long items0 = j0.rows * chunks, total = items0 + j1.rows * chunks;
    for (long long w = (long long)blockIdx.x * 8 + threadIdx.x / 32; w < total; w += (long long)gridDim.x * 8) {
        const bool second = w >= items0;
        const PackJob& j = second ? j1 : j0;
        const long long i = second ? w - items0 : w, r = i < (1ll << 32) ? (long long)((unsigned)i / chunks) : i / chunks;
        const int c0 = (int)(i - r * chunks) * 256;
        const bool live = !j.target || row_counts(rule, j.target[r]);
        const unsigned short* src = static_cast<const unsigned short*>(j.src) + r * j.ld + c0;
        unsigned short* dst = reinterpret_cast<unsigned short*>(j.dst) + r * pitch + c0;
        const int have = live ? cols - c0 : 0, want = pitch - c0;
        if (PAIRS) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = (e * 32 + lane) * 2;
                v[e] = c + 2 <= have ? *reinterpret_cast<const uint32_t*>(src + c) : c < have ? src[c] : 0u;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if ((e * 32 + lane) * 2 < want) *reinterpret_cast<uint32_t*>(dst + (e * 32 + lane) * 2) = v[e];
        } else {
            unsigned short v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e * 32 + lane < have ? src[e * 32 + lane] : (unsigned short)0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e * 32 + lane < want) dst[e * 32 + lane] = v[e];
        }
    }
}

// src (rows x cols, pitch ld) -> PLANES x rows x pitch BF16, four columns per thread, for up to two matrices
template <typename T, int PLANES>
__global__ void __launch_bounds__(256) xe_pack_kernel(const PackJob j0, const PackJob j1, int cols, int pitch, const RowRule rule) {
    pdl_wait();
    const unsigned quads = (unsigned)pitch / 4;
    const long long items0 = j0.rows * quads, total = items0 + j1.rows * quads;
    for (long long k = (long long)blockIdx.x * 256 + threadIdx.x; k < total; k += (long long)gridDim.x * 256) {
        const bool second = k >= items0;
        const PackJob& j = second ? j1 : j0;
        const long long i = second ? k - items0 : k;
        const long long r = i < (1ll << 32) ? (long long)((unsigned)i / quads) : i / quads;
        const int c = (int)(i - r * quads) * 4;
        const bool live = !j.target || row_counts(rule, j.target[r]);
        const T* src = static_cast<const T*>(j.src) + r * j.ld + c;
        T v[4];
        load4(v, src, live ? cols - c : 0);
        alignas(8) __nv_bfloat16 part[PLANES][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (PLANES == 3) xe_split3(to_float<T>(v[e]), part[0][e], part[1][e], part[2][e]);
            else part[0][e] = __float2bfloat16_rn(to_float<T>(v[e]));
        }
#pragma unroll
        for (int q = 0; q < PLANES; ++q)
            *reinterpret_cast<uint2*>(j.dst + (q * j.rows + r) * pitch + c) = *reinterpret_cast<const uint2*>(part[q]);
    }
}

// ---- rows --------------------------------------------------------------------------------------------------
struct RowArgs {
    RowRule rule;
    long long n;
    const long long* target;
    const float* dloss;         // n upstream gradients (WINO_NONE), or NULL
    float smooth;               // s
    float inv_v;                // 1 / v
    float* lse;                 // scratch
    float* lse_out;             // caller's, or NULL
    float* rowloss;             // scratch, or the caller's (WINO_NONE)
    float* rowg;                // a row's own weight in the gradient; 0: does not count
    XeLoss loss;                // written by the block that finishes last; loss NULL: left to the rows, or to a later kernel
    int* count;                 // [0] rows that count, [1] blocks that are done (both set to 0 by the kernel before)
    int* status;
};

// one thread per row: loss, lse, weight.  Returns whether the row counts.
__device__ __forceinline__ bool finish_row(const RowArgs& a, long long row, float lse, float zsum, float zt) {
    const long long t = a.target[row];
    const bool counts = row_counts(a.rule, t);
    float loss = (1.f - a.smooth) * (lse - zt);
    if (a.smooth > 0.f) loss += a.smooth * (lse - zsum * a.inv_v);
    if (!counts) {
        loss = row_ignored(a.rule, t) ? 0.f : __int_as_float(0x7fffffff);
        if (loss != 0.f) atomicCAS(a.status, 0, XE_STATUS_TARGET);
    }
    a.lse[row] = lse;
    a.rowloss[row] = loss;
    a.rowg[row] = counts ? (a.dloss ? a.dloss[row] : 1.f) : 0.f;
    if (a.lse_out) a.lse_out[row] = counts ? lse : 0.f;
    return counts;
}

// The block that finishes last sums the rows' losses (in the same order whichever block that is).  All threads call it; where
// warp 0 has written the block's losses, only that warp waits for its stores, else all do (EVERY_WARP).
template <int THREADS, bool EVERY_WARP = false>
__device__ __forceinline__ void finish_loss(const RowArgs& a) {
    if (!a.loss.loss) return;
    __shared__ int last;
    if (EVERY_WARP) {
        __threadfence();
        __syncthreads();
    }
    if (threadIdx.x < 32) {
        __threadfence();
        __syncwarp();
        if (threadIdx.x == 0) last = atomicAdd(a.count + 1, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    xe_sum_losses<THREADS>(a.loss);
}

// joins (maximum, sum) pairs
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
    const float mm = fmaxf(m, m2), ref = mm == -INFINITY ? 0.f : mm;
    s = s * xe_ex2((m - ref) * XE_LOG2E) + s2 * xe_ex2((m2 - ref) * XE_LOG2E);
    m = mm;
}

// 32 rows x 8 threads per row over the column tiles' statistics, eight tiles in flight per thread
__global__ void __launch_bounds__(256) xe_rows_from_stats_kernel(const float2* __restrict__ stats, const float* __restrict__ zsum,
                                                                 const float* __restrict__ zt, int tiles, const RowArgs a) {
    pdl_wait();
    __shared__ float2 red[8][32];
    __shared__ float redz[8][32];
    const int l = threadIdx.x % 32, g = threadIdx.x / 32;
    const long long row = (long long)blockIdx.x * 32 + l;
    float m = -INFINITY, s = 0.f, z = 0.f;
    if (row < a.n) {
        for (int i = g; i < tiles; i += 64) {
            float2 v[8];
            float mm = m;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = i + 8 * e < tiles ? stats[(long long)(i + 8 * e) * a.n + row] : make_float2(-INFINITY, 0.f);
                mm = fmaxf(mm, v[e].x);
            }
            const float ref = mm == -INFINITY ? 0.f : mm;
            s *= xe_ex2((m - ref) * XE_LOG2E);
            m = mm;
#pragma unroll
            for (int e = 0; e < 8; ++e) s += v[e].y * xe_ex2((v[e].x - ref) * XE_LOG2E);
            if (zsum) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (i + 8 * e < tiles) z += zsum[(long long)(i + 8 * e) * a.n + row];
            }
        }
    }
    red[g][l] = make_float2(m, s);
    redz[g][l] = z;
    __syncthreads();
    if (g == 0) {
        bool counts = false;
        if (row < a.n) {
            for (int i = 1; i < 8; ++i) {
                join(m, s, red[i][l].x, red[i][l].y);
                z += redz[i][l];
            }
            counts = finish_row(a, row, m + logf(s), z, row_counts(a.rule, a.target[row]) ? zt[row] : 0.f);
        }
        const unsigned live = __ballot_sync(0xffffffffu, counts);
        if (l == 0) atomicAdd(a.count, __popc(live));
    }
    finish_loss<256>(a);
}

// bias of columns c ... c + 3 (c a multiple of 4, the base 16-byte aligned); columns past v become -inf
__device__ __forceinline__ void add_bias(float (&e)[4], int c, int v, const float* __restrict__ bias) {
    if (c + 4 <= v) {
        if (bias) {
            const float4 b = __ldg(reinterpret_cast<const float4*>(bias + c));
            e[0] += b.x; e[1] += b.y; e[2] += b.z; e[3] += b.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (c + k >= v) e[k] = -INFINITY;
            else if (bias) e[k] += bias[c + k];
        }
    }
}

// sum of the parts of four logits and the bias
__device__ __forceinline__ void gather_logits(float (&e)[4], const float* zr, long long plane, int splits, int c, int v,
                                              const float* __restrict__ bias) {
    float4 q = *reinterpret_cast<const float4*>(zr + c);
    for (int i = 1; i + 8 <= splits; i += 8) {
        float4 o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = *reinterpret_cast<const float4*>(zr + (i + k) * plane + c);
#pragma unroll
        for (int k = 0; k < 8; ++k) { q.x += o[k].x; q.y += o[k].y; q.z += o[k].z; q.w += o[k].w; }
    }
    {
        const int i0 = 1 + (splits - 1) / 8 * 8;
        float4 o[7];                                     // the rest, in flight together
#pragma unroll
        for (int k = 0; k < 7; ++k)
            if (i0 + k < splits) o[k] = *reinterpret_cast<const float4*>(zr + (i0 + k) * plane + c);
#pragma unroll
        for (int k = 0; k < 7; ++k)
            if (i0 + k < splits) { q.x += o[k].x; q.y += o[k].y; q.z += o[k].z; q.w += o[k].w; }
    }
    e[0] = q.x; e[1] = q.y; e[2] = q.z; e[3] = q.w;
    add_bias(e, c, v, bias);
}

// logits of `count` groups of four columns, `step` columns apart; all loads of an unsplit product in flight together
template <bool SPLIT, int COUNT>
__device__ __forceinline__ void gather_groups(float (&e)[COUNT][4], const float* zr, long long plane, int splits, int c0, int step, int v,
                                              const float* __restrict__ bias) {
    if constexpr (!SPLIT) {
        float4 q[COUNT];
#pragma unroll
        for (int i = 0; i < COUNT; ++i)
            if (c0 + i * step < v) q[i] = *reinterpret_cast<const float4*>(zr + c0 + i * step);
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            e[i][0] = q[i].x; e[i][1] = q[i].y; e[i][2] = q[i].z; e[i][3] = q[i].w;
            add_bias(e[i], c0 + i * step, v, bias);
        }
    } else {
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            const int c = c0 + i * step;
            if (c < v) gather_logits(e[i], zr, plane, splits, c, v, bias);
            else e[i][0] = e[i][1] = e[i][2] = e[i][3] = -INFINITY;
        }
    }
}

// four columns of dz: floats (PLANES 0) or BF16 planes; d is used up
template <int PLANES>
__device__ __forceinline__ void store_dz(float (&d)[4], void* dz, long long n, long long row, int pitch, int c) {
    if constexpr (PLANES == 0) *reinterpret_cast<float4*>(static_cast<float*>(dz) + row * pitch + c) = make_float4(d[0], d[1], d[2], d[3]);
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(d[0], d[1]), hi = __floats2bfloat162_rn(d[2], d[3]);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(dz) + (p * n + row) * pitch + c) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        d[0] -= __low2float(lo); d[1] -= __high2float(lo);
        d[2] -= __low2float(hi); d[3] -= __high2float(hi);
    }
}

// Kept logits -> lse, loss and dz (PLANES BF16 planes; 0: floats, which may replace the first part of the logits) in one go.
// A block takes a run of rows; a thread holds the same 4 * QUADS columns of each in registers, from the sum of the parts to
// dz, and their column sums over the run.  v <= 4 * THREADS * QUADS.
// 1024 threads an SM (64 registers), fewer where the parts of the columns have to be in flight.
template <int THREADS, int QUADS, int PLANES, bool GRAD, bool SPLIT>
__global__ void __launch_bounds__(THREADS, (!SPLIT ? 1024 : QUADS > 1 ? 512 : 768) / THREADS)
xe_rows_kernel(const float* z, int splits, int v, int zpitch, const float* __restrict__ bias, const RowArgs a, const XeDzRule rule, void* dz, int dpitch,
               float* __restrict__ db_part) {
    pdl_wait();
    constexpr int WARPS = THREADS / 32;
    __shared__ float red[2][3][WARPS];          // two sets, used by turns: a row's second barrier frees the other set
    __shared__ float zt_s;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const long long r0 = blockIdx.x * a.n / gridDim.x, r1 = (blockIdx.x + 1) * a.n / gridDim.x, plane = a.n * zpitch;
    float sums[GRAD ? QUADS : 1][4];
#pragma unroll
    for (int q = 0; q < (GRAD ? QUADS : 1); ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[q][k] = 0.f;
    int live = 0;
    for (long long row = r0; row < r1; ++row) {
        const bool counts = row_counts(a.rule, a.target[row]);
        const int t = counts ? (int)a.target[row] : -1;
        float e[QUADS][4], m = -INFINITY, zsum = 0.f;
        gather_groups<SPLIT>(e, z + row * zpitch, plane, splits, threadIdx.x * 4, THREADS * 4, v, bias);
#pragma unroll
        for (int q = 0; q < QUADS; ++q) {
            const int c = (q * THREADS + threadIdx.x) * 4;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                m = fmaxf(m, e[q][k]);
                if (c + k < v) zsum += e[q][k];
                if (c + k == t) zt_s = e[q][k];
            }
        }
#pragma unroll
        for (int w = 16; w >= 1; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
        if (lane == 0) red[row & 1][0][warp] = m;
        __syncthreads();
        m = red[row & 1][0][0];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) m = fmaxf(m, red[row & 1][0][w]);
        const float ref = m == -INFINITY ? 0.f : m, zt = zt_s;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < QUADS; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) s += xe_ex2((e[q][k] - ref) * XE_LOG2E);
#pragma unroll
        for (int w = 16; w >= 1; w >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, w);
            zsum += __shfl_xor_sync(0xffffffffu, zsum, w);
        }
        if (lane == 0) { red[row & 1][1][warp] = s; red[row & 1][2][warp] = zsum; }
        __syncthreads();
        s = red[row & 1][1][0];
        zsum = red[row & 1][2][0];
#pragma unroll
        for (int w = 1; w < WARPS; ++w) { s += red[row & 1][1][w]; zsum += red[row & 1][2][w]; }
        const float lse = m + logf(s);
        if (threadIdx.x == 0) live += finish_row(a, row, lse, zsum, counts ? zt : 0.f);
        if constexpr (GRAD) {
            const float g = counts ? (a.dloss ? a.dloss[row] : 1.f) : 0.f;
#pragma unroll
            for (int q = 0; q < QUADS; ++q) {
                const int c = (q * THREADS + threadIdx.x) * 4;
                if (c < v) {
                    float d[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        d[k] = xe_ex2((e[q][k] - lse) * XE_LOG2E) * rule.pf - rule.smooth_all;
                        if (c + k == t) d[k] -= rule.smooth_t;
                        d[k] = g == 0.f || c + k >= v ? 0.f : d[k] * g;      // a row that does not count: exactly 0, whatever its logits
                        sums[q][k] += d[k];
                    }
                    store_dz<PLANES>(d, dz, a.n, row, dpitch, c);
                }
            }
        }
    }
    if (threadIdx.x == 0 && live) atomicAdd(a.count, live);
    if constexpr (GRAD && PLANES > 0) {
        if (db_part) {
#pragma unroll
            for (int q = 0; q < QUADS; ++q) {
                const int c = (q * THREADS + threadIdx.x) * 4;
                if (c < v) *reinterpret_cast<float4*>(db_part + (long long)blockIdx.x * dpitch + c) = make_float4(sums[q][0], sums[q][1], sums[q][2], sums[q][3]);
            }
        }
    }
    finish_loss<THREADS>(a);
}

// The same with a warp per row and no barriers, for v <= 512: lanes hold up to four groups of four columns.  A warp walks its
// run of rows; the block's warps add up their column sums at the end.
constexpr int XE_WARP_ROWS = 8;                    // warps per block
template <int PLANES, bool GRAD, bool SPLIT>
__global__ void __launch_bounds__(256) xe_warp_rows_kernel(const float* z, int splits, int v, int zpitch, const float* __restrict__ bias, const RowArgs a,
                                                           const XeDzRule rule, void* dz, int dpitch, float* __restrict__ db_part) {
    pdl_wait();
    constexpr int QUADS = 4;
    __shared__ __align__(16) float block_sums[XE_WARP_ROWS][128 * QUADS];
    __shared__ int block_live;
    if (threadIdx.x == 0) block_live = 0;
    __syncthreads();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const long long warps = (long long)gridDim.x * XE_WARP_ROWS, w0 = (long long)blockIdx.x * XE_WARP_ROWS + warp;
    const long long r0 = w0 * a.n / warps, r1 = (w0 + 1) * a.n / warps, plane = a.n * zpitch;
    float sums[QUADS][4];
#pragma unroll
    for (int q = 0; q < QUADS; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[q][k] = 0.f;
    int live = 0;
    for (long long row = r0; row < r1; ++row) {
        const bool counts = row_counts(a.rule, a.target[row]);
        const int t = counts ? (int)a.target[row] : -1;
        float e[QUADS][4], m = -INFINITY, zsum = 0.f, zt = 0.f;
        gather_groups<SPLIT>(e, z + row * zpitch, plane, splits, lane * 4, 128, v, bias);
#pragma unroll
        for (int q = 0; q < QUADS; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = q * 128 + lane * 4 + k;
                m = fmaxf(m, e[q][k]);
                if (c < v) zsum += e[q][k];
                if (c == t) zt = e[q][k];
            }
#pragma unroll
        for (int w = 16; w >= 1; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
        const float ref = m == -INFINITY ? 0.f : m;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < QUADS; ++q)
#pragma unroll
            for (int k = 0; k < 4; ++k) s += xe_ex2((e[q][k] - ref) * XE_LOG2E);
#pragma unroll
        for (int w = 16; w >= 1; w >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, w);
            zsum += __shfl_xor_sync(0xffffffffu, zsum, w);
        }
        if (counts) zt = __shfl_sync(0xffffffffu, zt, t % 128 / 4);
        const float lse = m + logf(s);
        if (lane == 0) live += finish_row(a, row, lse, zsum, zt);
        if constexpr (GRAD) {
            const float g = counts ? (a.dloss ? a.dloss[row] : 1.f) : 0.f;
#pragma unroll
            for (int q = 0; q < QUADS; ++q) {
                const int c = q * 128 + lane * 4;
                if (c < v) {
                    float d[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        d[k] = xe_ex2((e[q][k] - lse) * XE_LOG2E) * rule.pf - rule.smooth_all;
                        if (c + k == t) d[k] -= rule.smooth_t;
                        d[k] = g == 0.f || c + k >= v ? 0.f : d[k] * g;      // a row that does not count: exactly 0, whatever its logits
                        sums[q][k] += d[k];
                    }
                    store_dz<PLANES>(d, dz, a.n, row, dpitch, c);
                }
            }
        }
    }
    // one atomic per block: thousands of warps on one address would queue for longer than the rows take
    if (lane == 0 && live) atomicAdd(&block_live, live);
    __syncthreads();
    if (threadIdx.x == 0 && block_live) atomicAdd(a.count, block_live);
    if constexpr (GRAD) {
        if (db_part) {
#pragma unroll
            for (int q = 0; q < QUADS; ++q)
                *reinterpret_cast<float4*>(&block_sums[warp][q * 128 + lane * 4]) = make_float4(sums[q][0], sums[q][1], sums[q][2], sums[q][3]);
            __syncthreads();
            for (int c = threadIdx.x; c < v; c += 256) {
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < XE_WARP_ROWS; ++w) s += block_sums[w][c];
                db_part[(long long)blockIdx.x * dpitch + c] = s;
            }
        }
    }
    finish_loss<256, true>(a);
}

// The same for any v, in three kernels.  Statistics of split logits, 1024 columns of a row per block (the sum of the parts with
// the bias replaces the first); of unsplit ones they come with the product (XE_STATS_Z).
constexpr int XE_CHUNK = 1024;
__global__ void __launch_bounds__(256) xe_wide_stats_kernel(float* __restrict__ z, int splits, int v, int pitch, const float* __restrict__ bias, long long n,
                                                            const long long* __restrict__ target, float2* __restrict__ stats, float* __restrict__ zsums,
                                                            float* __restrict__ zt) {
    pdl_wait();
    __shared__ float red[3][8];
    const int chunks = (v + XE_CHUNK - 1) / XE_CHUNK, chunk = (int)(blockIdx.x % (unsigned)chunks);
    const long long row = blockIdx.x / (unsigned)chunks;
    const int c = chunk * XE_CHUNK + threadIdx.x * 4;
    const long long t = target[row];
    float* zr = z + row * pitch;
    float e[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, zsum = 0.f;
    if (c < v) {
        gather_logits(e, zr, n * pitch, splits, c, v, bias);
        *reinterpret_cast<float4*>(zr + c) = make_float4(e[0], e[1], e[2], e[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (c + i < v) zsum += e[i];
            if (c + i == t) zt[row] = e[i];
        }
    }
    float m = fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), ref = m == -INFINITY ? 0.f : m;
    float s = (xe_ex2((e[0] - ref) * XE_LOG2E) + xe_ex2((e[1] - ref) * XE_LOG2E)) + (xe_ex2((e[2] - ref) * XE_LOG2E) + xe_ex2((e[3] - ref) * XE_LOG2E));
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
        for (int i = 1; i < 8; ++i) {
            join(m, s, red[0][i], red[1][i]);
            zsum += red[2][i];
        }
        stats[chunk * n + row] = make_float2(m, s);
        if (zsums) zsums[chunk * n + row] = zsum;
    }
}

// dz (PLANES 0: floats, which may replace z), two classes per thread, 32 rows per block, with the block's column sums; z has
// the bias already
template <int PLANES>
__global__ void __launch_bounds__(128) xe_wide_dz_kernel(const float* z, int v, int zpitch, long long n, const float* __restrict__ lse,
                                                         const float* __restrict__ rowg, const long long* __restrict__ target, const XeDzRule rule,
                                                         void* dz, int dpitch, float* __restrict__ db_part) {
    pdl_wait();
    const unsigned cblocks = (unsigned)(v + 255) / 256, part = blockIdx.x / cblocks;
    const int c = (int)((blockIdx.x % cblocks) * 128 + threadIdx.x) * 2;
    if (c >= v) return;
    const long long r0 = (long long)part * XE_ROWS_PER_PART;
    const long long r1 = r0 + XE_ROWS_PER_PART < n ? r0 + XE_ROWS_PER_PART : n;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll 8
    for (long long r = r0; r < r1; ++r) {
        const float2 q = *reinterpret_cast<const float2*>(z + r * zpitch + c);
        const float l = lse[r], g = rowg[r];
        const long long t = target[r];
        float a = xe_ex2((q.x - l) * XE_LOG2E) * rule.pf - rule.smooth_all, b = xe_ex2((q.y - l) * XE_LOG2E) * rule.pf - rule.smooth_all;
        if (t == c) a -= rule.smooth_t;
        if (t == c + 1) b -= rule.smooth_t;
        a = g == 0.f ? 0.f : a * g;
        b = g == 0.f || c + 1 >= v ? 0.f : b * g;
        s0 += a;
        s1 += b;
        if constexpr (PLANES == 0) *reinterpret_cast<float2*>(static_cast<float*>(dz) + r * dpitch + c) = make_float2(a, b);
#pragma unroll
        for (int p = 0; p < PLANES; ++p) {
            const __nv_bfloat162 o = __floats2bfloat162_rn(a, b);
            *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(dz) + (p * n + r) * dpitch + c) = o;
            a -= __low2float(o);
            b -= __high2float(o);
        }
    }
    if (db_part) *reinterpret_cast<float2*>(db_part + (long long)part * dpitch + c) = make_float2(s0, s1);
}

// exponentials (kept in the place of dz) -> dz, eight classes per thread.  The target's probability comes from its logit in
// FP32, the others' from the exponential in 16 bits (xe_pack_exp): off by 2^-10 before dz itself is rounded.
__global__ void __launch_bounds__(256) xe_dz_from_exp_kernel(__nv_bfloat16* __restrict__ dz, int pitch, long long n, const float2* __restrict__ stats,
                                                             const float* __restrict__ zt, const float* __restrict__ lse, const float* __restrict__ rowg,
                                                             const long long* __restrict__ target, const XeDzRule rule) {
    pdl_wait();
    // a block takes 256 x 4 groups of a row at a time: one division per block, four loads in flight per thread
    const int octs = pitch / 8, spans = (octs + 1023) / 1024;
    for (long long b = blockIdx.x; b < n * spans; b += gridDim.x) {
        const long long r = b / spans;
        const int o0 = (int)(b - r * spans) * 1024 + threadIdx.x;
        uint4* at = reinterpret_cast<uint4*>(dz + r * pitch);
        uint4 q[4];                                       // everything that is read is asked for at once
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int o = o0 + i * 256;
            if (o < octs) {
                q[i] = at[o];
                f[i] = __ldg(&stats[(long long)(o / (XE_STAT_COLS / 8)) * n + r].x);
            }
        }
        const float g = __ldg(rowg + r), l = __ldg(lse + r), z_t = __ldg(zt + r);
        const int t = (int)__ldg(target + r), to = t >> 3;
        if (g == 0.f) {                                   // a row that does not count
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (o0 + i * 256 < octs) at[o0 + i * 256] = make_uint4(0, 0, 0, 0);
            continue;
        }
        const float gp = g * rule.pf, ga = g * rule.smooth_all;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int o = o0 + i * 256;
            if (o >= octs) break;
            const float h = xe_ex2((f[i] - l) * XE_LOG2E) * gp;
            uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 z = __ffma2_rn(xe_unpack_exp(w[e]), make_float2(h, h), make_float2(-ga, -ga));
                const __nv_bfloat162 v = __floats2bfloat162_rn(z.x, z.y);
                w[e] = *reinterpret_cast<const uint32_t*>(&v);
            }
            if (o == to) {                                // the target's own value
                const float pt = xe_ex2((z_t - l) * XE_LOG2E) * gp - ga - g * rule.smooth_t;
                const uint32_t b16 = __bfloat16_as_ushort(__float2bfloat16_rn(pt));
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if ((t & 7) >> 1 == k) w[k] = t & 1 ? (w[k] & 0xffffu) | b16 << 16 : (w[k] & 0xffff0000u) | b16;
            }
            at[o] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// dbias from the column sums of runs of rows (or from the rows of a float dz): COLS columns and 512 / COLS runs at a time
// per block; eight columns where there are few of them, 32 (whole lines) where there are many
template <int COLS>
__global__ void __launch_bounds__(512) xe_db_kernel(const float* __restrict__ part, int parts, int pitch, int cols, const XeScale scale, float* __restrict__ db) {
    pdl_wait();
    constexpr int RUNS = 512 / COLS;
    __shared__ float red[RUNS][COLS];
    const int l = threadIdx.x % COLS, g = threadIdx.x / COLS, c = blockIdx.x * COLS + l;
    float s = 0.f;
    if (c < cols) {
#pragma unroll 8
        for (int i = g; i < parts; i += RUNS) s += part[(long long)i * pitch + c];
    }
    red[g][l] = s;
    __syncthreads();
    if (g == 0 && c < cols) {
        for (int i = 1; i < RUNS; ++i) s += red[i][l];
        db[c] = s * xe_scale(scale);
    }
}

// out (rows x cols, pitch ld) = sum of `splits` float buffers (pitch `pitch`)
template <typename T>
__global__ void __launch_bounds__(256) xe_finish_kernel(const float* __restrict__ part, int splits, long long rows, int cols, int pitch, T* __restrict__ out,
                                                        long long ld) {
    pdl_wait();
    const int quads = (cols + 3) / 4;
    const long long total = rows * quads, plane = rows * pitch;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / quads;
        const int c = (int)(i - r * quads) * 4;
        float4 q = *reinterpret_cast<const float4*>(part + r * pitch + c);
#pragma unroll 8
        for (int s = 1; s < splits; ++s) {
            const float4 o = __ldg(reinterpret_cast<const float4*>(part + s * plane + r * pitch + c));
            q.x += o.x; q.y += o.y; q.z += o.z; q.w += o.w;
        }
        const float e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c + k < cols) out[r * ld + c + k] = from_float<T>(e[k]);
    }
}

// ---- few products: FP32 arithmetic on the caller's matrices --------------------------------------------------
// Below some millions of products a tensor-core launch is mostly set-up, and the operands fit the L2 many times over.
// Measured (GPU time of a call, BF16 / FP32X3, us): loss of 16 x 1024 x 1000 (16M products) 12.4 / 12.4 against 14.4 / 18.9 on
// tensor cores, of 512 x 256 x 256 (32M) 20.6 / 26.7 against 14.4 / 16.5; gradient of 32 x 4096 x 64 (8M) 18.5 / 20.6 against
// 22.7 / 28.8.  The gradient's sums run one after the other over rows or classes: with 256 of them 23.8 / 24.8 against
// 18.5 / 24.7, with 1000 of them 65 against 29.
// logits: a warp multiplies one class with eight rows, lanes along the features; blockIdx.z: part of the features
constexpr int XE_SMALL_ROWS = 8, XE_SMALL_SLICE = 2048;
constexpr int XE_SMALL_MAX = 128;                  // most rows and classes of the plain gradient
// acc[r] = sum over features k0 ... k1 - 1 of class j's weights with row r0 + r, lanes along the features; every lane gets the sums
template <typename T>
__device__ __forceinline__ void small_dots(float (&acc)[XE_SMALL_ROWS], const T* __restrict__ x, long long ldx, const T* __restrict__ wj, bool aligned,
                                           int r0, int n, int k0, int k1, int lane) {
    const T* row[XE_SMALL_ROWS];                               // rows past the last read it again
#pragma unroll
    for (int r = 0; r < XE_SMALL_ROWS; ++r) {
        row[r] = x + (long long)(r0 + r < n ? r0 + r : n - 1) * ldx;
        acc[r] = 0.f;
    }
    if (aligned && (k1 - k0) % 4 == 0) {
        // whole vectors: nine loads in flight per step, two steps
#pragma unroll 2
        for (int k = k0 + lane * 4; k < k1; k += 128) {
            float a[4], b[XE_SMALL_ROWS][4];
            load4_aligned(a, wj + k);
#pragma unroll
            for (int r = 0; r < XE_SMALL_ROWS; ++r) load4_aligned(b[r], row[r] + k);
#pragma unroll
            for (int r = 0; r < XE_SMALL_ROWS; ++r) acc[r] += (a[0] * b[r][0] + a[1] * b[r][1]) + (a[2] * b[r][2] + a[3] * b[r][3]);
        }
    } else {
#pragma unroll 4
        for (int k = k0 + lane; k < k1; k += 32) {
            const float a = to_float<T>(wj[k]);
#pragma unroll
            for (int r = 0; r < XE_SMALL_ROWS; ++r) acc[r] += a * to_float<T>(row[r][k]);
        }
    }
#pragma unroll
    for (int r = 0; r < XE_SMALL_ROWS; ++r)
#pragma unroll
        for (int s = 16; s >= 1; s >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], s);
}

template <typename T>
__global__ void __launch_bounds__(256) xe_small_logits_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ w, long long ldw, int n, int d, int v,
                                                              int zpitch, float* __restrict__ z, int* zero) {
    pdl_wait();
    const int lane = threadIdx.x % 32, j = blockIdx.x * 8 + threadIdx.x / 32, r0 = blockIdx.y * XE_SMALL_ROWS;
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x < 2) zero[threadIdx.x] = 0;
    if (j >= v) return;
    const int k0 = blockIdx.z * XE_SMALL_SLICE, k1 = k0 + XE_SMALL_SLICE < d ? k0 + XE_SMALL_SLICE : d;
    float acc[XE_SMALL_ROWS];
    small_dots(acc, x, ldx, w + j * ldw, ldx % 4 == 0 && ldw % 4 == 0, r0, n, k0, k1, lane);     // the bases are aligned
#pragma unroll
    for (int r = 0; r < XE_SMALL_ROWS; ++r)
        if (lane == r && r0 + r < n) z[((long long)blockIdx.z * n + r0 + r) * zpitch + j] = acc[r];
}

// Up to 128 classes that a block's 16 warps multiply in a few steps: logits, statistics and dz of eight rows in one kernel.  One
// launch fewer is 3.5 us of host time of a call that takes about 17.  A block that is the only one (n <= 8) sums the losses too.
constexpr int XE_TINY_WARPS = 16, XE_TINY_STEPS = 24;
template <typename T, bool GRAD>
__global__ void __launch_bounds__(32 * XE_TINY_WARPS) xe_tiny_kernel(const T* __restrict__ x, long long ldx, const T* __restrict__ w, long long ldw, int d, int v,
                                                                     int zpitch, const float* __restrict__ bias, const RowArgs a, const XeDzRule rule,
                                                                     float* __restrict__ dz) {
    pdl_wait();
    __shared__ float z[XE_SMALL_ROWS][XE_SMALL_MAX + 1];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r0 = blockIdx.x * XE_SMALL_ROWS, n = (int)a.n;
    const bool aligned = ldx % 4 == 0 && ldw % 4 == 0;
    for (int j = warp; j < v; j += XE_TINY_WARPS) {
        float acc[XE_SMALL_ROWS];
        small_dots(acc, x, ldx, w + j * ldw, aligned, r0, n, 0, d, lane);
        const float b = bias ? bias[j] : 0.f;
#pragma unroll
        for (int r = 0; r < XE_SMALL_ROWS; ++r)
            if (lane == r) z[r][j] = acc[r] + b;
    }
    __syncthreads();
    const long long row = r0 + warp;
    const bool mine = warp < XE_SMALL_ROWS && row < n, counts = mine && row_counts(a.rule, a.target[row]);
    if (mine) {
        const int t = counts ? (int)a.target[row] : -1;
        float e[4], m = -INFINITY, s = 0.f, zsum = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int c = q * 32 + lane;
            e[q] = c < v ? z[warp][c] : -INFINITY;
            if (c < v) zsum += e[q];
            m = fmaxf(m, e[q]);
        }
#pragma unroll
        for (int h = 16; h >= 1; h >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, h));
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int q = 0; q < 4; ++q) s += xe_ex2((e[q] - ref) * XE_LOG2E);
#pragma unroll
        for (int h = 16; h >= 1; h >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, h);
            zsum += __shfl_xor_sync(0xffffffffu, zsum, h);
        }
        const float lse = m + logf(s);
        if (lane == 0) finish_row(a, row, lse, zsum, counts ? z[warp][t] : 0.f);
        if constexpr (GRAD) {
            const float g = counts ? (a.dloss ? a.dloss[row] : 1.f) : 0.f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = q * 32 + lane;
                float v1 = xe_ex2((e[q] - lse) * XE_LOG2E) * rule.pf - rule.smooth_all;
                if (c == t) v1 -= rule.smooth_t;
                if (c < v) dz[row * zpitch + c] = g == 0.f ? 0.f : v1 * g;       // a row that does not count: exactly 0, whatever its logits
            }
        }
    }
    if (a.loss.loss) {
        const int live = __syncthreads_count(counts && lane == 0);
        if (threadIdx.x == 0) a.count[0] = live;
        __syncthreads();
        xe_sum_losses<32 * XE_TINY_WARPS>(a.loss);
    }
}

// out[o][k] = scale sum_c coef(o, c) M[c][k]: dx (o rows, c classes, M = W) and dW (o classes, c rows, M = x; and dbias),
// from dz in floats.  A block makes eight o by 128 k; its eight warps share the sum over c, whose coefficients sit in
// shared memory.  A row that does not count has nothing but zeros there and is not read.
constexpr int XE_SMALL_GRAD_SMEM = 8 * 8 * 128 * 4;
template <typename T>
struct SmallGrad {
    const T* x; const T* w;
    T* dx; T* dw;
    float* db;
    long long ldx, ldw, lddx, lddw;
    const float* dz;
    int n, d, v, dzpitch, kblocks, dx_blocks;
    XeScale scale;
    XeLoss loss;                      // summed by the last block
    RowRule rule;                     // n <= 256: every block counts the rows itself
    const long long* target;
    int* count;
};
template <typename T>
__global__ void __launch_bounds__(256) xe_small_grad_kernel(const SmallGrad<T> a) {
    pdl_wait();
    extern __shared__ __align__(16) float coef[];            // [c][8], then [warp][8][128] sums
    const int live = __syncthreads_count((int)threadIdx.x < a.n && row_counts(a.rule, a.target[threadIdx.x]));
    if (a.loss.loss && blockIdx.x == gridDim.x - 1) {
        if (threadIdx.x == 0) *a.count = live;
        __syncthreads();
        xe_sum_losses<256>(a.loss);
        return;
    }
    const bool is_dw = (int)blockIdx.x >= a.dx_blocks;
    const int b = is_dw ? blockIdx.x - a.dx_blocks : blockIdx.x;
    const int o0 = b / a.kblocks * 8, k = (b % a.kblocks) * 128 + (threadIdx.x % 32) * 4, warp = threadIdx.x / 32;
    const int outs = is_dw ? a.v : a.n, len = is_dw ? a.n : a.v;
    for (int i = threadIdx.x; i < len * 8; i += 256) {
        const int c = is_dw ? i / 8 : i % len, o = is_dw ? i % 8 : i / len;
        const bool in = o0 + o < outs;
        coef[c * 8 + o] = in ? a.dz[(long long)(is_dw ? c : o0 + o) * a.dzpitch + (is_dw ? o0 + o : c)] : 0.f;
    }
    __syncthreads();
    const float scale = xe_scale(a.scale, live);
    if (is_dw && a.db && k < 128 && threadIdx.x < 8 && o0 + threadIdx.x < outs) {
        float s = 0.f;
        for (int c = 0; c < len; ++c) s += coef[c * 8 + threadIdx.x];
        a.db[o0 + threadIdx.x] = s * scale;
    }
    T* out = is_dw ? a.dw : a.dx;
    if (!out) return;
    const T* m = is_dw ? a.x : a.w;
    const long long ldm = is_dw ? a.ldx : a.ldw, ldo = is_dw ? a.lddw : a.lddx;
    float acc[8][4];
#pragma unroll
    for (int o = 0; o < 8; ++o)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[o][e] = 0.f;
    if (k < a.d) {
#pragma unroll 4
        for (int c = warp; c < len; c += 8) {
            const float4 p = *reinterpret_cast<const float4*>(coef + c * 8), q = *reinterpret_cast<const float4*>(coef + c * 8 + 4);
            const float f[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
            if (p.x == 0.f && p.y == 0.f && p.z == 0.f && p.w == 0.f && q.x == 0.f && q.y == 0.f && q.z == 0.f && q.w == 0.f) continue;
            float v[4];
            load4f(v, m + c * ldm + k, a.d - k);
#pragma unroll
            for (int o = 0; o < 8; ++o)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[o][e] += f[o] * v[e];
        }
    }
    __syncthreads();
#pragma unroll
    for (int o = 0; o < 8; ++o) *reinterpret_cast<float4*>(coef + (warp * 8 + o) * 128 + (threadIdx.x % 32) * 4) = make_float4(acc[o][0], acc[o][1], acc[o][2], acc[o][3]);
    __syncthreads();
    // warp -> output row, lane -> columns
    if (o0 + warp < outs) {
        const int kb = (b % a.kblocks) * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int kk = i * 32 + threadIdx.x % 32;
            float s = 0.f;
#pragma unroll
            for (int g = 0; g < 8; ++g) s += coef[(g * 8 + warp) * 128 + kk];
            if (kb + kk < a.d) out[(long long)(o0 + warp) * ldo + kb + kk] = from_float<T>(s * scale);
        }
    }
}

// ---- few rows: FP32 products on the caller's matrices ----------------------------------------------------------
// FP32X3 with up to 8 rows, or up to 8 classes (for which read: x as W, and the other way round): the products are a read of
// W (twice) and a write of dW, and a tensor-core tile would be mostly empty.  In all three kernels a lane owns four features,
// 32 apart (single elements then make whole lines at any pitch and alignment), whose values of all rows (x, or the sums of dx) it
// holds in registers as packed pairs, and a warp walks over classes, one piece of 128 features of W or dW per class.
// Bound: HBM up to four rows (loss of 4 x 4096 x 32000 at 4.5 TB/s); beyond, the multiplications and, for the logits, the
// exchange of the lanes' sums (8 rows 3.0 TB/s).
constexpr int XF_ROWS = 8, XF_COLS = 128, XF_CLASSES = 128;      // most rows; features and classes of a block
struct FewArgs {
    const float* x; const float* w;       // the matrix of few rows (n), and the long one (v rows); classes and rows may change
                                          // places: then x is W, w is x, and dx and dW change places as well
    float* out;                           // z, dx or its parts, dW
    const float* dz;
    long long ldx, ldw, ldo, plane;       // plane: elements between the parts of z or dx
    long long zr, zj;                     // z and dz: elements from one row of x to the next, from one row of w to the next
    int n, d, v, splits;
    const float* xg; const float* wg;     // rows of x or w of weight 0 are not read, or NULL
    XeScale scale;
    int* zero;
};
// features k, k + 32, k + 64, k + 96 of one row
__device__ __forceinline__ void few_load(float (&v)[4], const float* row, int k, int d) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = k + 32 * e < d ? row[k + 32 * e] : 0.f;
}
template <int ROWS>
__device__ __forceinline__ void few_load_x(float2 (&xr)[ROWS][2], const FewArgs& p, int k, bool weigh) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        float v[4];
        const bool in = r < p.n && !(weigh && p.xg && p.xg[r] == 0.f);
        few_load(v, p.x + (in ? r * p.ldx : 0), k, in ? p.d : 0);
        xr[r][0] = make_float2(v[0], v[1]);
        xr[r][1] = make_float2(v[2], v[3]);
    }
}

// z: a block multiplies 128 classes with a part of the features, 128 at a time; the lanes' sums of a class meet in a halving
// exchange and add up in shared memory
template <int ROWS>
__global__ void __launch_bounds__(128) xe_few_logits_kernel(const FewArgs p) {
    pdl_wait();
    __shared__ float zs[XF_CLASSES][ROWS + 1];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, j0 = blockIdx.x * XF_CLASSES;
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 2) p.zero[threadIdx.x] = 0;
    for (int i = threadIdx.x; i < XF_CLASSES * (ROWS + 1); i += 128) (&zs[0][0])[i] = 0.f;
    __syncthreads();
    const int slices = (p.d + XF_COLS - 1) / XF_COLS, s0 = (int)((long long)blockIdx.y * slices / p.splits), s1 = (int)((long long)(blockIdx.y + 1) * slices / p.splits);
    const float* w = p.w;
    const int count = p.v - j0 < XF_CLASSES ? p.v - j0 : XF_CLASSES;
    for (int s = s0; s < s1; ++s) {
        const int k = s * XF_COLS + lane;
        float2 xr[ROWS][2];
        few_load_x<ROWS>(xr, p, k, false);
        constexpr int AHEAD = 4;                                   // pieces of W in flight per warp
        float wv[AHEAD][4];
        for (int c0 = warp; c0 < count; c0 += 4 * AHEAD) {
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int c = c0 + 4 * q;
                few_load(wv[q], w + (c < count ? (j0 + c) * p.ldw : 0), k, c < count ? p.d : 0);
            }
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int c = c0 + 4 * q;
                if (c >= count) break;
                float t[ROWS];
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    float2 m = __fmul2_rn(xr[r][0], make_float2(wv[q][0], wv[q][1]));
                    m = __ffma2_rn(xr[r][1], make_float2(wv[q][2], wv[q][3]), m);
                    t[r] = m.x + m.y;
                }
                // t[r] of lane l -> lane r (mod ROWS) holds the sum over lanes
#pragma unroll
                for (int h = ROWS / 2; h >= 1; h >>= 1) {
                    const bool up = lane & h;
#pragma unroll
                    for (int r = 0; r < h; ++r) {
                        const float send = up ? t[r] : t[r + h], keep = up ? t[r + h] : t[r];
                        t[r] = keep + __shfl_xor_sync(0xffffffffu, send, h);
                    }
                }
#pragma unroll
                for (int h = ROWS; h <= 16; h <<= 1) t[0] += __shfl_xor_sync(0xffffffffu, t[0], h);
                if (lane < ROWS) zs[c][lane] += t[0];              // this warp's class: nobody else's
            }
        }
    }
    __syncthreads();
    float* z = p.out + blockIdx.y * p.plane;
    for (int i = threadIdx.x; i < XF_CLASSES * p.n; i += 128) {
        const int r = i / XF_CLASSES, c = i % XF_CLASSES;
        if (c < count) z[r * p.zr + (j0 + c) * p.zj] = zs[c][r];
    }
}

// dz of 128 classes, [class][row], from rows of floats
template <int ROWS>
__device__ __forceinline__ void few_stage_dz(float (&ds)[XF_CLASSES][ROWS], const FewArgs& p, int j0) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int j = j0 + threadIdx.x;
        ds[threadIdx.x][r] = r < p.n && j < p.v ? p.dz[r * p.zr + j * p.zj] : 0.f;
    }
}

// dx = dz W: a block takes 128 features and a part of the classes; its warps' sums meet in shared memory
template <int ROWS>
__global__ void __launch_bounds__(128) xe_few_dx_kernel(const FewArgs p) {
    pdl_wait();
    __shared__ __align__(16) float ds[XF_CLASSES][ROWS];
    __shared__ float sums[4][XF_COLS];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, k = blockIdx.x * XF_COLS + lane;
    const int tiles = (p.v + XF_CLASSES - 1) / XF_CLASSES, t0 = (int)((long long)blockIdx.y * tiles / p.splits), t1 = (int)((long long)(blockIdx.y + 1) * tiles / p.splits);
    const float* w = p.w;
    float2 acc[ROWS][2];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) acc[r][0] = acc[r][1] = make_float2(0.f, 0.f);
    for (int t = t0; t < t1; ++t) {
        const int j0 = t * XF_CLASSES, count = p.v - j0 < XF_CLASSES ? p.v - j0 : XF_CLASSES;
        __syncthreads();
        few_stage_dz<ROWS>(ds, p, j0);
        __syncthreads();
        constexpr int AHEAD = 4;
        float wv[AHEAD][4];
        for (int c0 = warp; c0 < count; c0 += 4 * AHEAD) {
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int c = c0 + 4 * q;
                const bool in = c < count && !(p.wg && p.wg[j0 + c] == 0.f);
                few_load(wv[q], w + (in ? (j0 + c) * p.ldw : 0), k, in ? p.d : 0);
            }
#pragma unroll
            for (int q = 0; q < AHEAD; ++q) {
                const int c = c0 + 4 * q < count ? c0 + 4 * q : c0;        // past the last: zeros of W
                const float2 lo = make_float2(wv[q][0], wv[q][1]), hi = make_float2(wv[q][2], wv[q][3]);
#pragma unroll
                for (int r = 0; r < ROWS; r += 4) {
                    const float4 g = *reinterpret_cast<const float4*>(&ds[c][r]);
                    const float gv[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[r + e][0] = __ffma2_rn(make_float2(gv[e], gv[e]), lo, acc[r + e][0]);
                        acc[r + e][1] = __ffma2_rn(make_float2(gv[e], gv[e]), hi, acc[r + e][1]);
                    }
                }
            }
        }
    }
    const float scale = xe_scale(p.scale);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        __syncthreads();
        sums[warp][lane] = acc[r][0].x;
        sums[warp][lane + 32] = acc[r][0].y;
        sums[warp][lane + 64] = acc[r][1].x;
        sums[warp][lane + 96] = acc[r][1].y;
        __syncthreads();
        const int kk = blockIdx.x * XF_COLS + threadIdx.x;
        if (r < p.n && kk < p.d) {
            const float s = ((sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x])) * scale;
            const long long at = blockIdx.y * p.plane + r * p.ldo + kk;
            p.out[at] = s;
        }
    }
}

// dW = dz^T x: a block makes 128 classes x 128 features
template <int ROWS>
__global__ void __launch_bounds__(128) xe_few_dw_kernel(const FewArgs p) {
    pdl_wait();
    __shared__ __align__(16) float ds[XF_CLASSES][ROWS];
    const unsigned kblocks = (unsigned)(p.d + XF_COLS - 1) / XF_COLS;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, k = (int)(blockIdx.x % kblocks) * XF_COLS + lane, j0 = (int)(blockIdx.x / kblocks) * XF_CLASSES;
    const int count = p.v - j0 < XF_CLASSES ? p.v - j0 : XF_CLASSES;
    float2 xr[ROWS][2];
    few_load_x<ROWS>(xr, p, k, true);
    few_stage_dz<ROWS>(ds, p, j0);
    const float scale = xe_scale(p.scale);
    __syncthreads();
#pragma unroll 2
    for (int c = warp; c < count; c += 4) {
        float2 lo = make_float2(0.f, 0.f), hi = lo;
#pragma unroll
        for (int r = 0; r < ROWS; r += 4) {
            const float4 g = *reinterpret_cast<const float4*>(&ds[c][r]);
            const float gv[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                lo = __ffma2_rn(make_float2(gv[e], gv[e]), xr[r + e][0], lo);
                hi = __ffma2_rn(make_float2(gv[e], gv[e]), xr[r + e][1], hi);
            }
        }
        const float v[4] = {lo.x * scale, lo.y * scale, hi.x * scale, hi.y * scale};
        float* o = p.out + (long long)(j0 + c) * p.ldo + k;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k + 32 * e < p.d) o[32 * e] = v[e];
    }
}

unsigned loop_blocks(long long items) {
    const long long b = (items + 255) / 256, most = 16ll * sm_count();
    return (unsigned)(b < 1 ? 1 : b < most ? b : most);
}

// ---- plan ----------------------------------------------------------------------------------------------------
constexpr long long XE_SMALL_PRODUCTS = 16ll << 20;   // n v d up to which xe_small_* run
// Most logits and rows of the plain loss alone, whose warps make eight logits each whatever d is.  Measured, plain against tensor
// cores, BF16 / FP32X3, us: 512 x 64 x 100 10.4 / 11.2 against 10.6 / 13.4, 64 x 64 x 1000 10.2 / 11.6 against 10.0 / 13.2, 256 x 64 x 1000
// 24.3 / 28.5 against 10.0 / 14.0, 2000 x 800 x 10 15.8 (BF16) against 14.3, 500000 x 9 x 3 510 / 581 against 313 / 382.
constexpr long long XE_SMALL_LOGITS = 64ll << 10, XE_SMALL_ROWS_MAX = 1024;

struct Plan {
    int planes, es, dp;
    long long ldx, ldw, lddx, lddw;
    bool pack_x, pack_w;
    bool tiny, small, few, few_rows;     // FP32 arithmetic instead of tensor cores; few: of rows, else of classes
    bool thin, thin_rows;                // W (up to 128 rows) or x (up to 128 classes) is split inside the products (xe_thin)
    XeThinCut thin_z, thin_grad;
    int splits_few;                      // of the gradient of the matrix of few rows
    bool kept, exps;                     // floats of all logits, exponentials of all logits in 16 bits (else recomputed by piece)
    int splits_z, splits_dx, splits_dw, bn_z, bn_dx, bn_dw;
    int zpitch, piece, pieces, dzpitch, parts;
    bool dx_direct, dw_direct;           // the product's epilogue stores the caller's matrix
    int dpitch;                          // of float dx / dw buffers in the scratch
    size_t off_x, off_w, off_z, off_stats, off_zsum, off_zt, off_lse, off_rowloss, off_rowg, off_count, off_dz, off_db, off_dx, off_dw, total;
};

// parts of the contraction of an xe_few_* product: `tiles` blocks without splitting, `steps` pieces of the contraction;
// about eight blocks an SM
int few_split_count(long long tiles, long long steps) {
    const long long want = 8ll * sm_count();
    long long s = tiles > 0 ? (want + tiles - 1) / tiles : 1;
    if (s > steps) s = steps;
    if (s > 64) s = 64;
    return (int)(s < 1 ? 1 : s);
}

// blocks of xe_rows_kernel or xe_warp_rows_kernel, each with a run of rows: no more than fit the GPU at once (1024 threads an
// SM), and at least four rows each once every SM has a block, for the sake of the partial column sums
int row_blocks(long long n, int v) {
    if (v <= 512) {
        const long long most = 4ll * sm_count(), b = (n + XE_WARP_ROWS - 1) / XE_WARP_ROWS;
        return (int)(b < most ? b : most);
    }
    const long long most = (v <= 4096 ? 4ll : 2ll) * sm_count(), few = sm_count(), b = n / 4 < few ? (n < few ? n : few) : n / 4;
    return (int)(b < most ? b : most);
}
constexpr int XE_ROWS_MAX_V = 512 * 4 * 4;          // widest row of xe_rows_kernel: wider ones spill, and one block an SM is
                                                    // slower than two kernels (1024 x 21841: 130 us against 92)

// Parts of a contraction of `chunks` ring slots (times `products` plane pairs), and columns of a tile (256 or 128), so that
// the CTA pairs are filled in as few whole turns as possible.  Estimated time: turns of the slots (0.28 us each on a pair;
// 0.2 us for half the columns, which need 24 of the 32 KB) and of the epilogue (1.5 us; 0.75 us), and, for more than one part,
// writing and reading the floats of every part (5 TB/s) and, where `join` is set, a launch.
struct Cut {
    int splits, bn;
    double us;
};
Cut cut_product(long long rows, long long cols, long long chunks, int products, bool join) {
    const long long pairs = sm_count() < 4 ? 1 : sm_count() / 2;
    const double part_us = (double)rows * (double)cols * 8.0 / 5e6;
    Cut best = {1, XE_BN, 1e30};
    if (rows == 0) return best;
    for (int bn = XE_BN; bn >= 128; bn -= 128) {
        const long long tiles = ((rows + XE_BM - 1) / XE_BM) * ((cols + bn - 1) / bn);
        if (bn < XE_BN && tiles >= 8 * pairs) break;
        const double slot = bn == XE_BN ? 0.28 : 0.2, end = bn == XE_BN ? 1.5 : 0.75;
        for (long long s = 1; s <= chunks && s <= 64 && (s == 1 || tiles * s <= 4 * pairs); ++s) {
            const double us = (double)((tiles * s + pairs - 1) / pairs) * ((double)((chunks + s - 1) / s) * products * slot + end) +
                              (s > 1 || !join ? part_us * (double)s : 0.0) + (s > 1 && join ? 3.0 : 0.0);
            if (us < best.us * 0.97) best = {(int)s, bn, us};
        }
    }
    return best;
}

int build_plan(const wino_xent_desc* d, bool grad, Plan* out) {
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
    const Cut cz = cut_product(n, v, kd, products, false);
    p.splits_z = cz.splits;
    p.zpitch = round_up(d->v, 4);
    // what kept logits take beside them with gradients: dz, and the column sums of runs of rows
    const int kept_parts = d->v <= XE_ROWS_MAX_V ? row_blocks(n, d->v) : (int)((n + XE_ROWS_PER_PART - 1) / XE_ROWS_PER_PART);
    const long long dz_bytes = n * round_up(d->v, 8) * 2ll * p.planes, z_bytes = n * p.zpitch * 4ll;
    const long long db_bytes = grad && d->has_bias ? kept_parts * (round_up(d->v, 8) * 4ll) : 0, beside = (grad ? dz_bytes : 0) + db_bytes;
    const bool fits = z_bytes * p.splits_z + beside <= limit;
    const bool few_tiles = n * v <= 64ll * XE_BM * XE_BN;
    p.few_rows = n <= XF_ROWS;
    const long long long_tiles = ((p.few_rows ? v : n) + XF_CLASSES - 1) / XF_CLASSES, col_tiles = (d->d + XF_COLS - 1) / XF_COLS;
    const int few_splits = few_split_count(long_tiles, col_tiles);
    const int small_splits = (d->d + XE_SMALL_SLICE - 1) / XE_SMALL_SLICE;
    const long long piece_bytes = grad ? n * XE_BN * 2ll * p.planes : 0;        // the least that any gradient takes
    const bool small_fits = z_bytes * small_splits + db_bytes <= (limit > piece_bytes ? limit : piece_bytes);
    p.small = n > 0 && n * v <= XE_SMALL_PRODUCTS / d->d && small_fits &&
              (grad ? n <= XE_SMALL_MAX && v <= XE_SMALL_MAX : n * v <= XE_SMALL_LOGITS && n <= XE_SMALL_ROWS_MAX && v <= XE_ROWS_MAX_V);
    // Measured with gradients, against tensor cores that split W themselves, us: 8 x 2048 x 4000 53.3 / 62.7, 8 x 2048 x 20000
    // 158 / 193, 8000 x 2048 x 8 102 / 129; the same kernels for 16 rows 16 x 2048 x 20000 256 / 197, 8000 x 2048 x 16 145 / 125.
    p.few = !bf16 && !p.small && n > 0 && (p.few_rows || v <= XF_ROWS) && (p.few_rows ? v : n) * d->d >= 2ll << 20 && z_bytes * few_splits + db_bytes <= limit;
    // Measured, the long matrix split inside against beforehand, us: loss of 64 x 512 x 1000 16.4 / 16.4, 64 x 2048 x 1000 18.5 / 22.6, 64 x 2048 x 4000
    // 25.2 / 46.7, 128 x 2048 x 20000 84 / 208; gradient of 64 x 512 x 1000 34.9 / 30.8, 64 x 4096 x 300 43.0 / 44.0, 64 x 2048 x 1000
    // 39.8 / 45.1, 64 x 2048 x 20000 207 / 322.  A tile of 128 rows takes the products apart that one launch would share:
    // gradient of 128 x 512 x 20000 137 / 132, 128 x 2048 x 20000 232 / 382.  With few classes the same: loss of 8000 x 2048 x 64
    // 45.4 / 81.9; gradient of 4000 x 512 x 16 51.3 / 55.4, 8000 x 512 x 64 67.6 / 67.6, 4000 x 2048 x 128 100 / 94, 8000 x 2048 x 128 144 / 155.
    // Between them, near the threshold of 12M elements: 128 x 512 x 25000 143 / 153, 128 x 2048 x 6400 109 / 129, 6200 x 2048 x 128 127 / 128,
    // 25000 x 512 x 128 164 / 157.
    p.thin_rows = n <= 128 && (v > 128 || v >= n);
    const long long thin_n = p.thin_rows ? n : v, thin_m = p.thin_rows ? v : n;
    p.thin = !bf16 && !p.small && !p.few && n > 0 && thin_n <= 128 && thin_m * d->d >= (grad && thin_n > 64 ? 12ll << 20 : 1ll << 20);
    if (p.thin) {
        p.thin_z = xe_thin_cut((thin_m + 127) / 128, kd, (double)n * v * 8.0 / 5e6);
        p.thin_grad = xe_thin_cut(col_tiles, (thin_m + XE_BK - 1) / XE_BK, (double)thin_n * d->d * 8.0 / 5e6);
        p.thin = z_bytes * p.thin_z.parts + beside <= limit;
    }
    p.tiny = p.small && v <= XE_SMALL_MAX && (v + XE_TINY_WARPS - 1) / XE_TINY_WARPS * ((d->d + 127) / 128) <= XE_TINY_STEPS;
    // Logits are kept where the product is split, or has too few tiles for the GPU.  Elsewhere kept floats cost 14 bytes a
    // logit (18 in three parts), exponentials 6, against 2 d flops (12 d) for another product.  Measured, with gradients, kept
    // against computed again: floats 4096 x d x 20000 BF16 d = 512 363 / 316 us, 1024 498 / 500, 2048 841 / 941; FP32X3
    // 4096 x d x 12000 d = 128 484 / 465, 256 572 / 571, 512 891 / 995; exponentials d = 256 253 / 242, 512 303 / 304, 1024 440 / 495.
    if (p.small) {
        p.kept = true;
        p.pack_x = p.pack_w = false;
        p.splits_z = small_splits;
    } else if (p.few) {
        p.kept = true;
        p.pack_x = p.pack_w = false;
        p.splits_z = few_splits;
    } else if (p.thin) {
        p.kept = true;
        (p.thin_rows ? p.pack_w : p.pack_x) = false;
        p.splits_z = p.thin_z.parts;
    } else if (few_tiles && fits) p.kept = true;
    else if (grad && bf16 && !d->has_bias && dz_bytes <= limit && d->d >= 512) p.exps = true;
    else p.kept = grad && fits && d->d >= (bf16 ? 1024 : 256);
    if (!grad && p.splits_z == 1 && !p.small && !p.few && !p.thin) p.kept = false;          // statistics are all that is wanted
    if (!p.kept) p.splits_z = 1;
    // epilogues with statistics make them of 128 columns a warp
    p.bn_z = p.kept && (p.splits_z > 1 || d->v <= XE_ROWS_MAX_V) ? cz.bn : XE_BN;
    p.piece = d->v;
    p.pieces = 1;
    if (grad && !p.kept && !p.exps) {
        // dz, and partial column sums of 32 rows each
        long long most = limit / (n > 0 ? n * 2 * p.planes + (d->has_bias ? n / 8 : 0) : 1) / XE_BN * XE_BN;
        if (most < XE_BN) most = XE_BN;
        if (most < v) {
            p.pieces = (int)((v + most - 1) / most);
            p.piece = (int)round_up_ll((v + p.pieces - 1) / p.pieces, XE_BN);
            p.pieces = (int)((v + p.piece - 1) / p.piece);
        }
    }
    p.dzpitch = round_up(p.piece, 8);
    p.dpitch = round_up(d->d, 4);
    const Cut cx = cut_product(n, d->d, (p.piece + XE_BK - 1) / XE_BK, products, true), cw = cut_product(p.piece, d->d, (n + XE_BK - 1) / XE_BK, products, true);
    p.splits_dx = p.thin && p.thin_rows ? p.thin_grad.parts : cx.splits;
    p.splits_dw = p.thin && !p.thin_rows ? p.thin_grad.parts : cw.splits;
    p.bn_dx = cx.bn; p.bn_dw = cw.bn;
    p.splits_few = few_split_count(col_tiles, long_tiles);
    // more than one piece adds up in floats: in dx itself, or in the scratch
    p.dx_direct = p.splits_dx == 1 && (p.pieces == 1 || !bf16);
    p.dw_direct = p.splits_dw == 1;
    p.parts = p.kept ? kept_parts : (int)((n + XE_ROWS_PER_PART - 1) / XE_ROWS_PER_PART);
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
    p.off_count = take(8);               // rows that count, blocks that are done
    const size_t vtiles = (size_t)((v + XE_STAT_COLS - 1) / XE_STAT_COLS);
    p.off_zsum = take(d->label_smoothing > 0.f ? vtiles * un * 4 : 0);
    p.off_stats = take(vtiles * un * 8);
    p.off_z = take(p.kept ? un * p.zpitch * 4 * p.splits_z : 0);
    p.off_x = take(p.pack_x ? un * p.dp * 2 * p.planes : 0);
    p.off_w = take(p.pack_w ? (size_t)v * p.dp * 2 * p.planes : 0);
    if (grad) {
        p.off_dz = take(p.small || p.few ? 0 : un * p.dzpitch * 2 * p.planes);      // those two: in the place of the logits
        p.off_db = take(d->has_bias ? (size_t)p.parts * p.dzpitch * 4 : 0);
        p.off_dx = take(p.few ? (size_t)(p.few_rows ? n : v) * p.dpitch * 4 * p.splits_few : p.dx_direct ? 0 : un * p.dpitch * 4 * p.splits_dx);
        p.off_dw = take(p.few || p.dw_direct ? 0 : (size_t)p.piece * p.dpitch * 4 * p.splits_dw);
    }
    p.total = off + 256;
    *out = p;
    return WINO_OK;
}

// Every kernel of a call is launched with programmatic serialisation and waits for its predecessor itself, so that its blocks
// are set up as that one's leave.  Measured per call: 256 x 25088 x 1000 with gradients 70.8 -> 63.6 us, 512 x 2048 x 8000
// 85.8 -> 75.0 us.  No kernel lets its successor in any earlier: blocks that wait hold registers and shared memory (64.4 us, 83.3 us).
template <typename... KArgs, typename... Args>
int xe_launch(void (*kernel)(KArgs...), dim3 grid, int block, size_t smem, cudaStream_t st, Args... args) {
    count_launch();
    WINO_CUDA_CHECK(launch_kernel(kernel, grid, dim3((unsigned)block), smem, st, true, args...));
    return WINO_OK;
}

// A plan follows from the descriptor and the number of SMs alone; the last one of a thread is kept, since programs come
// back with the same descriptor step after step.
int make_plan(const wino_xent_desc* d, bool grad, Plan* out) {
    struct Last { wino_xent_desc d; bool grad; int sms; Plan plan; };
    static thread_local Last last = {};
    const int sms = sm_count();
    if (d && last.sms == sms && last.grad == grad && memcmp(&last.d, d, sizeof(*d)) == 0) { *out = last.plan; return WINO_OK; }
    const int rc = build_plan(d, grad, out);
    if (rc == WINO_OK) { memcpy(&last.d, d, sizeof(*d)); last.grad = grad; last.sms = sms; last.plan = *out; }
    return rc;
}

// planes: 0, 1, 3 as in xe_rows_kernel, -1 for statistics and loss alone
template <int THREADS, int QUADS>
int launch_rows(int planes, unsigned blocks, cudaStream_t st, const float* z, int splits, int v, int zpitch, const float* bias, const RowArgs& ra,
                 const XeDzRule& rule, void* dz, int dpitch, float* db_part) {
    auto go = [&](auto kernel) { return xe_launch(kernel, blocks, THREADS, 0, st, z, splits, v, zpitch, bias, ra, rule, dz, dpitch, db_part); };
    const bool split = splits > 1;
    if (planes < 0) return split ? go(xe_rows_kernel<THREADS, QUADS, 1, false, true>) : go(xe_rows_kernel<THREADS, QUADS, 1, false, false>);
    if (planes == 1) return split ? go(xe_rows_kernel<THREADS, QUADS, 1, true, true>) : go(xe_rows_kernel<THREADS, QUADS, 1, true, false>);
    if (planes == 3) return split ? go(xe_rows_kernel<THREADS, QUADS, 3, true, true>) : go(xe_rows_kernel<THREADS, QUADS, 3, true, false>);
    return split ? go(xe_rows_kernel<THREADS, QUADS, 0, true, true>) : go(xe_rows_kernel<THREADS, QUADS, 0, true, false>);
}

int launch_warp_rows(int planes, unsigned blocks, cudaStream_t st, const float* z, int splits, int v, int zpitch, const float* bias, const RowArgs& ra,
                     const XeDzRule& rule, void* dz, int dpitch, float* db_part) {
    auto go = [&](auto kernel) { return xe_launch(kernel, blocks, 32 * XE_WARP_ROWS, 0, st, z, splits, v, zpitch, bias, ra, rule, dz, dpitch, db_part); };
    const bool split = splits > 1;
    if (planes < 0) return split ? go(xe_warp_rows_kernel<1, false, true>) : go(xe_warp_rows_kernel<1, false, false>);
    if (planes == 1) return split ? go(xe_warp_rows_kernel<1, true, true>) : go(xe_warp_rows_kernel<1, true, false>);
    if (planes == 3) return split ? go(xe_warp_rows_kernel<3, true, true>) : go(xe_warp_rows_kernel<3, true, false>);
    return split ? go(xe_warp_rows_kernel<0, true, true>) : go(xe_warp_rows_kernel<0, true, false>);
}

template <typename T>
int launch_small_logits(const void* x, long long ldx, const void* w, long long ldw, const wino_xent_desc& d, const Plan& p, float* z, int* zero, cudaStream_t st) {
    const dim3 grid((unsigned)(d.v + 7) / 8, (unsigned)(d.n + XE_SMALL_ROWS - 1) / XE_SMALL_ROWS, (unsigned)p.splits_z);
    return xe_launch(xe_small_logits_kernel<T>, grid, 256, 0, st, (const T*)x, ldx, (const T*)w, ldw, d.n, d.d, d.v, p.zpitch, z, zero);
}

template <typename T>
int launch_small_grad(const void* x, const void* w, void* dx, void* dw, float* db, const wino_xent_desc& d, const Plan& p, const float* dz, const XeScale& scale,
                      const XeLoss& loss, const RowArgs& ra, cudaStream_t st) {
    SmallGrad<T> a;
    a.x = (const T*)x; a.w = (const T*)w; a.dx = (T*)dx; a.dw = (T*)dw; a.db = db;
    a.ldx = p.ldx; a.ldw = p.ldw; a.lddx = p.lddx; a.lddw = p.lddw;
    a.dz = dz; a.n = d.n; a.d = d.d; a.v = d.v; a.dzpitch = p.zpitch;
    a.kblocks = (d.d + 127) / 128;
    a.dx_blocks = dx ? (d.n + 7) / 8 * a.kblocks : 0;
    a.scale = scale;
    a.loss = loss;
    a.rule = ra.rule; a.target = ra.target; a.count = ra.count;
    const int dw_blocks = dw || db ? (d.v + 7) / 8 * a.kblocks : 0;
    return xe_launch(xe_small_grad_kernel<T>, (unsigned)(a.dx_blocks + dw_blocks + (loss.loss ? 1 : 0)), 256, XE_SMALL_GRAD_SMEM, st, a);
}

int launch_db(const float* part, int parts, int pitch, int cols, const XeScale& scale, float* db, cudaStream_t st) {
    if (cols < 4096) return xe_launch(xe_db_kernel<8>, (unsigned)(cols + 7) / 8, 512, 0, st, part, parts, pitch, cols, scale, db);
    return xe_launch(xe_db_kernel<32>, (unsigned)(cols + 31) / 32, 512, 0, st, part, parts, pitch, cols, scale, db);
}

int finish(const wino_xent_desc& d, const Plan& p, const float* buf, int splits, long long rows, void* out, long long ld, cudaStream_t st) {
    const unsigned blocks = loop_blocks(rows * ((d.d + 3) / 4));
    if (d.dtype == WINO_BF16) return xe_launch(xe_finish_kernel<__nv_bfloat16>, blocks, 256, 0, st, buf, splits, rows, d.d, p.dpitch, (__nv_bfloat16*)out, ld);
    return xe_launch(xe_finish_kernel<float>, blocks, 256, 0, st, buf, splits, rows, d.d, p.dpitch, (float*)out, ld);
}

FewArgs few_args(const void* x, const void* w, const wino_xent_desc& d, const Plan& p, const float* rowg) {
    FewArgs a = {};
    a.d = d.d;
    if (p.few_rows) {
        a.x = (const float*)x; a.w = (const float*)w;
        a.ldx = p.ldx; a.ldw = p.ldw;
        a.n = d.n; a.v = d.v; a.zr = p.zpitch; a.zj = 1;
        a.xg = rowg;
    } else {
        a.x = (const float*)w; a.w = (const float*)x;
        a.ldx = p.ldw; a.ldw = p.ldx;
        a.n = d.v; a.v = d.n; a.zr = 1; a.zj = p.zpitch;
        a.wg = rowg;
    }
    return a;
}

// the kernel for 4 or 8 rows
template <typename Pick>
int few_launch(int n, dim3 grid, cudaStream_t st, const FewArgs& a, Pick pick) {
    if (n <= 4) return xe_launch(pick(std::integral_constant<int, 4>()), grid, 128, 0, st, a);
    return xe_launch(pick(std::integral_constant<int, 8>()), grid, 128, 0, st, a);
}

int launch_few_logits(const void* x, const void* w, const wino_xent_desc& d, const Plan& p, float* z, int* zero, cudaStream_t st) {
    FewArgs a = few_args(x, w, d, p, nullptr);
    a.out = z; a.plane = (long long)d.n * p.zpitch;
    a.splits = p.splits_z;
    a.zero = zero;
    const dim3 grid((unsigned)((a.v + XF_CLASSES - 1) / XF_CLASSES), (unsigned)a.splits);
    return few_launch(a.n, grid, st, a, [](auto rows) { return xe_few_logits_kernel<decltype(rows)::value>; });
}

int launch_few_grad(const void* x, const void* w, void* dx, void* dw, const wino_xent_desc& d, const Plan& p, const float* dz, float* buf, const float* rowg,
                    const XeScale& scale, cudaStream_t st) {
    FewArgs a = few_args(x, w, d, p, rowg);
    a.dz = dz; a.scale = scale;
    const unsigned kblocks = (unsigned)((d.d + XF_COLS - 1) / XF_COLS), jblocks = (unsigned)((a.v + XF_CLASSES - 1) / XF_CLASSES);
    void* few = p.few_rows ? dx : dw;              // the gradient of the matrix of few rows, and of the long one
    void* full = p.few_rows ? dw : dx;
    const long long ld_few = p.few_rows ? p.lddx : p.lddw, ld_full = p.few_rows ? p.lddw : p.lddx;
    int rc;
    if (few) {
        const bool direct = p.splits_few == 1;
        a.out = direct ? (float*)few : buf; a.ldo = direct ? ld_few : p.dpitch; a.plane = (long long)a.n * p.dpitch;
        a.splits = p.splits_few;
        const dim3 grid(kblocks, (unsigned)a.splits);
        rc = few_launch(a.n, grid, st, a, [](auto rows) { return xe_few_dx_kernel<decltype(rows)::value>; });
        if (rc || (!direct && (rc = finish(d, p, buf, a.splits, a.n, few, ld_few, st)))) return rc;
    }
    if (full) {
        a.out = (float*)full; a.ldo = ld_full;
        const dim3 grid(kblocks * jblocks);
        rc = few_launch(a.n, grid, st, a, [](auto rows) { return xe_few_dw_kernel<decltype(rows)::value>; });
        if (rc) return rc;
    }
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
    if ((dx && (dx == x || dx == w)) || (dw && (dw == x || dw == w || dw == dx))) return fail(WINO_E_BADARG, "xent: a result in the place of another matrix");
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
    XeOperand ox = {x, n, d.d, p.ldx, n * p.ldx, p.planes, false}, ow = {w, v, d.d, p.ldw, v * p.ldw, p.planes, false};
    if (p.pack_x || p.pack_w) {
        PackJob jobs[2] = {};
        int k = 0;
        if (p.pack_x) {
            jobs[k++] = {x, p.ldx, n, reinterpret_cast<__nv_bfloat16*>(ws + p.off_x), grad && d.has_ignore ? target : nullptr};
            ox = {ws + p.off_x, n, d.d, p.dp, n * p.dp, p.planes, false};
        }
        if (p.pack_w) {
            jobs[k++] = {w, p.ldw, v, reinterpret_cast<__nv_bfloat16*>(ws + p.off_w), nullptr};
            ow = {ws + p.off_w, v, d.d, p.dp, v * p.dp, p.planes, false};
        }
        const unsigned blocks = loop_blocks((jobs[0].rows + jobs[1].rows) * (p.dp / 4));
        if (d.dtype == WINO_BF16 && ((p.pack_x && p.ldx % 8) || (p.pack_w && p.ldw % 8))) {
            const bool pairs = !(p.pack_x && p.ldx % 2) && !(p.pack_w && p.ldw % 2);
            const unsigned warp_blocks = loop_blocks((jobs[0].rows + jobs[1].rows) * ((p.dp + 255) / 256) * 32);
            rc = xe_launch(pairs ? xe_pack_rows_kernel<true> : xe_pack_rows_kernel<false>, warp_blocks, 256, 0, st, jobs[0], jobs[1], d.d, p.dp, rule);
        } else if (d.dtype == WINO_BF16) rc = xe_launch(xe_pack_kernel<__nv_bfloat16, 1>, blocks, 256, 0, st, jobs[0], jobs[1], d.d, p.dp, rule);
        else rc = xe_launch(xe_pack_kernel<float, 3>, blocks, 256, 0, st, jobs[0], jobs[1], d.d, p.dp, rule);
        if (rc) return rc;
    }

    const float s = d.label_smoothing, dz_factor = s <= 0.5f ? 1.f - s : 1.f;
    XeDzRule dzr;
    dzr.pf = 1.f / dz_factor;
    dzr.smooth_t = s <= 0.5f ? 1.f : 1.f - s;
    dzr.smooth_all = (float)((double)s / (double)v / (double)dz_factor);
    RowArgs ra;
    ra.rule = rule; ra.n = n; ra.target = target;
    ra.dloss = d.reduction == WINO_NONE ? dloss : nullptr;
    ra.smooth = s; ra.inv_v = (float)(1.0 / (double)v);
    ra.lse = f(p.off_lse); ra.lse_out = lse; ra.rowg = f(p.off_rowg);
    ra.rowloss = d.reduction == WINO_NONE ? loss : f(p.off_rowloss);
    ra.count = reinterpret_cast<int*>(ws + p.off_count);
    // the sum of the losses goes to the rows' last block, or, where gradients follow and a warp is done with it in good
    // time, to one that idles in their kernel
    const bool products = grad && (dx || dw || db);
    XeLoss sum;
    sum.loss = d.reduction == WINO_NONE ? nullptr : loss;
    sum.rowloss = ra.rowloss; sum.n = n; sum.count = ra.count;
    sum.mean = d.reduction == WINO_MEAN;
    const bool later = products && (dx || dw) && n <= 1024 && !p.few && (!p.thin || (p.thin_rows ? dw : dx));
    const bool tiny = p.tiny && (products ? d.n <= XE_SMALL_MAX : d.reduction == WINO_NONE || d.n <= XE_SMALL_ROWS);
    if (!later && !(tiny && products)) ra.loss = sum;
    if ((rc = status_word(&ra.status))) return rc;
    const float* b = d.has_bias ? bias : nullptr;
    const bool wide = d.v > XE_ROWS_MAX_V;
    __nv_bfloat16* dz = reinterpret_cast<__nv_bfloat16*>(ws + p.off_dz);
    float* db_part = db ? f(p.off_db) : nullptr;
    XeScale scale;
    scale.count = ra.count;
    scale.dloss = d.reduction == WINO_NONE ? nullptr : dloss;
    scale.factor = dz_factor;
    scale.mean = sum.mean;

    if (tiny) {
        float* z = f(p.off_z);
        const unsigned blocks = (unsigned)((n + XE_SMALL_ROWS - 1) / XE_SMALL_ROWS);
        auto go = [&](auto t) {
            using T = decltype(t);
            auto kernel = products ? xe_tiny_kernel<T, true> : xe_tiny_kernel<T, false>;
            return xe_launch(kernel, blocks, 32 * XE_TINY_WARPS, 0, st, (const T*)x, p.ldx, (const T*)w, p.ldw, d.d, d.v, p.zpitch, b, ra, dzr, z);
        };
        if ((rc = p.es == 2 ? go(__nv_bfloat16()) : go(float()))) return rc;
        if (!products) return WINO_OK;
        return p.es == 2 ? launch_small_grad<__nv_bfloat16>(x, w, dx, dw, db, d, p, z, scale, sum, ra, st)
                         : launch_small_grad<float>(x, w, dx, dw, db, d, p, z, scale, sum, ra, st);
    }
    XeThin thin = {};                  // the long matrix
    thin.l = (const float*)(p.thin_rows ? w : x); thin.rows = p.thin_rows ? v : n; thin.ldl = p.thin_rows ? p.ldw : p.ldx; thin.d = d.d;
    const bool kept_stats = p.kept && wide && p.splits_z == 1 && !p.few && !p.thin;
    XeProduct pz = {kept_stats ? XE_STATS_Z : p.kept ? XE_F32 : p.exps ? XE_STATS_E : XE_STATS, ox, ow, n, v, d.d, XeOutput()};
    pz.bn = p.bn_z;
    pz.out.zero = ra.count;
    if (p.kept && !kept_stats) {
        float* z = f(p.off_z);
        pz.out.ptr = z;
        pz.out.pitch = p.zpitch;
        pz.out.splits = p.splits_z;
        if (p.few) rc = launch_few_logits(x, w, d, p, z, ra.count, st);
        else if (p.thin) {
            XeThin t = thin;
            t.s = p.thin_rows ? ox : ow;
            t.out = z; t.plane = n * p.zpitch;
            t.out_s = p.thin_rows ? p.zpitch : 1; t.out_m = p.thin_rows ? 1 : p.zpitch;
            t.cut = p.thin_z;
            t.zero = ra.count;
            rc = xe_thin(t, st);
        } else if (!p.small) rc = xe_gemm(&pz, 1, st);
        else if (p.es == 2) rc = launch_small_logits<__nv_bfloat16>(x, p.ldx, w, p.ldw, d, p, z, ra.count, st);
        else rc = launch_small_logits<float>(x, p.ldx, w, p.ldw, d, p, z, ra.count, st);
        if (rc) return rc;
        if (wide) {
            const unsigned chunks = (unsigned)((v + XE_CHUNK - 1) / XE_CHUNK);
            float2* stats = reinterpret_cast<float2*>(ws + p.off_stats);
            float* zsum = d.label_smoothing > 0.f ? f(p.off_zsum) : nullptr;
            if ((rc = xe_launch(xe_wide_stats_kernel, chunks * (unsigned)n, 256, 0, st, z, p.splits_z, d.v, p.zpitch, b, n, target, stats, zsum, f(p.off_zt)))) return rc;
            rc = xe_launch(xe_rows_from_stats_kernel, (unsigned)((n + 31) / 32), 256, 0, st, stats, zsum, f(p.off_zt), (int)chunks, ra);
        } else {
            const unsigned blocks = (unsigned)row_blocks(n, d.v);
            auto rows_fn = d.v <= 512 ? launch_warp_rows : d.v <= 1024 ? launch_rows<256, 1> : d.v <= 2048 ? launch_rows<256, 2>
                         : d.v <= 4096 ? launch_rows<256, 4> : launch_rows<512, 4>;
            // floats in the place of the logits; column sums where there are more rows than the products' kernels add up
            float* few_db = p.few && !p.few_rows ? db_part : nullptr;
            if ((p.small || p.few) && products) rc = rows_fn(0, blocks, st, z, p.splits_z, d.v, p.zpitch, b, ra, dzr, z, p.zpitch, few_db);
            else rc = rows_fn(products ? p.planes : -1, blocks, st, z, p.splits_z, d.v, p.zpitch, b, ra, dzr, dz, p.dzpitch, db_part);
        }
    } else {
        pz.out.bias = b;
        pz.out.target = target;
        pz.out.stats = reinterpret_cast<float2*>(ws + p.off_stats);
        pz.out.zsum = d.label_smoothing > 0.f ? f(p.off_zsum) : nullptr;
        pz.out.zt = f(p.off_zt);
        if (kept_stats) {
            pz.out.ptr = f(p.off_z);
            pz.out.pitch = p.zpitch;
        } else if (p.exps) {
            pz.out.ptr = dz;
            pz.out.pitch = p.dzpitch;
        }
        if ((rc = xe_gemm(&pz, 1, st))) return rc;
        rc = xe_launch(xe_rows_from_stats_kernel, (unsigned)((n + 31) / 32), 256, 0, st, pz.out.stats, pz.out.zsum, pz.out.zt, (int)((v + XE_STAT_COLS - 1) / XE_STAT_COLS), ra);
    }
    if (rc) return rc;

    if (!products) return WINO_OK;
    if (p.small)
        return p.es == 2 ? launch_small_grad<__nv_bfloat16>(x, w, dx, dw, db, d, p, f(p.off_z), scale, later ? sum : XeLoss(), ra, st)
                         : launch_small_grad<float>(x, w, dx, dw, db, d, p, f(p.off_z), scale, later ? sum : XeLoss(), ra, st);
    if (p.few) {
        float* z = f(p.off_z);
        if (wide) {
            const unsigned grid = (unsigned)((v + 255) / 256) * (unsigned)((n + XE_ROWS_PER_PART - 1) / XE_ROWS_PER_PART);
            if ((rc = xe_launch(xe_wide_dz_kernel<0>, grid, 128, 0, st, z, d.v, p.zpitch, n, ra.lse, ra.rowg, target, dzr, z, p.zpitch, nullptr))) return rc;
        }
        if (db && (rc = p.few_rows ? launch_db(z, (int)n, p.zpitch, d.v, scale, db, st) : launch_db(db_part, p.parts, p.zpitch, d.v, scale, db, st))) return rc;
        return launch_few_grad(x, w, dx, dw, d, p, z, f(p.off_dx), ra.rowg, scale, st);
    }
    for (int i = 0; i < p.pieces; ++i) {
        const int v0 = i * p.piece, vc = d.v - v0 < p.piece ? d.v - v0 : p.piece;
        XeOperand wp = ow;                 // the piece's rows of W
        wp.ptr = static_cast<const char*>(ow.ptr) + (size_t)v0 * ow.pitch * 2;
        wp.rows = vc;
        if (p.kept && wide) {
            const unsigned grid = (unsigned)((vc + 255) / 256) * (unsigned)p.parts;
            if (p.planes == 1) rc = xe_launch(xe_wide_dz_kernel<1>, grid, 128, 0, st, f(p.off_z), vc, p.zpitch, n, ra.lse, ra.rowg, target, dzr, dz, p.dzpitch, db_part);
            else rc = xe_launch(xe_wide_dz_kernel<3>, grid, 128, 0, st, f(p.off_z), vc, p.zpitch, n, ra.lse, ra.rowg, target, dzr, dz, p.dzpitch, db_part);
        } else if (p.exps) {
            const long long spans = n * ((p.dzpitch / 8 + 1023) / 1024);
            rc = xe_launch(xe_dz_from_exp_kernel, (unsigned)(spans < 0x7fffffffll ? spans : 0x7fffffffll), 256, 0, st, dz, p.dzpitch, n, pz.out.stats, pz.out.zt,
                           ra.lse, ra.rowg, target, dzr);
        } else if (!p.kept) {
            XeProduct pd = {XE_DZ, ox, wp, n, vc, d.d, XeOutput()};
            pd.out.ptr = dz; pd.out.pitch = p.dzpitch;
            pd.out.bias = b ? b + v0 : nullptr;
            pd.out.target = target; pd.out.col_base = v0;
            pd.out.lse = ra.lse; pd.out.rowg = ra.rowg; pd.out.rule = dzr;
            pd.out.db_part = db_part; pd.out.db_pitch = p.dzpitch;
            if ((rc = xe_gemm(&pd, 1, st))) return rc;
        }
        if (rc) return rc;
        if (db && (rc = launch_db(db_part, p.parts, p.dzpitch, vc, scale, db + v0, st))) return rc;

        const XeOperand odz = {dz, n, vc, p.dzpitch, n * p.dzpitch, p.planes, false};
        const bool bf16 = p.planes == 1, first = i == 0, last = i == p.pieces - 1;
        XeProduct prod[2];
        int count = 0;
        auto product = [&](const XeOperand& a, const XeOperand& b, long long rows, long long k, bool direct, int splits, int bn, bool add, void* out,
                           long long ld, float* buf) {
            XeProduct& q = prod[count++];
            q = {direct && bf16 ? XE_BF16 : XE_F32, a, b, rows, d.d, k, XeOutput()};
            q.bn = bn;
            q.out.scale = scale;
            q.out.add = add;
            q.out.exact = direct;
            q.out.ptr = direct ? out : buf;
            q.out.pitch = direct ? ld : p.dpitch;
            const long long chunks = (k + XE_BK - 1) / XE_BK;          // a short last piece adds to fewer of the parts
            q.out.splits = direct ? 1 : chunks < splits ? (int)chunks : splits;
        };
        void* dw_at = static_cast<char*>(dw) + (size_t)v0 * p.lddw * p.es;
        const bool thin_dx = p.thin && p.thin_rows, thin_dw = p.thin && !p.thin_rows;
        if (thin_dx ? dx != nullptr : thin_dw && dw) {
            XeThin t = thin;
            t.along_rows = true;
            t.rowg = thin_dw ? ra.rowg : nullptr;
            t.s = odz;
            t.s.along_rows = thin_dw;
            const bool direct = thin_dx ? p.dx_direct : p.dw_direct;
            t.out = thin_dx ? (direct ? (float*)dx : f(p.off_dx)) : (direct ? (float*)dw : f(p.off_dw));
            t.out_s = !direct ? p.dpitch : thin_dx ? p.lddx : p.lddw; t.out_m = 1;
            t.plane = (thin_dx ? n : v) * p.dpitch;
            t.cut = p.thin_grad;
            t.scale = scale;
            if ((rc = xe_thin(t, st))) return rc;
        }
        if (dx && !thin_dx) {
            XeOperand wr = wp;
            wr.along_rows = true;
            product(odz, wr, n, vc, p.dx_direct, p.splits_dx, p.bn_dx, !first, dx, p.lddx, f(p.off_dx));
        }
        if (dw && !thin_dw) {
            XeOperand zr = odz, xr = ox;
            zr.along_rows = xr.along_rows = true;
            product(zr, xr, vc, n, p.dw_direct, p.splits_dw, p.bn_dw, false, dw_at, p.lddw, f(p.off_dw));
        }
        // Both in one launch where one of them has few tiles: the other fills the SMs that it leaves idle (256 x 25088 x 1000:
        // 46 -> 38 us).  With many turns of both there is nothing to fill, and the GPU runs at its power limit either way
        // (8192 x 4096 x 50021: 8.2 ms apart, 8.4 ms together).
        const long long tiles_x = (n + XE_BM - 1) / XE_BM * ((d.d + p.bn_dx - 1) / p.bn_dx) * p.splits_dx;
        const long long tiles_w = ((long long)vc + XE_BM - 1) / XE_BM * ((d.d + p.bn_dw - 1) / p.bn_dw) * p.splits_dw;
        if (first && later) prod[0].out.loss = sum;
        if (count == 2 && p.bn_dx == p.bn_dw && (tiles_x < tiles_w ? tiles_x : tiles_w) < sm_count()) {
            if ((rc = xe_gemm(prod, 2, st))) return rc;
        } else {
            for (int k = 0; k < count; ++k)
                if ((rc = xe_gemm(&prod[k], 1, st))) return rc;
        }
        if (dx && last && !p.dx_direct && (rc = finish(d, p, f(p.off_dx), p.splits_dx, n, dx, p.lddx, st))) return rc;
        if (dw && !p.dw_direct && (rc = finish(d, p, f(p.off_dw), p.splits_dw, vc, dw_at, p.lddw, st))) return rc;
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
