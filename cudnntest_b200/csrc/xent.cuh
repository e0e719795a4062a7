// Shared by the linear softmax cross entropy's products (xent_gemm.cu) and its driver and row kernels (xent.cu).
#pragma once

#include "ptx.cuh"

namespace wino {

constexpr int XE_BM = 256, XE_BN = 256, XE_BK = 64;      // tile of a CTA pair, contraction elements per ring slot
constexpr int XE_STATUS_TARGET = 100;                    // status word: a target outside 0 ... v-1

// A BF16 operand: `planes` matrices (parts of a split float operand, or one) of `rows` x `cols`, rows `pitch` and planes
// `plane_pitch` elements apart.  The contraction runs along the columns, or along the rows where `along_rows` is set.
struct XeOperand {
    const void* ptr;
    long long rows, cols, pitch, plane_pitch;
    int planes;
    bool along_rows;
};

// What the epilogue does with a 256 x 256 tile of the product (m rows x n columns)
enum XeEpilogue {
    XE_F32 = 0,       // scale, store floats or add them to what is there
    XE_BF16 = 1,      // scale, round and store
    XE_STATS = 2,     // per row and 128 columns: maximum, sum of exponentials (and of logits); the target's logit
    XE_STATS_E = 3,   // the same, and the exponentials exp(z - maximum) themselves, rounded to BF16
    XE_STATS_Z = 4,   // the same as XE_STATS, and the logits themselves (with the bias) as floats
    XE_DZ = 5,        // the gradient of the logits, rounded to BF16 (or split into three BF16 planes), and its column sums
};
constexpr int XE_STAT_COLS = 128;

// The gradient of a logit as it is stored: g ((p - s/v) / f - [target] (1 - s) / f), where f = 1 - s (1 if s > 1/2) and g is
// the row's weight without what all rows share.  The rest, f times the common factor, is applied to the finished products:
// a row's target has the value -1 + small, which BF16 holds well, where -(1 - s) / rows, alike in all rows, would be off by
// the same rounding in every one of them (measured: relative error of dx 3.7e-3 against 2.0e-3).
struct XeDzRule {
    float pf = 1.f;           // 1 / f
    float smooth_t = 1.f;     // (1 - s) / f
    float smooth_all = 0.f;   // s / v / f
};

// the factor all rows share: f of XeDzRule, the upstream gradient, 1 / (rows that count)
struct XeScale {
    const int* count = nullptr;       // NULL: 1
    const float* dloss = nullptr;     // NULL: 1
    float factor = 1.f;
    int mean = 0;
};
__device__ __forceinline__ float xe_scale(const XeScale& s, int n) {
    return s.factor * (s.dloss ? *s.dloss : 1.f) * (s.mean ? 1.f / (float)(n > 0 ? n : 1) : 1.f);
}
__device__ __forceinline__ float xe_scale(const XeScale& s) { return s.count ? xe_scale(s, *s.count) : 1.f; }

// the mean or sum of the rows' losses
struct XeLoss {
    float* loss = nullptr;            // NULL: nothing to do
    const float* rowloss = nullptr;
    long long n = 0;
    const int* count = nullptr;       // rows that count
    int mean = 0;
};
// by the first THREADS threads of a block, all of which call it (one warp: no barrier)
template <int THREADS>
__device__ __forceinline__ void xe_sum_losses(const XeLoss& a) {
    __shared__ double rs[THREADS / 32];
    const int tid = threadIdx.x % THREADS;
    double sum = 0;
#pragma unroll 8
    for (long long i = tid; i < a.n; i += THREADS) sum += __ldcg(a.rowloss + i);
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    if (THREADS > 32) {
        if (tid % 32 == 0) rs[tid / 32] = sum;
        __syncthreads();
        if (tid == 0)
            for (int i = 1; i < THREADS / 32; ++i) sum += rs[i];
    }
    if (tid == 0) {
        const int count = __ldcg(a.count);
        *a.loss = (float)(a.mean ? sum / (count > 0 ? count : 1) : sum);
    }
}

struct XeOutput {
    void* ptr = nullptr;            // XE_F32: [splits][m][pitch] floats; XE_BF16, XE_STATS_E, XE_STATS_Z: m rows; XE_DZ: [planes][m][pitch] BF16
    long long pitch = 0;
    int splits = 1;                 // parts of the contraction, one buffer each (XE_F32)
    bool add = false;               // XE_F32: add instead of store
    bool exact = false;             // nothing behind a row's last column may be written
    XeScale scale;                  // XE_F32, XE_BF16: what the product is multiplied by
    // XE_STATS*, XE_DZ
    const float* bias = nullptr;    // of column 0 of this product
    const long long* target = nullptr;
    int col_base = 0;               // class number of column 0
    float2* stats = nullptr;        // [n / 128][m] (maximum, sum)
    float* zsum = nullptr;          // [n / 128][m] sum of logits, or NULL
    float* zt = nullptr;            // [m] logit of the target
    const float* lse = nullptr;     // [m]
    const float* rowg = nullptr;    // [m] weight of a row, 0 for one that does not count
    XeDzRule rule;
    float* db_part = nullptr;       // [m / 32][db_pitch] column sums of 32 rows each, or NULL
    long long db_pitch = 0;
    int* zero = nullptr;            // two device words set to 0, or NULL
    XeLoss loss;                    // summed by a warp that has nothing else to do
};

// one product of a (m x k) and b (n x k)^T, contraction length k
struct XeProduct {
    XeEpilogue epi;
    XeOperand a, b;
    long long m, n, k;
    XeOutput out;
    int bn = XE_BN;                   // columns of a tile: 256, or 128 (XE_F32, XE_BF16)
};
// one or two products in one launch; two must have the same bn and epilogues XE_F32 or XE_BF16
int xe_gemm(const XeProduct* prod, int count, cudaStream_t st);

__device__ __forceinline__ float xe_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float XE_LOG2E = 1.4426950408889634f;

// v = p0 + p1 + p2 with BF16 parts (each remainder is rounded to nearest, so three parts hold 24 bits).  A float that
// rounds to BF16's infinity keeps its upper half instead; infinities and NaN stay in the first part.
__device__ __forceinline__ void xe_split3(float v, __nv_bfloat16& p0, __nv_bfloat16& p1, __nv_bfloat16& p2) {
    p0 = __float2bfloat16_rn(v);
    const uint32_t mag = __float_as_uint(v) & 0x7fffffffu;
    if (mag >= 0x7f7f8000u) {
        if (mag >= 0x7f800000u) { p1 = p2 = __float2bfloat16_rn(0.f); return; }
        p0 = __ushort_as_bfloat16((unsigned short)(__float_as_uint(v) >> 16));
    }
    const float r1 = v - __bfloat162float(p0);
    p1 = __float2bfloat16_rn(r1);
    p2 = __float2bfloat16_rn(r1 - __bfloat162float(p1));
}

}  // namespace wino
