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

// boxes of 64 columns (128 bytes, 128-byte swizzle): `share` rows for a K-major share, 64 rows (one contraction element each)
// for an MN-major one
int xe_operand_map(CUtensorMap* map, const XeOperand& o, unsigned share);

// MN-major tile with 128-byte swizzle: rows of 64 elements (128 bytes) along M or N, one row per contraction element,
// groups of 8 contraction elements 1 KiB apart, blocks of 64 M / N elements 8 KiB apart
__device__ __forceinline__ uint64_t smem_desc_mn128(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
    d |= (uint64_t)(8192 >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// what a wait that ran out was for
enum XeWaitCode {
    XE_WAIT_EMPTY = 51, XE_WAIT_FULL = 52, XE_WAIT_TMEM_EMPTY = 53, XE_WAIT_TMEM_FULL = 54,        // xent_gemm.cu
    XT_WAIT_EMPTY = 61, XT_WAIT_FULL = 62, XT_WAIT_TMEM_EMPTY = 63, XT_WAIT_TMEM_FULL = 64,        // xent_thin.cu
};

// What the epilogue does with a 256 x 256 tile of the product (m rows x n columns)
enum XeEpilogue {
    XE_F32 = 0,       // scale, store floats or add them to what is there
    XE_BF16 = 1,      // scale, round and store
    XE_STATS = 2,     // per row and 128 columns: maximum, sum of exponentials (and of logits); the target's logit
    XE_STATS_E = 3,   // the same, and the exponentials exp(z - maximum) themselves, in 16 bits (xe_pack_exp)
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

// how a product is shared: CTAs, and the buffers that hold pieces of the same tile
struct XeThinCut {
    int grid, parts;
};
// Product of a matrix L of floats as it lies with up to 128 rows s of BF16 planes (xent_thin.cu): out[s][row of L] = s L^T, or,
// where `along_rows` is set, out[s][column of L] = s L, the contraction along the rows of L.
struct XeThin {
    const float* l;
    long long rows, ldl;
    int d;                            // columns of L
    bool along_rows;
    const float* rowg = nullptr;      // rows of L with weight 0 are taken as zeros, or NULL
    XeOperand s;                      // its rows: 1 ... 128 (or its columns, where s.along_rows is set)
    float* out;                       // [parts][..]
    long long out_s, out_m, plane;    // elements from one row of s to the next, along the other extent, between buffers
    XeThinCut cut;
    XeScale scale;
    int* zero = nullptr;              // two device words set to 0, or NULL
};
int xe_thin(const XeThin& t, cudaStream_t st);
// for `tiles` tiles of 128 and a contraction of `chunks` times 64, where a buffer costs `part_us`
XeThinCut xe_thin_cut(long long tiles, long long chunks, double part_us);

__device__ __forceinline__ float xe_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float XE_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void prefetch_tensor_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// ties registers that tcgen05.ld fills to the wait before this: no use of them can be moved ahead of it
__device__ __forceinline__ void after_wait(uint32_t (&r)[16]) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                      "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 o = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&o);
}

// Two exponentials of at most 1 in a word, the first in the lower half: a float's sign and upper exponent bit are 0 there, so
// 16 bits hold its other 7 exponent bits and 9 of the fraction, two more than BF16 (rounded to nearest: off by 2^-10 of itself,
// where BF16 is off by 2^-8; dz, which is made of them, is rounded to BF16 afterwards).  NaN becomes some number.
__device__ __forceinline__ uint32_t xe_pack_exp(float lo, float hi) {
    return __byte_perm((__float_as_uint(lo) << 2) + 0x8000u, (__float_as_uint(hi) << 2) + 0x8000u, 0x7632);
}
__device__ __forceinline__ float2 xe_unpack_exp(uint32_t w) {
    return make_float2(__uint_as_float((w << 14) & 0x3fffc000u), __uint_as_float((w >> 2) & 0x3fffc000u));
}

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

// Two floats at once, the first in the lower half of each part; neither may be infinite or round to infinity (NaN may be there).
__device__ __forceinline__ void xe_split3_pair(float a, float b, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
    const float2 less = make_float2(-1.f, -1.f);           // (products with -1 are exact)
    p0 = pack_bf16(a, b);
    const float2 r1 = __ffma2_rn(make_float2(__uint_as_float(p0 << 16), __uint_as_float(p0 & 0xffff0000u)), less, make_float2(a, b));
    p1 = pack_bf16(r1.x, r1.y);
    const float2 r2 = __ffma2_rn(make_float2(__uint_as_float(p1 << 16), __uint_as_float(p1 & 0xffff0000u)), less, r1);
    p2 = pack_bf16(r2.x, r2.y);
}
constexpr float XE_SPLIT_MAX = 3.3895313892515355e38f;       // the largest BF16 value: floats up to it split like that

}  // namespace wino
