// Dropout with a mask that is computed where it is needed and never stored, forward and backward (the same linear map).
//
// Element e keeps its value, scaled by 65536 / (65536 - T), when 16 bits drawn for it are at least T = round(65536 p):
// p is met to 2^-17 and the scale belongs to the T that is used, so the expectation is exact.  The bits are lane e mod 8 of
// the eight 16-bit halves of Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011), counter (e div 8, offset), key = seed.
//
// Bound: one read and one write of the tensor.  Eight elements per Philox call rather than four (32 bits each): the ten
// rounds cost 20 wide multiplies, and at 4 bytes moved per BF16 element the multiplier would be the slower side with four.
#include <cmath>

#include "ptx.cuh"

namespace wino {

namespace {

constexpr int DO_THREADS = 256;

struct DropoutArgs {
    long long rows, cols, ldx, ldy;
    unsigned long long seed, offset;
    const unsigned long long* offset_dev;
    uint32_t threshold;
    float scale;
};

// the eight 16-bit lanes of group g, as four words (low half first)
__device__ __forceinline__ uint4 philox10(unsigned long long g, unsigned long long offset, unsigned long long seed) {
    uint32_t c0 = (uint32_t)g, c1 = (uint32_t)(g >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ unsigned long long dropout_offset(const DropoutArgs& a) {
    return a.offset + (a.offset_dev ? *a.offset_dev : 0ull);
}

// BF16 pair: a half is kept when its 16 random bits reach T
__device__ __forceinline__ uint32_t drop_pair(uint32_t v, uint32_t r, uint32_t t, float scale) {
    const float lo = __uint_as_float(v << 16) * scale, hi = __uint_as_float(v & 0xffff0000u) * scale;
    const __nv_bfloat162 o = __floats2bfloat162_rn((r & 0xffffu) >= t ? lo : 0.f, (r >> 16) >= t ? hi : 0.f);
    return *reinterpret_cast<const uint32_t*>(&o);
}

// Whole groups of eight, 16-byte accesses: cols, pitches and bases allow it (a dense matrix counts as one long row).
// groups_per_row is the number of groups in a row; the group index is the counter.
template <bool BF16>
__global__ void __launch_bounds__(DO_THREADS) dropout_vec_kernel(const void* xin, void* yout, const DropoutArgs a,
                                                                 long long groups_per_row) {
    const long long g = (long long)blockIdx.x * DO_THREADS + threadIdx.x;
    const long long total = a.rows * groups_per_row;
    if (g >= total) return;
    long long ox = g * 8, oy = g * 8;
    if (a.rows > 1) {
        const long long r = g / groups_per_row, c = (g - r * groups_per_row) * 8;
        ox = r * a.ldx + c;
        oy = r * a.ldy + c;
    }
    const uint32_t t = a.threshold;
    if (BF16) {
        const uint4 v = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(xin) + ox);
        const uint4 q = philox10((unsigned long long)g, dropout_offset(a), a.seed);
        uint4 o;
        o.x = drop_pair(v.x, q.x, t, a.scale);
        o.y = drop_pair(v.y, q.y, t, a.scale);
        o.z = drop_pair(v.z, q.z, t, a.scale);
        o.w = drop_pair(v.w, q.w, t, a.scale);
        *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(yout) + oy) = o;
    } else {
        const float4* x = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(xin) + ox);
        const float4 v0 = x[0], v1 = x[1];
        const uint4 q = philox10((unsigned long long)g, dropout_offset(a), a.seed);
        float4 o0, o1;
        o0.x = (q.x & 0xffffu) >= t ? v0.x * a.scale : 0.f;
        o0.y = (q.x >> 16) >= t ? v0.y * a.scale : 0.f;
        o0.z = (q.y & 0xffffu) >= t ? v0.z * a.scale : 0.f;
        o0.w = (q.y >> 16) >= t ? v0.w * a.scale : 0.f;
        o1.x = (q.z & 0xffffu) >= t ? v1.x * a.scale : 0.f;
        o1.y = (q.z >> 16) >= t ? v1.y * a.scale : 0.f;
        o1.z = (q.w & 0xffffu) >= t ? v1.z * a.scale : 0.f;
        o1.w = (q.w >> 16) >= t ? v1.w * a.scale : 0.f;
        float4* y = reinterpret_cast<float4*>(reinterpret_cast<float*>(yout) + oy);
        y[0] = o0;
        y[1] = o1;
    }
}

// Any width, pitch and alignment: a warp takes 256 consecutive elements.  Each lane draws the keep bits of one group, and
// lane l then handles elements l, l + 32, ... so that accesses stay coalesced; the bits come over by shuffles.
template <typename T>
__global__ void __launch_bounds__(DO_THREADS) dropout_any_kernel(const T* x, T* y, const DropoutArgs a) {
    const int lane = threadIdx.x % 32;
    const long long warp = (long long)blockIdx.x * (DO_THREADS / 32) + threadIdx.x / 32;
    const long long total = a.rows * a.cols, e0 = warp * 256;
    if (e0 >= total) return;
    const uint4 q = philox10((unsigned long long)(warp * 32 + lane), dropout_offset(a), a.seed);
    const uint32_t t = a.threshold;
    const uint32_t keep = ((q.x & 0xffffu) >= t ? 1u : 0u) | ((q.x >> 16) >= t ? 2u : 0u) | ((q.y & 0xffffu) >= t ? 4u : 0u) |
                          ((q.y >> 16) >= t ? 8u : 0u) | ((q.z & 0xffffu) >= t ? 16u : 0u) | ((q.z >> 16) >= t ? 32u : 0u) |
                          ((q.w & 0xffffu) >= t ? 64u : 0u) | ((q.w >> 16) >= t ? 128u : 0u);
    long long r = (e0 + lane) / a.cols, c = (e0 + lane) - r * a.cols;
    float v[8];
    long long oy[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        oy[i] = -1;
        if (e0 + i * 32 + lane < total) {
            v[i] = to_float<T>(x[r * a.ldx + c]);
            oy[i] = r * a.ldy + c;
        }
        c += 32;
        if (c >= a.cols) {
            if (a.cols >= 32) { c -= a.cols; ++r; }
            else { r += c / a.cols; c %= a.cols; }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = __shfl_sync(0xffffffffu, keep, i * 4 + lane / 8);
        if (oy[i] >= 0) y[oy[i]] = from_float<T>((bits >> (lane % 8)) & 1u ? v[i] * a.scale : 0.f);
    }
}

int run_dropout(const char* what, int dtype, long long rows, long long cols, long long ldx, long long ldy, float p,
                unsigned long long seed, unsigned long long offset, const unsigned long long* offset_dev, const void* x, void* y,
                cudaStream_t st) {
    if (dtype != WINO_FP32 && dtype != WINO_BF16) return fail(WINO_E_BADARG, "%s: dtype must be WINO_FP32 or WINO_BF16", what);
    if (rows < 0 || cols < 0 || (cols > 0 && rows > (1ll << 62) / cols)) return fail(WINO_E_BADARG, "%s: bad extents", what);
    if (!(p >= 0.f && p <= 1.f)) return fail(WINO_E_BADARG, "%s: p must lie in [0, 1]", what);
    if (rows == 0 || cols == 0) return WINO_OK;
    if (ldx < cols || ldy < cols) return fail(WINO_E_BADARG, "%s: a pitch is smaller than a row", what);
    if (!x || !y) return fail(WINO_E_BADARG, "%s: NULL pointer", what);
    const int es = dtype == WINO_BF16 ? 2 : 4;
    if (((uintptr_t)x | (uintptr_t)y) % es || (uintptr_t)offset_dev % 8) return fail(WINO_E_BADARG, "%s: misaligned pointer", what);
    if (x == y && ldx != ldy) return fail(WINO_E_BADARG, "%s: in place needs equal pitches", what);
    int rc = check_device();
    if (rc) return rc;
    DropoutArgs a;
    a.rows = rows; a.cols = cols; a.ldx = ldx; a.ldy = ldy;
    a.seed = seed; a.offset = offset; a.offset_dev = offset_dev;
    a.threshold = (uint32_t)floor((double)p * 65536.0 + 0.5);
    a.scale = a.threshold < 65536u ? (float)(65536.0 / (65536.0 - a.threshold)) : 0.f;
    const bool dense = ldx == cols && ldy == cols;
    const bool aligned = (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    const long long total = rows * cols;
    const bool vec = aligned && (dense ? total % 8 == 0 : cols % 8 == 0 && (ldx * es) % 16 == 0 && (ldy * es) % 16 == 0);
    long long gpr = 0, blocks;
    if (vec) {
        if (dense) { a.rows = 1; a.cols = a.ldx = a.ldy = total; }
        gpr = a.cols / 8;
        blocks = (total / 8 + DO_THREADS - 1) / DO_THREADS;
    } else {
        blocks = (total + 8ll * DO_THREADS - 1) / (8ll * DO_THREADS);
    }
    if (blocks > 0x7fffffffll) return fail(WINO_E_UNSUPPORTED, "%s: more than 2^42 elements", what);
    count_launch();
    if (vec) {
        if (dtype == WINO_BF16) dropout_vec_kernel<true><<<(unsigned)blocks, DO_THREADS, 0, st>>>(x, y, a, gpr);
        else dropout_vec_kernel<false><<<(unsigned)blocks, DO_THREADS, 0, st>>>(x, y, a, gpr);
    } else {
        if (dtype == WINO_BF16) dropout_any_kernel<__nv_bfloat16><<<(unsigned)blocks, DO_THREADS, 0, st>>>((const __nv_bfloat16*)x, (__nv_bfloat16*)y, a);
        else dropout_any_kernel<float><<<(unsigned)blocks, DO_THREADS, 0, st>>>((const float*)x, (float*)y, a);
    }
    WINO_CUDA_CHECK(cudaGetLastError());
    return WINO_OK;
}

}  // namespace

}  // namespace wino

extern "C" {

int wino_dropout_forward(int dtype, long long rows, long long cols, long long ldx, long long ldy, float p,
                         unsigned long long seed, unsigned long long offset, const unsigned long long* offset_dev,
                         const void* x, void* y, wino_stream_t stream) {
    return wino::run_dropout("dropout_forward", dtype, rows, cols, ldx, ldy, p, seed, offset, offset_dev, x, y, (cudaStream_t)stream);
}

int wino_dropout_backward(int dtype, long long rows, long long cols, long long lddy, long long lddx, float p,
                          unsigned long long seed, unsigned long long offset, const unsigned long long* offset_dev,
                          const void* dy, void* dx, wino_stream_t stream) {
    return wino::run_dropout("dropout_backward", dtype, rows, cols, lddy, lddx, p, seed, offset, offset_dev, dy, dx, (cudaStream_t)stream);
}

}  // extern "C"
