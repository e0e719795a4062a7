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
    unsigned long long offset;
    const unsigned long long* offset_dev;
    uint32_t keys[20];              // the generator's ten pairs of round keys
    uint32_t threshold_hi;          // T << 16
    float scale;
};

// the eight 16-bit lanes of group g, as four words (low half first)
__device__ __forceinline__ uint4 philox10(unsigned long long g, unsigned long long offset, const uint32_t (&keys)[20]) {
    uint32_t c0 = (uint32_t)g, c1 = (uint32_t)(g >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ keys[2 * r];
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ keys[2 * r + 1];
        c3 = (uint32_t)a;
    }
    return make_uint4(c0, c1, c2, c3);
}

// half >= T for both halves of a word without taking them apart: the upper one is compared in place, the lower one shifted up
__device__ __forceinline__ bool kept_hi(uint32_t r, const DropoutArgs& a) { return r >= a.threshold_hi; }
__device__ __forceinline__ bool kept_lo(uint32_t r, const DropoutArgs& a) { return (r << 16) >= a.threshold_hi; }

__device__ __forceinline__ unsigned long long dropout_offset(const DropoutArgs& a) {
    return a.offset + (a.offset_dev ? *a.offset_dev : 0ull);
}

__device__ __forceinline__ uint32_t drop_pair(uint32_t v, uint32_t r, const DropoutArgs& a) {
    const float lo = __uint_as_float(v << 16) * a.scale, hi = __uint_as_float(v & 0xffff0000u) * a.scale;
    const __nv_bfloat162 o = __floats2bfloat162_rn(kept_lo(r, a) ? lo : 0.f, kept_hi(r, a) ? hi : 0.f);
    return *reinterpret_cast<const uint32_t*>(&o);
}

// Whole groups of eight, 16-byte accesses: cols, pitches and bases allow it (a dense matrix counts as one long row).
// groups_per_row is the number of groups in a row; the group index is the counter.  A thread takes GROUPS groups, a block
// width apart, and has all their loads in flight before the first generator runs.
template <bool BF16, int GROUPS>
__global__ void __launch_bounds__(DO_THREADS) dropout_vec_kernel(const void* xin, void* yout, const DropoutArgs a, long long groups_per_row) {
    pdl_wait();
    const long long g0 = (long long)blockIdx.x * (DO_THREADS * GROUPS) + threadIdx.x;
    const long long total = a.rows * groups_per_row;
    uint4 v[GROUPS][BF16 ? 1 : 2];
    long long oy[GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        const long long g = g0 + i * DO_THREADS;
        oy[i] = -1;
        if (g < total) {
            long long ox = g * 8;
            oy[i] = ox;
            if (a.rows > 1) {
                const long long r = g / groups_per_row, c = (g - r * groups_per_row) * 8;
                ox = r * a.ldx + c;
                oy[i] = r * a.ldy + c;
            }
            const uint4* x = reinterpret_cast<const uint4*>(static_cast<const char*>(xin) + ox * (BF16 ? 2 : 4));
            v[i][0] = __ldcs(x);
            if (!BF16) v[i][BF16 ? 0 : 1] = __ldcs(x + 1);
        }
    }
    const unsigned long long offset = dropout_offset(a);
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        if (oy[i] < 0) continue;
        const uint4 q = philox10((unsigned long long)(g0 + i * DO_THREADS), offset, a.keys);
        uint4* y = reinterpret_cast<uint4*>(static_cast<char*>(yout) + oy[i] * (BF16 ? 2 : 4));
        if (BF16) {
            const uint4 w = v[i][0];
            __stcs(y, make_uint4(drop_pair(w.x, q.x, a), drop_pair(w.y, q.y, a), drop_pair(w.z, q.z, a), drop_pair(w.w, q.w, a)));
        } else {
            const uint32_t r[4] = {q.x, q.y, q.z, q.w};
            uint32_t o[8];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint4 w = v[i][BF16 ? 0 : e];
                const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t bits = r[e * 2 + k / 2];
                    o[e * 4 + k] = (k & 1 ? kept_hi(bits, a) : kept_lo(bits, a)) ? __float_as_uint(__uint_as_float(in[k]) * a.scale) : 0u;
                }
            }
            __stcs(y, make_uint4(o[0], o[1], o[2], o[3]));
            __stcs(y + 1, make_uint4(o[4], o[5], o[6], o[7]));
        }
    }
}

// Any width, pitch and alignment: a warp takes 256 consecutive elements.  Each lane draws the keep bits of one group, and
// lane l then handles elements l, l + 32, ... so that accesses stay coalesced; the bits come over by shuffles.
template <typename T>
__global__ void __launch_bounds__(DO_THREADS) dropout_any_kernel(const T* x, T* y, const DropoutArgs a) {
    pdl_wait();
    const int lane = threadIdx.x % 32;
    const long long warp = (long long)blockIdx.x * (DO_THREADS / 32) + threadIdx.x / 32;
    const long long total = a.rows * a.cols, e0 = warp * 256;
    if (e0 >= total) return;
    // one division (a 32-bit one where the tensor allows it)
    long long r = total < (1ll << 32) ? (long long)((uint32_t)e0 / (uint32_t)a.cols) : e0 / a.cols, c = e0 - r * a.cols;
    const bool inside = c + 256 <= a.cols && e0 + 256 <= total;       // most warps stay within a row
    T v[8];
    long long oy[8];
    if (inside) {
        const T* src = x + r * a.ldx + c + lane;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = src[i * 32];
    } else {
        c += lane;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (c >= a.cols) {
                if (a.cols >= 32) { c -= a.cols; ++r; }
                else { r += c / a.cols; c %= a.cols; }
            }
            oy[i] = -1;
            if (e0 + i * 32 + lane < total) {
                v[i] = x[r * a.ldx + c];
                oy[i] = r * a.ldy + c;
            }
            c += 32;
        }
    }
    const uint4 q = philox10((unsigned long long)(warp * 32 + lane), dropout_offset(a), a.keys);
    const uint32_t keep = (kept_lo(q.x, a) ? 1u : 0u) | (kept_hi(q.x, a) ? 2u : 0u) | (kept_lo(q.y, a) ? 4u : 0u) | (kept_hi(q.y, a) ? 8u : 0u) |
                    (kept_lo(q.z, a) ? 16u : 0u) | (kept_hi(q.z, a) ? 32u : 0u) | (kept_lo(q.w, a) ? 64u : 0u) | (kept_hi(q.w, a) ? 128u : 0u);
    T* dst = y + r * a.ldy + c + lane;                                // where inside
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t bits = __shfl_sync(0xffffffffu, keep, i * 4 + lane / 8);
        const T o = from_float<T>((bits >> (lane % 8)) & 1u ? to_float<T>(v[i]) * a.scale : 0.f);
        if (inside) dst[i * 32] = o;
        else if (oy[i] >= 0) y[oy[i]] = o;
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
    a.offset = offset; a.offset_dev = offset_dev;
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
    for (int r = 0; r < 10; ++r, k0 += 0x9E3779B9u, k1 += 0xBB67AE85u) { a.keys[2 * r] = k0; a.keys[2 * r + 1] = k1; }
    const uint32_t t = (uint32_t)floor((double)p * 65536.0 + 0.5);
    a.threshold_hi = t << 16;
    a.scale = t < 65536u ? (float)(65536.0 / (65536.0 - t)) : 0.f;
    if (t >= 65536u) {              // nothing is kept, and T << 16 has no room for it
        if (rows == 1 || ldy == cols) WINO_CUDA_CHECK(cudaMemsetAsync(y, 0, (size_t)rows * cols * es, st));
        else WINO_CUDA_CHECK(cudaMemset2DAsync(y, (size_t)ldy * es, 0, (size_t)cols * es, (size_t)rows, st));
        return WINO_OK;
    }
    const bool dense = ldx == cols && ldy == cols;
    const bool aligned = (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    const long long total = rows * cols;
    const bool vec = aligned && (dense ? total % 8 == 0 : cols % 8 == 0 && (ldx * es) % 16 == 0 && (ldy * es) % 16 == 0);
    long long gpr = 0, blocks;
    int groups = 1;
    if (vec) {
        if (dense) { a.rows = 1; a.cols = a.ldx = a.ldy = total; }
        gpr = a.cols / 8;
        // four (FP32: two) groups a thread once that still makes eight blocks an SM
        const int many = dtype == WINO_BF16 ? 4 : 2;
        if (total / 8 >= 8ll * DO_THREADS * many * sm_count()) groups = many;
        blocks = (total / 8 + DO_THREADS * groups - 1) / (DO_THREADS * groups);
    } else {
        blocks = (total + 8ll * DO_THREADS - 1) / (8ll * DO_THREADS);
    }
    if (blocks > 0x7fffffffll) return fail(WINO_E_UNSUPPORTED, "%s: more than 2^42 elements", what);
    count_launch();
    // launched with programmatic serialisation: the blocks are set up while the kernel before ends
    auto go = [&](auto kernel, auto... args) { return launch_kernel(kernel, dim3((unsigned)blocks), dim3(DO_THREADS), 0, st, true, args...); };
    if (vec) {
        WINO_CUDA_CHECK(go(dtype == WINO_BF16 ? (groups > 1 ? dropout_vec_kernel<true, 4> : dropout_vec_kernel<true, 1>)
                                              : (groups > 1 ? dropout_vec_kernel<false, 2> : dropout_vec_kernel<false, 1>), x, y, a, gpr));
    } else {
        WINO_CUDA_CHECK(dtype == WINO_BF16 ? go(dropout_any_kernel<__nv_bfloat16>, (const __nv_bfloat16*)x, (__nv_bfloat16*)y, a)
                                           : go(dropout_any_kernel<float>, (const float*)x, (float*)y, a));
    }
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
