// FP32X3 products of a long matrix L of floats with up to 128 rows s, for the linear softmax cross entropy: the logits of up to
// 128 rows (L = W) or classes (L = x), and the gradient with respect to the few.
//
// Splitting L into three BF16 parts beforehand writes and reads it three times over: 128 x 2048 x 21841 spent 84 us on that and
// another 110 us reading the parts.  Here the parts never leave the SM.  128 rows of L (or 128 columns, where the
// contraction runs along the rows) are the M of a CTA's MMAs; eight warps load 128 x 64 floats, two tiles ahead in registers,
// split them and store the parts into the swizzled tiles that tcgen05.mma reads, K-major or MN-major: either way 128 runs of 64
// floats, so nothing is transposed.  TMA brings the parts of s beside them.  Six products a tile: the five small ones add
// up in one accumulator, the large one in another, since the tensor cores truncate each sum they make; every 256
// elements of the contraction the two go to registers (eight more warps), where they are added rounded to nearest.
//
// The work is shared out in steps of 64 contraction elements, to all SMs alike: by whole tiles 171 of them on 148 SMs left some
// with half as much again (128 x 2048 x 21841: 92 -> 72 us).
//
// Bound: by bytes, one read of L: 128 x 2048 x 21841 72 us (2.5 TB/s), each way.  What holds it there is the splitting: a tile takes
// its warps about 1900 cycles, 700 of them arithmetic and stores, at two warps a scheduler.  Sixteen warps with half the floats each spill
// at the 72 registers that leaves them: 85 us.
#include <mutex>

#include "tcgen05.cuh"
#include "xent.cuh"

namespace wino {

namespace {

template <int N>
__device__ __forceinline__ void setmaxnreg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void setmaxnreg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }


constexpr int XT_WARPS = 8;                                        // that split; as many move accumulators
constexpr int XT_THREADS = 128 + 2 * 32 * XT_WARPS;                // TMA, MMA, two that idle; those that split; those that move
// Registers of a thread in these three groups, out of the launch's: three tiles of floats for the second, 64 sums for the third.
constexpr int XT_LAUNCH_REGS = 96, XT_REGS[3] = {40, 128, 88};
static_assert(128 * XT_REGS[0] + 32 * XT_WARPS * (XT_REGS[1] + XT_REGS[2]) <= XT_THREADS * XT_LAUNCH_REGS, "more registers than the launch has");
constexpr int XT_TILE = 128 * 128;                                 // bytes of one part of a tile of L
constexpr int XT_BLOCK = 4;                                        // tiles between two moves to registers

struct alignas(64) ThinParams {
    CUtensorMap tm_s;
    const float* l;
    long long rows, ldl, m, k;        // extents of the product: M, and the contraction
    int d, n;                         // columns of L, rows of s
    const float* rowg;
    int s_mn;
    int chunks, parts;                // steps of 64 of a tile; buffers that `out` has
    long long steps;                  // of all tiles
    uint32_t idesc;
    float* out;
    long long out_s, out_m, plane;
    XeScale scale;
    int* zero;
    int* status;
};

template <int NP>
struct ThinSmem {
    static constexpr int S_BYTES = NP * 128;                       // one part of 64 contraction elements of s
    static constexpr int STAGE = 3 * (XT_TILE + S_BYTES);
    static constexpr int STAGES = NP > 64 ? 2 : 3;
    static constexpr int BAR_OFF = STAGES * STAGE;
    static constexpr int SLOT_OFF = BAR_OFF + 8 * (2 * STAGES + 4);
    static constexpr int TOTAL = SLOT_OFF + 16 + 1024;
};

// loads that stay in the order written, ahead of what follows; v keeps its value where `in` is false
__device__ __forceinline__ void ldg1(float& v, const float* at) { asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(at)); }
__device__ __forceinline__ void ldg4(float& a, float& b, float& c, float& d, const float* at) {
    asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(a), "=f"(b), "=f"(c), "=f"(d) : "l"(at));
}
__device__ __forceinline__ void ldg1(float& v, const float* at, bool in) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %2, 0;\n@p ld.global.nc.f32 %0, [%1];\n}\n" : "+f"(v) : "l"(at), "r"((int)in));
}
__device__ __forceinline__ void ldg4(float& a, float& b, float& c, float& d, const float* at, bool in) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %5, 0;\n@p ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];\n}\n"
                 : "+f"(a), "+f"(b), "+f"(c), "+f"(d) : "l"(at), "r"((int)in));
}

// NP: rows of s, padded; ALONG_ROWS: the contraction runs along the rows of L; VEC: rows of L lie on 16-byte boundaries
template <int NP, bool ALONG_ROWS, bool VEC>
__global__ void __launch_bounds__(XT_THREADS, 1) xe_thin_kernel(const __grid_constant__ ThinParams p) {
    using L = ThinSmem<NP>;
    constexpr int STAGES = L::STAGES;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen_base = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bar_full = base + L::BAR_OFF, bar_empty = bar_full + 8 * STAGES;
    const uint32_t bar_tfull = bar_empty + 8 * STAGES, bar_tempty = bar_tfull + 16;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen_base + L::SLOT_OFF);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen_base + L::SLOT_OFF + 4);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

    if (threadIdx.x == 64) prefetch_tensor_map(&p.tm_s);
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bar_full + 8 * s, 1 + XT_WARPS);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_tfull + 8 * a, 1);
            mbar_init(bar_tempty + 8 * a, XT_WARPS);
        }
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(smem_u32((const void*)tmem_slot), 4 * NP);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    // Each CTA takes an even share of all steps, tile after tile: a piece of a tile, whole tiles, a piece of the last.  The
    // pieces of a tile go to one buffer each.
    const long long g1 = p.steps * (blockIdx.x + 1) / gridDim.x;
    struct Piece { long long next, tile; int c0, c1; };
    auto piece_at = [&](long long g) {                 // that begins with step g < g1
        Piece w;
        w.tile = g / p.chunks;
        w.c0 = (int)(g - w.tile * p.chunks);
        w.c1 = g1 - g < p.chunks - w.c0 ? w.c0 + (int)(g1 - g) : p.chunks;
        w.next = g + w.c1 - w.c0;
        return w;
    };
    const long long g0 = p.steps * blockIdx.x / gridDim.x;
    bool ok = true;
    int stage = 0;
    uint32_t phase = 0;

    if (warp < 4) {
        setmaxnreg_dec<XT_REGS[0]>();
        if (warp == 0) {                                   // s, by TMA
            const bool issuer = elect_one();
            pdl_wait();
            for (long long g = g0; ok && g < g1;) {
                const Piece w = piece_at(g);
                g = w.next;
                for (int c = w.c0; c < w.c1; ++c) {
                    if (!mbar_wait_warp(bar_empty + 8 * stage, phase ^ 1, abort_flag, p.status, XT_WAIT_EMPTY)) { ok = false; break; }
                    if (issuer) {
                        const uint32_t bar = bar_full + 8 * stage, dst = base + stage * L::STAGE + 3 * XT_TILE;
                        mbar_arrive_expect_tx(bar, 3 * L::S_BYTES);
#pragma unroll
                        for (int q = 0; q < 3; ++q) {
                            if (p.s_mn) {
                                tma_load_3d(dst + q * L::S_BYTES, &p.tm_s, bar, 0, c * XE_BK, q);
                                if (NP > 64) tma_load_3d(dst + q * L::S_BYTES + 8192, &p.tm_s, bar, 64, c * XE_BK, q);
                            } else {
                                tma_load_3d(dst + q * L::S_BYTES, &p.tm_s, bar, c * XE_BK, 0, q);
                            }
                        }
                    }
                    __syncwarp();
                    if (++stage == STAGES) { stage = 0; phase ^= 1; }
                }
            }
            if (!ok && issuer) drain_after_abort();
        } else if (warp == 1) {                            // MMAs
            const bool issuer = elect_one();
            const uint64_t l0 = ALONG_ROWS ? smem_desc_mn128(base) : smem_desc_k128(base);
            const uint64_t s0 = p.s_mn ? smem_desc_mn128(base + 3 * XT_TILE) : smem_desc_k128(base + 3 * XT_TILE);
            const uint64_t l_step = ALONG_ROWS ? 128 : 2, s_step = p.s_mn ? 128 : 2;      // 16 contraction elements
            int as = 0;
            uint32_t aphase = 0;
            for (long long g = g0; ok && g < g1;) {
                const Piece w = piece_at(g);
                g = w.next;
                for (int cb = w.c0; ok && cb < w.c1; cb += XT_BLOCK) {
                    const int steps = w.c1 - cb < XT_BLOCK ? w.c1 - cb : XT_BLOCK;
                    if (!mbar_wait_warp(bar_tempty + 8 * as, aphase ^ 1, abort_flag, p.status, XT_WAIT_TMEM_EMPTY)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t large = tmem_base + (uint32_t)(as * 2 * NP), small = large + NP;
                    for (int c = 0; c < steps; ++c) {
                        if (!mbar_wait_warp(bar_full + 8 * stage, phase, abort_flag, p.status, XT_WAIT_FULL)) { ok = false; break; }
                        tc_fence_after();
                        const uint64_t ld = l0 + (uint64_t)(stage * (L::STAGE >> 4)), sd = s0 + (uint64_t)(stage * (L::STAGE >> 4));
                        constexpr int pl[6] = {2, 1, 0, 1, 0, 0}, ps[6] = {0, 1, 2, 0, 1, 0};
#pragma unroll
                        for (int q = 0; q < 6; ++q)
#pragma unroll
                            for (int ks = 0; ks < XE_BK / 16; ++ks)
                                if (issuer)
                                    tc_mma<false>(q == 5 ? large : small, ld + pl[q] * (XT_TILE >> 4) + ks * l_step, sd + ps[q] * (L::S_BYTES >> 4) + ks * s_step,
                                                  p.idesc, c > 0 || ks > 0 || (q > 0 && q < 5) ? 1u : 0u);
                        if (issuer) tc_commit(bar_empty + 8 * stage);
                        if (++stage == STAGES) { stage = 0; phase ^= 1; }
                    }
                    if (ok && issuer) tc_commit(bar_tfull + 8 * as);
                    as ^= 1;
                    if (as == 0) aphase ^= 1;
                }
            }
        }
    } else if (warp < 4 + XT_WARPS) {                  // L
        setmaxnreg_inc<XT_REGS[1]>();
        const int cw = warp - 4;
        pdl_wait();
        if (p.zero && blockIdx.x == 0 && cw == 0 && lane < 2) p.zero[lane] = 0;
        // Run i of 16 of this warp: 64 floats from element (r, c) of L on.  VEC: half a warp per run, four floats a lane; else
        // a warp per run, two floats a lane.
        constexpr int PER = VEC ? 4 : 2, LOADS = 32 / PER, LANES = 64 / PER;
        const int sub = VEC ? lane / LANES : 0, off = (lane % LANES) * PER;
        const bool fours = VEC && p.d % 4 == 0;       // four floats of a row are all there, or none
        auto load = [&](float (&v)[32], long long m0, int chunk) {
            const int run0 = cw * 16 + sub;
            const long long r0 = ALONG_ROWS ? (long long)chunk * XE_BK + run0 % 64 : m0 + run0;
            const long long c0 = (ALONG_ROWS ? m0 + run0 / 64 * 64 : (long long)chunk * XE_BK) + off;
            const long long step = (VEC ? 2 : 1) * p.ldl, left = p.rows - r0;
            const float* at = p.l + r0 * p.ldl + c0;
            const bool weigh = ALONG_ROWS && p.rowg;
            if (left >= 16 && c0 - off + 64 <= p.d && !weigh) {        // all of this warp's floats are there
#pragma unroll
                for (int i = 0; i < LOADS; ++i, at += step) {
                    if constexpr (VEC) ldg4(v[PER * i], v[PER * i + 1], v[PER * i + PER - 2], v[PER * i + PER - 1], at);
                    else { ldg1(v[2 * i], at); ldg1(v[2 * i + 1], at + 1); }
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0.f;
            if (fours || (VEC && c0 - off + 64 <= p.d)) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i, at += step) {
                    const bool in = 2 * i < left && c0 < p.d && !(weigh && p.rowg[r0 + 2 * i] == 0.f);
                    ldg4(v[PER * i], v[PER * i + 1], v[PER * i + PER - 2], v[PER * i + PER - 1], at, in);
                }
            } else {
#pragma unroll
                for (int i = 0; i < LOADS; ++i, at += step) {
                    const int r = (VEC ? 2 : 1) * i;
                    const bool in = r < left && !(weigh && p.rowg[r0 + r] == 0.f);
#pragma unroll
                    for (int e = 0; e < PER; ++e) ldg1(v[PER * i + e], at + e, in && c0 + e < p.d);
                }
            }
        };
        auto store = [&](const float (&v)[32]) {
            // one look at the sizes of all: a branch for each pair left the warps waiting for themselves (2300 cycles a tile instead of 700)
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 32; i += 2) most = max3(most, fabsf(v[i]), fabsf(v[i + 1]));
            const bool far = most > XE_SPLIT_MAX;
            uint8_t* dst = gen_base + stage * L::STAGE + cw * 16 * 128;
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int run = VEC ? 2 * i + sub : i;
                uint8_t* at = dst + run * 128 + ((off / 8) ^ (run & 7)) * 16 + (off % 8) * 2;
                uint32_t part[3][PER / 2];
#pragma unroll
                for (int e = 0; e < PER / 2; ++e) xe_split3_pair(v[PER * i + 2 * e], v[PER * i + 2 * e + 1], part[0][e], part[1][e], part[2][e]);
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    if constexpr (VEC) *reinterpret_cast<uint2*>(at + q * XT_TILE) = make_uint2(part[q][0], part[q][PER / 2 - 1]);
                    else *reinterpret_cast<uint32_t*>(at + q * XT_TILE) = part[q][0];
                }
            }
            if (far) {                                 // this lane has an infinity, or something near the largest float: its floats again
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int run = VEC ? 2 * (i / 4) + sub : i / 2, o = off + i % PER;
                    __nv_bfloat16 part[3];
                    xe_split3(v[i], part[0], part[1], part[2]);
#pragma unroll
                    for (int q = 0; q < 3; ++q) *reinterpret_cast<__nv_bfloat16*>(dst + q * XT_TILE + run * 128 + ((o / 8) ^ (run & 7)) * 16 + (o % 8) * 2) = part[q];
                }
            }
        };
        auto put = [&](const float (&v)[32]) {
            if (!mbar_wait_warp(bar_empty + 8 * stage, phase ^ 1, abort_flag, p.status, XT_WAIT_EMPTY)) return false;
            store(v);
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_full + 8 * stage);
            if (++stage == STAGES) { stage = 0; phase ^= 1; }
            return true;
        };
        // two tiles of floats are on their way while a third is split
        long long g = g0;
        Piece w = piece_at(g0 < g1 ? g0 : 0);
        int c = w.c0;
        auto fetch = [&](float (&v)[32]) {             // the next tile, if there is one
            if (g >= g1) return;
            load(v, w.tile * 128, c);
            ++g;
            if (++c == w.c1 && g < g1) {
                w = piece_at(g);
                c = w.c0;
            }
        };
        const long long mine = g1 - g0;
        float va[32], vb[32], vc[32];
        fetch(va);
        fetch(vb);
        for (long long i = 0; i < mine; i += 3) {
            fetch(vc);
            if (!put(va)) break;
            fetch(va);
            if (i + 1 < mine && !put(vb)) break;
            fetch(vb);
            if (i + 2 < mine && !put(vc)) break;
        }
    } else {                                           // accumulators
        setmaxnreg_dec<XT_REGS[2]>();
        const int quarter = warp % 4, half = (warp - 4 - XT_WARPS) / 4;
        constexpr int COLS = NP / 2;                   // of an accumulator, per warp
        pdl_wait();
        const float scale = xe_scale(p.scale);
        int as = 0;
        uint32_t aphase = 0;
        for (long long g = g0; ok && g < g1;) {
            const Piece w = piece_at(g);
            g = w.next;
            float z[COLS];
#pragma unroll
            for (int i = 0; i < COLS; ++i) z[i] = 0.f;
            for (int cb = w.c0; cb < w.c1; cb += XT_BLOCK) {
                if (!mbar_wait_warp(bar_tfull + 8 * as, aphase, abort_flag, p.status, XT_WAIT_TMEM_FULL)) { ok = false; break; }
                tc_fence_after();
                const uint32_t src = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(as * 2 * NP + half * COLS);
#pragma unroll
                for (int j = 0; j < COLS / 8; ++j) {   // 16 of the small terms' sums, 16 of the large ones', and so on
                    uint32_t r[16];
                    tmem_ld_32x16(src + (j % 2 ? 0 : NP) + j / 2 * 16, r);
                    tmem_ld_wait();
                    after_wait(r);
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[j / 2 * 16 + i] += __uint_as_float(r[i]);
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_tempty + 8 * as);
                as ^= 1;
                if (as == 0) aphase ^= 1;
            }
            if (!ok) break;
            const long long m = w.tile * 128 + quarter * 32 + lane;
            // the CTA that has step x is the last one whose share begins at x or before
            auto owner = [&](long long x) { return (int)(((x + 1) * gridDim.x - 1) / p.steps); };
            const int piece = (int)blockIdx.x - owner(w.tile * p.chunks);
            if (m < p.m) {
                float* o = p.out + piece * p.plane + m * p.out_m + half * COLS * p.out_s;
                const int cols = p.n - half * COLS;
                auto store = [&](float f) {
                    if (p.out_s == 1) {                // a lane has a row's columns: rows and buffers are multiples of 16 bytes
#pragma unroll
                        for (int i = 0; i < COLS; i += 4) {
                            if (i + 4 <= cols) {
                                *reinterpret_cast<float4*>(o + i) = make_float4(z[i] * f, z[i + 1] * f, z[i + 2] * f, z[i + 3] * f);
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (i + e < cols) o[i + e] = z[i + e] * f;
                            }
                        }
                    } else {                           // the warp has 32 consecutive elements of a row
#pragma unroll
                        for (int i = 0; i < COLS; ++i)
                            if (i < cols) o[i * p.out_s] = z[i] * f;
                    }
                };
                store(scale);
                if (w.c1 == p.chunks) {                // the tile's last piece: zeros to the buffers without one
#pragma unroll
                    for (int i = 0; i < COLS; ++i) z[i] = 0.f;
                    for (int q = piece + 1; q < p.parts; ++q) {
                        o += p.plane;
                        store(1.f);
                    }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 4 * NP);
    }
}

template <int NP, bool ALONG_ROWS, bool VEC>
int run(const ThinParams& p, int grid, cudaStream_t st) {
    using L = ThinSmem<NP>;
    static_assert(L::TOTAL <= 232448, "shared memory budget of one CTA exceeded");
    static std::once_flag once[64];
    static int regs[64];
    int dev = 0;
    WINO_CUDA_CHECK(cudaGetDevice(&dev));
    cudaError_t attr_err = cudaSuccess;
    std::call_once(once[dev & 63], [&] {
        attr_err = cudaFuncSetAttribute(xe_thin_kernel<NP, ALONG_ROWS, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL);
        cudaFuncAttributes a;
        if (attr_err == cudaSuccess && (attr_err = cudaFuncGetAttributes(&a, xe_thin_kernel<NP, ALONG_ROWS, VEC>)) == cudaSuccess) regs[dev & 63] = a.numRegs;
    });
    WINO_CUDA_CHECK(attr_err);
    // with fewer the groups' shares would never all be there
    if (regs[dev & 63] < XT_LAUNCH_REGS) return fail(WINO_E_UNSUPPORTED, "xent: a kernel was built with %d registers", regs[dev & 63]);
    count_launch();
    WINO_CUDA_CHECK(launch_kernel(xe_thin_kernel<NP, ALONG_ROWS, VEC>, dim3((unsigned)grid), dim3(XT_THREADS), L::TOTAL, st, true, p));
    return WINO_OK;
}

}  // namespace

// most pieces of a tile when `grid` CTAs share the steps
static int pieces(long long tiles, long long chunks, long long grid) {
    const long long steps = tiles * chunks, share = steps / grid;
    if (steps % grid == 0 && (share % chunks == 0 || chunks % share == 0)) return (int)(share >= chunks ? 1 : chunks / share);
    return (int)(chunks < 2 ? 1 : (chunks - 2) / share + 2);
}

// All SMs, fewer with 2 ... 16 steps each, or so many that no tile, or each in as many even pieces, is cut: fewer buffers.
// Estimated time: 1.2 us a step, and per buffer its bytes and 0.2 us where the pieces are added up.
XeThinCut xe_thin_cut(long long tiles, long long chunks, double part_us) {
    const long long sms = sm_count(), steps = tiles * chunks;
    XeThinCut best = {0, 0};
    double best_us = 1e30;
    auto consider = [&](long long grid) {
        const int parts = pieces(tiles, chunks, grid);
        const double us = (double)((steps + grid - 1) / grid) * 1.2 + (part_us + 0.2) * parts;
        if (us < best_us) { best_us = us; best = {(int)grid, parts}; }
    };
    consider(steps < sms ? steps : sms);
    for (long long share = 2; share <= 16; ++share)
        if ((steps + share - 1) / share <= sms) consider((steps + share - 1) / share);
    for (long long k = 1; k <= chunks && k * tiles <= sms; ++k)
        if (chunks % k == 0) consider(k * tiles);
    return best;
}

int xe_thin(const XeThin& t, cudaStream_t st) {
    ThinParams p = {};
    int rc;
    const int n = (int)(t.s.along_rows ? t.s.cols : t.s.rows), np = n <= 64 ? 64 : 128;
    if (n < 1 || n > 128 || t.s.planes != 3) return fail(WINO_E_BADARG, "xent: no kernel for this product");
    if (t.out_s == 1 && ((((uintptr_t)t.out) & 15) || t.out_m % 4 || t.plane % 4)) return fail(WINO_E_BADARG, "xent: buffer rows must be multiples of 16 bytes");
    if ((rc = xe_operand_map(&p.tm_s, t.s, (unsigned)np))) return rc;
    p.l = t.l; p.rows = t.rows; p.ldl = t.ldl; p.d = t.d; p.n = n;
    p.m = t.along_rows ? t.d : t.rows;
    p.k = t.along_rows ? t.rows : t.d;
    p.rowg = t.rowg;
    p.s_mn = t.s.along_rows;
    const long long tiles = (p.m + 127) / 128;
    const int chunks = (int)((p.k + XE_BK - 1) / XE_BK);
    p.chunks = chunks;
    p.steps = tiles * chunks;
    p.parts = t.cut.parts;
    if (t.cut.grid < 1 || t.cut.grid > p.steps || t.cut.parts < pieces(tiles, chunks, t.cut.grid)) return fail(WINO_E_BADARG, "xent: bad parts of a product");
    p.idesc = make_idesc(OP_BF16, np, 128) | (t.along_rows ? 1u << 15 : 0u) | (p.s_mn ? 1u << 16 : 0u);
    p.out = t.out; p.out_s = t.out_s; p.out_m = t.out_m; p.plane = t.plane;
    p.scale = t.scale;
    p.zero = t.zero;
    if ((rc = status_word(&p.status))) return rc;
    const bool vec = t.ldl % 4 == 0 && ((uintptr_t)t.l & 15) == 0;
    if (np == 64) {
        if (t.along_rows) return vec ? run<64, true, true>(p, t.cut.grid, st) : run<64, true, false>(p, t.cut.grid, st);
        return vec ? run<64, false, true>(p, t.cut.grid, st) : run<64, false, false>(p, t.cut.grid, st);
    }
    if (t.along_rows) return vec ? run<128, true, true>(p, t.cut.grid, st) : run<128, true, false>(p, t.cut.grid, st);
    return vec ? run<128, false, true>(p, t.cut.grid, st) : run<128, false, false>(p, t.cut.grid, st);
}

}  // namespace wino
