// The products of the linear softmax cross entropy (sm_100a): logits z = x W^T, dx = dz W, dW = dz^T x, one kernel with
// the step that follows fused into its epilogue.
//
// CTA pairs (tcgen05.mma.cta_group::2, 256 x 256 tiles; 256 x 128 where tiles are few), for the reason given in gemm_tc_pair.cu: half of B comes from the
// partner's shared memory, so a 64-deep slice costs 32 KB of L2 reads per SM.  Operands are BF16; what changes between the
// three products is along which axis of the stored matrix the contraction runs:
//   z : x and W along their columns (K-major);  dx: dz along its columns, W along its rows;  dW: dz and x along their rows.
// An operand contracted along its rows is fetched as boxes of 64 columns x 64 rows and given to the MMA as an MN-major
// tile (transpose bit of the instruction descriptor, 8-row groups 1 KiB apart, 64-column blocks 8 KiB apart), so nothing
// is ever transposed in memory.
// FP32X3: each operand is three BF16 planes; a block of the contraction runs over six pairs of planes, the smallest
// products first so that they add up before the accumulator is large.
//
// The tensor cores truncate when they add to an accumulator, which over a contraction of 1000 elements biases a sum by
// some 10^-6 of itself.  So the contraction is cut into blocks (256 elements for FP32X3, 1024 for BF16); each block's sum is
// fetched from tensor memory and added to the tile's sums in registers, rounded to nearest, while the next block runs in
// the other accumulator.
//
// Roles as in gemm_tc_pair.cu: warp 0 TMA, warp 1 of the leader MMA, warps 2-9 epilogue: a warp holds 32 rows x 128 (64)
// columns of the tile in registers and gives the accumulator back before it works on them.  Tiles are walked in bands
// of eight row blocks, rows fastest, so that the pairs working at a time share both operands through the L2.
// Bound: tensor pipe for wide layers; the read of W (or the write of dW) where rows are few.
#include <mutex>

#include "tcgen05.cuh"
#include "xent.cuh"
#include "xent_turns.cuh"

namespace wino {

// boxes of 64 columns (128 bytes, 128-byte swizzle): `share` rows for a K-major share, 64 rows (one contraction element each)
// for an MN-major one
int xe_operand_map(CUtensorMap* map, const XeOperand& o, unsigned share) {
    const unsigned long long dims[3] = {(unsigned long long)o.cols, (unsigned long long)o.rows, (unsigned long long)o.planes};
    const unsigned long long strides[2] = {(unsigned long long)o.pitch * 2, (unsigned long long)o.plane_pitch * 2};
    const unsigned box[3] = {64u, o.along_rows ? 64u : share, 1u};
    return encode_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, o.ptr, dims, strides, box, 1);
}

namespace {

constexpr int XE_THREADS = 320;
constexpr int XE_TILE_BYTES = 128 * 128;             // a CTA's share of an operand per ring slot: 128 rows x 64 BF16
constexpr int XE_STAGE_TILE = 32 * 128;              // epilogue staging: 32 rows x 128 bytes
constexpr int XE_EPI_WARPS = 8;
constexpr int XE_BAND = 8;


struct alignas(64) XeProblem {
    CUtensorMap tm_a, tm_b, tm_out;
    long long m, n;
    unsigned units, tiles;            // work units: tiles * splits
    unsigned mpairs, nblocks, band;   // row blocks of 256, column blocks, tiles in a band of XE_BAND row blocks
    int splits, kchunks, part, part_over, pairs;   // a part has `part` ring slots, the first part_over parts one more
    int block;                        // ring slots per block of the contraction (and plane pair)
    unsigned char pa[6], pb[6];       // planes of a and b, one entry per partial product
    int a_mn, b_mn;                   // contracted along the rows of the stored matrix
    uint32_t idesc;
    int add, bf16;                    // XE_F32, XE_BF16 (one kernel for both)
    int plain;                        // rows that TMA cannot store: out_ptr, out_pitch
    void* out_ptr;
    long long out_pitch;
    XeScale scale;
    const float* bias;
    const long long* target;
    int col_base;
    float2* stats;
    float* zsum;
    float* zt;
    const float* lse;
    const float* rowg;
    XeDzRule rule;
    float* db_part;
    long long db_pitch;
};
struct XeParams {
    XeProblem prob[2];
    int lead;                         // units of the second product that a pair without a last unit of the first takes ahead
    int* zero;
    XeLoss loss;
    int* status;
};

template <int EPI, int PLANES, int BN>
struct XeSmem {
    static constexpr int B_BYTES = BN / 2 * 128;                          // a CTA's half of the rows of b per ring slot
    static constexpr int STAGES = EPI == XE_STATS || BN < 256 ? 6 : 5;
    static constexpr int A_OFF = 0;
    static constexpr int B_OFF = STAGES * XE_TILE_BYTES;
    static constexpr int STORE_OFF = B_OFF + STAGES * B_BYTES;
    static constexpr int BUF = EPI == XE_STATS ? 0 : XE_STAGE_TILE;
    static constexpr int NBUF = EPI >= XE_STATS ? 1 : 2;                  // staging tiles per epilogue warp
    static constexpr int BIAS_OFF = STORE_OFF + NBUF * XE_EPI_WARPS * BUF;               // 128 floats per epilogue warp
    static constexpr int BAR_OFF = BIAS_OFF + (EPI >= XE_STATS ? XE_EPI_WARPS * 512 : 0);
    static constexpr int SLOT_OFF = BAR_OFF + 8 * (2 * STAGES + 4);
    static constexpr int TOTAL = SLOT_OFF + 16 + 1024;
};

__device__ __forceinline__ void tma_reduce_add_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(src),
                 "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}

// packed FP32 pairs: one issue slot for two columns, each rounded like the scalar operation
__device__ __forceinline__ void add2(float& a, float& b, float c, float d) {
    const float2 r = __fadd2_rn(make_float2(a, b), make_float2(c, d));
    a = r.x; b = r.y;
}
__device__ __forceinline__ void mul2(float& a, float& b, float c) {
    const float2 r = __fmul2_rn(make_float2(a, b), make_float2(c, c));
    a = r.x; b = r.y;
}
__device__ __forceinline__ void fma2(float& a, float& b, float c, float d) {
    const float2 r = __ffma2_rn(make_float2(a, b), make_float2(c, c), make_float2(d, d));
    a = r.x; b = r.y;
}
// v[i] of lane l -> lane i returns the sum over lanes of v[i] (halving exchange, 31 shuffles); v is used up
__device__ __forceinline__ float column_sums(float* v, int lane) {
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) {
        const bool up = lane & w;
#pragma unroll
        for (int i = 0; i < w; ++i) {
            const float send = up ? v[i] : v[i + w], keep = up ? v[i + w] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
        }
    }
    return v[0];
}

template <int EPI, int PLANES, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(XE_THREADS, 1) xe_gemm_kernel(const __grid_constant__ XeParams pp) {
    using L = XeSmem<EPI, PLANES, BN>;
    constexpr int WCOLS = BN / 2;                     // columns of an epilogue warp
    constexpr int STAGES = L::STAGES;

    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;       // same offset in both CTAs of the pair
    uint8_t* gen_base = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t a_ring = base + L::A_OFF, b_ring = base + L::B_OFF;
    const uint32_t bar_full = base + L::BAR_OFF, bar_empty = bar_full + 8 * STAGES;
    const uint32_t bar_tfull = bar_empty + 8 * STAGES, bar_tempty = bar_tfull + 16;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen_base + L::SLOT_OFF);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen_base + L::SLOT_OFF + 4);

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t rank = cluster_ctarank();          // 0 = leader (issues the MMAs, owns the "full" and "tempty" barriers)

    if (threadIdx.x == 64) {       // descriptors on their way while the barriers are set up
        prefetch_tensor_map(&pp.prob[0].tm_a);
        prefetch_tensor_map(&pp.prob[0].tm_b);
        if (EPI != XE_STATS && !pp.prob[0].plain) prefetch_tensor_map(&pp.prob[0].tm_out);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(bar_full + 8 * s, 1);
            mbar_init(bar_empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_tfull + 8 * a, 1);
            mbar_init(bar_tempty + 8 * a, 2 * XE_EPI_WARPS);
        }
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc_pair(smem_u32((const void*)tmem_slot), 512);
    tc_fence_before();
    cluster_sync_all();            // barriers of both CTAs initialised before any remote arrive or TMA completion
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const unsigned pair = blockIdx.x / 2, npairs = gridDim.x / 2;

    const unsigned units0 = pp.prob[0].units;
    const XeTurns turns(units0, pp.prob[1].units, npairs, pp.lead, pair);
    auto unit_at = [&](unsigned i) { return turns.at(i); };

    // work unit -> problem, part of the contraction (ring slots c0 ... c1), tile
    struct Unit { int sp, mp, nb, c0, c1; };
    auto decode = [&](long long at, Unit& w) -> const XeProblem& {
        const bool second = at >= units0;
        const XeProblem& p = pp.prob[second];
        const unsigned u = second ? (unsigned)at - units0 : (unsigned)at, sp = u / p.tiles, t = u - sp * p.tiles;
        const unsigned b = t / p.band, first = b * XE_BAND, left = p.mpairs - first, height = left < XE_BAND ? left : XE_BAND;
        const unsigned in = t - b * p.band;
        w.sp = (int)sp;
        w.nb = (int)(in / height);
        w.mp = (int)(first + in - w.nb * height);
        w.c0 = (int)sp * p.part + ((int)sp < p.part_over ? (int)sp : p.part_over);
        w.c1 = w.c0 + p.part + ((int)sp < p.part_over ? 1 : 0);
        return p;
    };

    if (warp == 0) {
        const bool issuer = elect_one();
        const uint32_t full_leader = mapa_shared(bar_full, 0);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        long long u;
        for (unsigned i = 0; ok && (u = unit_at(i)) >= 0; ++i) {
            Unit w;
            const XeProblem& p = decode(u, w);
            if (i == 0) pdl_wait();        // all of the above ran under the predecessor; now its results are read
            const bool a_mn = p.a_mn, b_mn = p.b_mn;
            const int arow = (w.mp * 2 + (int)rank) * 128;             // this CTA's 128 rows of a
            const int brow = w.nb * BN + (int)rank * (BN / 2);           // this CTA's half of the rows of b
            for (int cb = w.c0; ok && cb < w.c1; cb += p.block) {
                const int ce = cb + p.block < w.c1 ? cb + p.block : w.c1;
                for (int q = 0; ok && q < p.pairs; ++q) {
                    const int pa = p.pa[q], pb = p.pb[q];
                    for (int kc = cb; kc < ce; ++kc) {
                        if (!mbar_wait_warp(bar_empty + 8 * stage, phase ^ 1, abort_flag, pp.status, XE_WAIT_EMPTY)) { ok = false; break; }
                        if (rank == 0 && issuer) mbar_arrive_expect_tx(bar_full + 8 * stage, 2 * (XE_TILE_BYTES + L::B_BYTES));
                        if (issuer) {
                            const uint32_t bar = full_leader + 8 * stage, as = a_ring + stage * XE_TILE_BYTES, bs = b_ring + stage * L::B_BYTES;
                            const int k0 = kc * XE_BK;
                            if (a_mn) {
                                tma_load_3d_pair(as, &p.tm_a, bar, arow, k0, pa);
                                tma_load_3d_pair(as + 8192, &p.tm_a, bar, arow + 64, k0, pa);
                            } else {
                                tma_load_3d_pair(as, &p.tm_a, bar, k0, arow, pa);
                            }
                            if (b_mn) {
                                tma_load_3d_pair(bs, &p.tm_b, bar, brow, k0, pb);
                                if (BN == 256) tma_load_3d_pair(bs + 8192, &p.tm_b, bar, brow + 64, k0, pb);
                            } else {
                                tma_load_3d_pair(bs, &p.tm_b, bar, k0, brow, pb);
                            }
                        }
                        if (++stage == STAGES) { stage = 0; phase ^= 1; }
                    }
                }
            }
        }
        if (!ok && issuer) drain_after_abort();
    } else if (warp == 1) {
        if (rank == 0) {   // warp-uniform loop, one elected lane issues the tcgen05 instructions
            const bool issuer = elect_one();
            int stage = 0, as = 0;
            uint32_t phase = 0, aphase = 0;
            bool ok = true;
            long long u;
            for (unsigned i = 0; ok && (u = unit_at(i)) >= 0; ++i) {
                Unit w;
                const XeProblem& p = decode(u, w);
                // 16 contraction elements further on: 32 bytes in a K-major row, 16 rows (2 KiB) in an MN-major tile
                const bool a_mn = p.a_mn, b_mn = p.b_mn;
                const uint64_t a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2;
                const uint64_t a0 = a_mn ? smem_desc_mn128(a_ring) : smem_desc_k128(a_ring), b0 = b_mn ? smem_desc_mn128(b_ring) : smem_desc_k128(b_ring);
                const uint32_t idesc = p.idesc;
                for (int cb = w.c0; ok && cb < w.c1; cb += p.block) {
                    const int steps = (cb + p.block < w.c1 ? p.block : w.c1 - cb) * p.pairs;
                    if (!mbar_wait_warp(bar_tempty + 8 * as, aphase ^ 1, abort_flag, pp.status, XE_WAIT_TMEM_EMPTY)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t d_tmem = tmem_base + (uint32_t)(as * BN);
                    for (int kc = 0; kc < steps; ++kc) {
                        if (!mbar_wait_warp(bar_full + 8 * stage, phase, abort_flag, pp.status, XE_WAIT_FULL)) { ok = false; break; }
                        tc_fence_after();
                        const uint64_t a_desc = a0 + (uint64_t)(stage * (XE_TILE_BYTES >> 4)), b_desc = b0 + (uint64_t)(stage * (L::B_BYTES >> 4));
#pragma unroll
                        for (int ks = 0; ks < XE_BK / 16; ++ks)
                            if (issuer) tc_mma_pair<false>(d_tmem, a_desc + ks * a_step, b_desc + ks * b_step, idesc, (kc | ks) ? 1u : 0u);
                        if (issuer) tc_commit_pair(bar_empty + 8 * stage, 3);       // frees the slot in both CTAs
                        if (++stage == STAGES) { stage = 0; phase ^= 1; }
                    }
                    if (ok && issuer) tc_commit_pair(bar_tfull + 8 * as, 3);        // this block's sums are ready in both CTAs
                    as ^= 1;
                    if (as == 0) aphase ^= 1;
                }
            }
        }
        if (blockIdx.x == 1 && pp.loss.loss) {        // the partner CTA's MMA warp has no other work
            pdl_wait();
            xe_sum_losses<32>(pp.loss);
        }
    } else {
        const int quarter = warp % 4;                 // tensor-memory lanes [32*quarter, 32*quarter + 32)
        const int half = (warp - 2) / 4;              // columns [WCOLS*half, WCOLS*half + WCOLS)
        uint8_t* stage_gen = gen_base + L::STORE_OFF + (warp - 2) * L::NBUF * L::BUF;
        const uint32_t stage_s = base + L::STORE_OFF + (warp - 2) * L::NBUF * L::BUF;
        const uint32_t tempty_leader = mapa_shared(bar_tempty, 0);
        float* bias_s = reinterpret_cast<float*>(gen_base + L::BIAS_OFF + (warp - 2) * 512);
        int as = 0;
        uint32_t aphase = 0, issued = 0;
        bool ok = true;
        pdl_wait();                                   // before anything is read or stored (the MMA warp does neither)
        if (pp.zero && blockIdx.x == 0 && warp == 2 && lane < 2) pp.zero[lane] = 0;
        // the staging buffer that is free next (its earlier store has been read out of shared memory)
        auto next_buffer = [&](bool plain = false) -> uint32_t {
            const uint32_t buf = L::NBUF == 1 ? 0 : issued & 1;
            if (plain) {                              // a use that no store follows: leave nothing outstanding behind it
                if (lane == 0) tma_store_wait_read<0>();
                __syncwarp();
            } else if (issued >= (uint32_t)L::NBUF) {
                if (lane == 0) tma_store_wait_read<L::NBUF - 1>();
                __syncwarp();
            }
            ++issued;
            return buf;
        };
        long long u;
        for (unsigned i = 0; ok && (u = unit_at(i)) >= 0; ++i) {
            Unit w;
            const XeProblem& p = decode(u, w);
            const long long row0 = (long long)(w.mp * 2 + (int)rank) * 128 + quarter * 32;
            const long long row = row0 + lane, wcol = (long long)w.nb * BN + half * WCOLS;

            // what the epilogue reads, on its way while the products run
            constexpr bool SOFTMAX = EPI >= XE_STATS;
            const bool live = row < p.m, whole = wcol + WCOLS <= p.n;
            long long target = -1;
            float lse = 0.f, g = 0.f;
            if constexpr (SOFTMAX) {
                if (live) target = p.target[row];
                if constexpr (EPI == XE_DZ) {
                    if (live) { lse = p.lse[row]; g = p.rowg[row]; }
                }
                if (p.bias) {                         // four columns per lane, to be read by all lanes
                    const float* b = p.bias + wcol + lane * 4;
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    const long long left = p.n - wcol - lane * 4;
                    if (left >= 4) v = __ldg(reinterpret_cast<const float4*>(b));
                    else if (left > 0) { v.x = b[0]; v.y = left > 1 ? b[1] : 0.f; v.z = left > 2 ? b[2] : 0.f; }
                    __syncwarp();
                    reinterpret_cast<float4*>(bias_s)[lane] = v;
                    __syncwarp();
                }
            }

            float z[WCOLS];                        // this thread's row of the tile
            for (int cb = w.c0; cb < w.c1; cb += p.block) {
                if (!mbar_wait_warp(bar_tfull + 8 * as, aphase, abort_flag, pp.status, XE_WAIT_TMEM_FULL)) { ok = false; break; }
                tc_fence_after();
                const uint32_t tsrc = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(as * BN + half * WCOLS);
                if (cb == w.c0) {
#pragma unroll
                    for (int j = 0; j < WCOLS / 32; ++j) tmem_ld_32x32(tsrc + j * 32, *reinterpret_cast<uint32_t(*)[32]>(&z[32 * j]));
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < WCOLS / 16; ++j) after_wait(*reinterpret_cast<uint32_t(*)[16]>(&z[16 * j]));
                } else {
#pragma unroll
                    for (int j = 0; j < WCOLS / 16; ++j) {
                        uint32_t r[16];
                        tmem_ld_32x16(tsrc + j * 16, r);
                        tmem_ld_wait();
                        after_wait(r);
#pragma unroll
                        for (int i = 0; i < 16; ++i) z[16 * j + i] += __uint_as_float(r[i]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(tempty_leader + 8 * as);       // this warp's share of the accumulator is in registers
                as ^= 1;
                if (as == 0) aphase ^= 1;
            }
            if (!ok) break;
            if (row0 >= p.m || wcol >= p.n) continue;

            // 64 columns of values, packed as BF16 pairs, to plane `plane` of the output
            auto stage64 = [&](const uint32_t (&w)[32], uint32_t buf) {
                uint4* dst = reinterpret_cast<uint4*>(stage_gen + buf * L::BUF + lane * 128);
#pragma unroll
                for (int j = 0; j < 8; ++j) dst[j ^ (lane & 7)] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
            };
            auto store64 = [&](uint32_t buf, long long col0, int plane) {
                fence_async_shared();
                __syncwarp();
                if (lane == 0) {
                    tma_store_3d(&p.tm_out, stage_s + buf * L::BUF, (int)col0, (int)row0, plane);
                    tma_store_commit();
                }
            };

            if constexpr (EPI == XE_F32) {
                const float scale = xe_scale(p.scale);
#pragma unroll
                for (int i = 0; i < WCOLS; ++i) z[i] *= scale;
            }
            // the warp's columns as floats, 32 at a time
            auto store_floats = [&]() {
#pragma unroll
                for (int chunk = 0; chunk < WCOLS / 32; ++chunk) {
                    const long long col0 = wcol + chunk * 32;
                    if (col0 < p.n) {
                        const uint32_t buf = next_buffer(p.plain);
                        float4* dst = reinterpret_cast<float4*>(stage_gen + buf * L::BUF + lane * 128);
                        const float* v = &z[chunk * 32];
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            dst[j ^ (lane & 7)] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                        if (p.plain) {                // row by row, 128 contiguous bytes per store
                            __syncwarp();
                            float* o = static_cast<float*>(p.out_ptr) + row0 * p.out_pitch + col0 + lane;
                            const int rows = p.m - row0 < 32 ? (int)(p.m - row0) : 32;
                            if (col0 + lane < p.n) {
                                const float* src = reinterpret_cast<const float*>(stage_gen + buf * L::BUF) + (lane & 3);
                                const long long pitch = p.out_pitch;
                                if (rows == 32 && !p.add) {
#pragma unroll
                                    for (int r = 0; r < 32; ++r) o[r * pitch] = src[r * 32 + ((lane >> 2) ^ (r & 7)) * 4];
                                } else {
                                    for (int r = 0; r < rows; ++r) {
                                        const float x = src[r * 32 + ((lane >> 2) ^ (r & 7)) * 4];
                                        o[r * pitch] = p.add ? o[r * pitch] + x : x;
                                    }
                                }
                            }
                            __syncwarp();
                            continue;
                        }
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0) {
                            if (p.add) tma_reduce_add_3d(&p.tm_out, stage_s + buf * L::BUF, (int)col0, (int)row0, w.sp);
                            else tma_store_3d(&p.tm_out, stage_s + buf * L::BUF, (int)col0, (int)row0, w.sp);
                            tma_store_commit();
                        }
                    }
                }
            };
            if constexpr (EPI == XE_F32) {
                if (!p.bf16) {
                    store_floats();
                    continue;
                }
#pragma unroll
                for (int h = 0; h < WCOLS / 64; ++h) {
                    if (wcol + h * 64 < p.n) {
                        const uint32_t buf = next_buffer(p.plain);
                        uint32_t pk[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) pk[i] = pack_bf16(z[64 * h + 2 * i], z[64 * h + 2 * i + 1]);
                        stage64(pk, buf);
                        if (p.plain) {                // row by row, two columns of 32 per row
                            __syncwarp();
                            const int rows = p.m - row0 < 32 ? (int)(p.m - row0) : 32;
                            const unsigned short* src = reinterpret_cast<const unsigned short*>(stage_gen + buf * L::BUF) + (lane & 7);
                            unsigned short* o = static_cast<unsigned short*>(p.out_ptr) + row0 * p.out_pitch + wcol + h * 64 + lane;
                            const bool in0 = wcol + h * 64 + lane < p.n, in1 = wcol + h * 64 + 32 + lane < p.n;
                            const long long pitch = p.out_pitch;
                            if (rows == 32 && __all_sync(0xffffffffu, in1)) {
#pragma unroll
                                for (int r = 0; r < 32; ++r) {
                                    o[r * pitch] = src[r * 64 + ((lane >> 3) ^ (r & 7)) * 8];
                                    o[r * pitch + 32] = src[r * 64 + (((lane >> 3) + 4) ^ (r & 7)) * 8];
                                }
                            } else {
                                for (int r = 0; r < rows; ++r) {
                                    if (in0) o[r * pitch] = src[r * 64 + ((lane >> 3) ^ (r & 7)) * 8];
                                    if (in1) o[r * pitch + 32] = src[r * 64 + (((lane >> 3) + 4) ^ (r & 7)) * 8];
                                }
                            }
                            __syncwarp();
                            continue;
                        }
                        store64(buf, wcol + h * 64, 0);
                    }
                }
            } else {
                if (p.bias) {
#pragma unroll
                    for (int j = 0; j < WCOLS / 4; ++j) {
                        const float4 b = reinterpret_cast<const float4*>(bias_s)[j];
                        add2(z[4 * j], z[4 * j + 1], b.x, b.y);
                        add2(z[4 * j + 2], z[4 * j + 3], b.z, b.w);
                    }
                }
                // column of the target among this warp's, -1 when it lies elsewhere
                const long long tl = target - p.col_base - wcol;
                const int tc = live && tl >= 0 && tl < WCOLS ? (int)tl : -1;
                const bool here = __any_sync(0xffffffffu, tc >= 0);
                if constexpr (EPI == XE_STATS || EPI == XE_STATS_E || EPI == XE_STATS_Z) {
                    if constexpr (EPI == XE_STATS_Z) store_floats();
                    if (here) {
                        float t = 0.f;
#pragma unroll
                        for (int i = 0; i < WCOLS; ++i) t = i == tc ? z[i] : t;
                        if (tc >= 0) p.zt[row] = t;
                    }
                    if (p.zsum) {
                        float t[4] = {0.f, 0.f, 0.f, 0.f};
                        if (whole) {                  // in pairs: a selection per element took 6152 x 64 x 32149 from 108 to 221 us
#pragma unroll
                            for (int i = 0; i < WCOLS; i += 2) add2(t[i & 2], t[(i & 2) + 1], z[i], z[i + 1]);
                        } else {
#pragma unroll
                            for (int i = 0; i < WCOLS; ++i) t[i & 3] += wcol + i < p.n ? z[i] : 0.f;
                        }
                        if (live) p.zsum[wcol / XE_STAT_COLS * p.m + row] = (t[0] + t[1]) + (t[2] + t[3]);
                    }
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < WCOLS; ++i) z[i] = wcol + i < p.n ? z[i] : -INFINITY;
                    }
                    float cm[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
                    for (int i = 4; i < WCOLS; i += 2) cm[i / 2 & 3] = max3(cm[i / 2 & 3], z[i], z[i + 1]);
                    const float mx = fmaxf(max3(cm[0], cm[1], cm[2]), cm[3]);
                    const float ref = mx == -INFINITY ? 0.f : mx;      // nothing but -inf: every term is 0
                    float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < WCOLS; i += 2) {
                        add2(z[i], z[i + 1], -ref, -ref);
                        mul2(z[i], z[i + 1], XE_LOG2E);
                        z[i] = xe_ex2(z[i]);
                        z[i + 1] = xe_ex2(z[i + 1]);
                        add2(t[i & 2], t[(i & 2) + 1], z[i], z[i + 1]);
                    }
                    if (live) p.stats[wcol / XE_STAT_COLS * p.m + row] = make_float2(mx, (t[0] + t[1]) + (t[2] + t[3]));
                    if constexpr (EPI == XE_STATS_E) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if (wcol + h * 64 < p.n) {
                                const uint32_t buf = next_buffer();
                                uint32_t pk[32];
#pragma unroll
                                for (int i = 0; i < 32; ++i) pk[i] = xe_pack_exp(z[64 * h + 2 * i], z[64 * h + 2 * i + 1]);
                                stage64(pk, buf);
                                store64(buf, wcol + h * 64, 0);
                            }
                        }
                    }
                } else {
                    const float gp = g * p.rule.pf, ga = g * p.rule.smooth_all;
#pragma unroll
                    for (int i = 0; i < WCOLS; i += 2) {
                        add2(z[i], z[i + 1], -lse, -lse);
                        mul2(z[i], z[i + 1], XE_LOG2E);
                        z[i] = xe_ex2(z[i]);
                        z[i + 1] = xe_ex2(z[i + 1]);
                        fma2(z[i], z[i + 1], gp, -ga);
                    }
                    if (__any_sync(0xffffffffu, g == 0.f)) {          // a row that does not count: exactly 0, whatever its logits
#pragma unroll
                        for (int i = 0; i < WCOLS; ++i) z[i] = g == 0.f ? 0.f : z[i];
                    }
                    if (here) {
                        const float gt = g * p.rule.smooth_t;
#pragma unroll
                        for (int i = 0; i < WCOLS; ++i) z[i] = i == tc ? z[i] - gt : z[i];
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (wcol + h * 64 < p.n) {
                            auto sums = [&]() {       // of this warp's 32 rows
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    const long long col = wcol + h * 64 + k * 32 + lane;
                                    float c[32];
#pragma unroll
                                    for (int i = 0; i < 32; ++i) c[i] = z[64 * h + 32 * k + i];
                                    const float cs = column_sums(c, lane);
                                    if (col < p.n) p.db_part[(row0 / 32) * p.db_pitch + col] = cs;
                                }
                            };
                            if (PLANES > 1 && p.db_part) sums();
#pragma unroll
                            for (int q = 0; q < PLANES; ++q) {        // round; several planes: keep the remainder for the next
                                const uint32_t buf = next_buffer();
                                uint4* dst = reinterpret_cast<uint4*>(stage_gen + buf * L::BUF + lane * 128);
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    uint32_t w4[4];
#pragma unroll
                                    for (int i = 0; i < 4; ++i) {
                                        float& v0 = z[64 * h + 8 * j + 2 * i];
                                        float& v1 = z[64 * h + 8 * j + 2 * i + 1];
                                        w4[i] = pack_bf16(v0, v1);
                                        if (q + 1 < PLANES) {
                                            v0 -= __uint_as_float(w4[i] << 16);
                                            v1 -= __uint_as_float(w4[i] & 0xffff0000u);
                                        }
                                    }
                                    dst[j ^ (lane & 7)] = make_uint4(w4[0], w4[1], w4[2], w4[3]);
                                }
                                store64(buf, wcol + h * 64, q);
                            }
                            if (PLANES == 1 && p.db_part) sums();
                        }
                    }
                }
            }
        }
        if (lane == 0) tma_store_wait_all();
    }

    // neither CTA may leave (or give back tensor memory) while its partner can still read its shared memory,
    // signal its barriers or run an MMA over both tensor memories
    tc_fence_before();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

// CTA pairs of a launch
unsigned launch_pairs(const XeParams& p) {
    const long long total = (long long)p.prob[0].units + p.prob[1].units, most = sm_count() < 4 ? 1 : sm_count() / 2;
    return (unsigned)(total < most ? total : most);
}

template <int EPI, int PLANES, int BN = XE_BN>
int run(const XeParams& p, cudaStream_t st) {
    using L = XeSmem<EPI, PLANES, BN>;
    static_assert(L::TOTAL <= 232448, "shared memory budget of one CTA exceeded");
    static std::once_flag once[64];
    int dev = 0;
    WINO_CUDA_CHECK(cudaGetDevice(&dev));
    cudaError_t attr_err = cudaSuccess;
    std::call_once(once[dev & 63], [&] {
        attr_err = cudaFuncSetAttribute(xe_gemm_kernel<EPI, PLANES, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::TOTAL);
    });
    WINO_CUDA_CHECK(attr_err);
    const unsigned pairs = launch_pairs(p);
    count_launch();
    WINO_CUDA_CHECK(launch_kernel(xe_gemm_kernel<EPI, PLANES, BN>, dim3(2 * pairs), dim3(XE_THREADS), L::TOTAL, st, true, p));
    return WINO_OK;
}

int make_problem(const XeProduct& x, XeProblem* out) {
    XeProblem& p = *out;
    const XeOutput& o = x.out;
    int rc;
    if ((rc = xe_operand_map(&p.tm_a, x.a, 128)) || (rc = xe_operand_map(&p.tm_b, x.b, (unsigned)x.bn / 2))) return rc;
    const bool f32 = x.epi == XE_F32 || x.epi == XE_STATS_Z;
    const int es = f32 ? 4 : 2;
    // a TMA store fills a row's last 16-byte unit with zeros behind the last column (measured), and wants such units as pitch
    p.plain = x.epi != XE_STATS && ((o.pitch * es) % 16 != 0 || (o.exact && (x.n * es) % 16 != 0));
    if (p.plain && (o.splits > 1 || x.epi > XE_BF16)) return fail(WINO_E_BADARG, "xent: buffer rows must be multiples of 16 bytes");
    if (x.epi == XE_STATS || p.plain) {
        p.tm_out = p.tm_a;
    } else {
        const int planes = f32 ? o.splits : x.epi == XE_DZ ? x.a.planes : 1;
        const unsigned long long dims[3] = {(unsigned long long)x.n, (unsigned long long)x.m, (unsigned long long)planes};
        const unsigned long long strides[2] = {(unsigned long long)o.pitch * es, (unsigned long long)(o.pitch * x.m) * es};
        const unsigned box[3] = {(unsigned)(128 / es), 32u, 1u};
        if ((rc = encode_tensor_map(&p.tm_out, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, o.ptr, dims, strides, box, 1)))
            return rc;
    }
    p.m = x.m; p.n = x.n;
    p.mpairs = (unsigned)((x.m + XE_BM - 1) / XE_BM);
    p.nblocks = (unsigned)((x.n + x.bn - 1) / x.bn);
    p.kchunks = (int)((x.k + XE_BK - 1) / XE_BK);
    p.splits = o.splits;
    p.part = p.kchunks / p.splits;
    p.part_over = p.kchunks % p.splits;
    const unsigned long long tiles = (unsigned long long)p.mpairs * p.nblocks;
    if (tiles * p.splits > 0x3fffffffull) return fail(WINO_E_UNSUPPORTED, "xent: more than 2^30 tiles");
    p.tiles = (unsigned)tiles;
    p.units = p.tiles * p.splits;
    p.band = XE_BAND * p.nblocks;
    p.block = x.a.planes == 3 ? 4 : 16;
    if (x.a.planes == 3) {
        static const unsigned char pa[6] = {2, 1, 0, 1, 0, 0}, pb[6] = {0, 1, 2, 0, 1, 0};
        p.pairs = 6;
        for (int i = 0; i < 6; ++i) { p.pa[i] = pa[i]; p.pb[i] = pb[i]; }
    } else {
        p.pairs = 1;
        p.pa[0] = p.pb[0] = 0;
    }
    p.a_mn = x.a.along_rows;
    p.b_mn = x.b.along_rows;
    p.idesc = make_idesc(OP_BF16, x.bn, XE_BM) | (p.a_mn ? 1u << 15 : 0u) | (p.b_mn ? 1u << 16 : 0u);
    p.add = o.add;
    p.bf16 = x.epi == XE_BF16;
    p.out_ptr = o.ptr; p.out_pitch = o.pitch;
    p.scale = o.scale;
    p.bias = o.bias; p.target = o.target; p.col_base = o.col_base;
    p.stats = o.stats; p.zsum = o.zsum; p.zt = o.zt;
    p.lse = o.lse; p.rowg = o.rowg; p.rule = o.rule;
    p.db_part = o.db_part; p.db_pitch = o.db_pitch;
    return WINO_OK;
}

}  // namespace

int xe_gemm(const XeProduct* prod, int count, cudaStream_t st) {
    static_assert(sizeof(XeParams) <= 4096, "kernel parameters");
    XeParams p;
    int rc;
    p.zero = prod[0].out.zero;
    p.loss = prod[0].out.loss;
    for (int i = 0; i < count; ++i)
        if ((rc = make_problem(prod[i], &p.prob[i]))) return rc;
    p.lead = 0;
    if (count == 1) {
        p.prob[1].units = 0;
    } else {
        // ring slots of a unit, and about six more for its epilogue; the product with the longer units goes first
        auto cost = [](const XeProblem& q) { return (double)q.kchunks / q.splits * q.pairs + 6.0; };
        if (cost(p.prob[0]) < cost(p.prob[1])) { const XeProblem t = p.prob[0]; p.prob[0] = p.prob[1]; p.prob[1] = t; }
        p.lead = (int)xe_turns_lead(p.prob[0].units, p.prob[1].units, launch_pairs(p), cost(p.prob[0]) / cost(p.prob[1]));
    }
    if ((rc = status_word(&p.status))) return rc;
    switch (prod[0].epi) {
        case XE_F32:
        case XE_BF16: return prod[0].bn == 128 ? run<XE_F32, 1, 128>(p, st) : run<XE_F32, 1>(p, st);
        case XE_STATS: return run<XE_STATS, 1>(p, st);
        case XE_STATS_Z: return run<XE_STATS_Z, 1>(p, st);
        case XE_STATS_E: return run<XE_STATS_E, 1>(p, st);
        case XE_DZ: return prod[0].a.planes == 3 ? run<XE_DZ, 3>(p, st) : run<XE_DZ, 1>(p, st);
    }
    return fail(WINO_E_BADARG, "xent: no kernel for this product");
}

}  // namespace wino
