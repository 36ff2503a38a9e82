// gk_grouped.cu -- bf16 / f16 products of rows grouped by expert, forward and both gradients.
//
//   forward / input gradient   C[i, :] = alpha A[i, :] B[g] + beta C[i, :],  off[g] <= i < off[g+1]
//   weight gradient            C[g]    = alpha A_g^T B_g + beta C[g]         (contraction over rows)
//
// Both are lowered to D[i, j] = sum_p P[i, p] Q[j, p] per group: P on the 128 TMEM lanes, Q on
// the MMA's N. P is always the side along C's columns (the weights' n, or B's columns), so a
// warp stores 32 consecutive elements of a row of C per instruction; Q is the ragged side of the
// forward product (the rows of A), so a group's last tile runs with N rounded up to 16 of its
// rows instead of a whole tile of rows.
//
// One persistent kernel: warp 1 issues tcgen05.mma kind::f16 (M = 128, N <= BN, f32
// accumulators, two TMEM buffers), the epilogue warps drain one accumulator while the next tile
// is computed, and a ring of shared-memory stages of 64 contraction elements in the 128-byte
// swizzle is filled by TMA (one producer thread). The tile schedule is computed on the device
// from the offsets (gk_group.cuh), so the host never waits for them.
//
// Operands that TMA cannot address (no unit stride, a pitch that is no multiple of 16 bytes, a
// base off a 16-byte boundary) are first copied to aligned scratch, line by line or transposed.
// (Loader warps that gather such operands inside the product were tried: at most 170 TFLOP/s and
// 1.5 TB/s, 143 us for 2000 x 2001 x 3001 against 46 us with the copies.)
//
// Operands lie K-major (the contraction contiguous: rows of A, weights stored n x k) or MN-major
// (weights stored k x n, both operands of the weight gradient); the MMA reads either from the
// boxes as they land. In the weight gradient the contraction ends where the group ends, in the
// middle of a stage: the stage's later MMAs are skipped, and warp 2 zeroes the rows between the
// end and the next multiple of 16 in both operands (they belong to other groups and may hold
// anything). The copies of such a stage complete on a barrier of warp 2's (rfull), and warp 2
// completes the stage's full[] when it is done, so the zeroing passes while earlier stages are
// multiplied. (Asked for by the MMA warp when it got there it cost 2 us a tile: 39 against 26
// us for 64 experts' gradients of 1024 x 512 over 65 rows.)
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdio.h>
#include <string.h>

#include <mutex>

#include "gemmkit_cuda.h"
#include "gk_engine.h"
#include "gk_group.cuh"
#include "gk_sm100.cuh"
#include "gk_store.cuh"
#include "gk_tc_common.cuh"

namespace gk {

namespace {

constexpr int GBK = 64;  // contraction elements per stage (one 128-byte swizzle row)
// MN-major stages: boxes of 64 rows (128 bytes) x 64 contraction indices, one after the other
// along the rows; an MMA reads 16 contraction indices = 16 lines of 128 bytes.
constexpr int MN_BOX = GBK * 128;
constexpr int MN_STEP = 16 * 128;

// Shared-memory matrix descriptor of an MN-major operand in such boxes: 128-byte swizzle atoms of
// 64 elements x 8 contraction indices; the next 64 elements are a box away (leading offset), the
// next 8 contraction indices 1024 bytes (stride offset).
__device__ __forceinline__ uint64_t sdesc_mn128(uint32_t saddr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(MN_BOX >> 4) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}

// The descriptors of an operand's stage 0 and the distances (in the descriptor's 16-byte units)
// between its MMAs' 16-element slices. The issuing thread has about 128 cycles per MMA: building
// the descriptors anew for each one held the products at 0.65 of what the tensor cores give.
struct OperandDesc {
    uint64_t base;
    uint32_t step;
    __device__ __forceinline__ OperandDesc(uint32_t saddr, int mn)
        : base(mn ? sdesc_mn128(saddr) : sdesc_kmajor_sw128(saddr)),
          step((mn ? MN_STEP : MMA_KB) >> 4) {}
    // slice ks of the stage that lies `off` bytes after stage 0
    __device__ __forceinline__ uint64_t at(uint32_t off, int ks) const {
        return base + (off >> 4) + static_cast<uint32_t>(ks) * step;
    }
};

// An operand: element (row r, contraction index p) of group g at
// ptr + g * gs + r * rs + p * ps.
struct GOperand {
    const uint16_t* ptr;
    int64_t rs, ps, gs;
};

struct GroupedParams {
    GOperand P, Q;
    int64_t np;               // rows of the P side (columns of C)
    int64_t nq;               // weight gradient: rows of the Q side; else unused
    int32_t kdim;             // forward: contraction length
    int32_t wgrad;            // 1: the contraction is ragged
    int32_t zero;             // 1: no product (k == 0 or alpha == 0): C <- beta C
    int32_t groups, rows, tiles_p, tiles_q;  // tiles_q: weight gradient only
    const int32_t* offsets;
    void* c;
    int64_t ldq, ldp, gsc;    // strides of C along the Q side, the P side and the groups
    float alpha, beta;
    int32_t p_mn, q_mn;       // TMA: the operand is MN-major
    int32_t p_z;              // TMA: 1 = the P operand has a group dimension
    int32_t p_4d, q_4d;       // TMA: MN-major boxes of a tile in one copy (see encode_mn4)
    int32_t f16;              // operands are f16 (else bf16)
    int32_t out_type;         // gk_dtype of C
    int32_t pieces;           // C leaves in 16-byte pieces (c_in_pieces)
    uint64_t timeout_ns;
    unsigned int* status;
};

template <int BN>
struct GroupedCfg {
    static constexpr int NEPI = BN >= 64 ? 8 : 4;
    static constexpr int EPI_W0 = 4;
    static constexpr int THREADS = 32 * (EPI_W0 + NEPI);
    static constexpr int WCOLS = BN / (NEPI / 4);
    static constexpr int P_BYTES = BM * BKB;
    static constexpr int Q_BYTES = BN * BKB;
    static constexpr int STAGE_BYTES = P_BYTES + Q_BYTES;
    static constexpr int TAB_BYTES = (2 * GROUP_TABLE_INTS * 4 + 15) / 16 * 16;
    static constexpr int BAR_BYTES = 512;
    static constexpr int EPI_BYTES = NEPI * EPI_BUF;
    static constexpr int RAW_STAGES =
        (SMEM_LIMIT - 1024 - BAR_BYTES - TAB_BYTES - EPI_BYTES) / STAGE_BYTES;
    static constexpr int STAGES = RAW_STAGES > 10 ? 10 : RAW_STAGES;
    static constexpr int OFF_EPI = STAGES * STAGE_BYTES;
    static constexpr int OFF_BARS = OFF_EPI + EPI_BYTES;
    static constexpr int OFF_TAB = OFF_BARS + BAR_BYTES;
    static constexpr int SMEM = 1024 + OFF_TAB + TAB_BYTES;
    static constexpr int TMEM_COLS = 2 * BN < 32 ? 32 : 2 * BN;
    static_assert(BN == 32 || BN == 64 || BN == 128 || BN == 256, "tile width");
    static_assert(STAGES >= 2 && SMEM <= SMEM_LIMIT, "shared memory budget");
    static_assert((3 * STAGES + 6) * 8 <= BAR_BYTES, "barrier area");
};

// One tile of the schedule as every role sees it.
struct GTile {
    int g, p0, q0;        // group, first row on the P and Q sides (inside the group)
    int qn;               // its Q rows
    int64_t qbase;        // first row of the Q operand / of C along the Q side
    int k0, nk;           // first contraction row (weight gradient) and contraction length
    int pb;               // its blocks of 256 P rows (tall pair tiles: 1 or 2)
};

// Q rows of a tile where `rows` of them are cut into tiles of at most BN: equal heights, rounded up
// to STEP. (Whole tiles of BN and a short last one would cost more: the short tile loads as
// much of P as a whole one, and is bound by that.)
template <int BN, int STEP>
__host__ __device__ __forceinline__ int tile_height(int rows) {
    const int tiles = (rows + BN - 1) / BN;
    const int h = (rows + tiles - 1) / tiles;
    return (h + STEP - 1) & ~(STEP - 1);
}

// The walk over tall tiles (2 TM P rows, p.tiles_p of them on the P side): where what is left after
// the last full wave of clusters would fill at most half of them, its tiles are walked in halves of
// TM rows, so that the last wave takes half the time.
template <int TM>
__device__ __forceinline__ bool next_tall(GroupWalk& w, const GroupedParams& p, GTile& t, int& tq) {
    const int rest = w.total % w.step;
    const int split = 2 * rest <= w.step ? w.total - rest : w.total;
    for (;;) {
        w.t += w.step;
        const int over = w.t - split;
        if (over >= 2 * (w.total - split)) return false;
        int tp;
        w.locate(over < 0 ? w.t : split + (over >> 1), p.tiles_p, tp, tq);
        t.p0 = tp * 2 * TM + (over >= 0 ? (over & 1) * TM : 0);
        if (t.p0 >= p.np) continue;  // the second half of a tile that has one
        t.pb = over < 0 && p.np - t.p0 > TM ? 2 : 1;
        return true;
    }
}

// PB: blocks of TM P rows in a tile.
template <int BN, int TM = BM, int PB = 1>
__device__ __forceinline__ bool next_tile(GroupWalk& w, const GroupedParams& p, GTile& t) {
    int tp, tq;
    if constexpr (PB == 1) {
        if (!w.next(p.tiles_p, tp, tq)) return false;
        t.p0 = tp * TM;
        t.pb = 1;
    } else {
        if (!next_tall<TM>(w, p, t, tq)) return false;
    }
    t.g = w.g;
    const int o0 = w.off[t.g], m = w.off[t.g + 1] - o0;
    const int qrows = p.wgrad ? static_cast<int>(p.nq) : m;
    const int h = tile_height<BN, 32>(qrows);
    t.q0 = tq * h;
    t.qn = min(h, qrows - t.q0);
    if (p.wgrad) {
        t.qbase = t.q0;
        t.k0 = o0;
        t.nk = p.zero ? 0 : m;
    } else {
        t.qbase = static_cast<int64_t>(o0) + t.q0;
        t.k0 = 0;
        t.nk = p.zero ? 0 : p.kdim;
    }
    return true;
}

// The factor of a tile's accumulators. An empty contraction is zero whatever alpha is (an infinity or
// a NaN too): C <- beta C.
__device__ __forceinline__ float tile_alpha(const GroupedParams& p, const GTile& t) {
    return t.nk > 0 ? p.alpha : 0.0f;
}

// Whether the stage of contraction block kb holds the end of its group inside 16 indices.
__device__ __forceinline__ bool ragged_stage(const GroupedParams& p, const GTile& t, int kb) {
    return p.wgrad && t.nk - kb < GBK && (t.nk & 15) != 0;
}

// Zeroes contraction indices [v, next multiple of 16) of `boxes` MN-major boxes (lines of 128 bytes).
__device__ __forceinline__ void zero_rows(uint8_t* box, int boxes, int v, int lane) {
    const int n = (16 - (v & 15)) * 8;  // 16-byte pieces per box
    for (int c = 0; c < boxes; ++c)
        for (int i = lane; i < n; i += 32)
            *reinterpret_cast<uint4*>(box + c * MN_BOX + v * 128 + i * 16) = make_uint4(0, 0, 0, 0);
}

template <int BN>
__global__ void __launch_bounds__(GroupedCfg<BN>::THREADS, 1)
    grouped_half_kernel(const __grid_constant__ CUtensorMap tmP,
                        const __grid_constant__ CUtensorMap tmQ, const GroupedParams p) {
    using C = GroupedCfg<BN>;
    constexpr int STAGES = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* sP = smem;
    uint8_t* sQ = smem + STAGES * C::P_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BARS);
    uint64_t* empty = full + STAGES;
    uint64_t* rfull = empty + STAGES;  // a stage that holds a group's ragged end has landed
    uint64_t* tfull = rfull + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* off = reinterpret_cast<int*>(smem + C::OFF_TAB);
    int* tile0 = off + GROUP_TABLE_INTS;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t tmo = p.timeout_ns;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
            mbar_init(&rfull[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], C::NEPI);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (threadIdx.x == 0 && !p.zero) {
        prefetch_tmap(&tmP);
        prefetch_tmap(&tmQ);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM_COLS);
        tmem_relinquish();
    }
    griddep_wait();  // the offsets, operands and C may belong to the previous kernel
    load_groups(p.offsets, p.groups, p.rows, off, tile0, blockIdx.x == 0 ? p.status : nullptr,
                [&](int m) {
                    return p.wgrad ? p.tiles_p * p.tiles_q : (m + BN - 1) / BN * p.tiles_p;
                });
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    GroupWalk walk(off, tile0, p.groups, blockIdx.x, gridDim.x);
    GTile t;

    if (warp == 0) {
        // ---------------- TMA producer (the whole warp, one lane issues) ----------------
        int stage = 0;
        uint32_t phase = 0, issued = 0, last_par = 0;
        bool ok = true;
        while (ok && next_tile<BN>(walk, p, t)) {
            const int pz = p.p_z ? t.g : 0;
            const int qb = static_cast<int>(t.qbase);
            for (int kb = 0; kb < t.nk; kb += GBK) {
                if (!warp_wait(&empty[stage], phase ^ 1u, abort_flag, p.status,
                               GK_DEV_TIMEOUT_PRODUCER, tmo)) {
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    uint64_t* fb = ragged_stage(p, t, kb) ? &rfull[stage] : &full[stage];
                    uint8_t* dp = sP + stage * C::P_BYTES;
                    uint8_t* dq = sQ + stage * C::Q_BYTES;
                    mbar_arrive_expect_tx(fb, C::STAGE_BYTES);
                    const int k = t.k0 + kb;
                    if (p.p_4d) {
                        tma_load_4d(dp, &tmP, fb, 0, k, t.p0 >> 6, pz);
                    } else if (p.p_mn) {
#pragma unroll
                        for (int c = 0; c < BM / 64; ++c)
                            tma_load_3d(dp + c * MN_BOX, &tmP, fb, t.p0 + 64 * c, k, pz);
                    } else {
                        tma_load_3d(dp, &tmP, fb, k, t.p0, pz);
                    }
                    if (p.q_4d) {
                        tma_load_4d(dq, &tmQ, fb, 0, k, qb >> 6, 0);
                    } else if (p.q_mn) {
#pragma unroll
                        for (int c = 0; c < BN / 64; ++c)
                            tma_load_3d(dq + c * MN_BOX, &tmQ, fb, qb + 64 * c, k, 0);
                    } else {
                        tma_load_3d(dq, &tmQ, fb, k, qb, 0);
                    }
                }
                __syncwarp();
                issued |= 1u << stage;
                last_par = (last_par & ~(1u << stage)) | (phase << stage);
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        griddep_launch_dependents();
        // every issued copy has landed before the CTA may exit
        int dummy = 0;
        for (int s = 0; s < STAGES; ++s)
            if (issued & (1u << s))
                mbar_wait(&full[s], (last_par >> s) & 1u, &dummy, p.status, GK_DEV_TIMEOUT_DRAIN,
                          tmo);
    } else if (warp == 2) {
        // ---------------- the contraction's ragged end (weight gradient) ----------------
        if (p.wgrad) {
            int blocks = 0;        // stages filled so far
            uint32_t parity = 0;   // rfull's, a bit per stage
            while (next_tile<BN>(walk, p, t)) {
                blocks += (t.nk + GBK - 1) / GBK;
                if ((t.nk & 15) == 0) continue;
                const int stage = (blocks - 1) % STAGES;
                if (!warp_wait(&rfull[stage], (parity >> stage) & 1u, abort_flag, p.status,
                               GK_DEV_TIMEOUT_PRODUCER, tmo))
                    break;
                parity ^= 1u << stage;
                const int v = t.nk & (GBK - 1);
                zero_rows(sP + stage * C::P_BYTES, BM / 64, v, lane);
                zero_rows(sQ + stage * C::Q_BYTES, BN / 64, v, lane);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[stage]);
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (the whole warp, one lane issues) ----------------
        int stage = 0;
        uint32_t phase = 0;
        const OperandDesc dP(smem_u32(sP), p.p_mn), dQ(smem_u32(sQ), p.q_mn);
        bool ok = true;
        for (int local = 0; ok && next_tile<BN>(walk, p, t); ++local) {
            const int acc = local & 1;
            const uint32_t aph = (local >> 1) & 1;
            if (!warp_wait(&tempty[acc], aph ^ 1u, abort_flag, p.status, GK_DEV_TIMEOUT_MMA, tmo))
                break;
            tc_fence_after();
            const uint32_t idesc = idesc_f16(BM, min(BN, (t.qn + 15) & ~15), p.f16 == 0) |
                                   (static_cast<uint32_t>(p.p_mn) << 15) |
                                   (static_cast<uint32_t>(p.q_mn) << 16);
            const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
            for (int kb = 0; kb < t.nk; kb += GBK) {
                if (!warp_wait(&full[stage], phase, abort_flag, p.status, GK_DEV_TIMEOUT_MMA, tmo)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t po = stage * C::P_BYTES, qo = stage * C::Q_BYTES;
                // the group's end: only the MMAs up to it (rounded up to 16) are issued
                const bool cut = p.wgrad && t.nk - kb < GBK;
                if (elect_one()) {
                    if (cut) {
                        const int steps = (t.nk - kb + 15) >> 4;
                        for (int ks = 0; ks < steps; ++ks)
                            mma_f16(d, dP.at(po, ks), dQ.at(qo, ks), idesc, (kb | ks) != 0 ? 1u : 0u);
                    } else {
#pragma unroll
                        for (int ks = 0; ks < GBK / 16; ++ks)
                            mma_f16(d, dP.at(po, ks), dQ.at(qo, ks), idesc, (kb | ks) != 0 ? 1u : 0u);
                    }
                    mma_commit(&empty[stage]);
                }
                __syncwarp();
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (!ok) break;
            if (elect_one()) mma_commit(&tfull[acc]);
            __syncwarp();
        }
        if (elect_one()) mma_commit(drain);  // every issued MMA has finished before TMEM is freed
        __syncwarp();
        int dummy = 0;
        mbar_wait(drain, 0, &dummy, p.status, GK_DEV_TIMEOUT_DRAIN, tmo);
    } else if (warp >= C::EPI_W0) {
        // ---------------- epilogue ----------------
        const int q = warp & 3;
        const int cbase = ((warp - C::EPI_W0) >> 2) * C::WCOLS;
        uint8_t* ebuf = smem + C::OFF_EPI + (warp - C::EPI_W0) * EPI_BUF;
        for (int local = 0; next_tile<BN>(walk, p, t); ++local) {
            const int acc = local & 1;
            const uint32_t aph = (local >> 1) & 1;
            if (!warp_wait(&tfull[acc], aph, abort_flag, p.status, GK_DEV_TIMEOUT_EPILOGUE, tmo))
                break;
            tc_fence_after();
            const int i0 = t.p0 + q * 32;  // the warp's first P row
            const int64_t at = (p.wgrad ? t.g * p.gsc : 0) + t.qbase * p.ldq + i0 * p.ldp;
            const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                                static_cast<uint32_t>(acc * BN + cbase);
            const int pn = static_cast<int>(min(static_cast<int64_t>(32), p.np - i0));
            const float alpha = tile_alpha(p, t);
            if (p.pieces) {
                store_cols16(tb, C::WCOLS, static_cast<uint16_t*>(p.c) + at + cbase * p.ldq, p.ldq,
                             t.qn - cbase, pn, alpha, p.out_type, ebuf, lane, t.nk > 0);
            } else {
                for (int c = 0; c < C::WCOLS && cbase + c < t.qn; c += 32) {
                    uint32_t v[32];
                    if (t.nk > 0) {
                        tmem_ld_x32(tb + c, v);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = 0u;
                    }
                    if (lane < pn)
                        store_any(p.c, p.out_type, at + lane * p.ldp + (cbase + c) * p.ldq, p.ldq, v,
                                  t.qn - cbase - c, alpha, p.beta);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[acc]);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

// ---- operands that TMA cannot address --------------------------------------------------------------
// (Plain loads: these kernels may start before the kernel that writes their source has ended, and
// only wait for it, so the source is not read-only for their lifetime.)

// The 16 bytes at byte offset a (0, 2 .. 14) of the 32 in (lo, hi).
__device__ __forceinline__ uint4 shift_bytes(const uint4& lo, const uint4& hi, uint32_t a) {
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (a & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (a & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const uint32_t b = (a & 2) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], b), __funnelshift_r(w[1], w[2], b),
                      __funnelshift_r(w[2], w[3], b), __funnelshift_r(w[3], w[4], b));
}

constexpr int RU = 4;  // 16-byte pieces of a lane in flight

// dst[g][l][e] = src[g * gs + l * pitch + e] for l < lines, e < len, zero for len <= e < dld (dld a
// multiple of 8): lines that start at any 2-byte address, to 16-byte aligned ones. A warp takes
// RU * 256 elements of a line; a piece is two aligned 16-byte loads shifted together (one where
// the line is aligned), or single elements where those would leave the source's bytes [lo, hi).
__global__ void __launch_bounds__(256)
    realign_lines_kernel(uint16_t* dst, int64_t dld, const uint16_t* src,
                         int64_t pitch, int64_t gs, int64_t lines, int64_t len, int64_t groups,
                         const uint8_t* lo, const uint8_t* hi) {
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t chunks = (dld + RU * 256 - 1) / (RU * 256);
    const int64_t units = groups * lines * chunks;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
         u < units; u += step) {
        const int64_t gl = u / chunks, c = u - gl * chunks;
        const int64_t g = gl / lines, l = gl - g * lines;
        const uint16_t* s = src + g * gs + l * pitch;
        uint16_t* d = dst + gl * dld;
        const int64_t e0 = c * (RU * 256) + lane * 8;
        const uint32_t a = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(s)) & 15u;
        uint4 x[RU], y[RU];
#pragma unroll
        for (int i = 0; i < RU; ++i) {
            const int64_t e = e0 + i * 256;
            const int n = static_cast<int>(min(static_cast<int64_t>(8), len - e));
            x[i] = y[i] = make_uint4(0, 0, 0, 0);
            if (n <= 0) continue;
            const uint8_t* p = reinterpret_cast<const uint8_t*>(s + e) - a;
            const bool two = a + 2 * n > 16;
            if (p >= lo && p + (two ? 32 : 16) <= hi) {
                x[i] = *reinterpret_cast<const uint4*>(p);
                if (two) y[i] = reinterpret_cast<const uint4*>(p)[1];
            } else {  // placed so that the shift below finds them
                uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k < n) {
                        const uint32_t at = a / 2 + k;
                        const uint32_t v = static_cast<uint32_t>(s[e + k]) << (16 * (at & 1));
#pragma unroll
                        for (uint32_t q = 0; q < 8; ++q)
                            if ((at >> 1) == q) w[q] |= v;
                    }
                x[i] = make_uint4(w[0], w[1], w[2], w[3]);
                y[i] = make_uint4(w[4], w[5], w[6], w[7]);
            }
        }
#pragma unroll
        for (int i = 0; i < RU; ++i) {
            const int64_t e = e0 + i * 256;
            if (e >= dld) break;
            uint4 q = shift_bytes(x[i], y[i], a);
            const int64_t n = len - e;
            q.x = n > 1 ? q.x : n > 0 ? q.x & 0xFFFFu : 0u;
            q.y = n > 3 ? q.y : n > 2 ? q.y & 0xFFFFu : 0u;
            q.z = n > 5 ? q.z : n > 4 ? q.z & 0xFFFFu : 0u;
            q.w = n > 7 ? q.w : n > 6 ? q.w & 0xFFFFu : 0u;
            *reinterpret_cast<uint4*>(d + e) = q;
        }
    }
}

// dst[g][l][e] = src[g * gs + l * sl + e * se], padded likewise, through a 32 x 32 tile: both sides
// are coalesced whichever source stride is small.
__global__ void __launch_bounds__(256)
    realign_any_kernel(uint16_t* dst, int64_t dld, const uint16_t* src,
                       int64_t sl, int64_t se, int64_t gs, int64_t lines, int64_t len,
                       int64_t groups) {
    __shared__ uint16_t tile[32][33];
    griddep_wait();
    griddep_launch_dependents();
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t te = (dld + 31) / 32, tl = (lines + 31) / 32;
    const bool e_fast = se <= sl;
    for (int64_t t = blockIdx.x; t < groups * tl * te; t += gridDim.x) {
        const int64_t g = t / (tl * te), r = t - g * tl * te;
        const int64_t l0 = r / te * 32, e0 = (r - r / te * te) * 32;
        for (int i = ty; i < 32; i += 8) {
            const int64_t l = l0 + (e_fast ? i : tx), e = e0 + (e_fast ? tx : i);
            const uint16_t v =
                l < lines && e < len ? src[g * gs + l * sl + e * se] : uint16_t{0};
            tile[e_fast ? i : tx][e_fast ? tx : i] = v;
        }
        __syncthreads();
        for (int i = ty; i < 32; i += 8) {
            const int64_t l = l0 + i, e = e0 + tx;
            if (l < lines && e < dld) dst[(g * lines + l) * dld + e] = tile[i][tx];
        }
        __syncthreads();
    }
}

// ---- the CTA-pair form ----------------------------------------------------------------------------
//
// Two CTAs of a cluster compute a tile of PB x 256 P rows x up to 256 Q rows with tcgen05
// cta_group::2: each loads its 128 rows of every P block and half of the Q rows (the peer's half is
// read from its shared memory by the MMA). The leader (even CTA) issues every MMA; barriers as in
// the engine's other pair kernel: full[] and tempty[] live in the leader, empty[] and tfull[] in
// both (one multicast commit each).
//   What bounds it is shared memory. A 256 x 256 tile needs 64 bytes of operands per SM and
// cycle of MMA from L2, and moves them through shared memory twice: all that it gives. Counted
// at 8192^3, a stage took 604 cycles for 512 of MMA, and shorter Q tiles took as long. PB = 2 loads
// 48 bytes per cycle instead (943k active cycles instead of 1070k for 907k of MMA; 746 -> 659
// us; 8 experts of 4096 -> 14336 over 8192 rows, skewed: 727 -> 659 us).
//   PB = 2 fills TMEM with one tile: accumulator b is P block b's. So that the MMAs need not wait for
// the epilogue, the two blocks run shifted at a tile's ends. The last TAIL stages run for block 0
// first, whose accumulator is then read while block 1's MMAs run; the next tile starts with block 0
// alone (up to LATE stages) until accumulator 1 is read. The epilogue takes an accumulator to
// registers, rounds and releases it before it stores, and stores without shared memory, which the
// MMAs need (28.6 instead of 29.8 us for 4096 x 1024 x 4096). TAIL 1 or 2 instead of 3 cost 1 to 2 %
// at contractions of 512, nothing at long ones. C of another layout or type, and beta, take PB = 1.

template <int PB>
struct GPairCfg {
    static constexpr int BN = 256;
    static constexpr int NEPI = 8;
    static constexpr int EPI_W0 = 4;
    static constexpr int THREADS = 32 * (EPI_W0 + NEPI);
    static constexpr int WCOLS = BN / 2;
    static constexpr int P_BYTES = PB * BM * BKB;
    static constexpr int Q_BYTES = BN / 2 * BKB;
    static constexpr int STAGE_BYTES = P_BYTES + Q_BYTES;
    static constexpr int TAB_BYTES = (2 * GROUP_TABLE_INTS * 4 + 15) / 16 * 16;
    static constexpr int BAR_BYTES = 256;
    static constexpr int EPI_BYTES = PB == 1 ? NEPI * EPI_BUF : 0;
    static constexpr int STAGES =
        (SMEM_LIMIT - 1024 - BAR_BYTES - TAB_BYTES - EPI_BYTES) / STAGE_BYTES;
    static constexpr int OFF_EPI = STAGES * STAGE_BYTES;
    static constexpr int OFF_BARS = OFF_EPI + EPI_BYTES;
    static constexpr int OFF_TAB = OFF_BARS + BAR_BYTES;
    static constexpr int SMEM = 1024 + OFF_TAB + TAB_BYTES;
    static constexpr int LATE = STAGES - 1, TAIL = 3;  // PB = 2: see above
    static_assert(STAGES >= 4 && (4 * STAGES + 6) * 8 <= BAR_BYTES, "barrier area");
};

template <int PB>
__global__ void __launch_bounds__(GPairCfg<PB>::THREADS, 1)
    grouped_pair_kernel(const __grid_constant__ CUtensorMap tmP,
                        const __grid_constant__ CUtensorMap tmQ, const GroupedParams p) {
    using C = GPairCfg<PB>;
    constexpr int STAGES = C::STAGES, BN = C::BN, TM = 2 * BM;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* sP = smem;
    uint8_t* sQ = smem + STAGES * C::P_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BARS);
    uint64_t* empty = full + STAGES;
    uint64_t* rfull = empty + STAGES;  // own half of a stage with a ragged end has landed
    uint64_t* peerz = rfull + STAGES;  // leader's: the peer has zeroed its half
    uint64_t* tfull = peerz + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* off = reinterpret_cast<int*>(smem + C::OFF_TAB);
    int* tile0 = off + GROUP_TABLE_INTS;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const uint64_t tmo = p.timeout_ns;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);  // the leader's producer; the peer's copies only add bytes
            mbar_init(&empty[s], 1);
            mbar_init(&rfull[s], 1);
            mbar_init(&peerz[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], 2 * C::NEPI);  // every epilogue warp of both CTAs
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_mbar_init();
        prefetch_tmap(&tmP);
        prefetch_tmap(&tmQ);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    griddep_wait();
    load_groups(p.offsets, p.groups, p.rows, off, tile0, blockIdx.x == 0 ? p.status : nullptr,
                [&](int m) {
                    return p.wgrad ? p.tiles_p * p.tiles_q : (m + BN - 1) / BN * p.tiles_p;
                });
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t full_l = mapa_shared(smem_u32(&full[0]), 0);
    const uint32_t tempty_l = mapa_shared(smem_u32(&tempty[0]), 0);
    const uint32_t rfull_own = mapa_shared(smem_u32(&rfull[0]), rank);
    GroupWalk walk(off, tile0, p.groups, blockIdx.x >> 1, gridDim.x >> 1);
    GTile t;

    if (warp == 0) {
        // ---------------- TMA producer (both CTAs; the whole warp, one lane issues) ------------
        int stage = 0;
        uint32_t phase = 0, issued = 0, last_par = 0;
        bool ok = true;
        while (ok && next_tile<BN, TM, PB>(walk, p, t)) {
            const int pz = p.p_z ? t.g : 0;
            const int p0 = t.p0 + static_cast<int>(rank) * BM;
            // the MMA's N, and this CTA's half of its rows
            const int n = min(BN, (t.qn + 31) & ~31);
            const int qb = static_cast<int>(t.qbase) + static_cast<int>(rank) * (n >> 1);
            for (int kb = 0; kb < t.nk; kb += GBK) {
                if (!warp_wait(&empty[stage], phase ^ 1u, abort_flag, p.status,
                               GK_DEV_TIMEOUT_PRODUCER, tmo)) {
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    // a ragged stage's halves complete on each CTA's own rfull
                    const bool ragged = ragged_stage(p, t, kb);
                    const uint32_t fb = (ragged ? rfull_own : full_l) + 8u * stage;
                    uint8_t* dq = sQ + stage * C::Q_BYTES;
                    const uint32_t bytes = t.pb * BM * BKB + C::Q_BYTES;
                    if (ragged)
                        mbar_arrive_expect_tx(&rfull[stage], bytes);
                    else if (leader)
                        mbar_arrive_expect_tx(&full[stage], 2 * bytes);
                    const int k = t.k0 + kb;
#pragma unroll
                    for (int b = 0; b < PB; ++b) {
                        if (b >= t.pb) break;
                        uint8_t* dp = sP + stage * C::P_BYTES + b * BM * BKB;
                        const int pr = p0 + b * TM;
                        if (p.p_4d) {
                            tma_load_4d_pair(dp, &tmP, fb, 0, k, pr >> 6, pz);
                        } else if (p.p_mn) {
#pragma unroll
                            for (int c = 0; c < BM / 64; ++c)
                                tma_load_3d_pair(dp + c * MN_BOX, &tmP, fb, pr + 64 * c, k, pz);
                        } else {
                            tma_load_3d_pair(dp, &tmP, fb, k, pr, pz);
                        }
                    }
                    if (p.q_4d) {
                        tma_load_4d_pair(dq, &tmQ, fb, 0, k, qb >> 6, 0);
                    } else if (p.q_mn) {
#pragma unroll
                        for (int c = 0; c < BN / 128; ++c)
                            tma_load_3d_pair(dq + c * MN_BOX, &tmQ, fb, qb + 64 * c, k, 0);
                    } else {
                        tma_load_3d_pair(dq, &tmQ, fb, k, qb, 0);
                    }
                }
                __syncwarp();
                issued |= 1u << stage;
                last_par = (last_par & ~(1u << stage)) | (phase << stage);
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        griddep_launch_dependents();
        if (leader) {  // its full barriers count both CTAs' copies
            int dummy = 0;
            for (int s = 0; s < STAGES; ++s)
                if (issued & (1u << s))
                    mbar_wait(&full[s], (last_par >> s) & 1u, &dummy, p.status,
                              GK_DEV_TIMEOUT_DRAIN, tmo);
        }
    } else if (warp == 1) {
        if (leader) {
            // ---------------- MMA issuer (leader; the whole warp, one lane issues) ----------------
            int stage = 0;
            uint32_t phase = 0;
            const OperandDesc dP(smem_u32(sP), p.p_mn), dQ(smem_u32(sQ), p.q_mn);
            bool ok = true;
            uint32_t idesc = 0;
            // the MMAs of a stage for the accumulator at d and the P block at `po`
            auto issue = [&](uint32_t d, uint32_t po, uint32_t qo, int kb, int nk) {
                if (p.wgrad && nk - kb < GBK) {
                    const int steps = (nk - kb + 15) >> 4;
                    for (int ks = 0; ks < steps; ++ks)
                        mma_f16_pair(d, dP.at(po, ks), dQ.at(qo, ks), idesc,
                                     (kb | ks) != 0 ? 1u : 0u);
                } else {
#pragma unroll
                    for (int ks = 0; ks < GBK / 16; ++ks)
                        mma_f16_pair(d, dP.at(po, ks), dQ.at(qo, ks), idesc,
                                     (kb | ks) != 0 ? 1u : 0u);
                }
            };
            int used1 = 0;  // tall tiles: those so far that used accumulator 1
            for (int local = 0; ok && next_tile<BN, TM, PB>(walk, p, t); ++local) {
                const int acc = PB == 1 ? local & 1 : 0;
                const uint32_t aph = (PB == 1 ? local >> 1 : local) & 1;
                if (!warp_wait(&tempty[acc], aph ^ 1u, abort_flag, p.status, GK_DEV_TIMEOUT_MMA,
                               tmo))
                    break;
                tc_fence_after();
                idesc = idesc_f16(TM, min(BN, (t.qn + 31) & ~31), p.f16 == 0) |
                        (static_cast<uint32_t>(p.p_mn) << 15) |
                        (static_cast<uint32_t>(p.q_mn) << 16);
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
                const bool two = PB == 2 && t.pb == 2;
                bool free1 = false;            // accumulator 1 is drained
                int late = 0, late0 = stage;   // stages that wait for block 1's MMAs, the first
                for (int kb = 0; kb < t.nk; kb += GBK) {
                    if (!warp_wait(&full[stage], phase, abort_flag, p.status, GK_DEV_TIMEOUT_MMA,
                                   tmo)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const bool last = kb + GBK >= t.nk;
                    if (elect_one()) {
                        issue(d, stage * C::P_BYTES, stage * C::Q_BYTES, kb, t.nk);
                        if (!two) mma_commit_pair_both(smem_u32(&empty[stage]), 0x3);
                        if (last) mma_commit_pair_both(smem_u32(&tfull[acc]), 0x3);
                    }
                    __syncwarp();
                    if (two) {
                        const bool must = ++late == C::LATE || last;
                        if (!free1) {
                            const uint32_t par = (used1 & 1) ^ 1u;
                            if (must) {
                                if (!warp_wait(&tempty[1], par, abort_flag, p.status,
                                               GK_DEV_TIMEOUT_MMA, tmo)) {
                                    ok = false;
                                    break;
                                }
                                free1 = true;
                            } else {
                                free1 = __all_sync(0xffffffffu, mbar_test(&tempty[1], par));
                            }
                            tc_fence_after();
                        }
                        if (must || (free1 && kb + C::TAIL * GBK < t.nk)) {
                            for (; late > 0; --late) {
                                if (elect_one()) {
                                    issue(d + BN, late0 * C::P_BYTES + BM * BKB,
                                          late0 * C::Q_BYTES, kb - (late - 1) * GBK, t.nk);
                                    mma_commit_pair_both(smem_u32(&empty[late0]), 0x3);
                                }
                                __syncwarp();
                                if (++late0 == STAGES) late0 = 0;
                            }
                        }
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                if (t.nk == 0) {  // an empty group's tile: its zeros are the epilogue's
                    if (two && !warp_wait(&tempty[1], (used1 & 1) ^ 1u, abort_flag, p.status,
                                          GK_DEV_TIMEOUT_MMA, tmo))
                        break;
                    if (elect_one()) mma_commit_pair_both(smem_u32(&tfull[acc]), 0x3);
                    __syncwarp();
                }
                if (two) {
                    if (elect_one()) mma_commit_pair_both(smem_u32(&tfull[1]), 0x3);
                    __syncwarp();
                    ++used1;
                }
            }
            if (elect_one()) mma_commit_pair(mapa_shared(smem_u32(drain), rank));
            __syncwarp();
            int dummy = 0;
            mbar_wait(drain, 0, &dummy, p.status, GK_DEV_TIMEOUT_DRAIN, tmo);
        }
    } else if (warp == 2) {
        // ---------------- the contraction's ragged end (both CTAs) ----------------
        // Each CTA's warp zeroes its own half; the leader's completes full[] once both have.
        if (p.wgrad) {
            const uint32_t peerz_l = mapa_shared(smem_u32(peerz), 0);
            int blocks = 0;        // stages filled so far
            uint32_t parity = 0;   // rfull's and peerz's, a bit per stage
            while (next_tile<BN, TM, PB>(walk, p, t)) {
                blocks += (t.nk + GBK - 1) / GBK;
                if ((t.nk & 15) == 0) continue;
                const int stage = (blocks - 1) % STAGES;
                const uint32_t par = (parity >> stage) & 1u;
                if (!warp_wait(&rfull[stage], par, abort_flag, p.status, GK_DEV_TIMEOUT_PRODUCER, tmo))
                    break;
                parity ^= 1u << stage;
                const int v = t.nk & (GBK - 1);
                zero_rows(sP + stage * C::P_BYTES, t.pb * (BM / 64), v, lane);
                zero_rows(sQ + stage * C::Q_BYTES, BN / 128, v, lane);
                fence_proxy_async_smem();
                __syncwarp();
                if (!leader) {
                    if (lane == 0) mbar_arrive_cluster(peerz_l + 8u * stage);
                    continue;
                }
                const bool ok = mbar_wait_cluster(&peerz[stage], par, abort_flag, p.status,
                                                  GK_DEV_TIMEOUT_PRODUCER, tmo);
                if (__any_sync(0xffffffffu, !ok)) break;
                if (lane == 0) mbar_arrive(&full[stage]);
            }
        }
    } else if (warp >= C::EPI_W0) {
        // ---------------- epilogue (both CTAs) ----------------
        const int q = warp & 3;
        const int cbase = ((warp - C::EPI_W0) >> 2) * C::WCOLS;
        uint8_t* ebuf = smem + C::OFF_EPI + (warp - C::EPI_W0) * EPI_BUF;
        if constexpr (PB == 2) {
            // Each accumulator goes to registers, rounded, before anything of it is stored: the
            // next tile's MMAs wait for that only.
            int used1 = 0;
            for (int local = 0; next_tile<BN, TM, PB>(walk, p, t); ++local) {
                bool ok = true;
                for (int b = 0; b < t.pb && ok; ++b) {
                    const uint32_t par = (b == 0 ? local : used1++) & 1;
                    if (!(ok = warp_wait(&tfull[b], par, abort_flag, p.status,
                                         GK_DEV_TIMEOUT_EPILOGUE, tmo)))
                        break;
                    tc_fence_after();
                    const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                                        static_cast<uint32_t>(b * BN + cbase);
                    uint32_t w[C::WCOLS / 2];
                    if (t.nk > 0) {
#pragma unroll
                        for (int k = 0; k < C::WCOLS; k += 32) {
                            uint32_t v[32];
                            tmem_ld_x32(tb + k, v);
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                w[k / 2 + i] = round_pair(v[2 * i], v[2 * i + 1], p.alpha, p.out_type);
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < C::WCOLS / 2; ++k) w[k] = 0u;
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster_relaxed(tempty_l + 8u * b);
                    const int i0 = t.p0 + b * TM + static_cast<int>(rank) * BM + q * 32;
                    const int pn = static_cast<int>(min(static_cast<int64_t>(32), p.np - i0));
                    uint16_t* c = static_cast<uint16_t*>(p.c) + (p.wgrad ? t.g * p.gsc : 0) +
                                  (t.qbase + cbase) * p.ldq + i0;
                    store_pairs(w, c, p.ldq, t.qn - cbase, pn, lane);
                }
                if (!ok) break;
            }
        } else {
            for (int local = 0; next_tile<BN, TM, PB>(walk, p, t); ++local) {
                const int acc = local & 1;
                const uint32_t aph = (local >> 1) & 1;
                if (!warp_wait(&tfull[acc], aph, abort_flag, p.status, GK_DEV_TIMEOUT_EPILOGUE, tmo))
                    break;
                tc_fence_after();
                const int i0 = t.p0 + static_cast<int>(rank) * BM + q * 32;  // the warp's first P row
                const int64_t at = (p.wgrad ? t.g * p.gsc : 0) + t.qbase * p.ldq + i0 * p.ldp;
                const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                                    static_cast<uint32_t>(acc * BN + cbase);
                const int pn = static_cast<int>(min(static_cast<int64_t>(32), p.np - i0));
                const float alpha = tile_alpha(p, t);
                if (p.pieces) {
                    store_cols16(tb, C::WCOLS, static_cast<uint16_t*>(p.c) + at + cbase * p.ldq, p.ldq,
                                 t.qn - cbase, pn, alpha, p.out_type, ebuf, lane, t.nk > 0);
                } else {
                    for (int c = 0; c < C::WCOLS && cbase + c < t.qn; c += 32) {
                        uint32_t v[32];
                        if (t.nk > 0) {
                            tmem_ld_x32(tb + c, v);
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[e] = 0u;
                        }
                        if (lane < pn)
                            store_any(p.c, p.out_type, at + lane * p.ldp + (cbase + c) * p.ldq, p.ldq, v,
                                      t.qn - cbase - c, alpha, p.beta);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(tempty_l + 8u * acc);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();  // neither CTA leaves while the other may still use its barriers or operands
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

template <int PB>
int launch_grouped_pair(const CUtensorMap& tp, const CUtensorMap& tq, const GroupedParams& p,
                        int grid, int pdl, cudaStream_t stream, char* err, size_t errlen) {
    using C = GPairCfg<PB>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(grouped_pair_kernel<PB>, C::SMEM, done);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof(cfg));
        cfg.gridDim = dim3(static_cast<unsigned>(grid));
        cfg.blockDim = dim3(C::THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl ? 2 : 1;
        e = cudaLaunchKernelEx(&cfg, grouped_pair_kernel<PB>, tp, tq, p);
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) {
        snprintf(err, errlen, "gemmkit: grouped kernel launch failed: %s", cudaGetErrorString(e));
        return GK_ECUDA;
    }
    return GK_OK;
}

template <int BN>
int launch_grouped(const CUtensorMap& tp, const CUtensorMap& tq, const GroupedParams& p, int grid,
                   int pdl, cudaStream_t stream, char* err, size_t errlen) {
    using C = GroupedCfg<BN>;
    auto kern = grouped_half_kernel<BN>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(kern, C::SMEM, done);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof(cfg));
        cfg.gridDim = dim3(static_cast<unsigned>(grid));
        cfg.blockDim = dim3(C::THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl ? 1 : 0;
        e = cudaLaunchKernelEx(&cfg, kern, tp, tq, p);
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) {
        snprintf(err, errlen, "gemmkit: grouped kernel launch failed: %s", cudaGetErrorString(e));
        return GK_ECUDA;
    }
    return GK_OK;
}

// Whether TMA can address a 16-bit operand of `rows` rows x `len` contraction indices x `groups`
// (1: no group dimension), and how it lies: 0 = K-major, 1 = MN-major, -1 = not at all. A stride
// along a dimension of one element says nothing.
int tma_major(const GOperand& o, int64_t rows, int64_t len, int64_t groups, bool mn_ok, bool k_ok) {
    if (reinterpret_cast<uintptr_t>(o.ptr) & 15) return -1;
    if (groups > 1 && (o.gs <= 0 || o.gs % 8)) return -1;
    const bool r1 = rows <= 1, p1 = len <= 1;
    if (k_ok && (o.ps == 1 || p1) && (r1 || (o.rs > 0 && o.rs % 8 == 0))) return 0;
    if (mn_ok && (o.rs == 1 || r1) && (p1 || (o.ps > 0 && o.ps % 8 == 0))) return 1;
    return -1;
}

// The tensor map of such an operand: 64 contiguous elements x `box` lines (a power of two) of one
// group. Strides along dimensions of one element are replaced by any valid one.
int encode_goperand(CUtensorMap* map, const GOperand& o, int major, int64_t rows, int64_t len,
                    int64_t groups, int box, char* err, size_t errlen) {
    const int64_t inner = major ? rows : len, outer = major ? len : rows;
    const int64_t ld = outer > 1 ? (major ? o.ps : o.rs) : (inner + 7) / 8 * 8;
    const int64_t gs = groups > 1 ? o.gs : ld;
    return encode_tmap_u16(map, o.ptr, inner, outer, groups, ld, gs, 64, box, err, errlen);
}

// Tile width along the Q side. Forward: the mean rows of a group; a group's last tile costs only
// its own rows on the tensor cores, so a wide tile loses little on short groups, but its stages
// are larger and fewer fit.
int grouped_bn(int64_t q) { return q <= 32 ? 32 : q <= 64 ? 64 : q <= 128 ? 128 : 256; }

// Scratch for realigned operands: stream-ordered memory from a pool of the engine's own on the
// current device, so that calls on several streams, and calls captured into several graphs, never
// share any (a captured call allocates and frees inside its graph). At every synchronisation the
// pool gives back what it holds beyond 1 / SCRATCH_SHARE of the device's memory (2.8 of 179 GiB), and
// gk_scratch_release the rest. (Held without a bound, one call with a large stack of odd weights
// kept its size from the process's other allocations for good. Mapping memory anew is not cheap:
// with a bound below its 0.94 GB a synchronised call with 8 weights of 4096 x 14336 took 2.3
// instead of 0.49 ms.)
constexpr size_t SCRATCH_SHARE = 64;

// The pool of device `dev`; with `make`, made at the first call (nullptr on failure).
cudaMemPool_t scratch_pool(int dev, bool make) {
    static std::mutex m;
    static cudaMemPool_t pools[64] = {};
    if (dev < 0 || dev >= 64) return nullptr;
    std::lock_guard<std::mutex> lock(m);
    if (!pools[dev] && make) {
        cudaMemPoolProps props;
        memset(&props, 0, sizeof(props));
        props.allocType = cudaMemAllocationTypePinned;
        props.handleTypes = cudaMemHandleTypeNone;
        props.location.type = cudaMemLocationTypeDevice;
        props.location.id = dev;
        size_t unused = 0, total = 0;
        cudaMemPool_t pool = nullptr;
        if (cudaMemGetInfo(&unused, &total) != cudaSuccess ||
            cudaMemPoolCreate(&pool, &props) != cudaSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        uint64_t keep = total / SCRATCH_SHARE;
        if (cudaMemPoolSetAttribute(pool, cudaMemPoolAttrReleaseThreshold, &keep) != cudaSuccess)
            cudaGetLastError();  // it then keeps nothing
        pools[dev] = pool;
    }
    return pools[dev];
}

// A realigned copy of an operand (rows x len x groups) in scratch memory, K-major or, with `mn`,
// MN-major; the operand is changed to describe it, and *scratch is what to free on the stream.
int realign(GOperand* o, int64_t rows, int64_t len, int64_t groups, bool mn, int pdl,
            cudaStream_t st, void** scratch) {
    const int64_t lines = mn ? len : rows, run = mn ? rows : len;
    const int64_t sl = mn ? o->ps : o->rs, se = mn ? o->rs : o->ps;
    const int64_t dld = (run + 7) / 8 * 8;
    // a captured allocation belongs to its graph, whichever pool it names (and a pool cannot be
    // created during a capture)
    const size_t bytes = static_cast<size_t>(groups * lines * dld * 2);
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    cudaError_t e = cudaStreamIsCapturing(st, &cap);
    if (e == cudaSuccess && cap != cudaStreamCaptureStatusNone) {
        e = cudaMallocAsync(scratch, bytes, st);
    } else if (e == cudaSuccess) {
        int dev = -1;
        cudaGetDevice(&dev);
        cudaMemPool_t pool = scratch_pool(dev, true);
        e = pool ? cudaMallocFromPoolAsync(scratch, bytes, pool, st) : cudaErrorMemoryAllocation;
        if (e == cudaErrorMemoryAllocation && pool) {  // once more, without what the pool holds unused
            cudaGetLastError();
            cudaMemPoolTrimTo(pool, 0);
            e = cudaMallocFromPoolAsync(scratch, bytes, pool, st);
        }
    }
    if (e != cudaSuccess) {
        cudaGetLastError();
        *scratch = nullptr;
        return api_err(e == cudaErrorMemoryAllocation ? GK_ENOMEM : GK_ECUDA,
                       "gemmkit: workspace allocation: %s", cudaGetErrorString(e));
    }
    uint16_t* dst = static_cast<uint16_t*>(*scratch);
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    const int64_t most = static_cast<int64_t>(sm_count()) * 8;
    if (se == 1 || run <= 1) {
        const int64_t units = groups * lines * ((dld + RU * 256 - 1) / (RU * 256));
        const int64_t blocks = (units + 7) / 8;
        cfg.gridDim = dim3(static_cast<unsigned>(blocks < most ? blocks : most));
        const uint8_t* lo = reinterpret_cast<const uint8_t*>(o->ptr);
        const uint8_t* hi = reinterpret_cast<const uint8_t*>(
            o->ptr + (groups - 1) * o->gs + (lines - 1) * sl + run);
        e = cudaLaunchKernelEx(&cfg, realign_lines_kernel, dst, dld, o->ptr, sl, o->gs, lines, run,
                               groups, lo, hi);
    } else {
        const int64_t tiles = groups * ((lines + 31) / 32) * ((dld + 31) / 32);
        cfg.gridDim = dim3(static_cast<unsigned>(tiles < most ? tiles : most));
        e = cudaLaunchKernelEx(&cfg, realign_any_kernel, dst, dld, o->ptr, sl, se, o->gs, lines, run,
                               groups);
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess)
        return api_err(GK_ECUDA, "gemmkit: pack kernel launch failed: %s", cudaGetErrorString(e));
    *o = mn ? GOperand{dst, 1, dld, lines * dld} : GOperand{dst, dld, 1, lines * dld};
    return GK_OK;
}

// Clusters of the pair kernel that are resident at once on the current device.
int pair_clusters() {
    static PerDevice<int> cache;
    int dev = 0;
    cudaGetDevice(&dev);
    return cache.get(dev, [] {
        cudaLaunchConfig_t q;
        memset(&q, 0, sizeof(q));
        q.gridDim = dim3(static_cast<unsigned>(sm_count() / 2 * 2));
        q.blockDim = dim3(GPairCfg<1>::THREADS);
        q.dynamicSmemBytes = GPairCfg<1>::SMEM;
        cudaLaunchAttribute a[1];
        a[0].id = cudaLaunchAttributeClusterDimension;
        a[0].val.clusterDim.x = 2;
        a[0].val.clusterDim.y = 1;
        a[0].val.clusterDim.z = 1;
        q.attrs = a;
        q.numAttrs = 1;
        int c = 0;
        if (cudaFuncSetAttribute(grouped_pair_kernel<1>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 GPairCfg<1>::SMEM) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&c, grouped_pair_kernel<1>, &q) != cudaSuccess || c <= 0) {
            cudaGetLastError();
            c = sm_count() / 2;
        }
        return c;
    });
}

int run_planned(GroupedParams p, int64_t gp, int64_t plen, int64_t qrows, cudaStream_t stream);

int run_grouped(GroupedParams p, cudaStream_t stream) {
    int dev = 0;
    int rc = api_check_device(&dev);
    if (rc) return rc;
    // TMA needs unit strides and 16-byte multiples; the forward product's Q rows start anywhere
    // (K-major only: their coordinate is the slow one), and so does the weight gradient's
    // contraction (MN-major only).
    const int64_t gp = p.P.gs != 0 ? p.groups : 1;
    const int64_t plen = p.wgrad ? p.rows : p.kdim;
    const int64_t qrows = p.wgrad ? p.nq : p.rows;
    void* scratch[2] = {nullptr, nullptr};
    if (!p.zero) {
        p.p_mn = tma_major(p.P, p.np, plen, gp, true, !p.wgrad);
        p.q_mn = tma_major(p.Q, qrows, plen, 1, p.wgrad != 0, !p.wgrad);
        const int pdl = api_pdl_enabled();
        if (p.p_mn < 0) {  // the contiguous side stays so where the product can read it
            p.p_mn = p.wgrad || (p.P.rs == 1 && p.P.ps != 1);
            rc = realign(&p.P, p.np, plen, gp, p.p_mn != 0, pdl, stream, &scratch[0]);
        }
        if (!rc && p.q_mn < 0) {
            p.q_mn = p.wgrad;
            rc = realign(&p.Q, qrows, plen, 1, p.q_mn != 0, pdl, stream, &scratch[1]);
        }
    }
    if (!rc) rc = run_planned(p, gp, plen, qrows, stream);
    for (void* s : scratch)
        if (s && cudaFreeAsync(s, stream) != cudaSuccess && !rc) {
            cudaGetLastError();
            rc = api_err(GK_ECUDA, "gemmkit: freeing the workspace failed");
        }
    return rc;
}

// Chooses the tiles and launches the product; both operands are ready for TMA.
int run_planned(GroupedParams p, int64_t gp, int64_t plen, int64_t qrows, cudaStream_t stream) {
    int rc = 0;
    p.p_z = gp > 1;
    const bool tma = !p.zero;
    const int64_t mean = (static_cast<int64_t>(p.rows) + p.groups - 1) / p.groups;
    const int64_t qside = p.wgrad ? p.nq : mean;
    // an upper bound of the tiles (the device computes the true number from the offsets)
    auto tiles_bound = [&](int64_t tm, int64_t bn) {
        const int64_t tq = p.wgrad ? (p.nq + bn - 1) / bn * p.groups
                                   : (static_cast<int64_t>(p.rows) + bn - 1) / bn + p.groups;
        return (p.np + tm - 1) / tm * tq;
    };
    const int clusters = pair_clusters();
    // The pair kernel where its 256 x 256 tiles are mostly full on both sides and keep every
    // cluster busy (a forward group that fills no whole tile still counts one in the bound)
    const int64_t pair_tiles = tiles_bound(2 * BM, 256) - (p.wgrad ? 0 : p.groups);
    const bool pair = tma && p.np > BM && qside > BM && pair_tiles >= clusters;
    const int bn = pair ? 256 : grouped_bn(p.wgrad && qside < 64 ? 64 : qside);
    p.pieces = c_in_pieces(p.c, p.out_type, p.ldq, p.ldp, p.gsc, p.np, p.beta);
    // 512-column tiles where C allows their epilogue and they do not leave more clusters idle: a
    // wave of halves takes about 11/12 of a wave of 256 x 256 tiles (46 against 50 us for
    // 4096 -> 4096 over 2048 rows, two each), but 4096 -> 9472 over 512 rows is one wave of 74 square
    // tiles and two of halves (30 against 44 us).
    const int64_t q_tiles = p.wgrad ? (p.nq + 255) / 256 * p.groups  // forward: about half a tile
                                    : (p.rows + 255) / 256 + (p.groups - 1) / 2;  // over per group
    const int64_t waves = ((p.np + 2 * BM - 1) / (2 * BM) * q_tiles + clusters - 1) / clusters;
    const int64_t tall_tiles = (p.np + 4 * BM - 1) / (4 * BM) * q_tiles, rest = tall_tiles % clusters;
    const int64_t half_waves = tall_tiles / clusters * 2 + (rest == 0 ? 0 : 2 * rest <= clusters ? 1 : 2);
    const bool tall = pair && p.pieces && p.np > 2 * BM && 11 * half_waves <= 12 * waves;
    const int tm = tall ? 4 * BM : pair ? 2 * BM : BM;
    const int64_t tiles = tiles_bound(tm, bn);
    if (tiles > INT32_MAX / 2)
        return set_last_error(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    p.tiles_p = static_cast<int>((p.np + tm - 1) / tm);
    p.tiles_q = static_cast<int>((p.nq + bn - 1) / bn);
    p.timeout_ns = wait_limit_ns((plen + GBK - 1) / GBK);
    p.status = device_status_ptr();
    const int pdl = api_pdl_enabled();
    char err[256] = "";
    CUtensorMap tmp, tmq;
    memset(&tmp, 0, sizeof(tmp));
    memset(&tmq, 0, sizeof(tmq));
    if (tma) {
        const int qbox = pair ? bn / 2 : bn;
        // Where the rows of an MN-major operand are whole 64-element chunks and every tile starts
        // on one, its boxes come in one copy (two 8 KB copies per operand and stage held the
        // ring back: 1339 against 1500 TFLOP/s at 8192^3).
        const int nq = static_cast<int>(p.nq);
        const int h = !p.wgrad ? 1 : bn == 256 ? tile_height<256, 32>(nq) : bn == 128
                          ? tile_height<128, 32>(nq) : tile_height<64, 32>(nq);
        p.p_4d = p.p_mn && p.np % 64 == 0;
        p.q_4d = p.q_mn && nq % 64 == 0 && h % (pair ? 128 : 64) == 0 && nq % h == 0;
        const int64_t pld = plen > 1 ? p.P.ps : p.np, qld = plen > 1 ? p.Q.ps : p.nq;
        if (p.p_4d)
            rc = encode_tmap_mn4(&tmp, p.P.ptr, p.np, plen, gp, pld, gp > 1 ? p.P.gs : pld, BM / 64, err,
                                 sizeof(err));
        else
            rc = encode_goperand(&tmp, p.P, p.p_mn, p.np, plen, gp, p.p_mn ? GBK : BM, err,
                                 sizeof(err));
        if (!rc && p.q_4d)
            rc = encode_tmap_mn4(&tmq, p.Q.ptr, p.nq, plen, 1, qld, qld, qbox / 64, err, sizeof(err));
        else if (!rc)
            rc = encode_goperand(&tmq, p.Q, p.q_mn, qrows, plen, 1, p.q_mn ? GBK : qbox, err,
                                 sizeof(err));
        if (rc) return set_last_error(rc, err);
    }
    if (pair) {
        // (tall tiles may be walked in halves)
        const int64_t units = tall ? 2 * tiles : tiles;
        const int grid = 2 * static_cast<int>(units < clusters ? units : clusters);
        rc = tall ? launch_grouped_pair<2>(tmp, tmq, p, grid, pdl, stream, err, sizeof(err))
                  : launch_grouped_pair<1>(tmp, tmq, p, grid, pdl, stream, err, sizeof(err));
        return rc ? set_last_error(rc, err) : GK_OK;
    }
    const int sms = sm_count();
    const int grid = static_cast<int>(tiles < sms ? tiles : sms);
    auto go = [&](auto bn_tag) {
        constexpr int BN = decltype(bn_tag)::value;
        return launch_grouped<BN>(tmp, tmq, p, grid, pdl, stream, err, sizeof(err));
    };
    switch (bn) {
        case 32: rc = go(std::integral_constant<int, 32>{}); break;
        case 64: rc = go(std::integral_constant<int, 64>{}); break;
        case 128: rc = go(std::integral_constant<int, 128>{}); break;
        default: rc = go(std::integral_constant<int, 256>{}); break;
    }
    return rc ? set_last_error(rc, err) : GK_OK;
}

// The checks that both grouped entries share.
int check_groups(size_t groups, const int32_t* offsets, size_t rows, int is_f16, int out_type) {
    if (groups < 1 || groups > MAX_GROUPS)
        return api_err(GK_EINVAL, "gemmkit: grouped products take 1 to %d groups (groups = %zu)",
                       MAX_GROUPS, groups);
    if (!offsets) return api_err(GK_EINVAL, "gemmkit: null offsets");
    if (int rc = api_check_aligned(offsets, 4, "offsets")) return rc;
    if (rows > INT32_MAX / 2)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    if (out_type != GK_F32 && out_type != (is_f16 ? GK_F16 : GK_BF16))
        return api_err(GK_EINVAL, "gemmkit: a grouped product writes f32 or its operands' type");
    return GK_OK;
}

// A stack of `groups` views at stride gs (elements): the slice must hold all of them.
int check_stack(size_t len, size_t groups, size_t rows, size_t cols, ptrdiff_t rs, ptrdiff_t cs,
                ptrdiff_t gs, const char* name) {
    int rc = api_check_view(len, rows, cols, rs, cs, name);
    if (rc) return rc;
    if (gs < 0)
        return api_err(GK_EINVAL, "gemmkit: %s group stride (%td) must not be negative", name, gs);
    if (groups > 1 && rows && cols) {
        const __int128 last = static_cast<__int128>(groups - 1) * gs + 1 +
                              static_cast<__int128>(rows - 1) * rs +
                              static_cast<__int128>(cols - 1) * cs;
        if (last > static_cast<__int128>(len))
            return api_err(GK_EINVAL,
                           "gemmkit: %s stack of %zu views %zux%zu (strides %td,%td, group stride "
                           "%td) does not fit its slice of %zu elements",
                           name, groups, rows, cols, rs, cs, gs, len);
    }
    return GK_OK;
}

}  // namespace

}  // namespace gk

using namespace gk;

extern "C" {

int gk_scratch_release(int device) {
    int prev = 0;
    cudaGetDevice(&prev);
    if (cudaSetDevice(device) != cudaSuccess) {
        cudaGetLastError();
        return api_err(GK_ENODEV, "gemmkit: bad device");
    }
    cudaMemPool_t pool = scratch_pool(device, false);
    cudaError_t e = cudaSuccess;
    if (pool) {  // what was freed is unused once the calls that used it have ended
        e = cudaDeviceSynchronize();
        if (e == cudaSuccess) e = cudaMemPoolTrimTo(pool, 0);
    }
    cudaSetDevice(prev);
    if (e != cudaSuccess)
        return api_err(GK_ECUDA, "gemmkit: releasing the scratch: %s", cudaGetErrorString(e));
    return GK_OK;
}

int gk_gemm_half_grouped(int is_f16, size_t groups, const int32_t* offsets, float alpha,
                         gk_matref a, gk_matref b, ptrdiff_t b_gs, float beta, gk_matmut c,
                         int out_type, gk_parallelism par, gk_stream_t stream) {
    (void)par;
    int rc = check_groups(groups, offsets, a.rows, is_f16, out_type);
    if (rc) return rc;
    const size_t so = out_type == GK_F32 ? 4 : 2;
    if ((rc = api_validate_gemm_views(a, b, c, 2, so))) return rc;
    if ((rc = check_stack(b.len, groups, b.rows, b.cols, b.rs, b.cs, b_gs, "B"))) return rc;
    if (a.cols > INT32_MAX / 2 || b.cols > INT32_MAX / 2)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    if (c.rows == 0 || c.cols == 0) return GK_OK;
    if (!c.data) return api_err(GK_EINVAL, "gemmkit: null C");
    const bool zero = a.cols == 0 || alpha == 0.0f;
    if (!zero && (!a.data || !b.data)) return api_err(GK_EINVAL, "gemmkit: null A or B");
    if ((rc = api_check_aligned(a.data, 2, "A")) || (rc = api_check_aligned(b.data, 2, "B")) ||
        (rc = api_check_aligned(c.data, so, "C")))
        return rc;
    GroupedParams p;
    memset(&p, 0, sizeof(p));
    p.P = GOperand{static_cast<const uint16_t*>(b.data), b.cs, b.rs, b_gs};
    p.Q = GOperand{static_cast<const uint16_t*>(a.data), a.rs, a.cs, 0};
    p.np = static_cast<int64_t>(b.cols);
    p.kdim = static_cast<int32_t>(a.cols);
    p.zero = zero;
    p.groups = static_cast<int>(groups);
    p.rows = static_cast<int>(a.rows);
    p.offsets = offsets;
    p.c = c.data;
    p.ldq = c.rs;
    p.ldp = c.cs;
    p.alpha = alpha;
    p.beta = beta;
    p.f16 = is_f16 != 0;
    p.out_type = out_type;
    return run_grouped(p, static_cast<cudaStream_t>(stream));
}

int gk_gemm_half_grouped_wgrad(int is_f16, size_t groups, const int32_t* offsets, float alpha,
                               gk_matref a, gk_matref b, float beta, gk_matmut c, ptrdiff_t c_gs,
                               int out_type, gk_parallelism par, gk_stream_t stream) {
    (void)par;
    int rc = check_groups(groups, offsets, a.rows, is_f16, out_type);
    if (rc) return rc;
    const size_t so = out_type == GK_F32 ? 4 : 2;
    // A^T B in gemmkit's frame: (A.cols x rows) (rows x B.cols)
    const gk_matref at{a.data, a.len, a.cols, a.rows, a.cs, a.rs};
    if ((rc = api_validate_gemm_views(at, b, c, 2, so))) return rc;
    const gk_matref cr{c.data, c.len, c.rows, c.cols, c.rs, c.cs};
    if ((rc = check_stack(cr.len, groups, cr.rows, cr.cols, cr.rs, cr.cs, c_gs, "C"))) return rc;
    if (a.cols > INT32_MAX / 2 || b.cols > INT32_MAX / 2)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    if (c.rows == 0 || c.cols == 0) return GK_OK;
    if (groups > 1) {  // no element of one group's C may be an element of another's
        size_t need = static_cast<size_t>((c.rows - 1) * c.rs + (c.cols - 1) * c.cs) + 1;
        if (static_cast<size_t>(c_gs) < need)
            return api_err(GK_EINVAL,
                           "gemmkit: the groups of C overlap or interleave (group stride %td, a group "
                           "spans %zu elements)",
                           c_gs, need);
    }
    if (!c.data) return api_err(GK_EINVAL, "gemmkit: null C");
    const bool zero = a.rows == 0 || alpha == 0.0f;
    if (!zero && (!a.data || !b.data)) return api_err(GK_EINVAL, "gemmkit: null A or B");
    if ((rc = api_check_aligned(a.data, 2, "A")) || (rc = api_check_aligned(b.data, 2, "B")) ||
        (rc = api_check_aligned(c.data, so, "C")))
        return rc;
    GroupedParams p;
    memset(&p, 0, sizeof(p));
    p.P = GOperand{static_cast<const uint16_t*>(b.data), b.cs, b.rs, 0};
    p.Q = GOperand{static_cast<const uint16_t*>(a.data), a.cs, a.rs, 0};
    p.np = static_cast<int64_t>(b.cols);
    p.nq = static_cast<int64_t>(a.cols);
    p.wgrad = 1;
    p.zero = zero;
    p.groups = static_cast<int>(groups);
    p.rows = static_cast<int>(a.rows);
    p.offsets = offsets;
    p.c = c.data;
    p.ldq = c.rs;
    p.ldp = c.cs;
    p.gsc = c_gs;
    p.alpha = alpha;
    p.beta = beta;
    p.f16 = is_f16 != 0;
    p.out_type = out_type;
    return run_grouped(p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
