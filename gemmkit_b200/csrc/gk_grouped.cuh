// gk_grouped.cuh -- bf16 / f16 products of rows grouped by expert, forward and both gradients.
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
// What becomes of the accumulators is a template argument (EPI): alpha acc + beta C here, the epilogues
// of a feed-forward layer in gk_epilogue.cuh.
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
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdio.h>
#include <string.h>

#include "gemmkit_cuda.h"
#include "gk_engine.h"
#include "gk_epilogue.cuh"
#include "gk_group.cuh"
#include "gk_sm100.cuh"
#include "gk_store.cuh"
#include "gk_tc_common.cuh"

namespace gk {

// An operand: element (row r, contraction index p) of group g at
// ptr + g * gs + r * rs + p * ps.
struct GOperand {
    const uint16_t* ptr;
    int64_t rs, ps, gs;
};

// A realigned copy of an operand (rows x len x groups) in scratch memory, K-major or, with `mn`,
// MN-major; the operand is changed to describe it, and *scratch is what to free on the stream.
int realign(GOperand* o, int64_t rows, int64_t len, int64_t groups, bool mn, int pdl,
            cudaStream_t st, void** scratch);

// dbias[g] from the sums of the tiles of `tile` rows that a backward epilogue left in `part`, `shares`
// slots of np columns each (gk_linear.cu; slice: see there).
int launch_sum_parts(const float* part, const int32_t* offsets, int groups, int rows, int tile,
                     int shares, int slice, int64_t np, const EpiArgs& e, cudaStream_t st);

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
    EpiArgs e;                // EPI_FWD, EPI_BWD
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
    int tq;               // its place among the group's tiles along the Q side
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
    t.tq = tq;
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

// The sums of a warp's columns, to slot `share` of its tile's: the tiles of a group follow each other
// along the Q side, so a group's slots are consecutive. Without slots (one tile along the Q side, its rows
// all in share 0) they are the gradient itself.
__device__ __forceinline__ void epi_sum(const GroupedParams& p, const GTile& t, const int* tile0,
                                        int i0, int pn, int share, int shares, float sum, int lane) {
    if (lane >= pn || !p.e.dbias) return;
    if (!p.e.part) {
        if (share == 0) store_sum(p.e, i0 + lane, sum);
        return;
    }
    const int64_t slot =
        static_cast<int64_t>(tile0[t.g] / p.tiles_p + t.tq) * shares + share;
    p.e.part[slot * p.np + i0 + lane] = sum;
}

// A warp's part of a tile through the epilogue: `wcols` columns (a multiple of 32) from TMEM address tb
// on, the tile's Q rows from cbase on; its sums go to slot `share` of the tile's `shares`.
template <int EPI>
__device__ __forceinline__ void epi_tile(const GroupedParams& p, const GTile& t, const int* tile0,
                                         uint32_t tb, int wcols, int cbase, int i0, int pn, int share,
                                         int shares, int lane) {
    const float alpha = tile_alpha(p, t);
    const float bias = epi_fwd(EPI) ? epi_bias(p.e, t.g, i0, pn, lane) : 0.0f;
    float sum = 0.0f;
    auto columns = [&](auto pairs) {
        constexpr bool PAIRS = decltype(pairs)::value;
        constexpr int N = 32;  // (with 16 the latencies of a block show: 1024 -> 8192 over 8192 rows 164 us, 153)
#pragma unroll 1
        for (int c = 0; c < wcols && cbase + c < t.qn; c += N) {
            const EpiAt at{i0, pn, t.qbase + cbase + c, t.qn - cbase - c};
            EpiSide<EPI, N> s;
            s.template load<PAIRS>(p.e, at, p.out_type == GK_F32, lane);
            uint32_t v[N];
            if (t.nk > 0) {
                tmem_ld_x32(tb + c, v);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = 0u;
            }
            s.template own<PAIRS>(p.e, lane);
            epi_columns<EPI, N, PAIRS>(p.e, p.c, p.out_type, p.ldq, p.ldp, at, v, s, alpha, bias, sum, lane);
        }
    };
    if (p.e.pairs)
        columns(std::true_type{});
    else
        columns(std::false_type{});
    if constexpr (epi_bwd(EPI)) epi_sum(p, t, tile0, i0, pn, share, shares, sum, lane);
}

// SPLIT: a cluster of up to eight CTAs computes one tile, each a run of its stages. Their accumulators are
// exchanged through shared memory once the ring is idle: 16 Q rows (a unit) go to CTA unit % cluster
// size, which adds them in the CTAs' order and runs the epilogue. For products with fewer tiles than the
// SMs hold: one row, 14336 -> 4096 in 32 tiles streams its weights through 128 SMs instead of 32 (83 ->
// 26 us).
template <int BN, int EPI, bool SPLIT = false>
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
    const int ctas = SPLIT ? static_cast<int>(cluster_ctas()) : 1;
    const int rank = SPLIT ? static_cast<int>(cluster_ctarank()) : 0;
    GroupWalk walk(off, tile0, p.groups, blockIdx.x / ctas, gridDim.x / ctas);
    GTile t;
    // the contraction indices of this CTA (a cluster's tile has more stages than the cluster CTAs)
    auto first_k = [&](int r) {
        return SPLIT ? (t.nk + GBK - 1) / GBK * r / ctas * GBK : 0;
    };
    auto last_k = [&]() { return SPLIT ? min(first_k(rank + 1), t.nk) : t.nk; };
    bool tile = false;  // SPLIT: this CTA's part of a tile is ready

    if (warp == 0) {
        // ---------------- TMA producer (the whole warp, one lane issues) ----------------
        int stage = 0;
        uint32_t phase = 0, issued = 0, last_par = 0;
        bool ok = true;
        while (ok && next_tile<BN>(walk, p, t)) {
            const int pz = p.p_z ? t.g : 0;
            const int qb = static_cast<int>(t.qbase);
            const int kend = last_k();
            for (int kb = first_k(rank); kb < kend; kb += GBK) {
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
            const int kb0 = first_k(rank), kend = last_k();
            for (int kb = kb0; kb < kend; kb += GBK) {
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
                            mma_f16(d, dP.at(po, ks), dQ.at(qo, ks), idesc, ((kb - kb0) | ks) != 0 ? 1u : 0u);
                    } else {
#pragma unroll
                        for (int ks = 0; ks < GBK / 16; ++ks)
                            mma_f16(d, dP.at(po, ks), dQ.at(qo, ks), idesc, ((kb - kb0) | ks) != 0 ? 1u : 0u);
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
            if constexpr (SPLIT) {
                tile = true;
                break;
            }
            const int i0 = t.p0 + q * 32;  // the warp's first P row
            const int64_t at = (p.wgrad ? t.g * p.gsc : 0) + t.qbase * p.ldq + i0 * p.ldp;
            const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                                static_cast<uint32_t>(acc * BN + cbase);
            const int pn = static_cast<int>(min(static_cast<int64_t>(32), p.np - i0));
            const float alpha = tile_alpha(p, t);
            if constexpr (EPI != EPI_STORE) {
                epi_tile<EPI>(p, t, tile0, tb, C::WCOLS, cbase, i0, pn, (warp - C::EPI_W0) >> 2,
                              C::NEPI / 4, lane);
            } else if (p.pieces) {
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

    if constexpr (SPLIT) {
        static_assert(EPI != EPI_STORE && BN <= 128, "the epilogues that a cluster shares");
        tc_fence_before();
        __syncwarp();
        cluster_sync();  // every CTA's MMAs are done, its ring is idle
        tc_fence_after();
        const int q = warp & 3, sets = C::NEPI / 4, set = (warp - C::EPI_W0) >> 2;
        const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
        const int units = tile ? (min(BN, t.qn) + 15) >> 4 : 0;
        // unit u of CTA r lies at ((u / ctas) * ctas + r) * UNIT of its owner's shared memory
        constexpr int UNIT = 16 * BM * 4;
        if (warp >= C::EPI_W0) {
            for (int u = set; u < units; u += sets) {
                const int owner = u % ctas;
                if (owner == rank) continue;
                uint32_t v[16];
                tmem_ld_cols16(tb + 16 * u, v);
                const uint32_t at =
                    mapa_shared(smem_u32(smem) + static_cast<uint32_t>((u - owner + rank) * UNIT), owner) +
                    static_cast<uint32_t>(q * 32 + lane) * 4u;
#pragma unroll
                for (int e = 0; e < 16; ++e) st_cluster_u32(at + e * BM * 4, v[e]);
            }
        }
        __syncwarp();
        cluster_sync();  // the units have arrived
        if (warp >= C::EPI_W0) {
            const int i0 = t.p0 + q * 32;
            const int pn = static_cast<int>(min(static_cast<int64_t>(32), p.np - i0));
            const float bias = tile && epi_fwd(EPI) ? epi_bias(p.e, t.g, i0, pn, lane) : 0.0f;
            float sum = 0.0f;
            for (int u = set * ctas + rank; u < units; u += sets * ctas) {
                const EpiAt at{i0, pn, t.qbase + 16 * u, t.qn - 16 * u};
                uint32_t v[16];
                tmem_ld_cols16(tb + 16 * u, v);
                float a[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) a[e] = 0.0f;
                for (int r = 0; r < ctas; ++r) {
                    const float* part = reinterpret_cast<const float*>(
                        smem + (u - rank + r) * UNIT + (q * 32 + lane) * 4);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        a[e] += r == rank ? __uint_as_float(v[e]) : part[e * BM];
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(a[e]);
                EpiSide<EPI, 16> s;
                auto columns = [&](auto pairs) {
                    constexpr bool PAIRS = decltype(pairs)::value;
                    s.template load<PAIRS>(p.e, at, p.out_type == GK_F32, lane);
                    s.template own<PAIRS>(p.e, lane);
                    epi_columns<EPI, 16, PAIRS>(p.e, p.c, p.out_type, p.ldq, p.ldp, at, v, s, p.alpha, bias,
                                                sum, lane);
                };
                if (p.e.pairs)
                    columns(std::true_type{});
                else
                    columns(std::false_type{});
            }
            if (epi_bwd(EPI) && tile)
                epi_sum(p, t, tile0, i0, pn, set * ctas + rank, sets * ctas, sum, lane);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::TMEM_COLS);
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

template <int PB, int EPI>
struct GPairCfg {
    static constexpr int BN = 256;
    // A whole epilogue on tall tiles keeps 64 accumulators a lane in registers (epi_tall); sixteen warps
    // do it, and the four others give up registers for it (setmaxnreg): 128 x 56 + 512 x 104 are 60416
    // of the 640 x 96 that the block is launched with.
    static constexpr bool SPLIT_REGS = EPI != EPI_STORE && PB == 2;
    static constexpr int NEPI = SPLIT_REGS ? 16 : 8;
    static constexpr int REGS_OTHER = 56, REGS_EPI = 104;
    static_assert(128 * REGS_OTHER + 32 * 16 * REGS_EPI <= 32 * 20 * 96, "registers of the block");
    static constexpr int EPI_W0 = 4;
    static constexpr int THREADS = 32 * (EPI_W0 + NEPI);
    static constexpr int WCOLS = BN / (NEPI / 4);
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

// A warp's 64 columns of a tall tile's accumulator through the epilogue: all of them go to registers
// and the accumulator is handed back before any of the arithmetic, which then passes under the MMAs.
// (C moves in pairs.)
template <int EPI>
__device__ __forceinline__ void epi_tall(const GroupedParams& p, const GTile& t, const int* tile0,
                                         uint32_t tb, int cbase, int i0, int pn, int share, int shares,
                                         uint32_t tempty, int lane) {
    uint32_t raw[4][16];
#pragma unroll
    for (int i = 0; i < 4; ++i) tmem_ld_cols16_nowait(tb + 16 * i, raw[i]);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 4; ++i) frag_fence(raw[i]);
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive_cluster_relaxed(tempty);
    if (pn <= 0) return;
    const float bias = epi_fwd(EPI) ? epi_bias(p.e, t.g, i0, pn, lane) : 0.0f;
    float sum = 0.0f;
    auto columns = [&](int c, const uint32_t(&v)[16]) {
        const EpiAt at{i0, pn, t.qbase + cbase + c, t.qn - cbase - c};
        if (at.n <= 0) return;
        EpiSide<EPI, 16> s;
        s.template load<true>(p.e, at, false, lane);
        s.template own<true>(p.e, lane);
        epi_columns<EPI, 16, true>(p.e, p.c, p.out_type, p.ldq, 1, at, v, s, p.alpha, bias, sum, lane);
    };
    // A loop, the accumulators moved up after each 32 columns: unrolled over all 128 the code left the
    // instruction cache behind (8192 x 4096 -> 14336 with GELU and z kept: 926 us,
    // now 680).
#pragma unroll 1
    for (int c = 0; c < 64 && cbase + c < t.qn; c += 32) {
        columns(c, raw[0]);
        columns(c + 16, raw[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) raw[i][j] = raw[i + 2][j];
    }
    if constexpr (epi_bwd(EPI)) epi_sum(p, t, tile0, i0, pn, share, shares, sum, lane);
}

template <int PB, int EPI>
__global__ void __launch_bounds__(GPairCfg<PB, EPI>::THREADS, 1)
    grouped_pair_kernel(const __grid_constant__ CUtensorMap tmP,
                        const __grid_constant__ CUtensorMap tmQ, const GroupedParams p) {
    using C = GPairCfg<PB, EPI>;
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

    // (Each role's branch sets its own registers: after a common point the compiler would have to
    // count on the smaller number.)
    if (warp == 0) {
        if constexpr (C::SPLIT_REGS) regs_dec<C::REGS_OTHER>();
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
        if constexpr (C::SPLIT_REGS) regs_dec<C::REGS_OTHER>();
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
        if constexpr (C::SPLIT_REGS) regs_dec<C::REGS_OTHER>();
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
        if constexpr (C::SPLIT_REGS) regs_inc<C::REGS_EPI>();
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
                    const int i0 = t.p0 + b * TM + static_cast<int>(rank) * BM + q * 32;
                    const int pn = static_cast<int>(min(static_cast<int64_t>(32), p.np - i0));
                    if constexpr (EPI != EPI_STORE) {
                        epi_tall<EPI>(p, t, tile0, tb, cbase, i0, pn, (warp - C::EPI_W0) >> 2,
                                      C::NEPI / 4, tempty_l + 8u * b, lane);
                    } else {
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
                    uint16_t* c = static_cast<uint16_t*>(p.c) + (p.wgrad ? t.g * p.gsc : 0) +
                                  (t.qbase + cbase) * p.ldq + i0;
                    store_pairs(w, c, p.ldq, t.qn - cbase, pn, lane);
                    }
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
                if constexpr (EPI != EPI_STORE) {
                    epi_tile<EPI>(p, t, tile0, tb, C::WCOLS, cbase, i0, pn, (warp - C::EPI_W0) >> 2,
                                  C::NEPI / 4, lane);
                } else if (p.pieces) {
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
    } else {
        if constexpr (C::SPLIT_REGS) regs_dec<C::REGS_OTHER>();
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();  // neither CTA leaves while the other may still use its barriers or operands
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

template <int PB, int EPI>
int launch_grouped_pair(const CUtensorMap& tp, const CUtensorMap& tq, const GroupedParams& p,
                        int grid, int pdl, cudaStream_t stream, char* err, size_t errlen) {
    using C = GPairCfg<PB, EPI>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(grouped_pair_kernel<PB, EPI>, C::SMEM, done);
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
        e = cudaLaunchKernelEx(&cfg, grouped_pair_kernel<PB, EPI>, tp, tq, p);
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) {
        snprintf(err, errlen, "gemmkit: grouped kernel launch failed: %s", cudaGetErrorString(e));
        return GK_ECUDA;
    }
    return GK_OK;
}

// ctas > 1: clusters that split the contraction (SPLIT).
template <int BN, int EPI, bool SPLIT = false>
int launch_grouped(const CUtensorMap& tp, const CUtensorMap& tq, const GroupedParams& p, int grid,
                   int ctas, int pdl, cudaStream_t stream, char* err, size_t errlen) {
    using C = GroupedCfg<BN>;
    auto kern = grouped_half_kernel<BN, EPI, SPLIT>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(kern, C::SMEM, done);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg;
        memset(&cfg, 0, sizeof(cfg));
        cfg.gridDim = dim3(static_cast<unsigned>(grid));
        cfg.blockDim = dim3(C::THREADS);
        cfg.dynamicSmemBytes = C::SMEM;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        int n = 0;
        if (SPLIT) {
            attr[n].id = cudaLaunchAttributeClusterDimension;
            attr[n].val.clusterDim.x = static_cast<unsigned>(ctas);
            attr[n].val.clusterDim.y = 1;
            attr[n++].val.clusterDim.z = 1;
        }
        if (pdl) {
            attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[n++].val.programmaticStreamSerializationAllowed = 1;
        }
        cfg.attrs = attr;
        cfg.numAttrs = static_cast<unsigned>(n);
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

// Clusters of the pair kernel that are resident at once on the current device.
template <int EPI>
int pair_clusters() {
    static PerDevice<int> cache;
    int dev = 0;
    cudaGetDevice(&dev);
    return cache.get(dev, [] {
        cudaLaunchConfig_t q;
        memset(&q, 0, sizeof(q));
        q.gridDim = dim3(static_cast<unsigned>(sm_count() / 2 * 2));
        q.blockDim = dim3(GPairCfg<1, EPI>::THREADS);
        q.dynamicSmemBytes = GPairCfg<1, EPI>::SMEM;
        cudaLaunchAttribute a[1];
        a[0].id = cudaLaunchAttributeClusterDimension;
        a[0].val.clusterDim.x = 2;
        a[0].val.clusterDim.y = 1;
        a[0].val.clusterDim.z = 1;
        q.attrs = a;
        q.numAttrs = 1;
        int c = 0;
        if (cudaFuncSetAttribute(grouped_pair_kernel<1, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 GPairCfg<1, EPI>::SMEM) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&c, grouped_pair_kernel<1, EPI>, &q) != cudaSuccess || c <= 0) {
            cudaGetLastError();
            c = sm_count() / 2;
        }
        return c;
    });
}

// How many CTAs share a tile's contraction: the most (8, 4 or 2) for which all clusters are resident at once
// and each CTA keeps four stages, else 1.
template <int BN, int EPI>
int split_ctas(int64_t tiles, int64_t stages) {
    for (int ctas = 8; ctas > 1; ctas /= 2) {
        if (stages < 4 * ctas || tiles * ctas > sm_count()) continue;
        static PerDevice<int> cache[3];
        int dev = 0;
        cudaGetDevice(&dev);
        const int clusters = cache[ctas == 8 ? 0 : ctas == 4 ? 1 : 2].get(dev, [ctas] {
            auto kern = grouped_half_kernel<BN, EPI, true>;
            cudaLaunchConfig_t q;
            memset(&q, 0, sizeof(q));
            q.gridDim = dim3(static_cast<unsigned>(sm_count() / ctas * ctas));
            q.blockDim = dim3(GroupedCfg<BN>::THREADS);
            q.dynamicSmemBytes = GroupedCfg<BN>::SMEM;
            cudaLaunchAttribute a[1];
            a[0].id = cudaLaunchAttributeClusterDimension;
            a[0].val.clusterDim.x = static_cast<unsigned>(ctas);
            a[0].val.clusterDim.y = 1;
            a[0].val.clusterDim.z = 1;
            q.attrs = a;
            q.numAttrs = 1;
            int c = 0;
            if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     GroupedCfg<BN>::SMEM) != cudaSuccess ||
                cudaOccupancyMaxActiveClusters(&c, kern, &q) != cudaSuccess || c <= 0) {
                cudaGetLastError();
                c = -1;
            }
            return c;
        });
        if (tiles <= clusters) return ctas;
    }
    return 1;
}

template <int EPI>
int run_planned(GroupedParams p, int64_t gp, int64_t plen, int64_t qrows, cudaStream_t stream);

template <int EPI>
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
    if (!rc) rc = run_planned<EPI>(p, gp, plen, qrows, stream);
    for (void* s : scratch) {
        const int fr = scratch_free(s, stream);
        if (!rc) rc = fr;
    }
    return rc;
}

// Chooses the tiles and launches the product; both operands are ready for TMA.
template <int EPI>
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
    const int clusters = pair_clusters<EPI>();
    // The pair kernel where its 256 x 256 tiles are mostly full on both sides and keep every
    // cluster busy (a forward group that fills no whole tile still counts one in the bound)
    const int64_t pair_tiles = tiles_bound(2 * BM, 256) - (p.wgrad ? 0 : p.groups);
    const bool pair = tma && p.np > BM && qside > BM && pair_tiles >= clusters;
    const int bn = pair ? 256 : grouped_bn(p.wgrad && qside < 64 ? 64 : qside);
    p.pieces = EPI == EPI_STORE
                   ? c_in_pieces(p.c, p.out_type, p.ldq, p.ldp, p.gsc, p.np, p.beta)
                   : p.e.pairs != 0;
    // 512-column tiles where C allows their epilogue and they do not leave more clusters idle: a
    // wave of halves takes about 11/12 of a wave of 256 x 256 tiles (46 against 50 us for
    // 4096 -> 4096 over 2048 rows, two each), but 4096 -> 9472 over 512 rows is one wave of 74 square
    // tiles and two of halves (30 against 44 us).
    const int64_t q_tiles = p.wgrad ? (p.nq + 255) / 256 * p.groups  // forward: about half a tile
                                    : (p.rows + 255) / 256 + (p.groups - 1) / 2;  // over per group
    const int64_t waves = ((p.np + 2 * BM - 1) / (2 * BM) * q_tiles + clusters - 1) / clusters;
    const int64_t tall_tiles = (p.np + 4 * BM - 1) / (4 * BM) * q_tiles, rest = tall_tiles % clusters;
    const int64_t half_waves = tall_tiles / clusters * 2 + (rest == 0 ? 0 : 2 * rest <= clusters ? 1 : 2);
    // A whole epilogue holds the next tile's second accumulator back (epi_tall): about 11000 to 13000 cycles a
    // tile forward and 22000 backward, where square tiles cost 184 cycles more a stage of 64. Measured
    // over 8192 rows, in tall and in square tiles: 1024 -> 8192 with GELU and z kept 172 and 153 us,
    // 4096 -> 14336 796 and 806, 8192 -> 8192 840 and 915; the gradient 2048 -> 8192 295 and 265,
    // 4096 -> 14336 835 and 800, 8192 -> 8192 885 and 944.
    const bool long_enough = EPI == EPI_STORE || plen >= (epi_fwd(EPI) ? 4096 : 8192);
    const bool tall = pair && long_enough && p.pieces && p.np > 2 * BM && 11 * half_waves <= 12 * waves;
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
    // Products with few tiles share them between clusters of CTAs; `few`: no more tiles than that, whatever
    // the groups are.
    const int64_t few = (p.np + BM - 1) / BM * ((p.rows + static_cast<int64_t>(p.groups) * (bn - 1)) / bn);
    int ctas = 1;
    if constexpr (EPI != EPI_STORE) {
        const int64_t stages = (plen + GBK - 1) / GBK;
        if (tma && !pair && bn <= 128)
            ctas = bn == 32   ? split_ctas<32, EPI>(few, stages)
                   : bn == 64 ? split_ctas<64, EPI>(few, stages)
                              : split_ctas<128, EPI>(few, stages);
    }
    auto launch = [&]() -> int {
        if (pair) {
            // (tall tiles may be walked in halves)
            const int64_t units = tall ? 2 * tiles : tiles;
            const int grid = 2 * static_cast<int>(units < clusters ? units : clusters);
            return tall ? launch_grouped_pair<2, EPI>(tmp, tmq, p, grid, pdl, stream, err, sizeof(err))
                        : launch_grouped_pair<1, EPI>(tmp, tmq, p, grid, pdl, stream, err, sizeof(err));
        }
        const int sms = sm_count();
        const int grid = static_cast<int>(tiles < sms ? tiles : sms);
        auto go = [&](auto bn_tag) {
            constexpr int BN = decltype(bn_tag)::value;
            if constexpr (EPI != EPI_STORE && BN <= 128)
                if (ctas > 1)
                    return launch_grouped<BN, EPI, true>(tmp, tmq, p, static_cast<int>(few) * ctas, ctas, pdl,
                                                         stream, err, sizeof(err));
            return launch_grouped<BN, EPI>(tmp, tmq, p, grid, 1, pdl, stream, err, sizeof(err));
        };
        switch (bn) {
            case 32: return go(std::integral_constant<int, 32>{});
            case 64: return go(std::integral_constant<int, 64>{});
            case 128: return go(std::integral_constant<int, 128>{});
            default: return go(std::integral_constant<int, 256>{});
        }
    };
    if constexpr (epi_bwd(EPI)) {
        // A single tile of up to 32 rows, in one CTA (or in one unit): its epilogue has the whole sums. A few
        // rows then need no scratch and no second kernel (17 -> 12 us of host time).
        const bool whole = !p.offsets && bn == 32 && (ctas == 1 || p.rows <= 16);
        if (p.e.dbias && !whole) {  // a slot for each share of each tile along the Q side
            const int shares = tall ? GPairCfg<2, EPI>::NEPI / 4 : (bn == 32 ? 1 : 2) * ctas;
            const int64_t slots = ((static_cast<int64_t>(p.rows) + bn - 1) / bn + p.groups) * shares;
            void* part = nullptr;
            if ((rc = scratch_alloc(&part, static_cast<size_t>(slots * p.np) * 4, stream))) return rc;
            p.e.part = static_cast<float*>(part);
            if ((rc = launch()))
                set_last_error(rc, err);
            else
                rc = launch_sum_parts(p.e.part, p.offsets, p.groups, p.rows, bn, shares, 0, p.np, p.e,
                                      stream);
            const int fr = scratch_free(part, stream);
            return rc ? rc : fr;
        }
    }
    rc = launch();
    return rc ? set_last_error(rc, err) : GK_OK;
}

// The checks that the grouped entries share.
inline int check_groups(size_t groups, const int32_t* offsets, size_t rows, int is_f16, int out_type) {
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
inline int check_stack(size_t len, size_t groups, size_t rows, size_t cols, ptrdiff_t rs, ptrdiff_t cs,
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
