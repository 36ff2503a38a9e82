// gk_store.cuh -- the epilogue of the grouped and the 4-bit products: alpha * acc + beta * C in
// f32, rounded once to the output type.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "gemmkit_cuda.h"
#include "gk_sm100.cuh"

namespace gk {

__device__ __forceinline__ float from_out(float x) { return x; }
__device__ __forceinline__ float from_out(__half x) { return __half2float(x); }
__device__ __forceinline__ float from_out(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void to_out(float* p, float x) { *p = x; }
__device__ __forceinline__ void to_out(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void to_out(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// CH of one thread's accumulators (its lane's P row, CH consecutive Q rows, `n` of them in C):
// alpha * acc + beta * C in f32, rounded once to the output type. A warp's stores of one Q row
// are 32 consecutive elements when C's P stride is 1.
template <int CH, typename T>
__device__ __forceinline__ void store_chunk(T* c, int64_t ldq, const uint32_t (&v)[32], int n,
                                            float alpha, float beta) {
    if (beta != 0.0f) {
#pragma unroll
        for (int e = 0; e < CH; ++e)
            if (e < n)
                to_out(c + e * ldq, fmaf(beta, from_out(c[e * ldq]), alpha * __uint_as_float(v[e])));
    } else if (n >= CH) {
#pragma unroll
        for (int e = 0; e < CH; ++e) to_out(c + e * ldq, alpha * __uint_as_float(v[e]));
    } else {
#pragma unroll
        for (int e = 0; e < CH; ++e)
            if (e < n) to_out(c + e * ldq, alpha * __uint_as_float(v[e]));
    }
}

// The same for C of type `type` (gk_dtype), the first of the CH at element `at`.
template <int CH = 32>
__device__ __forceinline__ void store_any(void* c, int type, int64_t at, int64_t ldq,
                                          const uint32_t (&v)[32], int n, float alpha, float beta) {
    if (type == GK_F32)
        store_chunk<CH>(static_cast<float*>(c) + at, ldq, v, n, alpha, beta);
    else if (type == GK_F16)
        store_chunk<CH>(static_cast<__half*>(c) + at, ldq, v, n, alpha, beta);
    else
        store_chunk<CH>(static_cast<__nv_bfloat16*>(c) + at, ldq, v, n, alpha, beta);
}

// ---- 16-bit rows of C in 16-byte pieces ------------------------------------------------------------
//
// The path for 16-bit C with P stride 1, 16-byte rows and no beta. A lane of the plain TMEM load
// holds one P row, so its stores are 2 bytes wide and a 32 x 32 block takes 32 of them, each with
// its address, conversion and product (a 256 x 256 tile: about 6000 cycles of an SM, more than the
// MMAs of an expert's weight gradient over 700 rows). Here the accumulators are loaded in
// the 16x256b layout (lane t: rows t / 4 and t / 4 + 8, two columns each), rounded in pairs,
// transposed through shared memory (2 KB per warp) by stmatrix, and leave in 16-byte pieces.

// 16 accumulator columns of the warp's 32 TMEM lanes, not waited for: r[0..7] lanes 0-15, r[8..15]
// lanes 16-31; of each eight, four registers per 8 columns.
__device__ __forceinline__ void tmem_ld_frag16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7])
        : "r"(taddr)
        : "memory");
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
        : "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr + (16u << 16))
        : "memory");
}

// After tcgen05.wait::ld: no use of the registers may be scheduled before it.
__device__ __forceinline__ void frag_fence(uint32_t (&r)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i += 8)
        asm volatile(""
                     : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]),
                       "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7]));
}

__device__ __forceinline__ uint32_t round_pair(uint32_t lo, uint32_t hi, float alpha, int type) {
    const float a = alpha * __uint_as_float(lo), b = alpha * __uint_as_float(hi);
    uint32_t w;
    if (type == GK_F16)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
    return w;
}

// A block of 16 Q rows x 32 P rows rounded to 16 bits, as stmatrix takes it.
struct Block16 {
    uint32_t w[8];
    __device__ __forceinline__ void round(const uint32_t (&r)[16], float alpha, int type) {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            w[4 * o] = round_pair(r[4 * o], r[4 * o + 1], alpha, type);
            w[4 * o + 1] = round_pair(r[4 * o + 2], r[4 * o + 3], alpha, type);
            w[4 * o + 2] = round_pair(r[8 + 4 * o], r[8 + 4 * o + 1], alpha, type);
            w[4 * o + 3] = round_pair(r[8 + 4 * o + 2], r[8 + 4 * o + 3], alpha, type);
        }
    }
    // Into the 1 KB at shared address sb, transposed: Q row q at q * 64, its 16-byte piece m (8 P
    // rows) at m ^ (q / 2 % 4), so that these stores and the loads of copy_out touch every
    // bank once.
    __device__ __forceinline__ void stage(uint32_t sb, int lane) const {
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            const int q = o * 8 + (lane & 7), m = lane >> 3;
            asm volatile(
                "stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                    sb + static_cast<uint32_t>(q * 64 + ((m ^ ((q >> 1) & 3)) << 4))),
                "r"(w[4 * o]), "r"(w[4 * o + 1]), "r"(w[4 * o + 2]), "r"(w[4 * o + 3])
                : "memory");
        }
    }
};

// A staged block to C: n of its Q rows exist in C, and the first pn of the warp's 32 P rows (a
// multiple of 8 when fewer than 32); c is the first Q row's first element, ldq the pitch.
__device__ __forceinline__ void copy_out(uint32_t sb, uint16_t* c, int64_t ldq, int n, int pn,
                                         int lane) {
#pragma unroll
    for (int o = 0; o < 2; ++o) {
        const int q = o * 8 + (lane >> 2), m = lane & 3;
        const uint4 v = ld_shared_v4(sb + static_cast<uint32_t>(q * 64 + ((m ^ ((q >> 1) & 3)) << 4)));
        if (q < n && m * 8 < pn) st_global_v4(c + q * ldq + m * 8, v.x, v.y, v.z, v.w);
    }
}

// ---- 16-bit rows of C without shared memory ----------------------------------------------------
//
// Two accumulator columns of one TMEM lane (P row) are rounded into a word; neighbouring lanes
// exchange halves, so that the even lane holds rows l, l + 1 of the even column and the odd lane
// those of the odd one, four bytes each: a store of the warp writes two Q rows of 64 bytes.
//   w[j]: columns 2 j and 2 j + 1 of this lane's P row (N words); n of the columns exist in C.
template <int N>
__device__ __forceinline__ void store_pairs(const uint32_t (&w)[N], uint16_t* c, int64_t ldq, int n,
                                            int pn, int lane) {
    const int odd = lane & 1;
    const uint32_t give = odd ? 0x5410u : 0x7632u;
    const uint32_t sel0 = odd ? 0x3254u : 0x5410u, sel1 = odd ? 0x3276u : 0x7610u;
    uint16_t* q = c + (lane & 30) + odd * ldq;
    const int left = (lane & 30) < pn ? n - odd : 0;  // columns of this lane: 0, 2, 4, ... < left
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const uint32_t got =
            __shfl_xor_sync(0xffffffffu, __byte_perm(w[j], w[j + 1], give), 1);
        const uint32_t x = __byte_perm(w[j], got, sel0), y = __byte_perm(w[j + 1], got, sel1);
        if (2 * j < left) *reinterpret_cast<uint32_t*>(q) = x;
        if (2 * j + 2 < left) *reinterpret_cast<uint32_t*>(q + 2 * ldq) = y;
        q += 4 * ldq;
    }
}

constexpr int EPI_BUF = 2048;  // shared memory per epilogue warp: two staged blocks

// `cols` accumulator columns (a multiple of 16) from TMEM address tb, of which the first n exist in
// C: two blocks at a time, the next two loaded while these are stored. have == false: zeros, TMEM
// not read.
__device__ __forceinline__ void store_cols16(uint32_t tb, int cols, uint16_t* c, int64_t ldq, int n,
                                             int pn, float alpha, int type, uint8_t* buf, int lane,
                                             bool have) {
    const int nb = (min(cols, n) + 15) >> 4;  // blocks with anything to store
    const uint32_t sb = smem_u32(buf);
    uint32_t a[16], b[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) a[i] = b[i] = 0u;
    if (have) {
        if (nb > 0) tmem_ld_frag16(tb, a);
        if (nb > 1) tmem_ld_frag16(tb + 16, b);
    }
#pragma unroll 1
    for (int k = 0; k < nb; k += 2) {
        Block16 x, y;
        if (have) {
            tmem_wait_ld();
            frag_fence(a);
            frag_fence(b);
        }
        x.round(a, alpha, type);
        y.round(b, alpha, type);
        if (have) {
            if (k + 2 < nb) tmem_ld_frag16(tb + 16 * (k + 2), a);
            if (k + 3 < nb) tmem_ld_frag16(tb + 16 * (k + 3), b);
        }
        x.stage(sb, lane);
        y.stage(sb + 1024, lane);
        __syncwarp();
        copy_out(sb, c + 16 * k * ldq, ldq, n - 16 * k, pn, lane);
        copy_out(sb + 1024, c + 16 * (k + 1) * ldq, ldq,
                 k + 1 < nb ? n - 16 * (k + 1) : 0, pn, lane);
        __syncwarp();  // the buffers are read before the next blocks are written
    }
}

// Whether C takes that path: 16-bit, P stride 1, every row start 16-byte aligned, the P side a whole
// number of pieces, no beta.
inline bool c_in_pieces(const void* c, int type, int64_t ldq, int64_t ldp, int64_t gsc, int64_t np,
                        float beta) {
    return type != GK_F32 && ldp == 1 && ldq % 8 == 0 && gsc % 8 == 0 && np % 8 == 0 &&
           (reinterpret_cast<uintptr_t>(c) & 15) == 0 && beta == 0.0f;
}

}  // namespace gk
