// gk_fp4.cu -- microscaled 4-bit floats: quantisation, the values back, and the product.
//
// A row is cut into blocks of consecutive elements that share one scale; the elements are e2m1
// (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte, the first in the low nibble.
//   mx  blocks of 32, the scale a power of two (e8m0):   2^(floor(log2 amax) - 2)
//   nv  blocks of 16, the scale e4m3 times a per-matrix f32 scale s:  e4m3(amax / (6 s))
//   element = e2m1(x / (block scale [* s])), ties to even, saturating at 6
// A block that holds an infinity or a NaN gets a NaN scale and zero elements.
//
// Layout. Elements: row-major, rows at a pitch of whole 16-byte pieces. Scales: the order in which
// the tensor cores take them from TMEM. A group of rows is cut into blocks of 128 rows (every
// group starts a new one); per block and 4 consecutive scales one 512-byte atom, the scale j of
// row r at (r % 32) * 16 + (r / 32 % 4) * 4 + j. An atom is copied to TMEM by one tcgen05.cp
// (32 lanes x 16 bytes, replicated to the four lane quarters): column r / 32 then holds the four
// scales of row r in lane r % 32. The atoms of a block follow each other along the row and cover
// a whole number of 256-element stages.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "gemmkit_cuda.h"
#include "gk_engine.h"
#include "gk_group.cuh"
#include "gk_sm100.cuh"
#include "gk_store.cuh"
#include "gk_tc_common.cuh"

namespace gk {

namespace {

constexpr int FBK = 256;  // elements per stage (128 bytes of codes)

template <int FMT>
struct Fp4 {
    static constexpr int BS = FMT == GK_FP4_MX ? 32 : 16;      // elements per scale
    static constexpr int ATOMS = FBK / (4 * BS);               // scale atoms per stage: 2 / 4
    static constexpr int SF_BYTES = ATOMS * 512;               // scales of 128 rows, one stage
};

// ---- conversions -------------------------------------------------------------------------------

// Eight f32 to e2m1 (round to nearest even, saturating), x[0] in the low nibble.
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float (&x)[8]) {
    uint32_t w;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(w)
        : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
    return w;
}

// y = x * m, two products an instruction.
__device__ __forceinline__ void scale8(const float (&x)[8], float m, float (&y)[8]) {
    uint64_t mm;
    asm("mov.b64 %0, {%1, %1};" : "=l"(mm) : "f"(m));
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%2, %3};\n\tmul.rn.f32x2 t, t, %4;\n\t"
            "mov.b64 {%0, %1}, t;\n\t}"
            : "=f"(y[i]), "=f"(y[i + 1])
            : "f"(x[i]), "f"(x[i + 1]), "l"(mm));
}

// Two f32 to e4m3 (round to nearest even, saturating): lo in the low byte.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
    uint16_t h;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(h) : "f"(hi), "f"(lo));
    return h;
}

__device__ __forceinline__ float e4m3_to_float(uint32_t b) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(b & 0xFFu)));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h2 & 0xFFFFu)));
}

// The values of two e2m1 codes (low nibble first).
__device__ __forceinline__ float2 e2m1x2_to_float(uint32_t byte) {
    uint32_t h2;
    asm("{\n\t.reg .b8 lo, hi;\n\tmov.b16 {lo, hi}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, lo;\n\t}"
        : "=r"(h2)
        : "h"(static_cast<uint16_t>(byte)));
    return __half22float2(*reinterpret_cast<const __half2*>(&h2));
}

// 2^(b - 127), b = 255: NaN
__device__ __forceinline__ float e8m0_to_float(uint32_t b) {
    return __uint_as_float(b == 255u ? 0x7FFFFFFFu : b == 0u ? 0x00400000u : b << 23);
}

struct NvScale {
    float s, inv6;  // the matrix scale, and 1 / (6 s) in f32
};

// The nv block scale, exactly: e4m3 of amax / (6 s). f32 gives the quotient within 2^-22; where
// both ends of that interval round alike, so does the exact quotient. Otherwise it lies next to
// the border between two codes, and amax is compared with border * 6 s, which f64 holds exactly
// (the border has 5 significant bits, 6 s has 26). The comparisons are rare and kept out of line:
// inlined eight times over they drove the loop out of the instruction cache.
__device__ __noinline__ uint32_t nv_scale_border(uint32_t lo, uint32_t hi, float amax, float s) {
    const double mid = 0.5 * (static_cast<double>(e4m3_to_float(lo)) + e4m3_to_float(hi));
    const double border = mid * (6.0 * static_cast<double>(s));
    const double a = static_cast<double>(amax);
    return a < border ? lo : a > border ? hi : (lo & 1u) ? hi : lo;
}
__device__ __forceinline__ uint32_t nv_block_scale(float amax, const NvScale& n) {
    const float q = amax * n.inv6;
    const uint32_t two = cvt_e4m3x2(q * (1.0f - 0x1p-21f), q * (1.0f + 0x1p-21f));
    const uint32_t lo = two & 0xFFu, hi = two >> 8;
    return lo == hi ? lo : nv_scale_border(lo, hi, amax, n.s);
}

// Eight elements over d = sb * s, decided exactly: the quotient in f32 within 2^-21 (r is 1 / d
// within 2^-22), and next to a border the sign of |x| - border * d. There d = hi + lo without
// error (sb has 4 significant bits), |x| - border * hi is a difference of near equals, exact in one
// fused step, and border * lo is exact. 16-bit inputs over a matrix scale of few digits meet
// borders often (a value in a hundred with s = 0.01), so only the elements concerned are looked
// at; out of line, to keep the loop in the instruction cache.
__device__ __noinline__ uint32_t nv_element_borders(uint32_t w, uint32_t w2, float x0, float x1,
                                                    float x2, float x3, float x4, float x5,
                                                    float x6, float x7, float sb, float s) {
    const float hi = __fmul_rn(sb, s), lo = __fmaf_rn(sb, s, -hi);
    uint32_t diff = w ^ w2;
    while (diff) {
        const int i = (__ffs(static_cast<int>(diff)) - 1) >> 2;
        diff &= ~(15u << (4 * i));
        const float a0 = i & 1 ? x1 : x0, a1 = i & 1 ? x3 : x2;
        const float a2 = i & 1 ? x5 : x4, a3 = i & 1 ? x7 : x6;
        const float b0 = i & 2 ? a1 : a0, b1 = i & 2 ? a3 : a2;
        const float x = fabsf(i & 4 ? b1 : b0);
        const uint32_t c = (w >> (4 * i)) & 15u, c2 = (w2 >> (4 * i)) & 15u;
        const float2 v = e2m1x2_to_float((c & 7u) | ((c2 & 7u) << 4));
        const float border = 0.5f * (v.x + v.y);
        const float t = __fmaf_rn(-border, hi, x), u = border * lo;
        if (t > u || (t == u && (c & 1u))) w = (w & ~(15u << (4 * i))) | (c2 << (4 * i));
    }
    return w;
}
__device__ __forceinline__ uint32_t nv_elements(const float (&x)[8], float r, float sb, float s) {
    float lo[8], hi[8];
    scale8(x, r * (1.0f - 0x1p-20f), lo);
    scale8(x, r * (1.0f + 0x1p-20f), hi);
    const uint32_t w = cvt_e2m1x8(lo), w2 = cvt_e2m1x8(hi);
    if (w == w2) return w;
    return nv_element_borders(w, w2, x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], sb, s);
}

// The largest magnitude of eight values, as bits (a NaN above every number).
__device__ __forceinline__ uint32_t absmax_bits(const float (&x)[8]) {
    float m;
    asm("{\n\t.reg .f32 a, b;\n\t"
        "max.NaN.abs.f32 a, %1, %2, %3;\n\t"
        "max.NaN.abs.f32 b, %4, %5, %6;\n\t"
        "max.NaN.abs.f32 a, a, %7, %8;\n\t"
        "max.NaN.f32 %0, a, b;\n\t}"
        : "=f"(m)
        : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
    return __float_as_uint(m);
}

__device__ __forceinline__ float fast_rcp(float x) {  // within 1 ulp, normal results
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// ---- where a row lies ----------------------------------------------------------------------------

struct Fp4View {
    uint8_t* data;
    uint8_t* scales;
    int64_t pitch;  // bytes between rows of codes
    int32_t rows, cols, groups, stages;  // stages: 256-element stages per row
    const int32_t* offsets;
    unsigned int* status;
};

// The group tables of a view in shared memory (blocks of 128 rows before each group); a single
// group without offsets needs none.
struct RowMap {
    int off[GROUP_TABLE_INTS];
    int blk[GROUP_TABLE_INTS];
};

__device__ __forceinline__ bool one_group(const Fp4View& v) { return v.groups == 1 && !v.offsets; }

// The 128-row scale block and the row inside it of row r, and r's group and place in the group;
// false for a row of no group.
__device__ __forceinline__ bool find_row(const Fp4View& v, const RowMap& m, int r, int& block,
                                         int& in, int& g, int& at) {
    if (one_group(v)) {
        g = 0;
        at = r;
        block = r >> 7;
        in = r & 127;
        return true;
    }
    if (r < m.off[0] || r >= m.off[v.groups]) return false;
    int lo = 0, hi = v.groups;  // off[lo] <= r < off[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (m.off[mid] <= r)
            lo = mid;
        else
            hi = mid;
    }
    g = lo;
    at = r - m.off[lo];
    block = m.blk[lo] + (at >> 7);
    in = at & 127;
    return true;
}

// Where the scales of row `in` of a 128-row block start; the scale sf lies sf / 4 * 512 + sf % 4 on.
template <int FMT>
__device__ __forceinline__ uint8_t* scale_row(const Fp4View& v, int block, int in) {
    return v.scales + static_cast<int64_t>(block) * v.stages * Fp4<FMT>::SF_BYTES + (in & 31) * 16 +
           (in >> 5) * 4;
}
__device__ __forceinline__ int scale_at(int sf) { return (sf >> 2) * 512 + (sf & 3); }

// ---- quantisation --------------------------------------------------------------------------------

// The kernels below start while the kernel that writes their input may still be running (they wait
// for it before they read), so the input is not read-only for their lifetime: plain loads, no
// read-only path and no __restrict__.

// One block's scale from the largest magnitude's bits (as f32): the scale byte, and what the
// elements are multiplied with.
template <int FMT>
__device__ __forceinline__ uint32_t block_scale(uint32_t amax_bits, const NvScale& nv, float& mul,
                                                float& sb) {
    sb = 0.0f;
    if constexpr (FMT == GK_FP4_MX) {
        const uint32_t e = amax_bits >> 23;
        const uint32_t b = e == 255u ? 255u : e > 2u ? e - 2u : 0u;
        mul = __uint_as_float((254u - b) << 23);  // 2^(127 - b); b <= 252 or 255 (unused then)
        return b;
    } else {
        if (amax_bits >= 0x7F800000u) {
            mul = 0.0f;
            return 0x7Fu;
        }
        const uint32_t b = nv_block_scale(__uint_as_float(amax_bits), nv);
        sb = e4m3_to_float(b);
        mul = b ? fast_rcp(sb * nv.s) : 0.0f;
        return b;
    }
}

template <int FMT>
__device__ __forceinline__ uint32_t block_codes(const float (&x)[8], uint32_t amax_bits, float mul,
                                                float sb, const NvScale& nv) {
    if (amax_bits >= 0x7F800000u) return 0u;
    if constexpr (FMT == GK_FP4_MX) {
        float y[8];
        scale8(x, mul, y);  // a power of two: exact
        return cvt_e2m1x8(y);
    } else {
        return nv_elements(x, mul, sb, nv.s);
    }
}

// E (8 or 16) elements of a row as loaded.
template <typename T, int E>
struct RawRow {
    static constexpr int N = static_cast<int>(sizeof(T)) * 8 / 16;  // pieces of 16 bytes in eight
    uint4 q[N * E / 8];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < N * E / 8; ++i) q[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    // element by element: any stride, zero at or past column `cols`
    __device__ __forceinline__ void load(const T* src, int64_t cs, int k, int cols) {
        T v[E];
#pragma unroll
        for (int i = 0; i < E; ++i)
            v[i] = k + i < cols ? src[static_cast<int64_t>(k + i) * cs] : T(0.0f);
        memcpy(q, v, sizeof(v));
    }
    // elements 8 h .. 8 h + 7
    __device__ __forceinline__ void values(int h, float (&x)[8]) const {
        T v[8];
        memcpy(v, q + h * N, sizeof(v));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f(v[i]);
    }
    static __device__ __forceinline__ float to_f(float v) { return v; }
    static __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
    static __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
};

// A warp takes QU steps of a row, a lane E elements of each: E / 8 stages of 256 elements a step,
// loads of 16 bytes, the block's maximum by shuffles, E / 2 bytes of codes stored. Elements past
// the row are zero, and so are the scales of blocks past it (the product reads whole stages).
//   E is 16 for many 16-bit rows read in whole pieces: the scale's arithmetic, a large part of the
// work in nv, is then done by one lane of a block (nv) or two (mx) instead of two or four.
// 8192 x 8192 of bf16: 31.9 us with 8, 28.3 with 16 (mx), 48.9 and 40.0 (nv). It is 8 for f32,
// where 16 would put a lane's loads 64 bytes from its neighbour's (4096 x 4096 in mx: 8.4 against
// 10.8 us), for rows read element by element (333 x 4099 of f32: 3.7 against 6.7 us), and for a
// few rows, where the longer chain of a lane shows (1 x 4096 in nv: 1.7 against 1.9 us).
//   A unit is 4 stages where that still gives every SM's warps one, so that enough loads are in
// flight, else one: for one row of 4096 more would only follow each other.
template <int FMT, typename T, int E, int QU>
__global__ void __launch_bounds__(256)
    quantize_fp4_kernel(const T* x, int64_t rs, int64_t cs, int64_t gs, int vec, Fp4View v,
                        NvScale nv) {
    __shared__ RowMap map;
    griddep_wait();
    griddep_launch_dependents();
    if (!one_group(v))
        load_groups(v.offsets, v.groups, v.rows, map.off, map.blk,
                    blockIdx.x == 0 ? v.status : nullptr, [](int m) { return (m + 127) >> 7; });
    constexpr int SPW = E / 8;               // stages a step
    constexpr int UNIT = QU * SPW;           // stages of a unit
    constexpr int LPS = 32 / SPW;            // lanes of a stage
    constexpr int LPB = Fp4<FMT>::BS / E;    // lanes of a block
    const int lane = threadIdx.x & 31, in_stage = lane % LPS;
    const uint32_t chunks = static_cast<uint32_t>(v.stages + UNIT - 1) / UNIT;  // of a row
    // units (row, chunk), counted in 64 bits only where 32 do not hold them
    const uint64_t units = static_cast<uint64_t>(v.rows) * chunks;
    const uint32_t step = gridDim.x * (blockDim.x >> 5);
    for (uint64_t u = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += step) {
        const int r = units >> 32 ? static_cast<int>(u / chunks)
                                  : static_cast<int>(static_cast<uint32_t>(u) / chunks);
        // this lane's first stage; its next ones lie SPW on
        const int st0 =
            static_cast<int>(u - static_cast<uint64_t>(r) * chunks) * UNIT + lane / LPS;
        int block, in, g, at;
        if (!find_row(v, map, r, block, in, g, at)) continue;
        // a stack's groups lie gs apart; ragged groups and a single one lie row after row
        const T* src = x + (v.offsets ? static_cast<int64_t>(r) * rs : g * gs + at * rs);
        uint8_t* dst = v.data + static_cast<int64_t>(r) * v.pitch +
                       static_cast<int64_t>(st0) * (FBK / 2) + in_stage * (E / 2);
        uint8_t* sp = scale_row<FMT>(v, block, in) +
                      static_cast<int64_t>(st0) * Fp4<FMT>::SF_BYTES + scale_at(in_stage / LPB);
        const int k0 = st0 * FBK + in_stage * E;
        RawRow<T, E> raw[QU];
        // a whole unit without a branch between its loads, so that they go out together
        if (vec && (st0 - lane / LPS + UNIT) * FBK <= v.cols) {
#pragma unroll
            for (int i = 0; i < QU; ++i) raw[i].load(src + k0 + i * SPW * FBK);
        } else {
#pragma unroll
            for (int i = 0; i < QU; ++i) {
                const int k = k0 + i * SPW * FBK;
                if (vec && k + E <= v.cols)
                    raw[i].load(src + k);
                else
                    raw[i].load(src, cs, k, v.cols);
            }
        }
#pragma unroll
        for (int i = 0; i < QU; ++i) {
            const int st = st0 + i * SPW;
            if (st - lane / LPS >= v.stages) break;
            float e[SPW][8];
            uint32_t m = 0;
#pragma unroll
            for (int h = 0; h < SPW; ++h) {
                raw[i].values(h, e[h]);
                m = max(m, absmax_bits(e[h]));
            }
#pragma unroll
            for (int d = 1; d < LPB; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
            float mul, sb;
            const uint32_t b = block_scale<FMT>(m, nv, mul, sb);
            uint32_t w[SPW];
#pragma unroll
            for (int h = 0; h < SPW; ++h) w[h] = block_codes<FMT>(e[h], m, mul, sb, nv);
            if (st >= v.stages) break;  // the second half's stage may lie past the row
            if (st * (FBK / 2) + in_stage * (E / 2) < v.pitch)
                memcpy(__builtin_assume_aligned(dst + i * SPW * (FBK / 2), sizeof(w)), w, sizeof(w));
            if (in_stage % LPB == 0)
                sp[i * SPW * Fp4<FMT>::SF_BYTES] =
                    static_cast<uint8_t>(st * FBK + in_stage * E < v.cols ? b : 0u);
        }
    }
}

// The values back, in f32: code * block scale (exact) [* s, rounded once]. A warp takes up to QU
// stages of a row; of each half stage a lane reads four codes and writes 16 bytes, so that a
// warp's stores are contiguous.
template <int FMT, int QU>
__global__ void __launch_bounds__(256)
    dequantize_fp4_kernel(Fp4View v, float s, float* out, int64_t rs, int64_t cs,
                          int vec) {
    __shared__ RowMap map;
    griddep_wait();
    griddep_launch_dependents();
    if (!one_group(v))
        load_groups(v.offsets, v.groups, v.rows, map.off, map.blk,
                    blockIdx.x == 0 ? v.status : nullptr, [](int m) { return (m + 127) >> 7; });
    const int lane = threadIdx.x & 31;
    const uint32_t chunks = static_cast<uint32_t>(v.stages + QU - 1) / QU;
    const uint64_t units = static_cast<uint64_t>(v.rows) * chunks;
    const uint32_t step = gridDim.x * (blockDim.x >> 5);
    for (uint64_t u = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += step) {
        const int r = units >> 32 ? static_cast<int>(u / chunks)
                                  : static_cast<int>(static_cast<uint32_t>(u) / chunks);
        const int st0 = static_cast<int>(u - static_cast<uint64_t>(r) * chunks) * QU;
        int block, in, g, at;
        if (!find_row(v, map, r, block, in, g, at)) continue;
        const uint8_t* src = v.data + static_cast<int64_t>(r) * v.pitch +
                             static_cast<int64_t>(st0) * (FBK / 2) + lane * 2;
        const uint8_t* sp = scale_row<FMT>(v, block, in) +
                            static_cast<int64_t>(st0) * Fp4<FMT>::SF_BYTES;
        const int k0 = st0 * FBK + lane * 4;
        uint32_t w[2 * QU], b[2 * QU];
#pragma unroll
        for (int i = 0; i < 2 * QU; ++i) {
            w[i] = b[i] = 0;
            if (k0 + i * 128 < v.cols) {
                w[i] = *reinterpret_cast<const uint16_t*>(src + i * 64);
                b[i] = sp[(i >> 1) * Fp4<FMT>::SF_BYTES +
                          scale_at(((i & 1) * 128 + lane * 4) / Fp4<FMT>::BS)];
            }
        }
        float* dst = out + r * rs + k0 * cs;
#pragma unroll
        for (int i = 0; i < 2 * QU; ++i) {
            const int left = v.cols - k0 - i * 128;  // columns from this lane's first on
            if (left <= 0) break;
            const float sb = FMT == GK_FP4_MX ? e8m0_to_float(b[i]) : e4m3_to_float(b[i]);
            const float2 lo = e2m1x2_to_float(w[i] & 255u), hi = e2m1x2_to_float(w[i] >> 8);
            float y[4] = {lo.x * sb, lo.y * sb, hi.x * sb, hi.y * sb};
            if (FMT != GK_FP4_MX) {
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] *= s;
            }
            float* d = dst + static_cast<int64_t>(i) * 128 * cs;
            if (vec && left >= 4) {
                *reinterpret_cast<float4*>(d) = make_float4(y[0], y[1], y[2], y[3]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < left) d[j * cs] = y[j];
            }
        }
    }
}

// Row-major codes (two a byte) and scales (one byte a block) into the layout above.
template <int FMT>
__global__ void __launch_bounds__(256)
    import_fp4_kernel(const uint8_t* codes, int64_t codes_ld,
                      const uint8_t* scales, int64_t scales_ld, Fp4View v) {
    __shared__ RowMap map;
    griddep_wait();
    if (!one_group(v))
        load_groups(v.offsets, v.groups, v.rows, map.off, map.blk,
                    blockIdx.x == 0 ? v.status : nullptr, [](int m) { return (m + 127) >> 7; });
    const int lane = threadIdx.x & 31;
    const uint32_t stages = static_cast<uint32_t>(v.stages);
    const uint64_t units = static_cast<uint64_t>(v.rows) * stages;
    const uint32_t step = gridDim.x * (blockDim.x >> 5);
    for (uint64_t u = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += step) {
        const int r = units >> 32 ? static_cast<int>(u / stages)
                                  : static_cast<int>(static_cast<uint32_t>(u) / stages);
        const int st = static_cast<int>(u - static_cast<uint64_t>(r) * stages);
        int block, in, g, at;
        if (!find_row(v, map, r, block, in, g, at)) continue;
        const int64_t byte = static_cast<int64_t>(st) * (FBK / 2) + lane * 4;
        if (byte < v.pitch) {
            uint32_t w = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int64_t k = (byte + i) * 2;
                uint32_t c = k < v.cols ? codes[r * codes_ld + byte + i] : 0u;
                if (k + 1 >= v.cols) c &= 15u;
                w |= c << (8 * i);
            }
            *reinterpret_cast<uint32_t*>(v.data + static_cast<int64_t>(r) * v.pitch + byte) = w;
        }
        constexpr int NSF = 4 * Fp4<FMT>::ATOMS;  // scales of a stage
        if (lane < NSF) {
            const int sf = st * NSF + lane;
            const bool in_row = sf * Fp4<FMT>::BS < v.cols;
            scale_row<FMT>(v, block, in)[static_cast<int64_t>(sf >> 2) * 512 + (sf & 3)] =
                in_row ? scales[r * scales_ld + sf] : 0;
        }
    }
}

// ---- the product -----------------------------------------------------------------------------------

struct Fp4GemmParams {
    const uint8_t* psf;       // scales of P (the weights) and Q (the rows of A)
    const uint8_t* qsf;
    int32_t np, npb;          // rows of P in a group, its 128-row scale blocks
    int32_t kdim, stages;     // contraction length, in 256-element stages
    int32_t zero;
    int32_t groups, rows, tiles_p;
    const int32_t* offsets;   // of A's rows (nullptr: equal groups)
    void* c;
    int64_t ldq, ldp;
    float alpha, beta;
    int32_t out_type;
    int32_t pieces;           // C leaves in 16-byte pieces (c_in_pieces)
    uint64_t timeout_ns;
    unsigned int* status;
};

// BN: rows of A per tile. A tile's scales start at a TMEM column of their own only where a 128-row
// scale block starts, so tiles of fewer rows serve calls that have no more rows than that (one
// tile per group); every other call takes tiles of 128 rows.
template <int FMT, int BN>
struct Fp4Cfg {
    static constexpr int NEPI = BN >= 64 ? 8 : 4;
    static constexpr int EPI_W0 = 4;
    static constexpr int THREADS = 32 * (EPI_W0 + NEPI);
    static constexpr int WCOLS = BN / (NEPI / 4);
    static constexpr int SF = Fp4<FMT>::SF_BYTES;
    static constexpr int P_BYTES = BM * BKB;
    static constexpr int Q_BYTES = BN * BKB;
    static constexpr int STAGE_BYTES = P_BYTES + Q_BYTES + 2 * SF;
    static constexpr int TAB_BYTES = (3 * GROUP_TABLE_INTS * 4 + 15) / 16 * 16;
    static constexpr int BAR_BYTES = 512;
    static constexpr int EPI_BYTES = NEPI * EPI_BUF;
    static constexpr int RAW_STAGES =
        (SMEM_LIMIT - 1024 - BAR_BYTES - TAB_BYTES - EPI_BYTES) / STAGE_BYTES;
    // TMEM: two accumulators, then each stage's scales (its own columns: they are free again when
    // the stage is)
    static constexpr int SF_COLS = 2 * 4 * Fp4<FMT>::ATOMS;
    static constexpr int TMEM_STAGES = (512 - 2 * BN) / SF_COLS;
    static constexpr int STAGES0 = RAW_STAGES > 10 ? 10 : RAW_STAGES;
    static constexpr int STAGES = STAGES0 > TMEM_STAGES ? TMEM_STAGES : STAGES0;
    // P | Q | scales of P | scales of Q | barriers | tables
    static constexpr int OFF_Q = STAGES * P_BYTES;
    static constexpr int OFF_SF = OFF_Q + STAGES * Q_BYTES;
    static constexpr int OFF_EPI = OFF_SF + STAGES * 2 * SF;
    static constexpr int OFF_BARS = OFF_EPI + EPI_BYTES;
    static constexpr int OFF_TAB = OFF_BARS + BAR_BYTES;
    static constexpr int SMEM = 1024 + OFF_TAB + TAB_BYTES;
    static constexpr int TMEM_COLS = 512;
    static_assert(BN == 32 || BN == 64 || BN == 128, "tile width");
    static_assert(STAGES >= 2 && SMEM <= SMEM_LIMIT, "shared memory budget");
    static_assert((3 * STAGES + 7) * 8 <= BAR_BYTES, "barrier area");
};

// Instruction descriptor of kind::mxf4 / mxf4nvf4: both operands e2m1 (1 at bits 7 and 10), K-major,
// N >> 3 at bit 17, the scales' type at bit 23 (1 = e8m0), M >> 4 at bit 24. The ids at bits 4
// and 29 pick the bytes of a scale column that an instruction of 64 elements uses: with a
// scale per 32, bytes 0-1 or 2-3 (ids 0, 2); with a scale per 16 all four (id 0).
template <int FMT>
__device__ __forceinline__ uint32_t idesc_fp4(int m, int n, int id) {
    return (static_cast<uint32_t>(id) << 4) | (1u << 7) | (1u << 10) |
           (static_cast<uint32_t>(n >> 3) << 17) | ((FMT == GK_FP4_MX ? 1u : 0u) << 23) |
           (static_cast<uint32_t>(m >> 4) << 24) | (static_cast<uint32_t>(id) << 29);
}

template <int FMT>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc,
                                        uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (FMT == GK_FP4_MX)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], "
            "[%5], p;\n\t}" ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb),
            "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, "
            "[%4], [%5], p;\n\t}" ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb),
            "r"(accumulate)
            : "memory");
}

// The descriptor of a 512-byte scale atom: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes
// apart.
__device__ __forceinline__ uint64_t sdesc_scales(uint32_t saddr) {
    return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) |
           (static_cast<uint64_t>(128u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46);
}

// One scale atom to four TMEM columns, replicated to the four lane quarters. Executes in order
// with the later MMAs of this thread.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
                 : "memory");
}

template <int FMT, int BN>
__global__ void __launch_bounds__(Fp4Cfg<FMT, BN>::THREADS, 1)
    fp4_gemm_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                    const Fp4GemmParams p) {
    using C = Fp4Cfg<FMT, BN>;
    constexpr int STAGES = C::STAGES;
    constexpr int ATOMS = Fp4<FMT>::ATOMS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* sP = smem;
    uint8_t* sQ = smem + C::OFF_Q;
    uint8_t* sSF = smem + C::OFF_SF;  // per stage: P's scales, then Q's
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BARS);
    uint64_t* empty = full + STAGES;
    uint64_t* sfull = empty + STAGES;  // a stage's scales are in TMEM
    uint64_t* tfull = sfull + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* off = reinterpret_cast<int*>(smem + C::OFF_TAB);
    int* tile0 = off + GROUP_TABLE_INTS;
    int* qblk = tile0 + GROUP_TABLE_INTS;  // scale blocks of Q before each group

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t tmo = p.timeout_ns;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
            mbar_init(&sfull[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], C::NEPI);
        }
        mbar_init(drain, 1);
        mbar_init(drain + 1, 1);
        *abort_flag = 0;
        fence_mbar_init();
        if (!p.zero) {
            prefetch_tmap(&tmP);
            prefetch_tmap(&tmQ);
        }
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, C::TMEM_COLS);
        tmem_relinquish();
    }
    griddep_wait();
    load_groups(p.offsets, p.groups, p.rows, off, qblk, blockIdx.x == 0 ? p.status : nullptr,
                [](int m) { return (m + 127) >> 7; });
    if (warp == 0)
        sum_groups(off, p.groups, tile0, [&](int m) { return (m + BN - 1) / BN * p.tiles_p; });
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    GroupWalk walk(off, tile0, p.groups, blockIdx.x, gridDim.x);
    int tp, tq;

    if (warp == 0) {
        // ---------------- producer (the whole warp, one lane issues) ----------------
        int stage = 0;
        uint32_t phase = 0, issued = 0, last_par = 0;
        bool ok = true;
        while (ok && walk.next(p.tiles_p, tp, tq)) {
            const int g = walk.g, q0 = tq * BN;
            const int64_t pb = static_cast<int64_t>(g) * p.npb + tp;
            const int64_t qb = static_cast<int64_t>(qblk[g]) + (q0 >> 7);
            const int prow = g * p.np + tp * BM, qrow = off[g] + q0;
            const int ns = p.zero ? 0 : p.stages;
            const uint8_t* ps = p.psf + pb * p.stages * C::SF;
            const uint8_t* qs = p.qsf + qb * p.stages * C::SF;
            for (int kb = 0; kb < ns; ++kb) {
                if (!warp_wait(&empty[stage], phase ^ 1u, abort_flag, p.status,
                               GK_DEV_TIMEOUT_PRODUCER, tmo)) {
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    uint64_t* fb = &full[stage];
                    mbar_arrive_expect_tx(fb, C::STAGE_BYTES);
                    tma_load_3d(sP + stage * C::P_BYTES, &tmP, fb, kb * (FBK / 4), prow, 0);
                    tma_load_3d(sQ + stage * C::Q_BYTES, &tmQ, fb, kb * (FBK / 4), qrow, 0);
                    uint8_t* sf = sSF + stage * 2 * C::SF;
                    bulk_load(sf, ps + static_cast<int64_t>(kb) * C::SF, C::SF, fb);
                    bulk_load(sf + C::SF, qs + static_cast<int64_t>(kb) * C::SF, C::SF, fb);
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
        int dummy = 0;
        for (int s = 0; s < STAGES; ++s)
            if (issued & (1u << s))
                mbar_wait(&full[s], (last_par >> s) & 1u, &dummy, p.status, GK_DEV_TIMEOUT_DRAIN,
                          tmo);
    } else if (warp == 1) {
        // ---------------- MMA issuer (the whole warp, one lane issues) ----------------
        const uint64_t dP = sdesc_kmajor_sw128(smem_u32(sP));
        const uint64_t dQ = sdesc_kmajor_sw128(smem_u32(sQ));
        constexpr uint32_t idesc_id2 = (2u << 4) | (2u << 29);  // both scale ids 2
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int local = 0; ok && walk.next(p.tiles_p, tp, tq); ++local) {
            const int acc = local & 1;
            const uint32_t aph = (local >> 1) & 1;
            if (!warp_wait(&tempty[acc], aph ^ 1u, abort_flag, p.status, GK_DEV_TIMEOUT_MMA, tmo))
                break;
            tc_fence_after();
            const int q0 = tq * BN, qn = off[walk.g + 1] - off[walk.g] - q0;
            const uint32_t idesc = idesc_fp4<FMT>(BM, min(BN, (qn + 15) & ~15), 0);
            const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
            const int ns = p.zero ? 0 : p.stages;
            for (int kb = 0; kb < ns; ++kb) {
                if (!warp_wait(&sfull[stage], phase, abort_flag, p.status, GK_DEV_TIMEOUT_MMA, tmo) ||
                    !warp_wait(&full[stage], phase, abort_flag, p.status, GK_DEV_TIMEOUT_MMA, tmo)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t tsf = tmem_base + static_cast<uint32_t>(2 * BN + stage * C::SF_COLS);
                const uint64_t ad = dP + ((stage * C::P_BYTES) >> 4);
                const uint64_t bd = dQ + ((stage * C::Q_BYTES) >> 4);
                // slice ks: 64 elements = 32 bytes; its scales
                auto slice = [&](int ks) {
                    const int atom = FMT == GK_FP4_MX ? ks >> 1 : ks;
                    mma_fp4<FMT>(d, ad + ks * 2, bd + ks * 2,
                                 idesc + (FMT == GK_FP4_MX ? (ks & 1) * idesc_id2 : 0u),
                                 tsf + 4 * atom, tsf + 4 * (ATOMS + atom), (kb | ks) != 0 ? 1u : 0u);
                };
                const int steps = (p.kdim - kb * FBK + 63) >> 6;
                if (elect_one()) {
                    if (steps >= 4) {
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) slice(ks);
                    } else {
#pragma unroll
                        for (int ks = 0; ks < 3; ++ks)
                            if (ks < steps) slice(ks);
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
        if (elect_one()) mma_commit(drain);
        __syncwarp();
        int dummy = 0;
        mbar_wait(drain, 0, &dummy, p.status, GK_DEV_TIMEOUT_DRAIN, tmo);
    } else if (warp == 2) {
        // ---------------- scales to TMEM ----------------
        // A stage's columns are its own: they are free when its shared memory was, which the
        // producer waited for before it filled the stage again.
        const uint64_t dS = sdesc_scales(smem_u32(sSF));
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        while (ok && walk.next(p.tiles_p, tp, tq)) {
            const int ns = p.zero ? 0 : p.stages;
            for (int kb = 0; kb < ns; ++kb) {
                if (!warp_wait(&full[stage], phase, abort_flag, p.status, GK_DEV_TIMEOUT_MMA, tmo)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint64_t sd = dS + ((stage * 2 * C::SF) >> 4);
                const uint32_t tsf = tmem_base + static_cast<uint32_t>(2 * BN + stage * C::SF_COLS);
                if (elect_one()) {
#pragma unroll
                    for (int a = 0; a < 2 * ATOMS; ++a) copy_scales(tsf + 4 * a, sd + 32 * a);
                    mma_commit(&sfull[stage]);
                }
                __syncwarp();
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        if (elect_one()) mma_commit(drain + 1);
        __syncwarp();
        int dummy = 0;
        mbar_wait(drain + 1, 0, &dummy, p.status, GK_DEV_TIMEOUT_DRAIN, tmo);
    } else if (warp >= C::EPI_W0) {
        // ---------------- epilogue ----------------
        const int q = warp & 3;
        const int cbase = ((warp - C::EPI_W0) >> 2) * C::WCOLS;
        uint8_t* ebuf = smem + C::OFF_EPI + (warp - C::EPI_W0) * EPI_BUF;
        for (int local = 0; walk.next(p.tiles_p, tp, tq); ++local) {
            const int acc = local & 1;
            const uint32_t aph = (local >> 1) & 1;
            if (!warp_wait(&tfull[acc], aph, abort_flag, p.status, GK_DEV_TIMEOUT_EPILOGUE, tmo))
                break;
            tc_fence_after();
            const int q0 = tq * BN, qn = off[walk.g + 1] - off[walk.g] - q0;
            const int i0 = tp * BM + q * 32;  // the warp's first P row
            const int64_t at = (static_cast<int64_t>(off[walk.g]) + q0) * p.ldq + i0 * p.ldp;
            const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                                static_cast<uint32_t>(acc * BN + cbase);
            const bool have = !p.zero;
            const int pn = min(32, p.np - i0);
            if (p.pieces) {
                store_cols16(tb, C::WCOLS, static_cast<uint16_t*>(p.c) + at + cbase * p.ldq, p.ldq,
                             qn - cbase, pn, p.alpha, p.out_type, ebuf, lane, have);
            } else {
                for (int c = 0; c < C::WCOLS && cbase + c < qn; c += 32) {
                    uint32_t v[32];
                    if (have) {
                        tmem_ld_x32(tb + c, v);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) v[e] = 0u;
                    }
                    if (lane < pn)
                        store_any(p.c, p.out_type, at + lane * p.ldp + (cbase + c) * p.ldq, p.ldq, v,
                                  qn - cbase - c, p.alpha, p.beta);
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

// ---- the CTA-pair form -----------------------------------------------------------------------------
//
// Two CTAs compute 256 P rows x up to 256 Q rows with cta_group::2, each loading its 128 rows of P
// and half of the Q rows (an SM then takes in 64 bytes of operands per cycle of MMA; the 128 x 128
// tile of the kernel above takes 128, all that shared memory gives). Each SM computes its 128
// rows times all Q rows, so both hold all of Q's scales.
//
// TMEM. Two 256-column accumulators and the scales need more than 512 columns, so the accumulators
// overlap by OVER columns: accumulator 0 is columns [0, 256), accumulator 1 [256 - OVER, 512 -
// OVER), the scales lie in the last OVER columns. The epilogue reads the shared columns first and
// hands them over (thead) before it stores anything; the next tile's MMAs wait for that, not for
// the rest. The scales have SLOTS slots; a slot is refilled once the MMAs of the stage that used it
// last have finished (their commit on empty[]). Warps 2 and 3 copy the scales to TMEM ahead of
// the MMA warp: issued between the MMAs by the same thread, the 12 (nv) or 6 (mx) copies of a
// stage took MMA issue time.

template <int FMT>
struct Fp4PairCfg {
    static constexpr int BN = 256;
    static constexpr int NEPI = 8;
    static constexpr int EPI_W0 = 4;
    static constexpr int THREADS = 32 * (EPI_W0 + NEPI);
    static constexpr int ATOMS = Fp4<FMT>::ATOMS;
    static constexpr int SF = Fp4<FMT>::SF_BYTES;
    static constexpr int P_BYTES = BM * BKB;
    static constexpr int Q_BYTES = BN / 2 * BKB;
    static constexpr int SF_STAGE = 3 * SF;  // P's block, Q's two blocks
    static constexpr int STAGE_BYTES = P_BYTES + Q_BYTES + SF_STAGE;
    static constexpr int TAB_BYTES = (3 * GROUP_TABLE_INTS * 4 + 15) / 16 * 16;
    static constexpr int BAR_BYTES = 256;
    static constexpr int EPI_BYTES = NEPI * EPI_BUF;
    static constexpr int STAGES =
        (SMEM_LIMIT - 1024 - BAR_BYTES - TAB_BYTES - EPI_BYTES) / STAGE_BYTES;
    static constexpr int OFF_Q = STAGES * P_BYTES;
    static constexpr int OFF_SF = OFF_Q + STAGES * Q_BYTES;
    static constexpr int OFF_EPI = OFF_SF + STAGES * SF_STAGE;
    static constexpr int OFF_BARS = OFF_EPI + EPI_BYTES;
    static constexpr int OFF_TAB = OFF_BARS + BAR_BYTES;
    static constexpr int SMEM = 1024 + OFF_TAB + TAB_BYTES;
    static constexpr int OVER = FMT == GK_FP4_MX ? 96 : 160;
    static constexpr int SF_COLS = 12 * ATOMS;         // 4 of P, 8 of Q per atom
    static constexpr int SLOTS = OVER / SF_COLS;       // mx 4, nv 3
    static constexpr int SF_COL0 = 512 - OVER;
    static_assert(SLOTS >= 2 && SLOTS <= STAGES && OVER % 32 == 0, "TMEM budget");
    static_assert((2 * STAGES + SLOTS + 11) * 8 <= BAR_BYTES && SMEM <= SMEM_LIMIT,
                  "shared memory budget");
};

template <int FMT>
__device__ __forceinline__ void mma_fp4_pair(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc,
                                             uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (FMT == GK_FP4_MX)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], "
            "[%5], p;\n\t}" ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb),
            "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, "
            "[%4], [%5], p;\n\t}" ::"r"(d), "l"(ad), "l"(bd), "r"(idesc), "r"(sfa), "r"(sfb),
            "r"(accumulate)
            : "memory");
}

// copy_scales in both CTAs of the pair, each from its own shared memory to its own TMEM.
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
                 : "memory");
}

template <int FMT>
__global__ void __launch_bounds__(Fp4PairCfg<FMT>::THREADS, 1)
    fp4_pair_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                    const __grid_constant__ CUtensorMap tmPS,
                    const __grid_constant__ CUtensorMap tmQS, const Fp4GemmParams p) {
    using C = Fp4PairCfg<FMT>;
    constexpr int STAGES = C::STAGES, BN = C::BN, ATOMS = C::ATOMS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* sP = smem;
    uint8_t* sQ = smem + C::OFF_Q;
    uint8_t* sSF = smem + C::OFF_SF;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BARS);
    uint64_t* empty = full + STAGES;
    uint64_t* tfull = empty + STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* thead = tempty + 2;
    uint64_t* sfull = thead + 2;  // a slot's scales are in TMEM
    uint64_t* drain = sfull + C::SLOTS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 3);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* off = reinterpret_cast<int*>(smem + C::OFF_TAB);
    int* tile0 = off + GROUP_TABLE_INTS;
    int* qblk = tile0 + GROUP_TABLE_INTS;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const uint64_t tmo = p.timeout_ns;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&tfull[a], 1);
            mbar_init(&tempty[a], 2 * C::NEPI);
            mbar_init(&thead[a], 2 * C::NEPI);
        }
        for (int s = 0; s < C::SLOTS; ++s) mbar_init(&sfull[s], 1);
        mbar_init(drain, 1);
        mbar_init(drain + 1, 1);
        mbar_init(drain + 2, 1);
        *abort_flag = 0;
        fence_mbar_init();
        prefetch_tmap(&tmP);
        prefetch_tmap(&tmQ);
        prefetch_tmap(&tmPS);
        prefetch_tmap(&tmQS);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512);
        tmem_relinquish_pair();
    }
    griddep_wait();
    load_groups(p.offsets, p.groups, p.rows, off, qblk, blockIdx.x == 0 ? p.status : nullptr,
                [](int m) { return (m + 127) >> 7; });
    if (warp == 0)
        sum_groups(off, p.groups, tile0, [&](int m) { return (m + BN - 1) / BN * p.tiles_p; });
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t full_l = mapa_shared(smem_u32(&full[0]), 0);
    const uint32_t tempty_l = mapa_shared(smem_u32(&tempty[0]), 0);
    const uint32_t thead_l = mapa_shared(smem_u32(&thead[0]), 0);
    GroupWalk walk(off, tile0, p.groups, blockIdx.x >> 1, gridDim.x >> 1);
    int tp, tq;

    if (warp == 0) {
        // ---------------- producer (both CTAs; the whole warp, one lane issues) ----------------
        int stage = 0;
        uint32_t phase = 0, issued = 0, last_par = 0;
        bool ok = true;
        while (ok && walk.next(p.tiles_p, tp, tq)) {
            const int g = walk.g, q0 = tq * BN;
            const int qn = off[g + 1] - off[g] - q0;
            const int half = min(BN, (qn + 31) & ~31) >> 1;  // Q rows of each CTA
            const int prow = g * p.np + tp * 2 * BM + static_cast<int>(rank) * BM;
            const int qrow = off[g] + q0 + static_cast<int>(rank) * half;
            // one stage of a 128-row scale block is SL lines of the scale maps (blocks that do
            // not exist belong to rows that are not stored)
            constexpr int SL = C::SF / 1024;
            const int pb = g * p.npb + tp * 2 + static_cast<int>(rank);
            const int qb = qblk[g] + (q0 >> 7);
            for (int kb = 0; kb < p.stages; ++kb) {
                if (!warp_wait(&empty[stage], phase ^ 1u, abort_flag, p.status,
                               GK_DEV_TIMEOUT_PRODUCER, tmo)) {
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    const uint32_t fb = full_l + 8u * stage;
                    if (leader) mbar_arrive_expect_tx(&full[stage], 2 * C::STAGE_BYTES);
                    uint8_t* sf = sSF + stage * C::SF_STAGE;
                    tma_load_3d_pair(sP + stage * C::P_BYTES, &tmP, fb, kb * (FBK / 4), prow, 0);
                    tma_load_3d_pair(sQ + stage * C::Q_BYTES, &tmQ, fb, kb * (FBK / 4), qrow, 0);
                    tma_load_3d_pair(sf, &tmPS, fb, 0, kb * SL, pb);
                    tma_load_3d_pair(sf + C::SF, &tmQS, fb, 0, kb * SL, qb);
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
        if (leader) {
            int dummy = 0;
            for (int s = 0; s < STAGES; ++s)
                if (issued & (1u << s))
                    mbar_wait(&full[s], (last_par >> s) & 1u, &dummy, p.status,
                              GK_DEV_TIMEOUT_DRAIN, tmo);
        }
    } else if (warp == 1) {
        if (leader) {
            // ---------------- MMA issuer (leader; the whole warp, one lane issues) ----------------
            const uint64_t dP = sdesc_kmajor_sw128(smem_u32(sP));
            const uint64_t dQ = sdesc_kmajor_sw128(smem_u32(sQ));
            constexpr uint32_t idesc_id2 = (2u << 4) | (2u << 29);
            int stage = 0, slot = 0;
            uint32_t phase = 0, slot_phase = 0;
            bool ok = true;
            for (int local = 0; ok && walk.next(p.tiles_p, tp, tq); ++local) {
                const int acc = local & 1;
                if (!warp_wait(&tempty[acc], ((local >> 1) & 1) ^ 1u, abort_flag, p.status,
                               GK_DEV_TIMEOUT_MMA, tmo) ||
                    (local > 0 && !warp_wait(&thead[acc ^ 1], ((local - 1) >> 1) & 1, abort_flag,
                                             p.status, GK_DEV_TIMEOUT_MMA, tmo)))
                    break;
                tc_fence_after();
                const int qn = off[walk.g + 1] - off[walk.g] - tq * BN;
                const uint32_t idesc = idesc_fp4<FMT>(2 * BM, min(BN, (qn + 31) & ~31), 0);
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc * (BN - C::OVER));
                for (int kb = 0; kb < p.stages; ++kb) {
                    if (!warp_wait(&sfull[slot], slot_phase, abort_flag, p.status,
                                   GK_DEV_TIMEOUT_MMA, tmo) ||
                        !warp_wait(&full[stage], phase, abort_flag, p.status, GK_DEV_TIMEOUT_MMA,
                                   tmo)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t tsf =
                        tmem_base + static_cast<uint32_t>(C::SF_COL0 + slot * C::SF_COLS);
                    const uint64_t ad = dP + ((stage * C::P_BYTES) >> 4);
                    const uint64_t bd = dQ + ((stage * C::Q_BYTES) >> 4);
                    auto slice = [&](int ks) {
                        const int atom = FMT == GK_FP4_MX ? ks >> 1 : ks;
                        mma_fp4_pair<FMT>(d, ad + ks * 2, bd + ks * 2,
                                          idesc + (FMT == GK_FP4_MX ? (ks & 1) * idesc_id2 : 0u),
                                          tsf + 4 * atom, tsf + 4 * ATOMS + 8 * atom,
                                          (kb | ks) != 0 ? 1u : 0u);
                    };
                    const int steps = (p.kdim - kb * FBK + 63) >> 6;
                    if (elect_one()) {
                        if (steps >= 4) {
#pragma unroll
                            for (int ks = 0; ks < 4; ++ks) slice(ks);
                        } else {
#pragma unroll
                            for (int ks = 0; ks < 3; ++ks)
                                if (ks < steps) slice(ks);
                        }
                        mma_commit_pair_both(smem_u32(&empty[stage]), 0x3);
                    }
                    __syncwarp();
                    if (++slot == C::SLOTS) {
                        slot = 0;
                        slot_phase ^= 1u;
                    }
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                if (elect_one()) mma_commit_pair_both(smem_u32(&tfull[acc]), 0x3);
                __syncwarp();
            }
            if (elect_one()) mma_commit_pair(mapa_shared(smem_u32(drain), rank));
            __syncwarp();
            int dummy = 0;
            mbar_wait(drain, 0, &dummy, p.status, GK_DEV_TIMEOUT_DRAIN, tmo);
        }
    } else if (warp == 2 || warp == 3) {
        if (leader) {
            // ---------------- scales to TMEM (leader, for both CTAs) ----------------
            // warp 2 takes the even stages of the ring's order, warp 3 the odd ones
            const uint64_t dS = sdesc_scales(smem_u32(sSF));
            uint64_t* done = drain + (warp - 1);
            int stage = 0, slot = 0, oldest = 0;  // oldest: the stage that used `slot` last
            uint32_t phase = 0, oldest_phase = 0, count = 0;
            bool ok = true;
            while (ok && walk.next(p.tiles_p, tp, tq)) {
                for (int kb = 0; kb < p.stages; ++kb, ++count) {
                    if ((count & 1u) == static_cast<uint32_t>(warp - 2)) {
                        // the MMAs of the slot's last user have finished
                        if ((count >= C::SLOTS &&
                             !warp_wait(&empty[oldest], oldest_phase, abort_flag, p.status,
                                        GK_DEV_TIMEOUT_MMA, tmo)) ||
                            !warp_wait(&full[stage], phase, abort_flag, p.status,
                                       GK_DEV_TIMEOUT_MMA, tmo)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t tsf =
                            tmem_base + static_cast<uint32_t>(C::SF_COL0 + slot * C::SF_COLS);
                        const uint64_t sd = dS + ((stage * C::SF_STAGE) >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int a = 0; a < ATOMS; ++a) {
                                copy_scales_pair(tsf + 4 * a, sd + a * 32);
                                copy_scales_pair(tsf + 4 * ATOMS + 8 * a,
                                                 sd + ((C::SF >> 4) + a * 32));
                                copy_scales_pair(tsf + 4 * ATOMS + 8 * a + 4,
                                                 sd + ((2 * C::SF >> 4) + a * 32));
                            }
                            mma_commit_pair(mapa_shared(smem_u32(&sfull[slot]), 0));
                        }
                        __syncwarp();
                    }
                    if (count >= C::SLOTS && ++oldest == STAGES) {
                        oldest = 0;
                        oldest_phase ^= 1u;
                    }
                    if (++slot == C::SLOTS) slot = 0;
                    if (++stage == STAGES) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (elect_one()) mma_commit_pair(mapa_shared(smem_u32(done), 0));
            __syncwarp();
            int dummy = 0;
            mbar_wait(done, 0, &dummy, p.status, GK_DEV_TIMEOUT_DRAIN, tmo);
        }
    } else if (warp >= C::EPI_W0) {
        // ---------------- epilogue (both CTAs) ----------------
        const int q = warp & 3;
        const int h = (warp - C::EPI_W0) >> 2;  // which half of the columns
        uint8_t* ebuf = smem + C::OFF_EPI + (warp - C::EPI_W0) * EPI_BUF;
        constexpr int HO = C::OVER / 2, HR = (BN - C::OVER) / 2;  // shared, other columns per warp
        static_assert(HO % 16 == 0 && HR % 16 == 0, "chunks of 16 columns");
        for (int local = 0; walk.next(p.tiles_p, tp, tq); ++local) {
            const int acc = local & 1;
            const uint32_t aph = (local >> 1) & 1;
            if (!warp_wait(&tfull[acc], aph, abort_flag, p.status, GK_DEV_TIMEOUT_EPILOGUE, tmo))
                break;
            tc_fence_after();
            const int q0 = tq * BN, qn = off[walk.g + 1] - off[walk.g] - q0;
            const int i0 = (tp * 2 + static_cast<int>(rank)) * BM + q * 32;  // its first P row
            const int64_t at = (static_cast<int64_t>(off[walk.g]) + q0) * p.ldq + i0 * p.ldp;
            const uint32_t tb = tmem_base + (static_cast<uint32_t>(q * 32) << 16) +
                                static_cast<uint32_t>(acc * (BN - C::OVER));
            const int pn = min(32, p.np - i0);
            // first the columns that the next accumulator shares: accumulator 0's last, 1's first
            const int s0 = (acc ? 0 : BN - C::OVER) + h * HO;
            const int r0 = (acc ? C::OVER : 0) + h * HR;
            auto shared_read = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(thead_l + 8u * acc);
            };
            if (p.pieces) {
                uint16_t* c = static_cast<uint16_t*>(p.c) + at;
                uint32_t v[HO / 16][16];
#pragma unroll
                for (int k = 0; k < HO / 16; ++k) tmem_ld_frag16(tb + s0 + 16 * k, v[k]);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < HO / 16; ++k) frag_fence(v[k]);
                shared_read();
#pragma unroll
                for (int k = 0; k < HO / 16; ++k) {
                    const int j = s0 + 16 * k;
                    if (j >= qn) continue;
                    const uint32_t sb = smem_u32(ebuf) + (k & 1) * 1024;
                    Block16 x;
                    x.round(v[k], p.alpha, p.out_type);
                    x.stage(sb, lane);
                    __syncwarp();
                    copy_out(sb, c + j * p.ldq, p.ldq, qn - j, pn, lane);
                }
                __syncwarp();
                store_cols16(tb + r0, HR, c + r0 * p.ldq, p.ldq, qn - r0, pn, p.alpha, p.out_type,
                             ebuf, lane, true);
            } else {
                const int64_t al = at + lane * p.ldp;
                uint32_t v[HO / 16][32];
#pragma unroll
                for (int k = 0; k < HO / 16; ++k) tmem_ld_chunk<16>(tb + s0 + 16 * k, v[k]);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < HO / 16; ++k) reg_fence<16>(v[k]);
                shared_read();
                if (lane < pn) {
#pragma unroll
                    for (int k = 0; k < HO / 16; ++k) {
                        const int j = s0 + 16 * k;
                        if (j < qn)
                            store_any<16>(p.c, p.out_type, al + j * p.ldq, p.ldq, v[k], qn - j,
                                          p.alpha, p.beta);
                    }
                }
                __syncwarp();
#pragma unroll 1
                for (int k = 0; k < HR && r0 + k < qn; k += 16) {
                    tmem_ld_x16(tb + r0 + k, v[0]);
                    if (lane < pn)
                        store_any<16>(p.c, p.out_type, al + (r0 + k) * p.ldq, p.ldq, v[0],
                                      qn - r0 - k, p.alpha, p.beta);
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster_relaxed(tempty_l + 8u * acc);
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512);
    }
}

// ---- host side ---------------------------------------------------------------------------------------

int64_t fp4_pitch(int64_t cols) { return ((cols + 1) / 2 + 15) / 16 * 16; }
int64_t fp4_stages(int64_t cols) { return (cols + FBK - 1) / FBK; }
int fp4_sf_bytes(int fmt) { return fmt == GK_FP4_MX ? Fp4<GK_FP4_MX>::SF_BYTES : Fp4<GK_FP4_NV>::SF_BYTES; }

// The checks of a 4-bit matrix; `name` in the messages.
int check_fp4(const gk_fp4_matrix* q, const char* name) {
    if (!q) return api_err(GK_EINVAL, "gemmkit: null 4-bit matrix %s", name);
    if (q->fmt != GK_FP4_MX && q->fmt != GK_FP4_NV)
        return api_err(GK_EINVAL, "gemmkit: %s: unknown 4-bit format %d", name, q->fmt);
    if (q->groups < 1 || q->groups > MAX_GROUPS)
        return api_err(GK_EINVAL, "gemmkit: %s: 1 to %d groups (groups = %zu)", name, MAX_GROUPS,
                       q->groups);
    if (q->rows > INT32_MAX / 2 || q->cols > INT32_MAX / 2)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    if (!q->offsets && q->rows % q->groups)
        return api_err(GK_EINVAL, "gemmkit: %s: %zu rows do not split into %zu equal groups", name,
                       q->rows, q->groups);
    // 2^-100 .. 2^100 keeps every quotient and product of the scales inside f32
    if (!(q->scale >= 0x1p-100f && q->scale <= 0x1p100f) || (q->fmt == GK_FP4_MX && q->scale != 1.0f))
        return api_err(GK_EINVAL, q->fmt == GK_FP4_MX
                                      ? "gemmkit: %s: the mx format has no matrix scale (must be 1)"
                                      : "gemmkit: %s: the matrix scale must lie in [2^-100, 2^100]",
                       name);
    if (int rc = api_check_aligned(q->offsets, 4, "offsets")) return rc;
    if (q->rows == 0 || q->cols == 0) return GK_OK;
    if (!q->data || !q->scales) return api_err(GK_EINVAL, "gemmkit: %s: null data or scales", name);
    if ((reinterpret_cast<uintptr_t>(q->data) | reinterpret_cast<uintptr_t>(q->scales)) & 15)
        return api_err(GK_EINVAL, "gemmkit: %s: data and scales must be 16-byte aligned", name);
    const size_t nd = gk_fp4_data_bytes(q->rows, q->cols);
    const size_t ns = gk_fp4_scale_bytes(q->fmt, q->groups, q->offsets != nullptr, q->rows, q->cols);
    if (q->data_len < nd || q->scales_len < ns)
        return api_err(GK_EINVAL,
                       "gemmkit: %s: %zux%zu in 4 bits needs %zu bytes of data and %zu of scales "
                       "(has %zu and %zu)",
                       name, q->rows, q->cols, nd, ns, q->data_len, q->scales_len);
    return GK_OK;
}

Fp4View view_of(const gk_fp4_matrix* q) {
    Fp4View v;
    memset(&v, 0, sizeof(v));
    v.data = q->data;
    v.scales = q->scales;
    v.pitch = fp4_pitch(static_cast<int64_t>(q->cols));
    v.rows = static_cast<int>(q->rows);
    v.cols = static_cast<int>(q->cols);
    v.groups = static_cast<int>(q->groups);
    v.stages = static_cast<int>(fp4_stages(static_cast<int64_t>(q->cols)));
    v.offsets = q->offsets;
    v.status = device_status_ptr();
    return v;
}

// A launch that may start while the previous kernel of the stream drains (the kernels wait for it
// before they touch memory).
template <typename... Args>
int launch_overlapped(int cluster, void (*kern)(Args...), int grid, int threads, size_t smem, cudaStream_t st,
                      Args... args) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (api_pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess)
        return api_err(GK_ECUDA, "gemmkit: 4-bit kernel launch failed: %s", cudaGetErrorString(e));
    return GK_OK;
}

// Blocks of 8 warps for `units` warp-sized units: up to 8 resident blocks on every SM.
int unit_grid(int64_t units) {
    const int64_t b = (units + 7) / 8, most = static_cast<int64_t>(sm_count()) * 8;
    return static_cast<int>(b < most ? b : most);
}

// Whether four stages per warp still give every SM 32 warps.
bool large_view(const Fp4View& v) {
    return static_cast<int64_t>(v.rows) * v.stages >= 4 * 32 * static_cast<int64_t>(sm_count());
}

template <int FMT, int BN>
int launch_fp4_gemm(const CUtensorMap& tp, const CUtensorMap& tq, const Fp4GemmParams& p, int grid,
                    cudaStream_t st) {
    using C = Fp4Cfg<FMT, BN>;
    auto kern = fp4_gemm_kernel<FMT, BN>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(kern, C::SMEM, done);
    if (e != cudaSuccess)
        return api_err(GK_ECUDA, "gemmkit: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    return launch_overlapped<CUtensorMap, CUtensorMap, Fp4GemmParams>(
        1, kern, grid, C::THREADS, C::SMEM, st, tp, tq, p);
}

// Clusters of the pair kernel that are resident at once on the current device (0 on failure).
template <int FMT>
int fp4_pair_clusters() {
    using C = Fp4PairCfg<FMT>;
    static PerDevice<int> cache;
    int dev = 0;
    cudaGetDevice(&dev);
    return cache.get(dev, [] {
        cudaLaunchConfig_t q;
        memset(&q, 0, sizeof(q));
        q.gridDim = dim3(static_cast<unsigned>(sm_count() / 2 * 2));
        q.blockDim = dim3(C::THREADS);
        q.dynamicSmemBytes = C::SMEM;
        cudaLaunchAttribute a[1];
        a[0].id = cudaLaunchAttributeClusterDimension;
        a[0].val.clusterDim.x = 2;
        a[0].val.clusterDim.y = 1;
        a[0].val.clusterDim.z = 1;
        q.attrs = a;
        q.numAttrs = 1;
        int c = 0;
        if (cudaFuncSetAttribute(fp4_pair_kernel<FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 C::SMEM) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&c, fp4_pair_kernel<FMT>, &q) != cudaSuccess || c <= 0) {
            cudaGetLastError();
            c = sm_count() / 2;
        }
        return c;
    });
}

template <int FMT>
int run_fp4_gemm(Fp4GemmParams p, const gk_fp4_matrix* a, const gk_fp4_matrix* b, cudaStream_t st) {
    // an upper bound of the tiles (the device computes the true number from the offsets)
    auto tiles_bound = [&](int64_t tm, int64_t bn) {
        return (p.np + tm - 1) / tm * ((static_cast<int64_t>(p.rows) + bn - 1) / bn + p.groups);
    };
    const int64_t mean = (static_cast<int64_t>(p.rows) + p.groups - 1) / p.groups;
    const int clusters = fp4_pair_clusters<FMT>();
    // The pair kernel where its 256 x 256 tiles are mostly full on both sides and keep every
    // cluster busy (a group that fills no whole tile still counts one in the bound).
    const bool pair = !p.zero && p.np > BM && mean > BM &&
                      tiles_bound(2 * BM, 256) - p.groups >= clusters;
    const int bn = pair ? 256 : p.rows <= 32 ? 32 : p.rows <= 64 ? 64 : 128;
    const int tm = pair ? 2 * BM : BM;
    const int64_t tiles = tiles_bound(tm, bn);
    const int64_t lines = fp4_sf_bytes(FMT) / 1024;
    const int64_t ablocks = (static_cast<int64_t>(p.rows) + 127) / 128 + p.groups;
    const int64_t bblocks = static_cast<int64_t>(p.groups) * p.npb;
    if (tiles > INT32_MAX / 2 || ablocks * p.stages * lines > INT32_MAX / 2 ||
        bblocks * p.stages * lines > INT32_MAX / 2 ||
        static_cast<int64_t>(p.groups) * p.np > INT32_MAX / 2)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    p.tiles_p = static_cast<int>((p.np + tm - 1) / tm);
    CUtensorMap tmp, tmq;
    memset(&tmp, 0, sizeof(tmp));
    memset(&tmq, 0, sizeof(tmq));
    char err[256] = "";
    int rc = 0;
    if (!p.zero) {
        // codes as 16-bit elements: four codes each, the pitch a multiple of 16 bytes
        const int64_t pe = fp4_pitch(p.kdim) / 2;
        rc = encode_tmap_u16(&tmp, b->data, pe, static_cast<int64_t>(b->rows), 1, pe, pe, 64, BM,
                             err, sizeof(err));
        if (!rc)
            rc = encode_tmap_u16(&tmq, a->data, pe, p.rows, 1, pe, pe, 64, pair ? 128 : bn, err,
                                 sizeof(err));
        if (rc) return set_last_error(rc, err);
    }
    if (pair) {
        using C = Fp4PairCfg<FMT>;
        // the scale buffers as blocks of lines of 1024 bytes; Q's two blocks come in one copy
        CUtensorMap tps, tqs;
        const int64_t bl = p.stages * lines;  // lines of a block
        rc = encode_tmap_lines(&tps, b->scales, bl, bblocks, static_cast<int>(lines), 1, err,
                               sizeof(err));
        const int64_t qblocks = static_cast<int64_t>(gk_fp4_scale_bytes(
                                    FMT, a->groups, a->offsets != nullptr, a->rows, a->cols)) /
                                (bl * 1024);
        if (!rc)
            rc = encode_tmap_lines(&tqs, a->scales, bl, qblocks, static_cast<int>(lines), 2, err,
                                   sizeof(err));
        if (rc) return set_last_error(rc, err);
        const int grid = 2 * static_cast<int>(tiles < clusters ? tiles : clusters);
        return launch_overlapped<CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, Fp4GemmParams>(
            2, fp4_pair_kernel<FMT>, grid, C::THREADS, C::SMEM, st, tmp, tmq, tps, tqs, p);
    }
    const int sms = sm_count();
    const int grid = static_cast<int>(tiles < sms ? tiles : sms);
    switch (bn) {
        case 32: return launch_fp4_gemm<FMT, 32>(tmp, tmq, p, grid, st);
        case 64: return launch_fp4_gemm<FMT, 64>(tmp, tmq, p, grid, st);
        default: return launch_fp4_gemm<FMT, 128>(tmp, tmq, p, grid, st);
    }
}

template <int FMT, typename T>
int run_quantize(const void* x, int64_t rs, int64_t cs, int64_t gs, const Fp4View& v, float scale,
                 cudaStream_t st) {
    // 16-byte loads: contiguous rows whose starts are all 16-byte aligned
    const int64_t es = sizeof(T);
    const bool rows1 = v.rows <= 1;
    const int vec = cs == 1 && !(reinterpret_cast<uintptr_t>(x) & 15) &&
                    (rows1 || (rs * es) % 16 == 0) &&
                    (v.offsets || v.groups == 1 || (gs * es) % 16 == 0);
    const NvScale nv{scale, 1.0f / (6.0f * scale)};
    auto go = [&](auto e_tag, auto unit_tag) {
        constexpr int E = decltype(e_tag)::value, UNIT = decltype(unit_tag)::value;
        return launch_overlapped<const T*, int64_t, int64_t, int64_t, int, Fp4View, NvScale>(
            1, quantize_fp4_kernel<FMT, T, E, UNIT * 8 / E>,
            unit_grid(static_cast<int64_t>(v.rows) * ((v.stages + UNIT - 1) / UNIT)), 256, 0, st,
            static_cast<const T*>(x), rs, cs, gs, vec, v, nv);
    };
    using std::integral_constant;
    const bool large = large_view(v);
    if constexpr (sizeof(T) == 2)
        if (vec && large) return go(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    return large ? go(integral_constant<int, 8>{}, integral_constant<int, 4>{})
                 : go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
}

}  // namespace

}  // namespace gk

using namespace gk;

extern "C" {

size_t gk_fp4_data_bytes(size_t rows, size_t cols) {
    return rows * static_cast<size_t>(fp4_pitch(static_cast<int64_t>(cols)));
}

size_t gk_fp4_scale_bytes(int fmt, size_t groups, int ragged, size_t rows, size_t cols) {
    if (groups == 0) groups = 1;
    const size_t blocks = ragged ? (rows + 127) / 128 + groups : groups * ((rows / groups + 127) / 128);
    return blocks * static_cast<size_t>(fp4_stages(static_cast<int64_t>(cols))) *
           static_cast<size_t>(fp4_sf_bytes(fmt));
}

int gk_quantize_fp4(gk_matref x, int x_type, ptrdiff_t x_gs, const gk_fp4_matrix* dst,
                    gk_stream_t stream) {
    int rc = check_fp4(dst, "the destination");
    if (rc) return rc;
    if (x_type != GK_F32 && x_type != GK_F16 && x_type != GK_BF16)
        return api_err(GK_EINVAL, "gemmkit: unknown element type %d", x_type);
    const bool stacked = !dst->offsets && dst->groups > 1;
    const size_t rows = stacked ? dst->rows / dst->groups : dst->rows;
    if (x.rows != rows || x.cols != dst->cols)
        return api_err(GK_EINVAL, "gemmkit: the source is %zux%zu, the 4-bit matrix holds %zux%zu%s",
                       x.rows, x.cols, rows, dst->cols, stacked ? " per group" : "");
    if ((rc = api_check_view(x.len, x.rows, x.cols, x.rs, x.cs, "X"))) return rc;
    if (x.rows == 0 || x.cols == 0) return GK_OK;
    if (!x.data) return api_err(GK_EINVAL, "gemmkit: null X");
    if ((rc = api_check_aligned(x.data, x_type == GK_F32 ? 4 : 2, "X"))) return rc;
    if (stacked) {
        const __int128 last = static_cast<__int128>(dst->groups - 1) * x_gs + 1 +
                              static_cast<__int128>(x.rows - 1) * x.rs +
                              static_cast<__int128>(x.cols - 1) * x.cs;
        if (x_gs < 0 || last > static_cast<__int128>(x.len))
            return api_err(GK_EINVAL, "gemmkit: X stack of %zu views %zux%zu (group stride %td) does "
                                      "not fit its slice of %zu elements",
                           dst->groups, x.rows, x.cols, x_gs, x.len);
    }
    const size_t es = x_type == GK_F32 ? 4 : 2;
    if (api_overlaps(x.data, x.len * es, dst->data, dst->data_len) ||
        api_overlaps(x.data, x.len * es, dst->scales, dst->scales_len) ||
        api_overlaps(dst->data, dst->data_len, dst->scales, dst->scales_len))
        return api_err(GK_EINVAL, "gemmkit: the 4-bit matrix aliases its source or itself");
    if ((rc = api_check_device(nullptr))) return rc;
    const Fp4View v = view_of(dst);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto fmt) {
        constexpr int F = decltype(fmt)::value;
        if (x_type == GK_F32)
            return run_quantize<F, float>(x.data, x.rs, x.cs, x_gs, v, dst->scale, st);
        if (x_type == GK_F16)
            return run_quantize<F, __half>(x.data, x.rs, x.cs, x_gs, v, dst->scale, st);
        return run_quantize<F, __nv_bfloat16>(x.data, x.rs, x.cs, x_gs, v, dst->scale, st);
    };
    return dst->fmt == GK_FP4_MX ? go(std::integral_constant<int, GK_FP4_MX>{})
                                 : go(std::integral_constant<int, GK_FP4_NV>{});
}

int gk_dequantize_fp4(const gk_fp4_matrix* q, gk_matmut out, gk_stream_t stream) {
    int rc = check_fp4(q, "the source");
    if (rc) return rc;
    if (out.rows != q->rows || out.cols != q->cols)
        return api_err(GK_EINVAL, "gemmkit: the 4-bit matrix holds %zux%zu, the output is %zux%zu",
                       q->rows, q->cols, out.rows, out.cols);
    if ((rc = api_check_view(out.len, out.rows, out.cols, out.rs, out.cs, "C"))) return rc;
    if (api_self_aliases(out.rows, out.cols, out.rs, out.cs))
        return api_err(GK_EINVAL, "gemmkit: C view aliases itself");
    if (out.rows == 0 || out.cols == 0) return GK_OK;
    if (!out.data) return api_err(GK_EINVAL, "gemmkit: null C");
    if ((rc = api_check_aligned(out.data, 4, "C"))) return rc;
    if (api_overlaps(out.data, out.len * 4, q->data, q->data_len) ||
        api_overlaps(out.data, out.len * 4, q->scales, q->scales_len))
        return api_err(GK_EINVAL, "gemmkit: C aliases the 4-bit matrix");
    if ((rc = api_check_device(nullptr))) return rc;
    const Fp4View v = view_of(q);
    const int vec = out.cs == 1 && !(reinterpret_cast<uintptr_t>(out.data) & 15) &&
                    (v.rows <= 1 || out.rs % 4 == 0);
    const int qu = large_view(v) ? 4 : 1;
    const int grid = unit_grid(static_cast<int64_t>(v.rows) * ((v.stages + qu - 1) / qu));
    auto kern = q->fmt == GK_FP4_MX
                    ? (qu == 4 ? dequantize_fp4_kernel<GK_FP4_MX, 4> : dequantize_fp4_kernel<GK_FP4_MX, 1>)
                    : (qu == 4 ? dequantize_fp4_kernel<GK_FP4_NV, 4> : dequantize_fp4_kernel<GK_FP4_NV, 1>);
    return launch_overlapped<Fp4View, float, float*, int64_t, int64_t, int>(
        1, kern, grid, 256, 0, static_cast<cudaStream_t>(stream), v, q->scale,
        static_cast<float*>(out.data), out.rs, out.cs, vec);
}

int gk_fp4_import(const uint8_t* codes, size_t codes_len, size_t codes_ld, const uint8_t* scales,
                  size_t scales_len, size_t scales_ld, const gk_fp4_matrix* dst,
                  gk_stream_t stream) {
    int rc = check_fp4(dst, "the destination");
    if (rc) return rc;
    if (dst->rows == 0 || dst->cols == 0) return GK_OK;
    const size_t bs = dst->fmt == GK_FP4_MX ? 32 : 16;
    const size_t cb = (dst->cols + 1) / 2, sb = (dst->cols + bs - 1) / bs;
    if (!codes || !scales) return api_err(GK_EINVAL, "gemmkit: null codes or scales");
    if (codes_ld < cb || scales_ld < sb || codes_len < (dst->rows - 1) * codes_ld + cb ||
        scales_len < (dst->rows - 1) * scales_ld + sb)
        return api_err(GK_EINVAL,
                       "gemmkit: %zux%zu in 4 bits takes rows of %zu code bytes and %zu scales (has "
                       "%zu at pitch %zu and %zu at pitch %zu)",
                       dst->rows, dst->cols, cb, sb, codes_len, codes_ld, scales_len, scales_ld);
    if (api_overlaps(codes, codes_len, dst->data, dst->data_len) ||
        api_overlaps(codes, codes_len, dst->scales, dst->scales_len) ||
        api_overlaps(scales, scales_len, dst->data, dst->data_len) ||
        api_overlaps(scales, scales_len, dst->scales, dst->scales_len) ||
        api_overlaps(dst->data, dst->data_len, dst->scales, dst->scales_len))
        return api_err(GK_EINVAL, "gemmkit: the 4-bit matrix aliases its source or itself");
    if ((rc = api_check_device(nullptr))) return rc;
    const Fp4View v = view_of(dst);
    const int grid = unit_grid(static_cast<int64_t>(v.rows) * v.stages);
    auto kern = dst->fmt == GK_FP4_MX ? import_fp4_kernel<GK_FP4_MX> : import_fp4_kernel<GK_FP4_NV>;
    return launch_overlapped<const uint8_t*, int64_t, const uint8_t*, int64_t, Fp4View>(
        1, kern, grid, 256, 0, static_cast<cudaStream_t>(stream), codes,
        static_cast<int64_t>(codes_ld), scales, static_cast<int64_t>(scales_ld), v);
}

int gk_gemm_fp4(float alpha, const gk_fp4_matrix* a, const gk_fp4_matrix* b, float beta, gk_matmut c,
                int out_type, gk_parallelism par, gk_stream_t stream) {
    (void)par;
    int rc;
    if ((rc = check_fp4(a, "A")) || (rc = check_fp4(b, "B"))) return rc;
    if (out_type != GK_F32 && out_type != GK_F16 && out_type != GK_BF16)
        return api_err(GK_EINVAL, "gemmkit: unknown element type %d", out_type);
    if (a->fmt != b->fmt)
        return api_err(GK_EINVAL, "gemmkit: A and B are held in different 4-bit formats");
    if (b->offsets) return api_err(GK_EINVAL, "gemmkit: B's groups must be equal (no offsets)");
    if (a->groups != b->groups)
        return api_err(GK_EINVAL, "gemmkit: A has %zu groups, B has %zu", a->groups, b->groups);
    const size_t n = b->rows / b->groups;
    if (a->cols != b->cols)
        return api_err(GK_EINVAL, "gemmkit: A.cols (%zu) != B.cols (%zu) (4-bit operands share k)",
                       a->cols, b->cols);
    if (a->rows != c.rows)
        return api_err(GK_EINVAL, "gemmkit: A.rows (%zu) != C.rows (%zu)", a->rows, c.rows);
    if (n != c.cols)
        return api_err(GK_EINVAL, "gemmkit: B.rows per group (%zu) != C.cols (%zu)", n, c.cols);
    if ((rc = api_check_view(c.len, c.rows, c.cols, c.rs, c.cs, "C"))) return rc;
    if (api_self_aliases(c.rows, c.cols, c.rs, c.cs))
        return api_err(GK_EINVAL,
                       "gemmkit: C view aliases itself (strides %td,%td map distinct elements to "
                       "the same memory); C must address each (i,j) uniquely",
                       c.rs, c.cs);
    const size_t cb = c.len * (out_type == GK_F32 ? 4 : 2);
    for (const gk_fp4_matrix* o : {a, b})
        if (o->rows && o->cols &&
            (api_overlaps(c.data, cb, o->data, o->data_len) ||
             api_overlaps(c.data, cb, o->scales, o->scales_len)))
            return api_err(GK_EINVAL, "gemmkit: C aliases A or B");
    const double scaled = static_cast<double>(alpha) * a->scale * b->scale;
    if (isfinite(alpha) && alpha != 0.0f &&
        !(fabs(scaled) >= 1.17549435e-38 && fabs(scaled) <= 3.4028234e38))
        return api_err(GK_EINVAL, "gemmkit: alpha times the matrix scales (%g) leaves f32", scaled);
    if (c.rows == 0 || c.cols == 0) return GK_OK;
    if (!c.data) return api_err(GK_EINVAL, "gemmkit: null C");
    if ((rc = api_check_aligned(c.data, out_type == GK_F32 ? 4 : 2, "C"))) return rc;
    if ((rc = api_check_device(nullptr))) return rc;
    Fp4GemmParams p;
    memset(&p, 0, sizeof(p));
    p.psf = b->scales;
    p.qsf = a->scales;
    p.np = static_cast<int>(n);
    p.npb = static_cast<int>((n + 127) / 128);
    p.kdim = static_cast<int>(a->cols);
    p.stages = static_cast<int>(fp4_stages(static_cast<int64_t>(a->cols)));
    p.zero = a->cols == 0 || alpha == 0.0f;
    p.groups = static_cast<int>(a->groups);
    p.rows = static_cast<int>(a->rows);
    p.offsets = a->offsets;
    p.c = c.data;
    p.ldq = c.rs;
    p.ldp = c.cs;
    // (an empty product is zero whatever alpha is, an infinity or a NaN too)
    p.alpha = p.zero ? 0.0f : static_cast<float>(scaled);
    p.beta = beta;
    p.out_type = out_type;
    p.pieces = c_in_pieces(c.data, out_type, c.rs, c.cs, 0, static_cast<int64_t>(n), beta);
    p.timeout_ns = wait_limit_ns(p.stages);
    p.status = device_status_ptr();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return a->fmt == GK_FP4_MX ? run_fp4_gemm<GK_FP4_MX>(p, a, b, st)
                               : run_fp4_gemm<GK_FP4_NV>(p, a, b, st);
}

}  // extern "C"
