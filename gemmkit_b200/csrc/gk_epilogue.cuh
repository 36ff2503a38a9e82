// gk_epilogue.cuh -- the epilogues of a feed-forward layer's products, on the accumulators of the
// grouped kernels (gk_grouped.cuh).
//
//   forward    z = alpha acc + bias;  C = act(z) + R, and z itself on demand
//   backward   C = alpha acc * act'(z);  the sums of C over a group's rows on demand
//
// All of it in f32 on the accumulators as they are, rounded once where it is stored. The backward
// pass takes z from a 16-bit matrix or from a checkpoint in 8 bits (gk_act8.cuh).
//
// A lane holds one P row (a column of C) and consecutive Q rows (rows of C), so a bias is one value
// a lane and a column sum one register. 16-bit matrices with unit column stride move in pairs: of
// two neighbouring lanes the even one reads and writes four bytes of the even Q rows, the odd one of
// the odd ones, half as many instructions as element by element; the halves are
// exchanged by one shuffle for four elements. The same lane reads an element of R (or z) and
// later stores that of C, so C may be R (or z) itself.
#pragma once

#include <stdint.h>

#include <type_traits>

#include "gemmkit_cuda.h"
#include "gk_act8.cuh"
#include "gk_f2.cuh"
#include "gk_sm100.cuh"
#include "gk_store.cuh"

namespace gk {

// What a kernel does with its accumulators; EPI_F16 is added where 16-bit matrices hold f16 (else bf16).
enum : int { EPI_STORE = 0, EPI_FWD = 1, EPI_BWD = 2, EPI_F16 = 4 };
constexpr bool epi_fwd(int epi) { return (epi & 3) == EPI_FWD; }
constexpr bool epi_bwd(int epi) { return (epi & 3) == EPI_BWD; }
constexpr bool epi_f16(int epi) { return (epi & EPI_F16) != 0; }

struct EpiArgs {
    int32_t act;              // gk_act
    float slope;              // LeakyReLU's
    const void* bias;         // forward; nullptr: none
    int64_t bias_gs;          // elements from one group's bias to the next's
    int32_t bias_type;        // gk_dtype of the bias (forward) or of the sums (backward)
    int32_t pairs;            // every 16-bit matrix of the epilogue moves in pairs (see above)
    const void* side;         // forward: R, of C's type; backward: z, of the operands' type
    int64_t sq, sp;           // its strides along the Q side (rows) and the P side (columns)
    uint16_t* z;              // forward: where z is kept, of the operands' type; nullptr: nowhere
    int64_t zq, zp;
    Act8View z8;              // backward: z as a checkpoint (codes != nullptr)
    void* dbias;              // backward: sums over the rows of each group; nullptr: none
    int64_t dbias_gs;
    float* part;              // backward: the tiles' sums
};

// ---- activations ------------------------------------------------------------------------------------
//
// ReLU and LeakyReLU as in the engine's other epilogues (fused_apply: a NaN becomes 0). GELU and SiLU
// keep a NaN; magnitudes beyond 100 count as 100 where only the limit is left of them, so that an
// infinity gives the limit instead of inf * 0.
//   GELU is z Phi(z). With q = Phi(-|z|): max(z, 0) - |z| q, and its derivative 1/2 +- (1/2 - q) + z phi(z).
// q comes from Abramowitz and Stegun's formula 7.1.26 for erfc (five terms in t = 1 / (1 + p x) times
// exp(-x^2), at most 1.5e-7 off, so q is 7.5e-8 off and its terms' roundings), whose exponential is
// phi's too: 10 and 12 instructions an element, two elements at a time, where erff and a second
// exponential took about 45.
//   Its tanh form is z sigma(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3), since (1 + tanh u) / 2 = sigma(2 u);
// SiLU is z sigma(z). sigma(t) = 1 / (1 + 2^(-t log2 e)) by the hardware's exponential and reciprocal
// (2^-22 and 2^-23 relative), the argument's rounding |t| 2^-24 on top. All of it is below a
// hundredth of a 16-bit rounding.

// min(|x|, |y|) with the product's sign (here: x clamped to +-y), a NaN kept.
__device__ __forceinline__ float clamp_nan(float x, float y) {
    float r;
    asm("min.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float rcp_hw(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ F2 clamp2(F2 x, float y) { return F2(clamp_nan(x.lo(), y), clamp_nan(x.hi(), y)); }
__device__ __forceinline__ F2 max2(F2 x, float y) { return F2(max_nan(x.lo(), y), max_nan(x.hi(), y)); }
__device__ __forceinline__ F2 exp2_2(F2 x) { return F2(exp2_hw(x.lo()), exp2_hw(x.hi())); }
__device__ __forceinline__ F2 rcp2(F2 x) { return F2(rcp_hw(x.lo()), rcp_hw(x.hi())); }

constexpr float LOG2E = 1.44269504f, RSQRT_2PI = 0.39894228f;
constexpr float GELU_C = 0.044715f, GELU_2K = 1.59576912f;  // 2 sqrt(2 / pi)

// 1 / (1 + 2^w)
__device__ __forceinline__ F2 sigma2(F2 w) { return rcp2(add2(exp2_2(w), F2(1.0f))); }

// Phi(-|z|) for |z| <= 100, from n = -|z|, and e = exp(-z^2 / 2) = phi(z) sqrt(2 pi).
__device__ __forceinline__ F2 normal_tail(F2 n, F2& e) {
    const F2 t = rcp2(fma2(n, F2(-0.3275911f * 0.70710678f), F2(1.0f)));
    e = exp2_2(mul2(mul2(n, n), F2(-0.5f * LOG2E)));
    F2 y = fma2(F2(0.5f * 1.061405429f), t, F2(0.5f * -1.453152027f));
    y = fma2(y, t, F2(0.5f * 1.421413741f));
    y = fma2(y, t, F2(0.5f * -0.284496736f));
    y = fma2(y, t, F2(0.5f * 0.254829592f));
    return mul2(mul2(y, t), e);
}
__device__ __forceinline__ F2 minus_abs(F2 z) {
    F2 r;
    r.v = z.v | 0x8000000080000000ull;
    return r;
}

template <int ACT>
__device__ __forceinline__ F2 act_value(F2 z, float slope) {
    if constexpr (ACT == GK_ACT_RELU) {
        return F2(z.lo() > 0.0f ? z.lo() : 0.0f, z.hi() > 0.0f ? z.hi() : 0.0f);
    } else if constexpr (ACT == GK_ACT_LEAKY_RELU) {
        return fma2(F2(slope), F2(z.lo() < 0.0f ? z.lo() : 0.0f, z.hi() < 0.0f ? z.hi() : 0.0f),
                    F2(z.lo() > 0.0f ? z.lo() : 0.0f, z.hi() > 0.0f ? z.hi() : 0.0f));
    } else if constexpr (ACT == GK_ACT_GELU) {
        const F2 n = minus_abs(clamp2(z, 100.0f));
        F2 e;
        return fma2(n, normal_tail(n, e), max2(z, 0.0f));
    } else if constexpr (ACT == GK_ACT_GELU_TANH) {
        z = max2(z, -100.0f);
        const F2 m = fma2(F2(-GELU_2K * LOG2E * GELU_C), mul2(z, z), F2(-GELU_2K * LOG2E));
        return mul2(z, sigma2(mul2(z, m)));
    } else if constexpr (ACT == GK_ACT_SILU) {
        z = max2(z, -100.0f);
        return mul2(z, sigma2(mul2(z, F2(-LOG2E))));
    } else {
        return z;
    }
}

// s (1 - s)
__device__ __forceinline__ F2 s_1_s(F2 s) { return mul2(s, fma2(s, F2(-1.0f), F2(1.0f))); }

template <int ACT>
__device__ __forceinline__ F2 act_slope(F2 z, float slope) {
    if constexpr (ACT == GK_ACT_RELU) {
        return F2(z.lo() > 0.0f ? 1.0f : 0.0f, z.hi() > 0.0f ? 1.0f : 0.0f);
    } else if constexpr (ACT == GK_ACT_LEAKY_RELU) {
        return F2(z.lo() > 0.0f ? 1.0f : slope, z.hi() > 0.0f ? 1.0f : slope);
    } else if constexpr (ACT == GK_ACT_GELU) {
        z = clamp2(z, 100.0f);
        F2 e;
        const F2 q = normal_tail(minus_abs(z), e);
        const F2 half = fma2(q, F2(-1.0f), F2(0.5f));
        return fma2(mul2(z, F2(RSQRT_2PI)), e,
                    add2(F2(copysignf(half.lo(), z.lo()), copysignf(half.hi(), z.hi())), F2(0.5f)));
    } else if constexpr (ACT == GK_ACT_GELU_TANH) {
        z = clamp2(z, 100.0f);
        const F2 z2 = mul2(z, z);
        const F2 m = fma2(F2(-GELU_2K * LOG2E * GELU_C), z2, F2(-GELU_2K * LOG2E));
        const F2 s = sigma2(mul2(z, m));
        return fma2(mul2(z, s_1_s(s)), fma2(F2(3.0f * GELU_C * GELU_2K), z2, F2(GELU_2K)), s);
    } else if constexpr (ACT == GK_ACT_SILU) {
        z = clamp2(z, 100.0f);
        const F2 s = sigma2(mul2(z, F2(-LOG2E)));
        return fma2(z, s_1_s(s), s);
    } else {
        return F2(1.0f);
    }
}

// f(the activation as a constant), compiled for each of them.
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
    switch (act) {
        case GK_ACT_RELU: f(std::integral_constant<int, GK_ACT_RELU>{}); break;
        case GK_ACT_LEAKY_RELU: f(std::integral_constant<int, GK_ACT_LEAKY_RELU>{}); break;
        case GK_ACT_GELU: f(std::integral_constant<int, GK_ACT_GELU>{}); break;
        case GK_ACT_GELU_TANH: f(std::integral_constant<int, GK_ACT_GELU_TANH>{}); break;
        case GK_ACT_SILU: f(std::integral_constant<int, GK_ACT_SILU>{}); break;
        default: f(std::integral_constant<int, GK_ACT_NONE>{}); break;
    }
}

// ---- 16-bit pairs ------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi, int f16) {
    uint32_t w;
    if (f16)
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    else
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
    return w;
}

__device__ __forceinline__ float half_lo(uint32_t w, int f16) {
    return f16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xFFFFu)))
               : __uint_as_float(w << 16);
}
__device__ __forceinline__ float half_hi(uint32_t w, int f16) {
    return f16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16)))
               : __uint_as_float(w & 0xFFFF0000u);
}

// The loads of that layout, not yet exchanged: N words hold the 2 N columns of this lane pair.
template <int N>
__device__ __forceinline__ void load_pairs(uint32_t (&w)[N], const uint16_t* c, int64_t ldq, int n,
                                           int pn, int lane) {
    const int odd = lane & 1;
    const uint16_t* q = c + (lane & 30) + odd * ldq;
    if (n >= 2 * N && pn >= 32) {  // (the warp's; no predicates)
        const uint32_t step = static_cast<uint32_t>(ldq) * 4u;  // one multiply-add an address
#pragma unroll
        for (int j = 0; j < N; ++j)
            w[j] = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(q) +
                                                      static_cast<uint64_t>(step) * j);
        return;
    }
    const int left = (lane & 30) < pn ? n - odd : 0;
#pragma unroll
    for (int j = 0; j < N; ++j, q += 2 * ldq)
        w[j] = 2 * j < left ? *reinterpret_cast<const uint32_t*>(q) : 0u;
}

// The exchange: w[j] becomes columns 2 j and 2 j + 1 of this lane's own P row (and back: the exchange undoes
// itself).
template <int N>
__device__ __forceinline__ void own_pairs(uint32_t (&w)[N], int lane) {
    const int odd = lane & 1;
    const uint32_t give = odd ? 0x5410u : 0x7632u;
    const uint32_t sel0 = odd ? 0x3254u : 0x5410u, sel1 = odd ? 0x3276u : 0x7610u;
#pragma unroll
    for (int j = 0; j < N; j += 2) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, __byte_perm(w[j], w[j + 1], give), 1);
        w[j] = __byte_perm(w[j], got, sel0);
        w[j + 1] = __byte_perm(w[j + 1], got, sel1);
    }
}

// 2 N columns of this lane's own P row, rounded, into a matrix that moves in pairs; w is used up.
template <int N>
__device__ __forceinline__ void put_pairs(uint32_t (&w)[N], uint16_t* c, int64_t ldq, int n, int pn,
                                          int lane) {
    own_pairs(w, lane);
    const int odd = lane & 1;
    uint16_t* q = c + (lane & 30) + odd * ldq;
    if (n >= 2 * N && pn >= 32) {
        const uint32_t step = static_cast<uint32_t>(ldq) * 4u;
#pragma unroll
        for (int j = 0; j < N; ++j)
            *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(q) +
                                         static_cast<uint64_t>(step) * j) = w[j];
        return;
    }
    const int left = (lane & 30) < pn ? n - odd : 0;
#pragma unroll
    for (int j = 0; j < N; ++j, q += 2 * ldq)
        if (2 * j < left) *reinterpret_cast<uint32_t*>(q) = w[j];
}

// ---- a warp's accumulators ----------------------------------------------------------------------------

// Where a warp's columns lie: P rows i0 .. i0 + pn - 1 of C exist (a lane each), Q rows r .. r + n - 1.
struct EpiAt {
    int i0, pn;
    int64_t r;
    int n;
};

// N columns of the matrix that the epilogue reads beside the accumulators, all loads issued together:
// R, or z in 16 bits (pairs, or element by element), or z in 8 bits.
template <int EPI, int N>
struct EpiSide {
    uint32_t w[N / 2];
    uint32_t sb;  // z in 8 bits: lane e holds the exponent byte of column e
    // PAIRS: see EpiArgs; an f32 R (f32: C is) is read where it is used.
    template <bool PAIRS>
    __device__ __forceinline__ void load(const EpiArgs& e, const EpiAt& at, bool f32, int lane) {
        if (epi_bwd(EPI) && e.z8.codes) {
#pragma unroll
            for (int j = 0; j < N / 4; ++j) {
                const int c = 4 * j + (lane >> 3);
                w[j] = at.pn > 0 && c < at.n
                           ? *reinterpret_cast<const uint32_t*>(
                                 e.z8.codes + (at.r + c) * e.z8.codes_ld + at.i0 + (lane & 7) * 4)
                           : 0u;
            }
            sb = at.pn > 0 && lane < N && lane < at.n
                     ? e.z8.exps[(at.r + lane) * e.z8.exps_ld + (at.i0 >> 5)]
                     : 0u;
        } else if (e.side) {
            if constexpr (PAIRS) {
                load_pairs(w, static_cast<const uint16_t*>(e.side) + at.r * e.sq + at.i0, e.sq, at.n,
                           at.pn, lane);
            } else if (!f32 || epi_bwd(EPI)) {
                const uint16_t* s = static_cast<const uint16_t*>(e.side) + at.r * e.sq +
                                    (at.i0 + lane) * e.sp;
                const int n = lane < at.pn ? at.n : 0;
                uint16_t v[N];
#pragma unroll
                for (int c = 0; c < N; ++c) v[c] = c < n ? s[c * e.sq] : uint16_t{0};
#pragma unroll
                for (int j = 0; j < N / 2; ++j)
                    w[j] = v[2 * j] | (static_cast<uint32_t>(v[2 * j + 1]) << 16);
            }
        }
    }
    // After load(): the pairs' exchange, or this lane's byte positions.
    template <bool PAIRS>
    __device__ __forceinline__ void own(const EpiArgs& e, int lane) {
        if (epi_bwd(EPI) && e.z8.codes) {
#pragma unroll
            for (int j = 0; j < N / 4; ++j) w[j] ^= 0x80808080u;
            sb = __float_as_uint(act8_unit(sb));
        } else if (PAIRS && e.side) {
            own_pairs(w, lane);
        }
    }
    // Columns c and c + 1 (c even) of this lane's P row.
    __device__ __forceinline__ F2 z8(int c, int lane) const {
        float v[2], unit[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t x = __shfl_sync(0xffffffffu, w[c / 4], ((c + i) % 4) * 8 + (lane >> 2));
            v[i] = act8_raw(x, lane & 3);
            unit[i] = __uint_as_float(__shfl_sync(0xffffffffu, sb, c + i));
        }
        return mul2(add2(F2(v[0], v[1]), F2(-8388736.0f)), F2(unit[0], unit[1]));
    }
    __device__ __forceinline__ F2 half(int c) const {
        return F2(half_lo(w[c / 2], epi_f16(EPI)), half_hi(w[c / 2], epi_f16(EPI)));
    }
};

// N accumulators of each lane (f32 bits), their side loaded and owned, through the activation and into
// C: a row of C is 32 P rows of the warp. `sum` gains the stored columns (backward).
template <int EPI, int N, bool PAIRS>
__device__ __forceinline__ void epi_columns(const EpiArgs& e, void* c, int out_type,
                                            int64_t ldq, int64_t ldp, const EpiAt& at,
                                            const uint32_t (&v)[N], const EpiSide<EPI, N>& s,
                                            float alpha, float bias, float& sum, int lane) {
    constexpr bool f16 = epi_f16(EPI);
    F2 y[N / 2];  // two columns each
    const bool live = lane < at.pn;
    const int64_t own = (at.i0 + lane) * ldp + at.r * ldq;  // element by element
    if constexpr (epi_fwd(EPI)) {
#pragma unroll
        for (int j = 0; j < N / 2; ++j)
            y[j] = fma2(F2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), F2(alpha), F2(bias));
        if (e.z) {
            uint32_t zw[N / 2];
#pragma unroll
            for (int j = 0; j < N / 2; ++j) zw[j] = pack_half2(y[j].lo(), y[j].hi(), f16);
            if constexpr (PAIRS) {
                put_pairs(zw, e.z + at.r * e.zq + at.i0, e.zq, at.n, at.pn, lane);
            } else {
                uint16_t* z = e.z + (at.i0 + lane) * e.zp + at.r * e.zq;
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (live && j < at.n)
                        z[j * e.zq] = static_cast<uint16_t>(zw[j / 2] >> (16 * (j & 1)));
            }
        }
        with_act(e.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) y[j] = act_value<decltype(act)::value>(y[j], e.slope);
        });
        if (e.side) {
            if (PAIRS || out_type != GK_F32) {
#pragma unroll
                for (int j = 0; j < N / 2; ++j) y[j] = add2(y[j], s.half(2 * j));
            } else {
                const float* r = static_cast<const float*>(e.side) + (at.i0 + lane) * e.sp +
                                 at.r * e.sq;
                const int n = live ? at.n : 0;
#pragma unroll
                for (int j = 0; j < N; j += 2)
                    y[j / 2] = add2(y[j / 2], F2(j < n ? r[j * e.sq] : 0.0f,
                                                 j + 1 < n ? r[(j + 1) * e.sq] : 0.0f));
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < N / 2; ++j)
            y[j] = mul2(F2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), F2(alpha));
        with_act(e.act, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
            if constexpr (ACT != GK_ACT_NONE) {
                if (e.z8.codes) {
#pragma unroll
                    for (int j = 0; j < N / 2; ++j)
                        y[j] = mul2(y[j], act_slope<ACT>(s.z8(2 * j, lane), e.slope));
                } else {
#pragma unroll
                    for (int j = 0; j < N / 2; ++j)
                        y[j] = mul2(y[j], act_slope<ACT>(s.half(2 * j), e.slope));
                }
            }
        });
        if (at.n >= N) {  // (rows past the tile hold anything)
            F2 a = y[0];
#pragma unroll
            for (int j = 1; j < N / 2; ++j) a = add2(a, y[j]);
            sum += a.lo() + a.hi();
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (j < at.n) sum += j & 1 ? y[j / 2].hi() : y[j / 2].lo();
        }
    }
    if constexpr (PAIRS) {
        uint32_t w[N / 2];
#pragma unroll
        for (int j = 0; j < N / 2; ++j) w[j] = pack_half2(y[j].lo(), y[j].hi(), f16);
        put_pairs(w, static_cast<uint16_t*>(c) + at.r * ldq + at.i0, ldq, at.n, at.pn, lane);
    } else if (out_type == GK_F32) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (live && j < at.n)
                static_cast<float*>(c)[own + j * ldq] = j & 1 ? y[j / 2].hi() : y[j / 2].lo();
    } else {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const uint32_t w = pack_half2(y[j / 2].lo(), y[j / 2].hi(), f16);
            uint16_t* o = static_cast<uint16_t*>(c) + own + j * ldq;
            if (live && j < at.n) *o = static_cast<uint16_t>(w);
            if (live && j + 1 < at.n) o[ldq] = static_cast<uint16_t>(w >> 16);
        }
    }
}

// A column's sum to element `at` of the sums.
__device__ __forceinline__ void store_sum(const EpiArgs& e, int64_t at, float y) {
    if (e.bias_type == GK_F32)
        to_out(static_cast<float*>(e.dbias) + at, y);
    else if (e.bias_type == GK_F16)
        to_out(static_cast<__half*>(e.dbias) + at, y);
    else
        to_out(static_cast<__nv_bfloat16*>(e.dbias) + at, y);
}

// The bias of this lane's P row.
__device__ __forceinline__ float epi_bias(const EpiArgs& e, int g, int i0, int pn, int lane) {
    if (!e.bias || lane >= pn) return 0.0f;
    const int64_t i = g * e.bias_gs + i0 + lane;
    if (e.bias_type == GK_F32) return static_cast<const float*>(e.bias)[i];
    const uint32_t w = static_cast<const uint16_t*>(e.bias)[i];
    return half_lo(w, e.bias_type == GK_F16);
}

}  // namespace gk
