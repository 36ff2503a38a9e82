// gk_act8.cu -- activations kept in 8 bits for the backward pass (gk_act8.cuh): quantisation, the values
// back, and the weight gradient from them.
//
// A block of 32 elements of a row shares a power of two:
//   e = floor(log2 max |x|), at least -127;  code = x 2^(6 - e), half to even, clamped to +-127
// Powers of two keep both directions exact: x 2^(6 - e) has the digits of x, and a code times 2^(e - 6)
// has at most 7, so bf16 and f32 hold every value, and f16 where the source was f16 (a block whose
// unit lies below f16's 2^-24 holds multiples of that already). The backward pass therefore
// multiplies what the checkpoint stands for, with no second rounding.
//
// Both kernels move each byte once and are bound by memory. The matrix is a run of pieces of E elements,
// row after row; a lane takes AU of them, 32 pieces apart, all of their loads issued together (so short
// rows fill warps too). Quantising, E is 16 where the elements have 16 bits, 8 in f32: 16-byte loads, a
// block's maximum over two or four lanes. The other way E makes 16 bytes of output, so that a warp's
// store writes whole sectors (with 16 elements a lane, two half sectors each, 8192 x 8192 of bf16 took 45
// instead of 36 us; quantising it takes 36).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "gemmkit_cuda.h"
#include "gk_act8.cuh"
#include "gk_engine.h"
#include "gk_f2.cuh"
#include "gk_launch.h"
#include "gk_sm100.cuh"
#include "gk_store.cuh"

namespace gk {

namespace {

constexpr int AU = 4;  // pieces of a lane

template <typename T>
constexpr int piece() {
    return sizeof(T) == 2 ? 16 : 8;
}

template <typename T>
struct Piece {  // its elements as they lie in memory
    static constexpr int E = piece<T>(), W = E * sizeof(T) / 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const T* x) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const uint4 v = ld_global_v4(reinterpret_cast<const uint32_t*>(x) + i);
            w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
        }
    }
    // element by element, zeros from n on
    __device__ __forceinline__ void load(const T* x, int64_t cs, int n) {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0u;
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (i < n) {
                if constexpr (sizeof(T) == 4)
                    w[i] = __float_as_uint(x[i * cs]);
                else
                    w[i / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(x)[i * cs])
                                << (16 * (i & 1));
            }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (std::is_same_v<T, float>) {
            return __uint_as_float(w[i]);
        } else if constexpr (std::is_same_v<T, __half>) {
            return __half2float(__ushort_as_half(static_cast<unsigned short>(w[i / 2] >> (16 * (i & 1)))));
        } else {
            return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        }
    }
};

// The largest magnitude of a piece, as f32 bits; 16-bit magnitudes compare as integers, two at a time.
template <typename T>
__device__ __forceinline__ uint32_t largest(const Piece<T>& x) {
    uint32_t m = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int k = 0; k < Piece<T>::W; ++k) m = max(m, x.w[k] & 0x7FFFFFFFu);
    } else {
#pragma unroll
        for (int k = 0; k < Piece<T>::W; ++k) m = __vmaxu2(m, x.w[k] & 0x7FFF7FFFu);
        m = max(m & 0xFFFFu, m >> 16);
        m = std::is_same_v<T, __half>
                ? __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))))
                : m << 16;
    }
    return m;
}

// x clamped to +-127 (one instruction: the smaller magnitude with the product's sign).
__device__ __forceinline__ float clamp_127(float x) {
    float r;
    asm("min.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(127.0f));
    return r;
}

// Where a lane's pieces lie, 32 apart: `per` of them make the whole blocks of a row. Divided once, in 64
// bits only where 32 do not hold the pieces.
struct At {
    int64_t r;
    uint32_t i;  // piece of the row
    __device__ __forceinline__ At(uint64_t piece, uint32_t per, bool wide) {
        r = wide ? piece / per : static_cast<uint32_t>(piece) / per;
        i = static_cast<uint32_t>(piece - r * per);
    }
    __device__ __forceinline__ void next(uint32_t per, uint32_t rows32, uint32_t rest32) {
        r += rows32;
        i += rest32;
        if (i >= per) {
            i -= per;
            ++r;
        }
    }
};

struct Act8Out {
    int8_t* codes;
    uint8_t* exps;
    int64_t codes_ld, exps_ld;
    int64_t rows;
    int32_t cols;
};

// vec: rows of x are contiguous and start on 16-byte boundaries.
template <typename T>
__global__ void __launch_bounds__(256, 4)
    quantize_act8_kernel(const T* x, int64_t rs, int64_t cs, int vec, Act8Out q) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int E = piece<T>(), LANES = ACT8_BLOCK / E;  // lanes of a block
    const int lane = threadIdx.x & 31;
    const uint32_t per = static_cast<uint32_t>((q.cols + 31) / 32 * LANES);
    const uint64_t pieces = static_cast<uint64_t>(q.rows) * per;
    const bool wide = pieces + 32 * AU > 0xFFFFFFFFull;
    const uint32_t rows32 = 32 / per, rest32 = 32 % per;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * (blockDim.x >> 5) * (32 * AU);
    for (uint64_t u = static_cast<uint64_t>(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * (32 * AU);
         u < pieces; u += step) {
        Piece<T> raw[AU];
        At at(u + lane, per, wide);
        const At first = at;
#pragma unroll
        for (int i = 0; i < AU; ++i, at.next(per, rows32, rest32)) {
            const int c = static_cast<int>(at.i) * E;
            const T* src = x + at.r * rs;
            if (at.r < q.rows && vec && c + E <= q.cols)
                raw[i].load(src + c);
            else
                raw[i].load(src + c * cs, cs, at.r < q.rows ? q.cols - c : 0);
        }
        at = first;
#pragma unroll
        for (int i = 0; i < AU; ++i, at.next(per, rows32, rest32)) {
            if (u + 32 * i >= pieces) break;  // the whole warp
            uint32_t m = largest(raw[i]);
#pragma unroll
            for (int d = 1; d < LANES; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
            const uint32_t b = m >> 23;  // the biased exponent is e + 127; 255: an infinity or a NaN
            float v[E];
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] = raw[i].value(k);
            // x 2^(6 - e), in two exact steps where 2^(6 - e) would not be a normal number
            if (__any_sync(0xffffffffu, b < 64)) {
#pragma unroll
                for (int k = 0; k < E; ++k) v[k] = b < 64 ? v[k] * 0x1p64f : v[k];
            }
            const F2 mul(__uint_as_float((b < 64 ? 196u - b : 260u - b) << 23));
            F2 s[E / 2];
#pragma unroll
            for (int k = 0; k < E / 2; ++k) s[k] = mul2(F2(v[2 * k], v[2 * k + 1]), mul);
            // Below 128 in magnitude: only a block whose largest value's digits begin 1.9921875 holds one
            // that would round to 128.
            if (__any_sync(0xffffffffu, (m & 0x7FFFFFu) >= 0x7F0000u)) {
#pragma unroll
                for (int k = 0; k < E / 2; ++k) s[k] = F2(clamp_127(s[k].lo()), clamp_127(s[k].hi()));
            }
            // 1.5 2^23 + s: rounded to an integer, half to even, its low byte the code
            uint32_t w[E / 4];
#pragma unroll
            for (int h = 0; h < E / 4; ++h) {
                const F2 y0 = add2(s[2 * h], F2(12582912.0f)), y1 = add2(s[2 * h + 1], F2(12582912.0f));
                w[h] = b == 255 ? 0u
                                : __byte_perm(__byte_perm(__float_as_uint(y0.lo()),
                                                          __float_as_uint(y0.hi()), 0x0040),
                                              __byte_perm(__float_as_uint(y1.lo()),
                                                          __float_as_uint(y1.hi()), 0x0040),
                                              0x5410);
            }
            if (at.r >= q.rows) continue;
            const int c = static_cast<int>(at.i) * E;
            int8_t* dst = q.codes + at.r * q.codes_ld + c;
            if constexpr (E == 16)
                st_global_v4(dst, w[0], w[1], w[2], w[3]);
            else
                *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
            if (lane % LANES == 0) q.exps[at.r * q.exps_ld + (c >> 5)] = static_cast<uint8_t>(b);
        }
    }
}

// vec: rows of out are contiguous and start on 16-byte boundaries.
template <typename T>
__global__ void __launch_bounds__(256)
    dequantize_act8_kernel(Act8View q, int64_t rows, int32_t cols, T* out, int64_t rs, int64_t cs,
                           int vec) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int E = 16 / sizeof(T), AU = 8;  // whole sectors are stored
    const int lane = threadIdx.x & 31;
    const uint32_t per = static_cast<uint32_t>((cols + E - 1) / E);
    const uint64_t pieces = static_cast<uint64_t>(rows) * per;
    const bool wide = pieces + 32 * AU > 0xFFFFFFFFull;
    const uint32_t rows32 = 32 / per, rest32 = 32 % per;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * (blockDim.x >> 5) * (32 * AU);
    for (uint64_t u = static_cast<uint64_t>(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * (32 * AU);
         u < pieces; u += step) {
        uint32_t w[AU][E / 4], b[AU];
        At at(u + lane, per, wide);
        const At first = at;
#pragma unroll
        for (int i = 0; i < AU; ++i, at.next(per, rows32, rest32)) {
            // (past the end the first piece again: no branch between the loads)
            const bool in = at.r < rows;
            const int c = in ? static_cast<int>(at.i) * E : 0;
            const int64_t r = in ? at.r : 0;
            const int8_t* src = q.codes + r * q.codes_ld + c;
            if constexpr (E == 8) {
                const uint2 v = *reinterpret_cast<const uint2*>(src);
                w[i][0] = v.x, w[i][1] = v.y;
            } else {
                w[i][0] = *reinterpret_cast<const uint32_t*>(src);
            }
            b[i] = q.exps[r * q.exps_ld + (c >> 5)];
        }
        at = first;
#pragma unroll
        for (int i = 0; i < AU; ++i, at.next(per, rows32, rest32)) {
            if (at.r >= rows) break;
            const int c = static_cast<int>(at.i) * E, n = cols - c;
            const F2 unit(act8_unit(b[i]));
            float v[E];
#pragma unroll
            for (int k = 0; k < E; k += 2) {
                const uint32_t x = w[i][k / 4] ^ 0x80808080u;
                const F2 y = mul2(add2(F2(act8_raw(x, k & 3), act8_raw(x, (k & 3) + 1)), F2(-8388736.0f)),
                                  unit);
                v[k] = y.lo();
                v[k + 1] = y.hi();
            }
            T* o = out + at.r * rs + c * cs;
            if (vec && n >= E) {
                uint32_t p[E * sizeof(T) / 4];
#pragma unroll
                for (int h = 0; h < static_cast<int>(E * sizeof(T) / 4); ++h) {
                    if constexpr (sizeof(T) == 4)
                        p[h] = __float_as_uint(v[h]);
                    else
                        p[h] = round_pair(__float_as_uint(v[2 * h]), __float_as_uint(v[2 * h + 1]), 1.0f,
                                          std::is_same_v<T, __half> ? GK_F16 : GK_BF16);
                }
#pragma unroll
                for (int h = 0; h < static_cast<int>(E * sizeof(T) / 4); h += 4)
                    st_global_v4(reinterpret_cast<uint32_t*>(o) + h, p[h], p[h + 1], p[h + 2], p[h + 3]);
            } else {
#pragma unroll
                for (int k = 0; k < E; ++k)
                    if (k < n) to_out(o + k * cs, v[k]);
            }
        }
    }
}

// Blocks for pieces of e elements, `au` a lane.
dim3 piece_grid(int64_t rows, int64_t cols, int e, int au) {
    const int64_t blocks = (rows * ((cols + 31) / 32 * (32 / e)) + 256 * au - 1) / (256 * au);
    const int64_t most = static_cast<int64_t>(sm_count()) * 4;  // what is resident
    return dim3(static_cast<unsigned>(blocks < most ? blocks : most));
}

bool whole_rows(const void* p, int64_t rows, int64_t rs, int64_t cs, size_t es) {
    return cs == 1 && (rows <= 1 || rs * static_cast<int64_t>(es) % 16 == 0) &&
           (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

template <typename T>
int quantize(const gk_matref& x, const Act8Out& q, cudaStream_t st) {
    return launch_overlapped(quantize_act8_kernel<T>, piece_grid(q.rows, q.cols, piece<T>(), AU), 256, st,
                             static_cast<const T*>(x.data), static_cast<int64_t>(x.rs),
                             static_cast<int64_t>(x.cs),
                             whole_rows(x.data, q.rows, x.rs, x.cs, sizeof(T)) ? 1 : 0, q);
}

template <typename T>
int dequantize(const gk_act8_matrix& q, void* out, int64_t rs, int64_t cs, cudaStream_t st) {
    const Act8View v{q.codes, q.exps, static_cast<int64_t>(q.codes_ld), static_cast<int64_t>(q.exps_ld)};
    const int64_t rows = static_cast<int64_t>(q.rows);
    return launch_overlapped(dequantize_act8_kernel<T>, piece_grid(rows, static_cast<int64_t>(q.cols), 16 / sizeof(T), 8),
                             256, st, v, rows, static_cast<int32_t>(q.cols), static_cast<T*>(out), rs, cs,
                             whole_rows(out, rows, rs, cs, sizeof(T)) ? 1 : 0);
}

int check_type(int type) {
    if (type != GK_F32 && type != GK_F16 && type != GK_BF16)
        return api_err(GK_EINVAL, "gemmkit: unknown element type %d", type);
    return GK_OK;
}

size_t view_bytes(size_t rows, size_t cols, ptrdiff_t rs, ptrdiff_t cs, size_t es) {
    return rows && cols ? ((rows - 1) * rs + (cols - 1) * cs + 1) * es : 0;
}

}  // namespace

int check_act8(const gk_act8_matrix* q, const char* name) {
    if (!q) return api_err(GK_EINVAL, "gemmkit: null %s", name);
    if (q->rows > INT32_MAX / 2 || q->cols > INT32_MAX / 2 || q->codes_ld > INT64_MAX / 4 ||
        q->exps_ld > INT64_MAX / 4)
        return api_err(GK_EINVAL, "gemmkit: problem dimensions exceed the engine's limits");
    if (q->rows == 0 || q->cols == 0) return GK_OK;
    if (!q->codes || !q->exps) return api_err(GK_EINVAL, "gemmkit: null codes or exponents of %s", name);
    const size_t blocks = (q->cols + ACT8_BLOCK - 1) / ACT8_BLOCK;
    if (q->codes_ld % ACT8_BLOCK || q->codes_ld < q->cols)
        return api_err(GK_EINVAL,
                       "gemmkit: the pitch of %s's codes (%zu) must be a multiple of 32 that holds its "
                       "%zu columns",
                       name, q->codes_ld, q->cols);
    if (q->rows > 1 && q->exps_ld < blocks)
        return api_err(GK_EINVAL, "gemmkit: the pitch of %s's exponents (%zu) must hold %zu blocks", name,
                       q->exps_ld, blocks);
    if (reinterpret_cast<uintptr_t>(q->codes) & 15)
        return api_err(GK_EINVAL, "gemmkit: the codes of %s must be 16-byte aligned", name);
    const unsigned __int128 codes = static_cast<unsigned __int128>(q->rows - 1) * q->codes_ld + blocks * 32;
    const unsigned __int128 exps = static_cast<unsigned __int128>(q->rows - 1) * q->exps_ld + blocks;
    if (codes > q->codes_len || exps > q->exps_len)
        return api_err(GK_EINVAL, "gemmkit: %s of %zux%zu needs %zu bytes of codes (has %zu) and %zu of "
                       "exponents (has %zu)",
                       name, q->rows, q->cols, static_cast<size_t>(codes), q->codes_len,
                       static_cast<size_t>(exps), q->exps_len);
    return GK_OK;
}

}  // namespace gk

using namespace gk;

extern "C" {

int gk_quantize_act8(gk_matref x, int x_type, const gk_act8_matrix* dst, gk_stream_t stream) {
    int rc = check_act8(dst, "the destination");
    if (rc || (rc = check_type(x_type)) ||
        (rc = api_check_view(x.len, x.rows, x.cols, x.rs, x.cs, "X")))
        return rc;
    if (x.rows != dst->rows || x.cols != dst->cols)
        return api_err(GK_EINVAL, "gemmkit: the source is %zux%zu, the 8-bit matrix holds %zux%zu", x.rows,
                       x.cols, dst->rows, dst->cols);
    if (x.rows == 0 || x.cols == 0) return GK_OK;
    if (!x.data) return api_err(GK_EINVAL, "gemmkit: null X");
    const size_t es = x_type == GK_F32 ? 4 : 2;
    if ((rc = api_check_aligned(x.data, es, "X"))) return rc;
    const size_t bytes = view_bytes(x.rows, x.cols, x.rs, x.cs, es);
    if (api_overlaps(x.data, bytes, dst->codes, dst->codes_len) ||
        api_overlaps(x.data, bytes, dst->exps, dst->exps_len) ||
        api_overlaps(dst->codes, dst->codes_len, dst->exps, dst->exps_len))
        return api_err(GK_EINVAL, "gemmkit: the 8-bit matrix aliases its source or itself");
    int dev = 0;
    if ((rc = api_check_device(&dev))) return rc;
    const Act8Out q{dst->codes, dst->exps, static_cast<int64_t>(dst->codes_ld),
                    static_cast<int64_t>(dst->exps_ld), static_cast<int64_t>(dst->rows),
                    static_cast<int32_t>(dst->cols)};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return x_type == GK_F32   ? quantize<float>(x, q, st)
           : x_type == GK_F16 ? quantize<__half>(x, q, st)
                              : quantize<__nv_bfloat16>(x, q, st);
}

int gk_dequantize_act8(const gk_act8_matrix* q, gk_matmut out, int out_type, gk_stream_t stream) {
    int rc = check_act8(q, "the source");
    if (rc || (rc = check_type(out_type)) ||
        (rc = api_check_view(out.len, out.rows, out.cols, out.rs, out.cs, "C")))
        return rc;
    if (out.rows != q->rows || out.cols != q->cols)
        return api_err(GK_EINVAL, "gemmkit: the 8-bit matrix holds %zux%zu, the output is %zux%zu", q->rows,
                       q->cols, out.rows, out.cols);
    if (api_self_aliases(out.rows, out.cols, out.rs, out.cs))
        return api_err(GK_EINVAL, "gemmkit: C view aliases itself");
    if (out.rows == 0 || out.cols == 0) return GK_OK;
    if (!out.data) return api_err(GK_EINVAL, "gemmkit: null C");
    const size_t es = out_type == GK_F32 ? 4 : 2;
    if ((rc = api_check_aligned(out.data, es, "C"))) return rc;
    const size_t bytes = view_bytes(out.rows, out.cols, out.rs, out.cs, es);
    if (api_overlaps(out.data, bytes, q->codes, q->codes_len) ||
        api_overlaps(out.data, bytes, q->exps, q->exps_len))
        return api_err(GK_EINVAL, "gemmkit: C aliases the 8-bit matrix");
    int dev = 0;
    if ((rc = api_check_device(&dev))) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return out_type == GK_F32   ? dequantize<float>(*q, out.data, out.rs, out.cs, st)
           : out_type == GK_F16 ? dequantize<__half>(*q, out.data, out.rs, out.cs, st)
                                : dequantize<__nv_bfloat16>(*q, out.data, out.rs, out.cs, st);
}

int gk_gemm_act8_wgrad(int is_f16, size_t groups, const int32_t* offsets, float alpha,
                       const gk_act8_matrix* a, gk_matref b, float beta, gk_matmut c,
                       ptrdiff_t c_gs, int out_type, gk_parallelism par, gk_stream_t stream) {
    (void)par;
    int rc = check_act8(a, "A");
    if (rc) return rc;
    // A's values, in memory that the call takes and gives back
    const size_t ld = (a->cols + 7) / 8 * 8;
    gk_matref av{nullptr, a->rows * ld, a->rows, a->cols, static_cast<ptrdiff_t>(ld), 1};
    if ((rc = check_wgrad(is_f16, groups, offsets, true, alpha, av, b, c, c_gs, out_type))) return rc;
    const size_t cb = view_bytes(c.rows, c.cols, c.rs, c.cs, out_type == GK_F32 ? 4 : 2) +
                      (groups - 1) * c_gs * (out_type == GK_F32 ? 4 : 2);
    if (c.data && (api_overlaps(c.data, cb, a->codes, a->codes_len) ||
                   api_overlaps(c.data, cb, a->exps, a->exps_len)))
        return api_err(GK_EINVAL, "gemmkit: C aliases A or B");
    if (c.rows == 0 || c.cols == 0) return GK_OK;
    int dev = 0;
    if ((rc = api_check_device(&dev))) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    void* scratch = nullptr;
    if (a->rows && alpha != 0.0f) {
        if ((rc = scratch_alloc(&scratch, a->rows * ld * 2, st))) return rc;
        rc = is_f16 ? dequantize<__half>(*a, scratch, static_cast<int64_t>(ld), 1, st)
                    : dequantize<__nv_bfloat16>(*a, scratch, static_cast<int64_t>(ld), 1, st);
        av.data = scratch;
    }
    // The product's lanes lie along C's columns; where C's rows are the contiguous side it is
    // computed transposed.
    if (!rc && c.rs == 1 && c.cs != 1) {
        const gk_matmut ct{c.data, c.len, c.cols, c.rows, c.cs, c.rs};
        rc = run_wgrad(is_f16, groups, offsets, alpha, b, av, beta, ct, c_gs, out_type, st);
    } else if (!rc) {
        rc = run_wgrad(is_f16, groups, offsets, alpha, av, b, beta, c, c_gs, out_type, st);
    }
    const int fr = scratch_free(scratch, st);
    return rc ? rc : fr;
}

}  // extern "C"
