// gk_store.cuh -- the epilogue of the grouped and the 4-bit products: alpha * acc + beta * C in
// f32, rounded once to the output type.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "gemmkit_cuda.h"

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

}  // namespace gk
