// gk_act8.cuh -- a matrix in 8 bits with a power of two per 32 elements of a row, as device code reads
// it: element (r, c) is codes[r * codes_ld + c] * 2^(exps[r * exps_ld + c / 32] - 133), the MXINT8 of the
// OCP Microscaling Formats specification v1.0 (a scale 2^(byte - 127) and elements of 1/64). An
// exponent byte of 255 makes its elements NaN.
#pragma once

#include <stdint.h>

#include "gk_sm100.cuh"

namespace gk {

constexpr int ACT8_BLOCK = 32;

struct Act8View {
    const int8_t* codes;   // 16-byte aligned, codes_ld a multiple of 32 and no less than the columns
    const uint8_t* exps;
    int64_t codes_ld, exps_ld;
};

// The value of a code of 1 under an exponent byte.
__device__ __forceinline__ float act8_unit(uint32_t b) {
    const uint32_t bits = b >= 7 ? (b - 6) << 23 : 1u << (b + 16);  // 2^(b - 133), subnormal below 7
    return __uint_as_float(b == 255 ? 0x7FFFFFFFu : bits);
}

// Code k (0 .. 3) of a word of four, each with its sign bit flipped (word ^ 0x80808080), as a float:
// placed under the exponent of 2^23 it reads 2^23 + 128 + code. (Two instructions at full rate;
// a conversion from an integer runs at a quarter of it.)
__device__ __forceinline__ float act8_raw(uint32_t flipped, int k) {  // 2^23 + 128 + code
    return __uint_as_float(__byte_perm(flipped, 0x4B000000u, 0x7650u | k));
}
__device__ __forceinline__ float act8_code(uint32_t flipped, int k) {
    return act8_raw(flipped, k) - 8388736.0f;
}

}  // namespace gk
