// exl3b200_mx4.cuh -- MXFP4 on the device: blocks of 32 values, each an e2m1 code (two a byte, the lower index in the
// low nibble), times one power of two held as E8M0 (2^(code - 127); 255 is NaN).
//
// A block's scale is 2^(floor(log2 amax) - 2), so its largest magnitude lands in [4, 8) of e2m1's grid
// 0 .5 1 1.5 2 3 4 6: floor(log2) is the exponent field of amax's f32 bits, and the division by the scale is exact.
// Values are rounded to nearest, ties to the even mantissa, those above 6 saturate. amax = 0 and exponents below
// 2^-127 take code 0; a block that holds a NaN or an infinity takes code 255 and zero codes.
#pragma once
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "exl3b200_rows.cuh"

namespace exl3b {

constexpr uint32_t kMx4Nan = 255;

// The magnitude's f32 bits, ordered as unsigned integers: finite < infinity < NaN, so a maximum keeps a NaN.
__device__ __forceinline__ uint32_t mx4_mag(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t mx4_scale_code(uint32_t mag) {
    const uint32_t e = mag >> 23;
    return e == 255 ? kMx4Nan : e > 2 ? e - 2 : 0u;
}
__device__ __forceinline__ float mx4_inv_scale(uint32_t code) {   // 2^(127 - code); code <= 252
    return __uint_as_float((254u - code) << 23);
}
__device__ __forceinline__ float mx4_scale(uint32_t code) {       // 2^(code - 127); 2^-127 is subnormal
    return code == kMx4Nan ? __uint_as_float(0x7FFFFFFFu) : code ? __uint_as_float(code << 23) : __uint_as_float(1u << 22);
}
// Eight values of a block of scale code `code` as eight codes, v[0] in the lowest nibble.
__device__ __forceinline__ uint32_t mx4_pack8(const float v[8], uint32_t code) {
    if (code == kMx4Nan) return 0u;
    const float s = mx4_inv_scale(code);
    uint32_t r;
    asm("{\n .reg .b8 a, b, c, d;\n"
        " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        " mov.b32 %0, {a, b, c, d};\n}\n"
        : "=r"(r)
        : "f"(v[0] * s), "f"(v[1] * s), "f"(v[2] * s), "f"(v[3] * s), "f"(v[4] * s), "f"(v[5] * s), "f"(v[6] * s),
          "f"(v[7] * s));
    return r;
}
// The four lanes of an aligned quad hold a block's 32 values, eight each: its scale code, in all four.
__device__ __forceinline__ uint32_t mx4_quad_code(const float v[8]) {
    uint32_t m = mx4_mag(v[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max(m, mx4_mag(v[i]));
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    return mx4_scale_code(m);
}

}  // namespace exl3b
