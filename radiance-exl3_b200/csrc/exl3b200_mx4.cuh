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

// ------------------------------------------------------------------------------------------ rows of 8 values
// dtype codes: RAD_F32 1, RAD_F16 2, RAD_BF16 3 (include/rad_types.h).
template <int DT>
struct El;
template <>
struct El<1> {
    typedef float T;
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct El<2> {
    typedef __half T;
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <>
struct El<3> {
    typedef __nv_bfloat16 T;
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// Eight consecutive values at a 16-byte aligned address.
__device__ __forceinline__ void ld8(const float* p, float v[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <int DT>
__device__ __forceinline__ void st8(void* p, const float v[8]) {
    if constexpr (DT == 1) {
        *static_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *(static_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        typedef typename El<DT>::T T;
        uint4 a;
        T* e = reinterpret_cast<T*>(&a);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = El<DT>::from(v[i]);
        *static_cast<uint4*>(p) = a;
    }
}

}  // namespace exl3b
