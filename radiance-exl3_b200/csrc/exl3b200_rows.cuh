// exl3b200_rows.cuh -- rows of f32, f16 or bf16 values, eight at a time. sm_100a.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "exl3b200_dense.h"

namespace exl3b {

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

// Eight values as they lie in memory.
template <int DT>
struct Raw {
    typedef typename El<DT>::T T;
    uint4 q[DT == 1 ? 2 : 1];
    __device__ __forceinline__ void clear() {
        q[0] = make_uint4(0u, 0u, 0u, 0u);
        if (DT == 1) q[DT == 1] = q[0];
    }
    __device__ __forceinline__ void fetch(const T* p) {
        q[0] = *reinterpret_cast<const uint4*>(p);
        if (DT == 1) q[DT == 1] = *(reinterpret_cast<const uint4*>(p) + 1);
    }
    __device__ __forceinline__ void set(int e, T v) { reinterpret_cast<T*>(q)[e] = v; }
    __device__ __forceinline__ void get(float x[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = El<DT>::to(reinterpret_cast<const T*>(q)[e]);
    }
};

// Vector i's row and place in it; BIG: vectors past 2^31, a 64-bit division.
template <bool BIG>
__device__ __forceinline__ void row_of(int64_t i, const Exl3bDiv& v, int64_t* row, int* vec) {
    if (BIG) {
        *row = i / v.d;
        *vec = (int)(i - *row * v.d);
    } else {
        const uint32_t n = (uint32_t)i, q = exl3b_div_of(n, v);
        *row = q;
        *vec = (int)(n - q * v.d);
    }
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

}  // namespace exl3b
