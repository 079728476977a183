// exl3b200_f8.cu -- FP8 rows: f32, f16 or bf16 values to e4m3 codes with an f32 scale for each 128 values of a row, and back.
// sm_100a.
//
// A block's scale is m / 448, m the block's largest magnitude but no less than 2^-110 (so that the scale and 448 / m are
// normal numbers), and a code the e4m3 value nearest x * (448 / m), ties to even: f32 numbers, each quotient and product
// rounded to nearest once. pow2: the least power of two from that scale on, and x divided by it, which is exact. A block that
// holds a NaN or an infinity has scale NaN and codes 0.
//
// HBM bound: sixteen lanes hold a block, eight values each, and a thread takes kUnroll blocks' worth, all loaded before the
// first is used. Measured on one B200 (copies at 6.5 TB/s), 20480 x 4096 bf16: there 40.0 us, 6.4 TB/s, back 38.8 us, 6.6 TB/s;
// 20480 x 2048 f32 31.3 and 43.9 us; 9000 x 640 bf16, whose scales lie apart, 4.5 us (latency); 64 x 2048: a launch each, 1.9 us.
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "exl3b200_chain.cuh"
#include "exl3b200_dense.h"
#include "exl3b200_rows.cuh"

using namespace exl3b;

namespace {

constexpr int kUnroll = 4;
constexpr uint32_t kInf = 0x7F800000u;

// The largest magnitude of eight values as f32 bits, which order as integers (a NaN above infinity).
template <int DT>
__device__ __forceinline__ uint32_t top_of(const Raw<DT>& x) {
    if constexpr (DT == RAD_F32) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            m = max(max(max(m, x.q[i].x & 0x7FFFFFFFu), x.q[i].y & 0x7FFFFFFFu), max(x.q[i].z & 0x7FFFFFFFu, x.q[i].w & 0x7FFFFFFFu));
        return m;
    } else {
        const uint32_t k = 0x7FFF7FFFu;
        uint32_t m = max_u16x2(max_u16x2(x.q[0].x & k, x.q[0].y & k), max_u16x2(x.q[0].z & k, x.q[0].w & k));
        m = max(m & 0xFFFFu, m >> 16);
        return DT == RAD_BF16 ? m << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    }
}

// Four values, rounded to e4m3, v[0] in the lowest byte.
__device__ __forceinline__ uint32_t e4m3x4(const float v[4]) {
    uint32_t r;
    asm("{\n .reg .b16 a, b;\n cvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n"
        " mov.b32 %0, {a, b};\n}\n"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
    return r;
}

// A row is nb blocks of 16 lanes; lane c of the row holds values 8 c .. 8 c + 7, if the row has them. FLAT: whole blocks, and
// rows without gaps in all three arrays, so that a lane's number is its place (with rows and places worked out, 20480 x 4096
// bf16 takes 50.5 us where it takes 40.0).
template <int DT, bool BIG, bool FLAT>
__global__ void __launch_bounds__(256) k_f8_quantize(const void* x, int64_t x_pitch, int64_t n_lane, Exl3bDiv div, int cols,
                                                     uint8_t* q, int64_t q_pitch, float* s, int64_t s_pitch, int pow2) {
    typedef typename El<DT>::T T;
    chain_wait();
    chain_next();
    const int64_t i0 = (int64_t)blockIdx.x * (256 * kUnroll) + threadIdx.x;
    Raw<DT> v[kUnroll];
    int64_t row[kUnroll];
    int c[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        v[u].clear();
        if constexpr (FLAT) {
            if (i0 + 256 * u < n_lane) v[u].fetch(static_cast<const T*>(x) + 8 * (i0 + 256 * u));
        } else {
            row_of<BIG>(i0 + 256 * u, div, &row[u], &c[u]);
            if (i0 + 256 * u < n_lane && 8 * c[u] < cols) v[u].fetch(static_cast<const T*>(x) + row[u] * x_pitch + 8 * c[u]);
        }
    }
    uint32_t m[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        m[u] = top_of<DT>(v[u]);
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) m[u] = max(m[u], __shfl_xor_sync(0xFFFFFFFFu, m[u], d));
    }
    // one quotient a lane: lane u of the sixteen has block u's scale, lane 4 + u what its values are multiplied by
    static_assert(kUnroll == 4, "lanes");
    const int lane = threadIdx.x & 31, at = lane & 15;
    const uint32_t mine = at & 2 ? (at & 1 ? m[3] : m[2]) : (at & 1 ? m[1] : m[0]);
    const float top = fmaxf(__uint_as_float(mine), 0x1p-110f);
    float quot = __fdiv_rn(at & 4 ? 448.f : top, at & 4 ? top : 448.f);
    if (pow2) {                                               // lane 4 + u has to know lane u's
        const uint32_t b = (__float_as_uint(__shfl_sync(0xFFFFFFFFu, quot, lane & ~4)) + 0x7FFFFFu) & kInf;
        quot = __uint_as_float(at & 4 ? (254u << 23) - b : b);
    }
    if (mine >= kInf) quot = __uint_as_float(0x7FFFFFFFu);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const float inv = __shfl_sync(0xFFFFFFFFu, quot, (lane & 16) + 4 + u);
        if (i0 + 256 * u >= n_lane) continue;
        float f[8];
        v[u].get(f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __fmul_rn(f[e], inv);
        const uint2 w = m[u] >= kInf ? make_uint2(0u, 0u) : make_uint2(e4m3x4(f), e4m3x4(f + 4));
        if constexpr (FLAT) {
            *reinterpret_cast<uint2*>(q + 8 * (i0 + 256 * u)) = w;
            if (at == u) s[(i0 + 256 * u) >> 4] = quot;
        } else {
            if (8 * c[u] < cols) *reinterpret_cast<uint2*>(q + row[u] * q_pitch + 8 * c[u]) = w;
            if (at == u) s[row[u] * s_pitch + (c[u] >> 4)] = quot;
        }
    }
}

// Vectors of eight codes, a row's laid end to end.
template <int DT, bool BIG>
__global__ void __launch_bounds__(256) k_f8_dequantize(const uint8_t* q, int64_t q_pitch, const float* s, int64_t s_pitch,
                                                       int64_t n_vec, Exl3bDiv div, void* y, int64_t y_pitch) {
    typedef typename El<DT>::T T;
    chain_wait();
    chain_next();
    const int64_t i0 = (int64_t)blockIdx.x * (256 * kUnroll) + threadIdx.x;
    uint2 n[kUnroll];
    float scale[kUnroll];
    int64_t row[kUnroll];
    int c[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        row_of<BIG>(i0 + 256 * u, div, &row[u], &c[u]);
        if (i0 + 256 * u >= n_vec) continue;
        n[u] = *reinterpret_cast<const uint2*>(q + row[u] * q_pitch + 8 * c[u]);
        scale[u] = s[row[u] * s_pitch + (c[u] >> 4)];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        if (i0 + 256 * u >= n_vec) continue;
        float v[8];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const uint32_t w = h < 2 ? n[u].x : n[u].y;
            uint32_t r;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)(w >> (16 * (h & 1)))));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
            v[2 * h] = __fmul_rn(f.x, scale[u]);
            v[2 * h + 1] = __fmul_rn(f.y, scale[u]);
        }
        st8<DT>(static_cast<T*>(y) + row[u] * y_pitch + 8 * c[u], v);
    }
}

}  // namespace

#define EXL3B_F8_ROWS(KERN, DT, ...)                                                                                       \
    do {                                                                                                                   \
        if (n < (1ll << 31) - 1024) return chain_launch(KERN<DT, false>, dim3(grid), dim3(256), 0, 1, st, __VA_ARGS__);    \
        return chain_launch(KERN<DT, true>, dim3(grid), dim3(256), 0, 1, st, __VA_ARGS__);                                 \
    } while (0)

extern "C" {

int exl3b_cuda_f8_quantize(const void* x, int dtype, int64_t x_pitch, int64_t rows, int64_t cols, uint8_t* q, int64_t q_pitch,
                           float* s, int64_t s_pitch, int pow2, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t nb = (cols + 127) / 128, n = rows * nb * 16;
    const unsigned grid = (unsigned)((n + 256 * kUnroll - 1) / (256 * kUnroll));
    const Exl3bDiv div = exl3b_div((uint32_t)(nb * 16));
    const bool flat = cols % 128 == 0 && x_pitch == cols && q_pitch == cols && s_pitch == nb;
#define EXL3B_F8_QUANT(DT)                                                                                                        \
    do {                                                                                                                          \
        auto kern = flat ? k_f8_quantize<DT, true, true> : n < (1ll << 31) - 1024 ? k_f8_quantize<DT, false, false>               \
                                                                                  : k_f8_quantize<DT, true, false>;               \
        return chain_launch(kern, dim3(grid), dim3(256), 0, 1, st, x, x_pitch, n, div, (int)cols, q, q_pitch, s, s_pitch, pow2);  \
    } while (0)
    if (dtype == RAD_F32) EXL3B_F8_QUANT(RAD_F32);
    if (dtype == RAD_F16) EXL3B_F8_QUANT(RAD_F16);
    EXL3B_F8_QUANT(RAD_BF16);
#undef EXL3B_F8_QUANT
}

int exl3b_cuda_f8_dequantize(const uint8_t* q, int64_t q_pitch, const float* s, int64_t s_pitch, int64_t rows, int64_t cols,
                             void* y, int dtype, int64_t y_pitch, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t n = rows * (cols / 8);
    const unsigned grid = (unsigned)((n + 256 * kUnroll - 1) / (256 * kUnroll));
    const Exl3bDiv div = exl3b_div((uint32_t)(cols / 8));
    if (dtype == RAD_F32) EXL3B_F8_ROWS(k_f8_dequantize, RAD_F32, q, q_pitch, s, s_pitch, n, div, y, y_pitch);
    if (dtype == RAD_F16) EXL3B_F8_ROWS(k_f8_dequantize, RAD_F16, q, q_pitch, s, s_pitch, n, div, y, y_pitch);
    EXL3B_F8_ROWS(k_f8_dequantize, RAD_BF16, q, q_pitch, s, s_pitch, n, div, y, y_pitch);
}

}  // extern "C"
