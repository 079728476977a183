// exl3b200_norm.cu -- the row-wise operators around an expert block: block_norm (the norm behind a block with its gate
// and residual scale, and the norm before the next, one pass over the row), MXFP4 quantisation and its reverse, and the
// one-time layout of a weight's scales. sm_100a.
#include "exl3b200_dense.h"
#include "exl3b200_mx4.cuh"

#include <type_traits>

using namespace exl3b;

namespace {

// ------------------------------------------------------------------------------------------ block_norm
// Row t, all in f32:  n = branch * rsqrt(mean(branch^2) + post_eps) * post_w;  r = res_scale * res + gate * n;
// y = r * rsqrt(mean(r^2) + pre_eps) * pre_w. HBM bound: every input is read once and every output written once.
// `tpr` threads hold a row in registers (VPT vectors of eight values each), so the second mean needs no second read;
// short rows share a block (blockDim.y rows). Rows whose addresses or width rule out 16-byte vectors take the same code
// over single values, a thread's values blockDim.x apart.
template <int DT, int BT, int VPT, bool VEC>
__global__ void __launch_bounds__(1024) k_block_norm(const Exl3bNormOp p) {
    typedef typename El<DT>::T T;
    typedef typename El<BT>::T B;
    __shared__ float part[2][32];
    const int tpr = blockDim.x, tid = threadIdx.x;
    const int wid = (threadIdx.y * tpr + tid) >> 5, w0 = threadIdx.y * tpr >> 5, nw = tpr >> 5;
    const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const bool live = row < p.rows;
    const int H = (int)p.cols;
    auto at = [&](int v, int e) { return VEC ? (v * tpr + tid) * 8 + e : (v * 8 + e) * tpr + tid; };
    auto load = [&](auto dt, const void* base, int64_t pitch, int v, float x[8]) {
        constexpr int D = decltype(dt)::value;
        typedef typename El<D>::T E;
        const E* q = static_cast<const E*>(base) + pitch * row;
        if (VEC) {
            if (at(v, 0) < H) ld8<D>(q + at(v, 0), x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (at(v, e) < H) x[e] = El<D>::to(q[at(v, e)]);
        }
    };
    auto store = [&](void* base, int64_t pitch, int v, const float x[8]) {
        T* q = static_cast<T*>(base) + pitch * row;
        if (VEC) {
            if (at(v, 0) < H) st8<DT>(q + at(v, 0), x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (at(v, e) < H) q[at(v, e)] = El<DT>::from(x[e]);
        }
    };
    // the row's sum of squares, in every thread of the row, summed in the same order whatever the block's shape
    auto mean_square = [&](const float x[VPT][8], int slot) {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(x[v][e], x[v][e], s);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
        if ((tid & 31) == 0) part[slot][wid] = s;
        __syncthreads();
        s = part[slot][w0];
        for (int w = 1; w < nw; ++w) s += part[slot][w0 + w];
        return s / (float)H;
    };
    const std::integral_constant<int, DT> stream_dt;
    const std::integral_constant<int, BT> branch_dt;

    float r[VPT][8], res[VPT][8];
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) r[v][e] = res[v][e] = 0.f;
    if (live) {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            if (p.branch) load(branch_dt, p.branch, p.branch_pitch, v, r[v]);
            if (p.res) load(stream_dt, p.res, p.res_pitch, v, res[v]);
        }
    }
    if (p.post_w) {
        const float s = __frsqrt_rn(mean_square(r, 0) + p.post_eps);
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            float w[8] = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };
            load(stream_dt, p.post_w, 0, v, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) r[v][e] = r[v][e] * s * w[e];
        }
    }
    if (p.gate_kind == EXL3B_GATE_TOKEN) {
        const float g = live ? 1.f / (1.f + expf(-static_cast<const float*>(p.gate)[row])) : 0.f;
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) r[v][e] *= g;
    } else if (p.gate_kind != EXL3B_GATE_NONE && live) {
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            float g[8] = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };
            load(stream_dt, p.gate, p.gate_kind == EXL3B_GATE_ELEMENT ? p.gate_pitch : 0, v, g);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                r[v][e] *= p.gate_kind == EXL3B_GATE_ELEMENT ? 1.f / (1.f + expf(-g[e])) : g[e];
        }
    }
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[v][e] = p.res ? fmaf(res[v][e], p.res_scale, r[v][e]) : r[v][e];
        if (p.out && live) store(p.out, p.out_pitch, v, r[v]);
    }
    if (!p.pre_w) return;
    const float s = __frsqrt_rn(mean_square(r, 1) + p.pre_eps);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        float w[8] = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };
        load(stream_dt, p.pre_w, 0, v, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) r[v][e] = r[v][e] * s * w[e];
        if (p.y && live) store(p.y, p.y_pitch, v, r[v]);
        if (VEC && p.q) {      // four neighbouring lanes hold a block of 32
            const uint32_t code = mx4_quad_code(r[v]);
            if (live && at(v, 0) < H) {
                *reinterpret_cast<uint32_t*>(p.q + row * p.q_pitch + at(v, 0) / 2) = mx4_pack8(r[v], code);
                if ((tid & 3) == 0) p.q_scales[row * p.qs_pitch + at(v, 0) / 32] = (uint8_t)code;
            }
        }
    }
}

template <int DT, int BT>
int launch_norm(const Exl3bNormOp* p, bool vec, cudaStream_t st) {
    const int64_t n8 = (p->cols + 7) / 8;
    const int vpt = n8 <= 1024 ? 1 : n8 <= 2048 ? 2 : 4;
    const int tpr = (int)(((n8 + vpt - 1) / vpt + 31) / 32 * 32);
    const int rpb = tpr >= 128 ? 1 : 128 / tpr;
    const int64_t grid = (p->rows + rpb - 1) / rpb;
    const dim3 block(tpr, rpb);
    if (vec) {
        if (vpt == 1) k_block_norm<DT, BT, 1, true><<<(unsigned)grid, block, 0, st>>>(*p);
        else if (vpt == 2) k_block_norm<DT, BT, 2, true><<<(unsigned)grid, block, 0, st>>>(*p);
        else k_block_norm<DT, BT, 4, true><<<(unsigned)grid, block, 0, st>>>(*p);
    } else {
        if (vpt == 1) k_block_norm<DT, BT, 1, false><<<(unsigned)grid, block, 0, st>>>(*p);
        else if (vpt == 2) k_block_norm<DT, BT, 2, false><<<(unsigned)grid, block, 0, st>>>(*p);
        else k_block_norm<DT, BT, 4, false><<<(unsigned)grid, block, 0, st>>>(*p);
    }
    return cudaGetLastError() == cudaSuccess ? 0 : -6;
}

// ------------------------------------------------------------------------------------------ MXFP4 rows
// HBM bound: 16-byte loads, eight values a thread, a block's scale from four neighbouring lanes. blockIdx.y walks the
// rows (grid-stride), blockIdx.x the row's vectors.
template <int DT>
__global__ void __launch_bounds__(256) k_mx4_quantize(const void* x, int64_t x_pitch, int64_t rows, int cols,
                                                      uint8_t* q, int64_t q_pitch, uint8_t* qs, int64_t qs_pitch) {
    typedef typename El<DT>::T T;
    const int c = (blockIdx.x * 256 + threadIdx.x) * 8;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        float v[8] = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };
        if (c < cols) ld8<DT>(static_cast<const T*>(x) + row * x_pitch + c, v);
        const uint32_t code = mx4_quad_code(v);
        if (c < cols) {
            *reinterpret_cast<uint32_t*>(q + row * q_pitch + c / 2) = mx4_pack8(v, code);
            if ((threadIdx.x & 3) == 0) qs[row * qs_pitch + c / 32] = (uint8_t)code;
        }
    }
}

// e2m1 code -> f32: the sign bit, then 0 .5 1 1.5 2 3 4 6 from a packed table of halves of those values' doubles.
__device__ __forceinline__ float e2m1_value(uint32_t n) {
    const float m = 0.5f * (float)((0xC8643210u >> ((n & 7u) * 4)) & 15u);
    return n & 8u ? -m : m;
}

template <int DT>
__global__ void __launch_bounds__(256) k_mx4_dequantize(const uint8_t* q, int64_t q_pitch, const uint8_t* qs,
                                                        int64_t qs_pitch, int64_t rows, int cols, void* y,
                                                        int64_t y_pitch) {
    typedef typename El<DT>::T T;
    const int c = (blockIdx.x * 256 + threadIdx.x) * 8;
    if (c >= cols) return;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const uint32_t n = *reinterpret_cast<const uint32_t*>(q + row * q_pitch + c / 2);
        const float s = mx4_scale(qs[row * qs_pitch + c / 32]);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = e2m1_value(n >> (4 * i)) * s;
        st8<DT>(static_cast<T*>(y) + row * y_pitch + c, v);
    }
}

// A weight's row-major scales [E][rows][cols / 32] -> the tiles the product's kernel copies whole: per expert, per block
// of 128 weight rows, per 128 input columns 512 bytes, row r's four scales at (r % 32) * 16 + (r / 32) * 4. With
// silu_mul a block is 64 gate rows then their 64 up rows. Rows and columns past the weight's get code 0.
__global__ void __launch_bounds__(256) k_mx4_tile(const uint8_t* s, int64_t s_pitch, int64_t e_pitch, int64_t rows,
                                                  int64_t cols, int act, int64_t n_blk, int64_t n_k, int64_t total,
                                                  uint32_t* out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t tile = i >> 7;
        const int w = (int)(i & 127), r = (w >> 2) + 32 * (w & 3);       // word w: row r's four scales
        const int64_t kb = tile % n_k, blk = tile / n_k % n_blk, e = tile / n_k / n_blk;
        const int64_t half = rows / 2, j = blk * 64 + (r & 63);
        const int64_t row = act ? (j < half ? (r < 64 ? j : half + j) : rows) : blk * 128 + r;
        uint32_t v = 0;
        for (int b = 0; b < 4; ++b) {
            const int64_t c = kb * 4 + b;
            if (row < rows && c < cols / 32) v |= (uint32_t)s[e * e_pitch + row * s_pitch + c] << (8 * b);
        }
        out[i] = v;
    }
}

}  // namespace

extern "C" {

int exl3b_cuda_block_norm(const Exl3bNormOp* p, int dtype, int branch_dtype, int vec, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype * 4 + branch_dtype) {
    case 1 * 4 + 1: return launch_norm<1, 1>(p, vec, st);
    case 1 * 4 + 2: return launch_norm<1, 2>(p, vec, st);
    case 1 * 4 + 3: return launch_norm<1, 3>(p, vec, st);
    case 2 * 4 + 1: return launch_norm<2, 1>(p, vec, st);
    case 2 * 4 + 2: return launch_norm<2, 2>(p, vec, st);
    case 2 * 4 + 3: return launch_norm<2, 3>(p, vec, st);
    case 3 * 4 + 1: return launch_norm<3, 1>(p, vec, st);
    case 3 * 4 + 2: return launch_norm<3, 2>(p, vec, st);
    case 3 * 4 + 3: return launch_norm<3, 3>(p, vec, st);
    default: return -2;
    }
}

int exl3b_cuda_mx4_quantize(const void* x, int dtype, int64_t x_pitch, int64_t rows, int64_t cols, uint8_t* q,
                            int64_t q_pitch, uint8_t* qs, int64_t qs_pitch, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((cols / 8 + 255) / 256), (unsigned)(rows < 65535 ? rows : 65535));
    if (dtype == 1) k_mx4_quantize<1><<<grid, 256, 0, st>>>(x, x_pitch, rows, (int)cols, q, q_pitch, qs, qs_pitch);
    else if (dtype == 2) k_mx4_quantize<2><<<grid, 256, 0, st>>>(x, x_pitch, rows, (int)cols, q, q_pitch, qs, qs_pitch);
    else k_mx4_quantize<3><<<grid, 256, 0, st>>>(x, x_pitch, rows, (int)cols, q, q_pitch, qs, qs_pitch);
    return cudaGetLastError() == cudaSuccess ? 0 : -6;
}

int exl3b_cuda_mx4_dequantize(const uint8_t* q, int64_t q_pitch, const uint8_t* qs, int64_t qs_pitch, int64_t rows,
                              int64_t cols, void* y, int dtype, int64_t y_pitch, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)((cols / 8 + 255) / 256), (unsigned)(rows < 65535 ? rows : 65535));
    if (dtype == 1) k_mx4_dequantize<1><<<grid, 256, 0, st>>>(q, q_pitch, qs, qs_pitch, rows, (int)cols, y, y_pitch);
    else if (dtype == 2) k_mx4_dequantize<2><<<grid, 256, 0, st>>>(q, q_pitch, qs, qs_pitch, rows, (int)cols, y, y_pitch);
    else k_mx4_dequantize<3><<<grid, 256, 0, st>>>(q, q_pitch, qs, qs_pitch, rows, (int)cols, y, y_pitch);
    return cudaGetLastError() == cudaSuccess ? 0 : -6;
}

int exl3b_cuda_mx4_tile(const uint8_t* s, int64_t s_pitch, int64_t e_pitch, int64_t n_expert, int64_t rows, int64_t cols,
                        int act, int64_t n_blk, int64_t n_k, void* out, void* stream) {
    const int64_t total = n_expert * n_blk * n_k * 128;
    const int64_t want = (total + 255) / 256;
    k_mx4_tile<<<(unsigned)(want < 65536 ? want : 65536), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        s, s_pitch, e_pitch, rows, cols, act, n_blk, n_k, total, static_cast<uint32_t*>(out));
    return cudaGetLastError() == cudaSuccess ? 0 : -6;
}

}  // extern "C"
