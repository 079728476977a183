// exl3b200_norm.cu -- the row-wise operators around an expert block: block_norm (the norm behind a block with its gate
// and residual scale, and the norm before the next, one pass over the row), MXFP4 quantisation and its reverse, and the
// one-time layout of a weight's scales. sm_100a.
#include "exl3b200_chain.cuh"
#include "exl3b200_dense.h"
#include "exl3b200_mx4.cuh"

#include <type_traits>

using namespace exl3b;

namespace {

// ------------------------------------------------------------------------------------------ block_norm
// Row t, all in f32:  n = branch * rsqrt(mean(branch^2) + post_eps) * post_w;  r = res_scale * res + gate * n;
// y = r * rsqrt(mean(r^2) + pre_eps) * pre_w. HBM bound: every input is read once and every output written once.
// `tpr` threads hold a row (VPT vectors of eight values each), so the second mean needs no second read of HBM; short rows
// share a block (blockDim.y rows). A row's fixed cost -- two reductions, its addresses -- is paid by fewer
// instructions the more values a thread holds (the kernel is near the issue limit: 640 instructions a warp and 256 values
// with one vector a thread, half of that with four); few short rows take one vector, since there a row's latency counts.
// Rows whose addresses or width rule out 16-byte vectors take the same code over single values, a thread's values
// blockDim.x apart.
// What a thread holds is in registers for 16-byte rows of up to 8192 values (an f32 row with an element gate: but for 100
// bytes). Not so for longer rows, whose 1024 threads have 64 registers each (24 bytes of a thread's values go through local
// memory in f16, 200 to 310 in bf16 and f32), and for single values, put into their words one by one (280 to 570 bytes, f32
// 680 to 1020; over 8192 values 1000 to 1490).
// Measured on one B200 (copies at 6.5 TB/s): 16384 rows of 4096, f32 branch, token gate, both norms, bf16 and MXFP4 out:
// 126 us, 5.6 TB/s. 2048 rows of 2560 in f16 with an element gate: 14.6 us, 3.6 TB/s: 14 rows an SM, too few rounds of
// load, two reductions and store to hide one another. One row of 2048: 2.8 us, a launch. f32 branch, both norms, bf16:
// 4096 rows of 2048 in 19 us, of 2047 in 103 (local memory); 2048 of 8192 in 34 us, 5.0 TB/s; 1024 of 16384 in 51 (f16: 35).
// r / (1 + e^-g), within 2^-19 of the value down to the bottom of f32's range. From kGateLow up both functions are the
// special-function unit's; below it, rare enough for a branch, the rounding of the exponential's argument would pass that
// bound, and below -60, where 1 + e^-g is e^-g to every bit, r e^(g/2) e^(g/2) stays in range while the value does.
constexpr float kGateLow = -16.f;
__device__ __forceinline__ float sigmoid(float g) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + __expf(-g)));
    return r;
}
__device__ __forceinline__ float gated(float r, float g) {
    if (!(g < kGateLow)) return r * sigmoid(g);
    const float e = expf(g < -60.f ? 0.5f * g : -g);
    return g < -60.f ? r * e * e : r / (1.f + e);
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

template <int DT, int BT, int VPT, int MAXT, bool VEC>
__global__ void __launch_bounds__(MAXT, MAXT <= 512 ? 2 : 1) k_block_norm(const Exl3bNormOp p) {
    typedef typename El<DT>::T T;
    typedef typename El<BT>::T B;
    constexpr int NW = MAXT / 32;                       // partial sums a row; those of warps it lacks stay zero
    __shared__ __align__(16) float part[2][2][MAXT > 512 ? 1 : 4][NW];
    const int tpr = blockDim.x, tid = threadIdx.x, ty = threadIdx.y;
    const int H = (int)p.cols;
    const float inv_h = 1.f / (float)H;
    for (int i = ty * tpr + tid; i < (int)(sizeof part / 4); i += tpr * blockDim.y) (&part[0][0][0][0])[i] = 0.f;
    chain_wait();
    chain_next();
    __syncthreads();
    const std::integral_constant<int, DT> stream_dt;
    const std::integral_constant<int, BT> branch_dt;
    auto at = [&](int v, int e) { return VEC ? (v * tpr + tid) * 8 + e : (v * 8 + e) * tpr + tid; };
    // a row's values (`q` its address), or zeros where there are none
    auto load = [&](auto dt, const void* row_at, int v, auto& x) {
        const auto* q = static_cast<const typename El<decltype(dt)::value>::T*>(row_at);
        x.clear();
        if (!q) return;
        if (VEC) {
            if (at(v, 0) < H) x.fetch(q + at(v, 0));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (at(v, e) < H) x.set(e, q[at(v, e)]);
        }
    };
    auto store = [&](T* q, int v, const float x[8]) {
        if (VEC) {
            if (at(v, 0) < H) st8<DT>(q + at(v, 0), x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (at(v, e) < H) q[at(v, e)] = El<DT>::from(x[e]);
        }
    };
    // the row's mean square, in every thread of the row; two buffers in turn, so that one barrier a sum does
    int turn = 0;
    auto mean_square = [&](const float x[VPT][8], int slot) {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf(x[v][e], x[v][e], s);
#pragma unroll
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
        float* sums = part[slot][turn][ty];
        if ((tid & 31) == 0) sums[tid >> 5] = s;
        __syncthreads();
        s = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w += 4) {
            const float4 f = *reinterpret_cast<const float4*>(sums + w);
            s += (f.x + f.y) + (f.z + f.w);
        }
        return s * inv_h;
    };
    const bool gates = p.gate_kind == EXL3B_GATE_ELEMENT || p.gate_kind == EXL3B_GATE_CHANNEL;
    const int64_t step = (int64_t)gridDim.x * blockDim.y;
    int64_t row = (int64_t)blockIdx.x * blockDim.y + ty;
    for (int64_t first = (int64_t)blockIdx.x * blockDim.y; first < p.rows; first += step, row += step, turn ^= 1) {
        const bool live = row < p.rows;
        const T* res_at = p.res && live ? static_cast<const T*>(p.res) + row * p.res_pitch : nullptr;
        const B* branch_at = p.branch && live ? static_cast<const B*>(p.branch) + row * p.branch_pitch : nullptr;
        const T* gate_at = !gates || !live ? nullptr
                           : static_cast<const T*>(p.gate) + (p.gate_kind == EXL3B_GATE_ELEMENT ? row * p.gate_pitch : 0);
        const float token = p.gate_kind == EXL3B_GATE_TOKEN && live ? static_cast<const float*>(p.gate)[row] : 0.f;
        // An element gate's registers leave few rows in flight: the next row's lines are asked into L2 meanwhile (9600 x 4096
        // 77.8 and 73.7 us, 2048 x 2560 15.5 without; not for 128 threads a row, 4096 x 2048 19.7 and 20.6; the other gates
        // gain nothing)
        if (VEC && p.gate_kind == EXL3B_GATE_ELEMENT && tpr > 128 && row + step < p.rows) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                const int c = at(v, 0);
                if (c < H && c % (128 / (int)sizeof(T)) == 0) {
                    prefetch_l2(gate_at + step * p.gate_pitch + c);
                    if (p.res) prefetch_l2(res_at + step * p.res_pitch + c);
                }
                if (p.branch && c < H && c % (128 / (int)sizeof(B)) == 0) prefetch_l2(branch_at + step * p.branch_pitch + c);
            }
        }
        // the row's loads first (the longest rows have registers for the branch alone)
        constexpr bool AHEAD = MAXT <= 512;
        float r[VPT][8];
        Raw<DT> res[VPT], gate[VPT];
        {
            Raw<BT> b[VPT];
#pragma unroll
            for (int v = 0; v < VPT; ++v) load(branch_dt, branch_at, v, b[v]);
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                if (AHEAD) load(stream_dt, res_at, v, res[v]);
                if (AHEAD && VPT <= 2) load(stream_dt, gate_at, v, gate[v]);
            }
#pragma unroll
            for (int v = 0; v < VPT; ++v) b[v].get(r[v]);
        }
        if (p.post_w) {
            Raw<DT> w[VPT];
#pragma unroll
            for (int v = 0; v < VPT; ++v) load(stream_dt, p.post_w, v, w[v]);
            const float s = __frsqrt_rn(mean_square(r, 0) + p.post_eps);
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                float f[8];
                w[v].get(f);
#pragma unroll
                for (int e = 0; e < 8; ++e) r[v][e] = r[v][e] * s * f[e];
            }
        }
        if (p.gate_kind == EXL3B_GATE_TOKEN) {
            const bool far = token < -60.f;                  // as gated: e^(g/2) twice
            const float f = gated(1.f, far ? 0.5f * token : token);
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) r[v][e] = far ? r[v][e] * f * f : r[v][e] * f;
        } else if (gates) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                float f[8];
                if (!AHEAD || VPT > 2) load(stream_dt, gate_at, v, gate[v]);
                gate[v].get(f);
                if (p.gate_kind == EXL3B_GATE_ELEMENT) {
                    float least = f[0];
#pragma unroll
                    for (int e = 1; e < 8; ++e) least = fminf(least, f[e]);
                    if (least < kGateLow) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) r[v][e] = gated(r[v][e], f[e]);
                        continue;
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = sigmoid(f[e]);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) r[v][e] *= f[e];
            }
        }
        if (p.res) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                float f[8];
                if (!AHEAD) load(stream_dt, res_at, v, res[v]);
                res[v].get(f);
#pragma unroll
                for (int e = 0; e < 8; ++e) r[v][e] = fmaf(f[e], p.res_scale, r[v][e]);
            }
        }
        if (p.out && live) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) store(static_cast<T*>(p.out) + row * p.out_pitch, v, r[v]);
        }
        if (!p.pre_w) continue;
        Raw<DT> w[VPT];
#pragma unroll
        for (int v = 0; v < VPT; ++v) load(stream_dt, p.pre_w, v, w[v]);
        const float s = __frsqrt_rn(mean_square(r, 1) + p.pre_eps);
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            float f[8];
            w[v].get(f);
#pragma unroll
            for (int e = 0; e < 8; ++e) r[v][e] = r[v][e] * s * f[e];
        }
        if (p.y && live) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) store(static_cast<T*>(p.y) + row * p.y_pitch, v, r[v]);
        }
        if (VEC && p.q) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) {      // four neighbouring lanes hold a block of 32
                const uint32_t code = mx4_quad_code(r[v]);
                if (live && at(v, 0) < H) {
                    *reinterpret_cast<uint32_t*>(p.q + row * p.q_pitch + at(v, 0) / 2) = mx4_pack8(r[v], code);
                    if ((tid & 3) == 0) p.q_scales[row * p.qs_pitch + at(v, 0) / 32] = (uint8_t)code;
                }
            }
        }
    }
}

template <int DT, int BT, int VPT, int MAXT>
int launch_norm_t(const Exl3bNormOp* p, bool vec, int sm_count, cudaStream_t st) {
    const int64_t n8 = (p->cols + 7) / 8;
    const int tpr = (int)(((n8 + VPT - 1) / VPT + 31) / 32 * 32);
    const int rpb = tpr >= 128 || MAXT > 512 ? 1 : 128 / tpr;
    const int64_t want = (p->rows + rpb - 1) / rpb, room = (int64_t)sm_count * (2048 / (tpr * rpb));
    const unsigned grid = (unsigned)(want < room ? want : room);
    const dim3 block(tpr, rpb);
    return vec ? chain_launch(k_block_norm<DT, BT, VPT, MAXT, true>, dim3(grid), block, 0, 1, st, *p)
               : chain_launch(k_block_norm<DT, BT, VPT, MAXT, false>, dim3(grid), block, 0, 1, st, *p);
}

template <int DT, int BT>
int launch_norm(const Exl3bNormOp* p, bool vec, int sm_count, cudaStream_t st) {
    const int64_t n8 = (p->cols + 7) / 8;
    // one B200, f32 branch, both norms: 2400 x 2048 in 20.5 / 15.1 / 14.5 us at 1 / 2 / 4 vectors a thread, 9600 x 4096 in
    // 100 / 80 / 72; an element gate's registers turn the last two round (9600 x 4096, bf16 branch: 111 / 95 / 112); one
    // row of 2048 in 2.9 / 3.5 / 3.6, of 4096 in 4.1 / 4.2 / 3.5; 9600 rows of 256 in 9.0 / 11.1 / 14.6
    if (n8 <= 32 || (n8 <= 256 && p->rows < 2 * (int64_t)sm_count)) return launch_norm_t<DT, BT, 1, 256>(p, vec, sm_count, st);
    if (n8 > 1024) return launch_norm_t<DT, BT, 4, 1024>(p, vec, sm_count, st);
    if (p->gate_kind == EXL3B_GATE_ELEMENT) return launch_norm_t<DT, BT, 2, 512>(p, vec, sm_count, st);
    return launch_norm_t<DT, BT, 4, 256>(p, vec, sm_count, st);
}

// ------------------------------------------------------------------------------------------ MXFP4 rows
// HBM bound: a thread takes kUnroll vectors of eight values, 256 vectors apart in the rows laid end to end (whatever the
// width, every lane has work), all loaded before the first is used; a block's scale comes from four neighbouring lanes.
// Measured on one B200, 20480 x 4096 in bf16: quantised in 37 us (5.7 TB/s), back in 34 us (6.2 TB/s): HBM's bytes; 64 x
// 2048: 2.8 us each, a launch.
constexpr int kUnroll = 4;

// The scale code of a block whose 32 values four neighbouring lanes hold. 16-bit types: the magnitudes two a word, which
// order as integers too.
template <int DT>
__device__ __forceinline__ uint32_t quad_code(const Raw<DT>& x) {
    if constexpr (DT == 1) {
        float v[8];
        x.get(v);
        return mx4_quad_code(v);
    } else {
        const uint32_t k = 0x7FFF7FFFu;
        uint32_t m = max_u16x2(max_u16x2(x.q[0].x & k, x.q[0].y & k), max_u16x2(x.q[0].z & k, x.q[0].w & k));
        m = max_u16x2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        m = max_u16x2(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
        m = max(m & 0xFFFFu, m >> 16);
        return mx4_scale_code(DT == 3 ? m << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)m))));
    }
}

template <int DT, bool BIG>
__global__ void __launch_bounds__(256) k_mx4_quantize(const void* x, int64_t x_pitch, int64_t n_vec, Exl3bDiv div,
                                                      uint8_t* q, int64_t q_pitch, uint8_t* qs, int64_t qs_pitch) {
    typedef typename El<DT>::T T;
    chain_wait();
    chain_next();
    const int64_t i0 = (int64_t)blockIdx.x * (256 * kUnroll) + threadIdx.x;
    Raw<DT> v[kUnroll];
    int64_t row[kUnroll];
    int c[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        row_of<BIG>(i0 + 256 * u, div, &row[u], &c[u]);
        v[u].clear();
        if (i0 + 256 * u < n_vec) v[u].fetch(static_cast<const T*>(x) + row[u] * x_pitch + 8 * c[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const uint32_t code = quad_code<DT>(v[u]);
        if (i0 + 256 * u >= n_vec) continue;
        float f[8];
        v[u].get(f);
        *reinterpret_cast<uint32_t*>(q + row[u] * q_pitch + 4 * c[u]) = mx4_pack8(f, code);
        if ((threadIdx.x & 3) == 0) qs[row[u] * qs_pitch + (c[u] >> 2)] = (uint8_t)code;
    }
}

// Eight e2m1 codes -> f32. As f16 the values 0 .5 1 1.5 2 3 4 6 have zero low bytes: a byte permutation looks four high
// bytes up at once, another the signs.
__device__ __forceinline__ void e2m1_unpack8(uint32_t n, float v[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t c = n >> (16 * h);
        const uint32_t b = __byte_perm(0x3E3C3800u, 0x46444240u, c & 0x7777u) | __byte_perm(0x8000u, 0u, (c >> 3) & 0x1111u);
        const uint32_t p0 = __byte_perm(b, 0u, 0x1404), p1 = __byte_perm(b, 0u, 0x3424);
        const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&p0));
        const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&p1));
        v[4 * h] = f0.x;
        v[4 * h + 1] = f0.y;
        v[4 * h + 2] = f1.x;
        v[4 * h + 3] = f1.y;
    }
}

// Eight e2m1 codes times 2^(code - 127) in bf16: both bytes of a value looked up, then one product of pairs, which rounds
// (below the normal range) as the f32 product would.
__device__ __forceinline__ uint4 e2m1_bf16x8(uint32_t n, uint32_t code) {
    const uint32_t bits = code == kMx4Nan ? 0x7FFFu : code ? code << 7 : 0x40u;
    const __nv_bfloat162 s = __halves2bfloat162(__ushort_as_bfloat16((unsigned short)bits), __ushort_as_bfloat16((unsigned short)bits));
    uint32_t w[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t c = n >> (16 * h), m = c & 0x7777u;
        const uint32_t hi = __byte_perm(0x3F3F3F00u, 0x40404040u, m) | __byte_perm(0x8000u, 0u, (c >> 3) & 0x1111u);
        const uint32_t lo = __byte_perm(0xC0800000u, 0xC0804000u, m);
        w[2 * h] = __byte_perm(lo, hi, 0x5140);
        w[2 * h + 1] = __byte_perm(lo, hi, 0x7362);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), s);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int DT, bool BIG>
__global__ void __launch_bounds__(256) k_mx4_dequantize(const uint8_t* q, int64_t q_pitch, const uint8_t* qs,
                                                        int64_t qs_pitch, int64_t n_vec, Exl3bDiv div, void* y,
                                                        int64_t y_pitch) {
    typedef typename El<DT>::T T;
    chain_wait();
    chain_next();
    const int64_t i0 = (int64_t)blockIdx.x * (256 * kUnroll) + threadIdx.x;
    uint32_t n[kUnroll], s[kUnroll];
    int64_t row[kUnroll];
    int c[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        row_of<BIG>(i0 + 256 * u, div, &row[u], &c[u]);
        n[u] = s[u] = 0;
        if (i0 + 256 * u >= n_vec) continue;
        n[u] = *reinterpret_cast<const uint32_t*>(q + row[u] * q_pitch + 4 * c[u]);
        s[u] = qs[row[u] * qs_pitch + (c[u] >> 2)];
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        if (i0 + 256 * u >= n_vec) continue;
        T* d = static_cast<T*>(y) + row[u] * y_pitch + 8 * c[u];
        if (DT == 3) {
            *reinterpret_cast<uint4*>(d) = e2m1_bf16x8(n[u], s[u]);
            continue;
        }
        const float scale = mx4_scale(s[u]);
        float v[8];
        e2m1_unpack8(n[u], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= scale;
        st8<DT>(d, v);
    }
}

// A weight's row-major scales [E][rows][cols / 32] -> the tiles the product's kernel copies whole: per expert, per block
// of 128 weight rows, per 128 input columns 512 bytes, row r's four scales at (r % 32) * 16 + (r / 32) * 4. With
// silu_mul a block is 64 gate rows and their 64 up rows, 16 of each in turn. Rows and columns past the weight's get code 0.
__global__ void __launch_bounds__(256) k_mx4_tile(const uint8_t* s, int64_t s_pitch, int64_t e_pitch, int64_t rows,
                                                  int64_t cols, int act, int64_t n_blk, int64_t n_k, int64_t total,
                                                  uint32_t* out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t tile = i >> 7;
        const int w = (int)(i & 127), r = (w >> 2) + 32 * (w & 3);       // word w: row r's four scales
        const int64_t kb = tile % n_k, blk = tile / n_k % n_blk, e = tile / n_k / n_blk;
        const int64_t half = rows / 2, j = blk * 64 + (r >> 5) * 16 + (r & 15);
        const int64_t row = act ? (j < half ? (r & 16 ? half + j : j) : rows) : blk * 128 + r;
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

int exl3b_cuda_block_norm(const Exl3bNormOp* p, int dtype, int branch_dtype, int vec, int sm_count, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype * 4 + branch_dtype) {
    case 1 * 4 + 1: return launch_norm<1, 1>(p, vec, sm_count, st);
    case 1 * 4 + 2: return launch_norm<1, 2>(p, vec, sm_count, st);
    case 1 * 4 + 3: return launch_norm<1, 3>(p, vec, sm_count, st);
    case 2 * 4 + 1: return launch_norm<2, 1>(p, vec, sm_count, st);
    case 2 * 4 + 2: return launch_norm<2, 2>(p, vec, sm_count, st);
    case 2 * 4 + 3: return launch_norm<2, 3>(p, vec, sm_count, st);
    case 3 * 4 + 1: return launch_norm<3, 1>(p, vec, sm_count, st);
    case 3 * 4 + 2: return launch_norm<3, 2>(p, vec, sm_count, st);
    case 3 * 4 + 3: return launch_norm<3, 3>(p, vec, sm_count, st);
    default: return -2;
    }
}

#define EXL3B_MX4_ROWS(KERN, DT, ...)                                                                        \
    do {                                                                                                     \
        if (n_vec < (1ll << 31) - 1024) return chain_launch(KERN<DT, false>, dim3(grid), dim3(256), 0, 1, st, __VA_ARGS__); \
        return chain_launch(KERN<DT, true>, dim3(grid), dim3(256), 0, 1, st, __VA_ARGS__);                   \
    } while (0)

int exl3b_cuda_mx4_quantize(const void* x, int dtype, int64_t x_pitch, int64_t rows, int64_t cols, uint8_t* q,
                            int64_t q_pitch, uint8_t* qs, int64_t qs_pitch, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t n_vec = rows * (cols / 8);
    const unsigned grid = (unsigned)((n_vec + 256 * kUnroll - 1) / (256 * kUnroll));
    const Exl3bDiv div = exl3b_div((uint32_t)(cols / 8));
    if (dtype == 1) EXL3B_MX4_ROWS(k_mx4_quantize, 1, x, x_pitch, n_vec, div, q, q_pitch, qs, qs_pitch);
    else if (dtype == 2) EXL3B_MX4_ROWS(k_mx4_quantize, 2, x, x_pitch, n_vec, div, q, q_pitch, qs, qs_pitch);
    else EXL3B_MX4_ROWS(k_mx4_quantize, 3, x, x_pitch, n_vec, div, q, q_pitch, qs, qs_pitch);
}

int exl3b_cuda_mx4_dequantize(const uint8_t* q, int64_t q_pitch, const uint8_t* qs, int64_t qs_pitch, int64_t rows,
                              int64_t cols, void* y, int dtype, int64_t y_pitch, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t n_vec = rows * (cols / 8);
    const unsigned grid = (unsigned)((n_vec + 256 * kUnroll - 1) / (256 * kUnroll));
    const Exl3bDiv div = exl3b_div((uint32_t)(cols / 8));
    if (dtype == 1) EXL3B_MX4_ROWS(k_mx4_dequantize, 1, q, q_pitch, qs, qs_pitch, n_vec, div, y, y_pitch);
    else if (dtype == 2) EXL3B_MX4_ROWS(k_mx4_dequantize, 2, q, q_pitch, qs, qs_pitch, n_vec, div, y, y_pitch);
    else EXL3B_MX4_ROWS(k_mx4_dequantize, 3, q, q_pitch, qs, qs_pitch, n_vec, div, y, y_pitch);
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
