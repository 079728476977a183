// exl3b200_route.cu -- router: which experts a token goes to, and with what weights. sm_100a.
//
//   s[e] = exp(l[e] - max l) / sum_j exp(l[j] - max l)   or   1 / (1 + exp(-l[e]))            (score)
//   c[e] = s[e] + bias[e]                                                                     (what is compared)
//   the group_keep groups of n_expert / n_group neighbouring experts with the largest sums of their group_top largest c stay,
//   and of their experts the top_k with the largest c, descending; ties go to the lower group and the lower expert
//   w = s of the chosen ones, divided by their sum if asked, times scale
//
// A warp holds a token, its lanes the experts in order: a lane's are neighbours, and a group has lanes of its own (as many as
// a power of two of groups leaves each), so that a group's maximum is a few shuffles and the lower of two lanes has the lower
// experts. Experts that are masked (a logit or a c that is -inf or NaN) have key 0, below every other key.
//
// Choices are made as the real numbers order them, not as their roundings do: without a bias and without sums of two, the
// logits themselves are compared (both scores grow with them), else c in 64 bits.
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include "exl3b200_chain.cuh"
#include "exl3b200_dense.h"
#include "exl3b200_rows.cuh"
#include "exl3b200_sort.cuh"

using namespace exl3b;

namespace {

constexpr uint32_t kAll = 0xFFFFFFFFu;

// Keys: unsigned integers that order as the numbers do; -0 is keyed as +0. 0 is left for masked experts.
__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t b = __float_as_uint(f == 0.f ? 0.f : f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(double f) {
    const uint64_t b = (uint64_t)__double_as_longlong(f == 0. ? 0. : f);
    return (b >> 63) ? ~b : (b | 1ull << 63);
}
__device__ __forceinline__ double value_of(uint64_t k) {
    return __longlong_as_double((long long)((k >> 63) ? (k & ~(1ull << 63)) : ~k));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ uint64_t warp_max(uint64_t k) {
    const uint32_t hi = __reduce_max_sync(kAll, (uint32_t)(k >> 32));
    const uint32_t lo = __reduce_max_sync(kAll, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
    return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(kAll, v, m);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(kAll, v, m);
    return v;
}
__device__ __forceinline__ float warp_max_of(float v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, m));
    return v;
}

// The keys of experts outside the kept groups to 0. Called by whole warps.
template <int RPL, typename K>
__device__ __forceinline__ void keep_groups(const Exl3bRouteOp& p, K key[RPL], int lane) {
    K a = 0, b = 0;                                            // the lane's, then the group's, two largest
#pragma unroll
    for (int q = 0; q < RPL; ++q) {
        const K lo = min(a, key[q]);
        a = max(a, key[q]);
        b = max(b, lo);
    }
    for (int m = 1; m < p.group_lanes; m <<= 1) {
        const K oa = __shfl_xor_sync(kAll, a, m), ob = __shfl_xor_sync(kAll, b, m);
        b = max(min(a, oa), max(b, ob));
        a = max(a, oa);
    }
    if constexpr (sizeof(K) == 8) {
        if (p.group_top == 2 && b) a = key_of(value_of(a) + value_of(b));
    }
    const int g = lane / p.group_lanes;
    int ahead = 0;
    for (int j = 0; j < p.n_group; ++j) {
        const K o = __shfl_sync(kAll, a, j * p.group_lanes);
        ahead += o > a || (o == a && j < g);
    }
    if (ahead >= p.group_keep) {
#pragma unroll
        for (int q = 0; q < RPL; ++q) key[q] = 0;
    }
}

// The expert of lane r's round, r < top_k: the largest key left, the lowest expert among equals; -1 when none is left.
template <int RPL, typename K>
__device__ __forceinline__ int pick(K key[RPL], int e0, int top_k, int lane) {
    K best;
    int at;
    auto look = [&]() {
        best = key[0];
        at = 0;
#pragma unroll
        for (int q = 1; q < RPL; ++q)
            if (key[q] > best) {
                best = key[q];
                at = q;
            }
    };
    look();
    int mine = -1;
    for (int r = 0; r < top_k; ++r) {
        const K top = warp_max(best);
        if (top == 0) break;
        const int from = __ffs(__ballot_sync(kAll, best == top)) - 1;
        const int id = __shfl_sync(kAll, e0 + at, from);
        if (lane == r) mine = id;
        if (lane == from) {
#pragma unroll
            for (int q = 0; q < RPL; ++q)
                if (q == at) key[q] = 0;
            look();
        }
    }
    return mine;
}

// 1 / (1 + e^-z); below -20 its exponential, which it is to within 2^-28, and which stays in range while the value does.
__device__ __forceinline__ float sigmoid(float z) { return z < -20.f ? expf(z) : 1.f / (1.f + expf(-z)); }

// One token, by a whole warp.
template <int RPL, int DT, bool WIDE>
__device__ __forceinline__ void route(const Exl3bRouteOp& p, int64_t t, int lane) {
    typedef typename El<DT>::T T;
    const T* row = static_cast<const T*>(p.logits) + t * p.logits_pitch;
    const int g = lane / p.group_lanes, j = lane % p.group_lanes;
    const int first = j * p.lane_experts, left = p.group_size - first;
    const int n = g < p.n_group ? max(min(left, p.lane_experts), 0) : 0, e0 = g * p.group_size + first;
    float l[RPL];                                              // NaN as -inf; +inf as the largest number, which it stands for
    float top = -INFINITY;
#pragma unroll
    for (int q = 0; q < RPL; ++q) {
        const float v = q < n ? El<DT>::to(row[e0 + q]) : -INFINITY;
        l[q] = v == v ? fminf(v, FLT_MAX) : -INFINITY;
        top = fmaxf(top, l[q]);
    }
    const bool softmax = p.score == EXL3B_SCORE_SOFTMAX;
    if (softmax) top = fmaxf(warp_max_of(top), -FLT_MAX);      // a row with nothing in it: any number does
    int id;
    if constexpr (WIDE) {
        double s[RPL];
        double sum = 0.;
#pragma unroll
        for (int q = 0; q < RPL; ++q) {
            s[q] = softmax ? exp((double)l[q] - (double)top) : 1. / (1. + exp(-(double)l[q]));
            sum += s[q];
        }
        if (softmax) sum = warp_sum(sum);
        uint64_t key[RPL];
#pragma unroll
        for (int q = 0; q < RPL; ++q) {
            const double c = (softmax ? s[q] / sum : s[q]) + (p.bias && q < n ? (double)p.bias[e0 + q] : 0.);
            key[q] = l[q] > -INFINITY && c > -INFINITY ? key_of(c) : 0;
        }
        if (p.group_keep < p.n_group) keep_groups<RPL>(p, key, lane);
        id = pick<RPL>(key, e0, p.top_k, lane);
    } else {
        uint32_t key[RPL];
#pragma unroll
        for (int q = 0; q < RPL; ++q) key[q] = l[q] > -INFINITY ? key_of(l[q]) : 0;
        if (p.group_keep < p.n_group) keep_groups<RPL>(p, key, lane);
        id = pick<RPL>(key, e0, p.top_k, lane);
    }
    // lane r has round r's expert. Renormalised weights come from the chosen logits alone; softmax's, and those of sigmoids all
    // below -20, less the largest of them, in range however small the scores are
    float z = -INFINITY;
    if (id >= 0) z = fminf(El<DT>::to(row[id]), FLT_MAX);
    float w;
    if (softmax || p.renorm) {
        const float most = fmaxf(warp_max_of(z), -FLT_MAX);
        if (softmax && !p.renorm) {
            float sum = 0.f;
#pragma unroll
            for (int q = 0; q < RPL; ++q) sum += expf(l[q] - top);
            w = expf(z - top) / warp_sum(sum);
        } else {
            w = softmax || most < -20.f ? expf(z - most) : sigmoid(z);
            w /= warp_sum(w);
        }
    } else {
        w = sigmoid(z);
    }
    if (lane < p.top_k) {
        p.ids[t * p.top_k + lane] = id;
        p.w[t * p.top_k + lane] = id < 0 ? 0.f : w * p.scale;
    }
}

template <int RPL, int DT, bool WIDE>
__global__ void __launch_bounds__(128) k_route(const Exl3bRouteOp p) {
    chain_wait();
    chain_next();
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (t < p.n_tok) route<RPL, DT, WIDE>(p, t, threadIdx.x & 31);
}

// A few tokens: their routing and the whole sort in one block.
constexpr int kFusedTokens = 32;
template <int RPL, int DT, bool WIDE>
__global__ void __launch_bounds__(512) k_route_sort(const Exl3bRouteOp p) {
    extern __shared__ int sm[];
    chain_wait();
    chain_next();
    for (int64_t t = threadIdx.x >> 5; t < p.n_tok; t += 16) route<RPL, DT, WIDE>(p, t, threadIdx.x & 31);
    __syncthreads();
    scatter_block(p.ids, p.n_tok * p.top_k, p.n_local, p.expert_base, p.sorted_tok, p.expert_offset, sm);
}

template <int RPL, int DT, bool WIDE>
int launch(const Exl3bRouteOp* p, int fused, cudaStream_t st) {
    if (!fused) return chain_launch(k_route<RPL, DT, WIDE>, dim3((unsigned)((p->n_tok + 3) / 4)), dim3(128), 0, 1, st, *p);
    auto kern = k_route_sort<RPL, DT, WIDE>;
    const size_t smem = (size_t)(p->n_local + 1) * 4 + (size_t)32 * p->n_local * 4;
    if (smem > 48 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return -6;
    return chain_launch(kern, dim3(1), dim3(512), smem, 1, st, *p);
}
template <int RPL, int DT>
int launch_wide(const Exl3bRouteOp* p, int fused, cudaStream_t st) {
    const bool wide = p->bias || (p->group_keep < p->n_group && p->group_top == 2);
    return wide ? launch<RPL, DT, true>(p, fused, st) : launch<RPL, DT, false>(p, fused, st);
}
template <int RPL>
int launch_type(const Exl3bRouteOp* p, int dtype, int fused, cudaStream_t st) {
    return dtype == RAD_F32 ? launch_wide<RPL, RAD_F32>(p, fused, st)
           : dtype == RAD_F16 ? launch_wide<RPL, RAD_F16>(p, fused, st) : launch_wide<RPL, RAD_BF16>(p, fused, st);
}

}  // namespace

extern "C" {

// Whether the sort comes in the same launch: few tokens, the placement's table in shared memory.
int exl3b_route_fuses(int64_t n_tok, int64_t n_local) { return n_tok <= kFusedTokens && n_local <= kPlaceFastExperts; }

int exl3b_cuda_route(const Exl3bRouteOp* p, int dtype, int fused, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->lane_experts <= 8) return launch_type<8>(p, dtype, fused, st);
    if (p->lane_experts <= 16) return launch_type<16>(p, dtype, fused, st);
    if (p->lane_experts <= 32) return launch_type<32>(p, dtype, fused, st);
    return launch_type<64>(p, dtype, fused, st);
}

}  // extern "C"
