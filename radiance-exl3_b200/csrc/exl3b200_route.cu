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
// Choices are made as the real numbers order them, not as their roundings do. Without a bias and without sums of two the
// logits are compared (both scores grow with them), else c. Each expert has a 32-bit key that orders as the number does, but
// for its last bits, which hold the expert's place in the lane: one maximum finds both. 16-bit logits that are compared leave
// room for the whole expert, and their keys are exact. Where two neighbours among the chosen ones, or the last chosen and the
// next, or the worst group kept and the best one dropped, are nearer than the keys and the f32 scores behind them can tell,
// the token is routed again with 64-bit scores, exactly (`again`). How often that is, by the thresholds below at N(0, 1.5)
// logits: two tokens in a thousand with a bias (256 experts, eight chosen, sums of two; or 512, ten chosen); f32 softmax sums
// of two without a bias 0.3 % (256 experts, eight chosen) and 1.8 % (512, sixteen). 16-bit logits hold equal ones, which sums
// of two without a bias, having c for keys, take for too near: f16 4 % and 14 % there, bf16 29 % and 71 %.
//
// Bound by instructions, about a thousand a token in this case, and by their latency: a round is a maximum over the warp, its
// lane and that lane's next key. Measured on one B200: 16384 tokens, 256 experts, sigmoid, bias, four of eight groups, eight
// chosen 26 us (all in 64 bits 43), of which the tokens routed again, a few us each at the grid's end, are 2 to 5; the 17 MB
// of logits alone are 2.7. Softmax without the bias 28 us in f32, 31 in f16, 49 in bf16; bf16, 512 experts, sixteen chosen
// 201. One token of 512 experts with its sort 5.6 us. A lane's sixteen keys (257 to 512 experts) lie in local memory where
// they are sorted, but for 16-bit logits compared by themselves without the sort of the tokens: a frame of 64 bytes; the
// forms for over 1024 experts with that sort spill up to 380 bytes.
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <type_traits>

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
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }
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
template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(kAll, v, m);
    return v;
}
__device__ __forceinline__ float warp_max_of(float v) {
#pragma unroll
    for (int m = 16; m; m >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, m));
    return v;
}

// 1 / (1 + e^-z); below -20 its exponential, which it is to within 2^-28, and which stays in range while the value does.
__device__ __forceinline__ float sigmoid(float z) { return z < -20.f ? expf(z) : 1.f / (1.f + expf(-z)); }

// e^x from the special-function unit: within 2^-22 + 1.3 |x| 2^-24 of the value (the product's rounding, and the constant's,
// which is 2^-26 of it).
__device__ __forceinline__ float exp_near(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.44269504f));
    return r;
}
__device__ __forceinline__ float sigmoid_near(float z) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + exp_near(-z)));
    return r;
}

// A logit: NaN as -inf, +inf as the largest number, which it stands for.
__device__ __forceinline__ float logit_of(float v) { return v == v ? fminf(v, FLT_MAX) : -INFINITY; }

// The experts of a lane: n from e0 on.
struct Span {
    int e0, n;
};
__device__ __forceinline__ Span span_of(const Exl3bRouteOp& p, int lane) {
    const int g = lane >> p.group_shift, first = (lane - (g << p.group_shift)) * p.lane_experts;
    return Span{ g * p.group_size + first, g < p.n_group ? max(min(p.group_size - first, p.lane_experts), 0) : 0 };
}

// The two largest of a lane's keys -> those of its group's lanes.
template <typename K>
__device__ __forceinline__ void group_top(const Exl3bRouteOp& p, K& a, K& b) {
    for (int m = 1; m >> p.group_shift == 0; m <<= 1) {
        const K oa = __shfl_xor_sync(kAll, a, m), ob = __shfl_xor_sync(kAll, b, m);
        b = max(min(a, oa), max(b, ob));
        a = max(a, oa);
    }
}
// Whether the lane's group is among the group_keep with the largest score, the lower one among equals.
template <typename K>
__device__ __forceinline__ bool group_kept(const Exl3bRouteOp& p, K score, int lane) {
    const int g = lane >> p.group_shift;
    int ahead = 0;
    for (int j = 0; j < p.n_group; ++j) {
        const K o = __shfl_sync(kAll, score, j << p.group_shift);
        ahead += o > score || (o == score && j < g);
    }
    return ahead < p.group_keep;
}

// The choice in 64 bits: lane r's is round r's expert, -1 when none is left. A lane of up to 16 experts holds their keys; of
// more, it works them out as often as it looks at them.
template <int RPL, int DT, bool WIDE>
__device__ __noinline__ int again(const Exl3bRouteOp& p, const typename El<DT>::T* row, float top, int lane) {
    constexpr bool HOLD = RPL <= 16;
    const Span s = span_of(p, lane);
    const bool softmax = p.score == EXL3B_SCORE_SOFTMAX;
    auto each = [&](auto&& f) {                                // of the lane's experts
        if constexpr (HOLD) {
#pragma unroll
            for (int q = 0; q < RPL; ++q) f(q);
        } else {
            for (int q = 0; q < s.n; ++q) f(q);
        }
    };
    auto logit = [&](int q) { return q < s.n ? logit_of(El<DT>::to(row[s.e0 + q])) : -INFINITY; };
    double sum = 0.;
    if (WIDE && softmax) {
        each([&](int q) { sum += exp((double)logit(q) - (double)top); });
        sum = warp_sum(sum);
    }
    auto key = [&](int q) -> uint64_t {
        const float l = logit(q);
        double c = l;
        if (WIDE) {
            c = softmax ? exp((double)l - (double)top) / sum : 1. / (1. + exp(-(double)l));
            if (p.bias && q < s.n) c += (double)p.bias[s.e0 + q];
        }
        return l > -INFINITY && c > -INFINITY ? key_of(c) : 0;
    };
    uint64_t held[HOLD ? RPL : 1];
    if constexpr (HOLD) each([&](int q) { held[q] = key(q); });
    uint64_t taken = 0;                                        // of the lane's experts
    auto left = [&](int q) -> uint64_t {
        if (taken >> q & 1) return 0;
        if constexpr (HOLD) return held[q];
        else return key(q);
    };
    if (p.group_keep < p.n_group) {
        uint64_t a = 0, b = 0;
        each([&](int q) {
            const uint64_t k = left(q);
            b = max(b, min(a, k));
            a = max(a, k);
        });
        group_top(p, a, b);
        if (p.group_top == 2 && b) a = key_of(value_of(a) + value_of(b));
        if (!group_kept(p, a, lane)) taken = ~0ull;
    }
    int mine = -1;
    for (int r = 0; r < p.top_k; ++r) {
        uint64_t best = 0;
        int at = 0;
        each([&](int q) {
            const uint64_t k = left(q);
            if (k > best) {
                best = k;
                at = q;
            }
        });
        const uint64_t most = warp_max(best);
        if (most == 0) break;
        const int from = __ffs(__ballot_sync(kAll, best == most)) - 1;
        const int id = __shfl_sync(kAll, s.e0 + at, from);
        if (lane == r) mine = id;
        if (lane == from) taken |= 1ull << at;
    }
    return mine;
}

// A lane's n values from p on as f32; `vec`: n is all of them or none, 16 bytes aligned.
template <int N, typename T>
__device__ __forceinline__ void load_lane(const T* p, int n, bool vec, float (&v)[N]) {
    constexpr int V = 16 / (int)sizeof(T);
    typedef El<sizeof(T) == 4 ? RAD_F32 : std::is_same<T, __half>::value ? RAD_F16 : RAD_BF16> E;
    if (N >= V && vec) {
#pragma unroll
        for (int q = 0; q + V <= N; q += V) {
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (q < n) w = *reinterpret_cast<const uint4*>(p + q);
#pragma unroll
            for (int i = 0; i < V; ++i) v[q + i] = E::to(reinterpret_cast<const T*>(&w)[i]);
        }
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = q < n ? E::to(p[q]) : 0.f;
    }
}

// Descending, by Batcher's odd-even merges.
template <int N>
__device__ __forceinline__ void sort_down(uint32_t (&k)[N]) {
#pragma unroll
    for (int p = 1; p < N; p <<= 1)
#pragma unroll
        for (int q = p; q; q >>= 1)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t hi = max(k[i + j], k[i + j + q]), lo = min(k[i + j], k[i + j + q]);
                        k[i + j] = hi;
                        k[i + j + q] = lo;
                    }
}

// One token, by a whole warp; its ids also to `local` (shared memory), if given.
template <int RPL, int DT, bool WIDE>
__device__ __forceinline__ void route(const Exl3bRouteOp& p, int64_t t, int lane, int32_t* local = nullptr) {
    typedef typename El<DT>::T T;
    constexpr bool EXACT = !WIDE && DT != RAD_F32;             // the keys are: 16 bits and the expert
    constexpr uint32_t LOW = EXACT ? 0xFFFFu : RPL <= 8 ? 7u : RPL <= 16 ? 15u : RPL <= 32 ? 31u : 63u;
    constexpr bool SORT = RPL <= 16;                           // a lane's keys are sorted, or searched each round
    const T* row = static_cast<const T*>(p.logits) + t * p.logits_pitch;
    const Span span = span_of(p, lane);
    const int n = span.n, e0 = span.e0;
    const bool softmax = p.score == EXL3B_SCORE_SOFTMAX;
    float l[RPL], bias[WIDE ? RPL : 1];
    load_lane<RPL>(row + e0, n, p.vec & 1, l);
    if (WIDE) {
        if (p.bias) load_lane<WIDE ? RPL : 1>(p.bias + e0, n, p.vec & 2, bias);
        else
#pragma unroll
            for (int q = 0; q < RPL; ++q) bias[WIDE ? q : 0] = 0.f;
    }
#pragma unroll
    for (int q = 0; q < RPL; ++q) l[q] = q < n ? logit_of(l[q]) : -INFINITY;
    float top = 0.f, inv = 1.f;                                // softmax: the largest logit, one over the sum
    if (softmax && (WIDE || !p.renorm)) {
        top = -INFINITY;
#pragma unroll
        for (int q = 0; q < RPL; ++q) top = fmaxf(top, l[q]);
        top = fmaxf(warp_max_of(top), -FLT_MAX);               // a row with nothing in it: any number does
        float sum = 0.f;
#pragma unroll
        for (int q = 0; q < RPL; ++q) sum += expf(l[q] - top);
        inv = 1.f / warp_sum(sum);
    }
    uint32_t key[RPL];
#pragma unroll
    for (int q = 0; q < RPL; ++q) {
        float c = l[q];
        if (WIDE) {
            c = (softmax ? exp_near(c - top) * inv : sigmoid_near(c)) + bias[WIDE ? q : 0];
        }
        const bool in = l[q] > -INFINITY && c > -INFINITY;
        if constexpr (DT == RAD_F16 && EXACT) {                // f16's own order: its 19 significant bits of an f32 are too many
            const uint32_t h = __half_as_ushort(__float2half_rn(c == 0.f ? 0.f : c));     // the largest f32: +inf, as it was
            key[q] = in ? ((h & 0x8000u) ? ~h & 0xFFFFu : h | 0x8000u) << 16 | (LOW - (uint32_t)(e0 + q)) : 0u;
        } else {
            if (EXACT && c == FLT_MAX) c = INFINITY;           // bf16's own largest number has the same 16 bits
            key[q] = in ? (key_of(c) & ~LOW) | (LOW - (uint32_t)(EXACT ? e0 + q : q)) : 0u;
        }
    }
    // Nearer than this two c cannot be told apart: twice an f32 score's error and, relative to c, its own rounding and the bits of
    // the key that hold a place. A sigmoid s is off by s (1 - s) (2^-22 + 1.3 |z| 2^-24) for the exponential and s 1.5 2^-23 for
    // the sum and the reciprocal, below 1.1 2^-22 in all. A softmax's exponentials are off by 2^-22 + 0.9 2^-24 of the largest
    // score, `inv`, at most (|x| e^x is below 0.37, and the difference x is rounded too), the quotient and the product by one
    // rounding each, their sum (the same way for all) by as much as a term and one rounding a term, at most 69 of 2^-24: 90 of
    // 2^-24 for a difference, where 256 are taken.
    const float near = softmax ? 0x1p-16f * inv : 0x1p-20f;
    constexpr float near_rel = 0x1p-22f + (float)(LOW + 1) * 0x1p-23f;
    bool unsure = false;
    auto compare = [&](uint32_t hi, uint32_t lo, float times) {
        if constexpr (WIDE) {
            const float a = value_of(hi & ~LOW), b = value_of(lo & ~LOW);
            unsure = unsure || !(a - b > times * (near + near_rel * fmaxf(fabsf(a), fabsf(b))));
        } else if constexpr (!EXACT) {
            unsure = unsure || ((hi ^ lo) & ~LOW) == 0;
        }
    };
    if (SORT) sort_down(key);
    if (p.group_keep < p.n_group) {
        uint32_t a = key[0], b = key[1];
        if (!SORT) {
            a = b = 0;
#pragma unroll
            for (int q = 0; q < RPL; ++q) {
                b = max(b, min(a, key[q]));
                a = max(a, key[q]);
            }
        }
        group_top(p, a, b);
        const bool two = WIDE && p.group_top == 2;
        if (two && b) a = key_of(value_of(a & ~LOW) + value_of(b & ~LOW));
        const bool kept = group_kept(p, a, lane);
        if (!EXACT) {                                          // a sum's error is its terms', whose magnitudes it may not show
            const uint32_t worst = ~warp_max(kept && lane >> p.group_shift < p.n_group ? ~a : 0u), best = warp_max(kept ? 0u : a);
            float size = 0.f;
            if (two && b) size = fabsf(value_of(b & ~LOW)) + fabsf(value_of(a));
            if (two) size = warp_max_of(size);
            if (best) compare(worst, best, 2.f);
            if (two && best) unsure = unsure || !(value_of(worst) - value_of(best) > 2.f * near + 4.f * near_rel * size);
        }
        if (!kept) {
#pragma unroll
            for (int q = 0; q < RPL; ++q) key[q] = 0;
        }
    }
    auto largest = [&]() {
        uint32_t m = key[0];
        if (!SORT) {
#pragma unroll
            for (int q = 1; q < RPL; ++q) m = max(m, key[q]);
        }
        return m;
    };
    uint32_t best = largest(), last = 0;
    int id = -1;
    for (int r = 0; r <= p.top_k; ++r) {
        const uint32_t most = warp_max(best);
        if (most == 0) break;
        if (r > 0) compare(last, most, 1.f);
        if (r == p.top_k) break;
        last = most;
        const int from = __ffs(__ballot_sync(kAll, best == most)) - 1;
        const int at = (int)(LOW - (most & LOW)), here = EXACT ? at : __shfl_sync(kAll, e0, from) + at;
        if (lane == r) id = here;
        const bool win = lane == from;
        if (SORT) {
#pragma unroll
            for (int q = 0; q < RPL; ++q) key[q] = win ? (q + 1 < RPL ? key[(q + 1) % RPL] : 0u) : key[q];
        } else {
#pragma unroll
            for (int q = 0; q < RPL; ++q) key[q] = win && key[q] == most ? 0u : key[q];
        }
        best = largest();
    }
    if (!EXACT && unsure) id = again<RPL, DT, WIDE>(p, row, top, lane);
    // lane r has round r's expert. Renormalised weights come from the chosen logits alone; softmax's, and those of sigmoids all
    // below -20, less the largest of them, in range however small the scores are
    float z = -INFINITY;
    if (id >= 0) z = fminf(El<DT>::to(row[id]), FLT_MAX);
    float w;
    if (p.renorm) {
        const float most = fmaxf(warp_max_of(z), -FLT_MAX);
        w = softmax || most < -20.f ? expf(z - most) : sigmoid(z);
        w /= warp_sum(w);
    } else {
        w = softmax ? expf(z - top) * inv : sigmoid(z);
    }
    if (lane < p.top_k) {
        p.ids[t * p.top_k + lane] = id;
        p.w[t * p.top_k + lane] = id < 0 ? 0.f : w * p.scale;
        if (local) local[t * p.top_k + lane] = id;
    }
}

template <int RPL, int DT, bool WIDE>
__global__ void __launch_bounds__(128) k_route(const __grid_constant__ Exl3bRouteOp p) {
    chain_wait();
    chain_next();
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (t < p.n_tok) route<RPL, DT, WIDE>(p, t, threadIdx.x & 31);
}

// A few tokens: their routing and the whole sort in one launch. A cluster of CTAs routes, a token a warp; its first CTA, to
// whose shared memory they write the ids, sorts as moe_scatter does: experts counted, the counts summed up, and each pair placed
// behind those of its expert in earlier warps (whose leading lanes note their counts, a row a warp) and lanes. The others are done
// when they have routed: nothing reads their shared memory. A CTA for each four tokens, up to eight of them: a warp a scheduler as
// long as it goes (32 tokens of 512 experts 7.4 us, all in one CTA 14.6, in two launches 9.7).
constexpr int kFusedTokens = 128, kFusedThreads = 512, kFusedWarps = kFusedThreads / 32;
__host__ __device__ __forceinline__ int64_t fused_ids(int64_t pairs) { return (pairs + 3) / 4 * 4; }
constexpr int kFusedBytes = 200 * 1024;          // the most that a sort takes
size_t fused_bytes(int64_t pairs, int64_t n_local) { return (size_t)(fused_ids(pairs) + n_local + 1 + (pairs + 31) / 32 * n_local) * 4; }
template <int RPL, int DT, bool WIDE>
__global__ void __launch_bounds__(kFusedThreads) k_route_sort(const __grid_constant__ Exl3bRouteOp p) {
    extern __shared__ int sm[];
    __shared__ int wtot[32];
    int* const ids = sm;                                       // [n_tok * top_k]
    const int tid = threadIdx.x, lane = tid & 31, E = p.n_local, P = (int)p.n_tok * p.top_k;
    int* const cnt = sm + fused_ids(P);                        // [n_local + 1], then [warps of pairs][n_local]
    int* const wcnt = cnt + E + 1;
    const bool several = gridDim.x > 1, first = blockIdx.x == 0;
    if (several) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    if (first)
        for (int x = tid; x < E + 1 + (P + 31) / 32 * E; x += kFusedThreads) cnt[x] = 0;
    chain_wait();
    chain_next();
    int* to = ids;
    if (several) {
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");                // the first CTA is there
        if (!first) asm volatile("mapa.u64 %0, %1, 0;" : "=l"(to) : "l"(ids));
    }
    for (int64_t t = blockIdx.x + gridDim.x * (tid >> 5); t < p.n_tok; t += gridDim.x * kFusedWarps)
        route<RPL, DT, WIDE>(p, t, lane, to);
    if (several) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        if (!first) return;
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
    for (int f0 = 0; f0 < P; f0 += kFusedThreads) {
        const int f = f0 + tid, e = f < P ? local_expert(ids[f], p.expert_base, E) : -1;
        const unsigned peers = __match_any_sync(kAll, e);
        if (e >= 0 && lane == __ffs(peers) - 1) {
            wcnt[(f >> 5) * E + e] = __popc(peers);
            atomicAdd(&cnt[e], __popc(peers));
        }
    }
    __syncthreads();
    const int live = block_scan_excl(cnt, E, wtot);
    for (int e = tid; e < E; e += kFusedThreads) {
        int at = cnt[e];
        p.expert_offset[e] = at;
        for (int w = 0; w < (P + 31) / 32; ++w) {
            const int c = wcnt[w * E + e];
            if (c) {
                wcnt[w * E + e] = at;
                at += c;
            }
        }
    }
    if (tid == 0) p.expert_offset[E] = live;
    for (int f = live + tid; f < P; f += kFusedThreads) p.sorted_tok[f] = -1;
    __syncthreads();
    for (int f0 = 0; f0 < P; f0 += kFusedThreads) {
        const int f = f0 + tid, e = f < P ? local_expert(ids[f], p.expert_base, E) : -1;
        const unsigned peers = __match_any_sync(kAll, e);
        if (e >= 0) p.sorted_tok[wcnt[(f >> 5) * E + e] + __popc(peers & ((1u << lane) - 1u))] = f;
    }
}

template <int RPL, int DT, bool WIDE>
int launch(const Exl3bRouteOp* p, int fused, cudaStream_t st) {
    if (!fused) return chain_launch(k_route<RPL, DT, WIDE>, dim3((unsigned)((p->n_tok + 3) / 4)), dim3(128), 0, 1, st, *p);
    auto kern = k_route_sort<RPL, DT, WIDE>;
    const size_t smem = fused_bytes(p->n_tok * p->top_k, p->n_local);
    // 48 KB, the static array among them, need no asking. The same limit whatever this call needs: a smaller one would fail another
    // thread's launch between its own two steps
    if (smem > 40 * 1024) {
        static bool allowed[64];                              // once a device
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -6;
        if (!allowed[dev] && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFusedBytes) != cudaSuccess)
            return -6;
        allowed[dev] = true;
    }
    const int ctas = (int)(p->n_tok > 28 ? 8 : (p->n_tok + 3) / 4);
    return chain_launch(kern, dim3(ctas), dim3(kFusedThreads), smem, ctas, st, *p);
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

// Whether the sort comes in the same launch: few tokens, the placement's table in shared memory. The table is one CTA's work, so
// that from 64 tokens on a large one costs more than a launch: one launch against two at 64 tokens of 512 experts, ten each, 9.7
// and 10.3 us, at 96 of them 11.2 and 10.8; at 128 of 256 experts, eight each (37 KB), 10.0 and 10.3.
int exl3b_route_fuses(int64_t n_tok, int64_t top_k, int64_t n_local) {
    return n_tok <= kFusedTokens && n_local <= kPlaceFastExperts &&
           fused_bytes(n_tok * top_k, n_local) <= (size_t)(n_tok <= 64 ? kFusedBytes : 40 * 1024);
}

int exl3b_cuda_route(const Exl3bRouteOp* p, int dtype, int fused, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->lane_experts <= 8) return launch_type<8>(p, dtype, fused, st);
    if (p->lane_experts <= 16) return launch_type<16>(p, dtype, fused, st);
    if (p->lane_experts <= 32) return launch_type<32>(p, dtype, fused, st);
    return launch_type<64>(p, dtype, fused, st);
}

}  // extern "C"
