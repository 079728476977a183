// exl3b200_sort.cuh -- the stable counting sort of flattened (token, slot) pairs by expert, as one block does it: the whole
// sort of few pairs (scatter_block), and a chunk's placement in the large sort. sm_100a.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace exl3b {

// Exclusive scan of cnt[0 .. n) in place (block-wide: each thread a run, warp shuffles, warp totals); returns the
// total to every thread. `wtot` holds blockDim.x / 32 ints.
__device__ __forceinline__ int block_scan_excl(int* cnt, int n, int* wtot) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    const int per = (n + blockDim.x - 1) / blockDim.x;
    const int e0 = tid * per, e1 = e0 + per < n ? e0 + per : n;
    int sum = 0;
    for (int e = e0; e < e1; ++e) sum += cnt[e];
    int incl = sum;
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, incl, d);
        if (lane >= d) incl += v;
    }
    if (lane == 31) wtot[warp] = incl;
    __syncthreads();
    int base = 0, total = 0;
    for (int w = 0; w < nw; ++w) {
        const int v = wtot[w];
        if (w < warp) base += v;
        total += v;
    }
    int acc = base + incl - sum;
    for (int e = e0; e < e1; ++e) {
        const int v = cnt[e];
        cnt[e] = acc;
        acc += v;
    }
    __syncthreads();
    return total;
}

// A negative id is no expert's, also where a rank's first expert is a negative number.
__device__ __forceinline__ int local_expert(int32_t id, int64_t base, int n_expert) {
    const int64_t e = (int64_t)id - base;
    return id >= 0 && e >= 0 && e < n_expert ? (int)e : -1;
}

// Stable placement of one chunk of up to 1024 pairs (one a thread, in order), the running per-expert
// positions in `run` (shared). Warps go one after another, so pairs of one expert land in flat order.
__device__ __forceinline__ void place_chunk(const int32_t* ids, int64_t c0, int64_t n_pairs, int64_t base, int n_expert,
                                            int* run, int32_t* sorted_tok) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    const int64_t f = c0 + tid;
    const int e = f < n_pairs ? local_expert(ids[f], base, n_expert) : -1;
    const unsigned peers = __match_any_sync(0xFFFFFFFFu, e);
    const int rank = __popc(peers & ((1u << lane) - 1u));
    const int leader = __ffs(peers) - 1;
    for (int w = 0; w < nw; ++w) {
        if (warp == w && e >= 0) {
            sorted_tok[run[e] + rank] = (int32_t)f;
            __syncwarp(peers);
            if (lane == leader) run[e] += __popc(peers);
        }
        __syncthreads();
    }
}

// The same placement without the warp-by-warp walk: each warp's leader lanes record their expert's count in the
// warp's row of `wcnt` ([32 warps][n_expert], shared, all zero on entry), one pass turns every expert's column into
// the warps' first positions (and advances `run`), and every pair is then stored at once. Leaves `wcnt` zero.
__device__ __forceinline__ void place_chunk_fast(const int32_t* ids, int64_t c0, int64_t n_pairs, int64_t base,
                                                 int n_expert, int* run, int* wcnt, int32_t* sorted_tok) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
    const int64_t f = c0 + tid;
    const int e = f < n_pairs ? local_expert(ids[f], base, n_expert) : -1;
    const unsigned peers = __match_any_sync(0xFFFFFFFFu, e);
    const int rank = __popc(peers & ((1u << lane) - 1u));
    const bool leader = lane == __ffs(peers) - 1;
    if (e >= 0 && leader) wcnt[warp * n_expert + e] = __popc(peers);
    __syncthreads();
    for (int x = tid; x < n_expert; x += blockDim.x) {
        int acc = run[x];
        for (int w = 0; w < nw; ++w) {
            const int c = wcnt[w * n_expert + x];
            if (c) {
                wcnt[w * n_expert + x] = acc;
                acc += c;
            }
        }
        run[x] = acc;
    }
    __syncthreads();
    if (e >= 0) sorted_tok[wcnt[warp * n_expert + e] + rank] = (int32_t)f;
    __syncthreads();
    if (e >= 0 && leader) wcnt[warp * n_expert + e] = 0;
    __syncthreads();
}

// The fast placement's table fits shared memory up to this many experts ([32][n_expert] ints).
constexpr int kPlaceFastExperts = 1024;

// The whole sort in one block (few pairs): histogram, scan, stable placement, tail of -1.
// `ids` carries no __restrict__: a fused router writes the ids earlier in the same kernel, so they must not be
// read through the read-only (non-coherent) path.
__device__ __forceinline__ void scatter_block(const int32_t* ids, int64_t n_pairs, int n_expert,
                                              int64_t base, int32_t* __restrict__ sorted_tok,
                                              int32_t* __restrict__ off, int* sm) {
    int* cnt = sm;                 // [n_expert + 1]
    const int tid = threadIdx.x;
    for (int e = tid; e <= n_expert; e += blockDim.x) cnt[e] = 0;
    __syncthreads();
    for (int64_t f = tid; f < n_pairs; f += blockDim.x) {
        const int e = local_expert(ids[f], base, n_expert);
        if (e >= 0) atomicAdd(&cnt[e], 1);
    }
    __syncthreads();
    __shared__ int wtot[32];
    const int live = block_scan_excl(cnt, n_expert, wtot);
    for (int e = tid; e < n_expert; e += blockDim.x) off[e] = cnt[e];
    if (tid == 0) off[n_expert] = live;
    for (int64_t f = live + tid; f < n_pairs; f += blockDim.x) sorted_tok[f] = -1;
    if (n_expert <= kPlaceFastExperts) {
        int* wcnt = sm + n_expert + 1;   // [32][n_expert]
        for (int x = tid; x < 32 * n_expert; x += blockDim.x) wcnt[x] = 0;
        __syncthreads();
        for (int64_t c0 = 0; c0 < n_pairs; c0 += blockDim.x)
            place_chunk_fast(ids, c0, n_pairs, base, n_expert, cnt, wcnt, sorted_tok);
    } else {
        for (int64_t c0 = 0; c0 < n_pairs; c0 += blockDim.x)
            place_chunk(ids, c0, n_pairs, base, n_expert, cnt, sorted_tok);
    }
}

}  // namespace exl3b
