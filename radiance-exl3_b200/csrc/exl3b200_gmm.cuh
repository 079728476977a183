// exl3b200_gmm.cuh -- what the kernels of grouped_mm share: the units of work and their table, tensor memory, TMA, the sorted
// rows' loads, the epilogue's arithmetic and stores, and on the host the weight's tensor map. sm_100a only.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "exl3b200_decode.cuh"
#include "exl3b200_dense.h"

namespace exl3b {

constexpr int kXWarp0 = 4, kXWarps = 4, kEpiWarp0 = 8;
constexpr int kRowB = 128;                       // bytes of k a stage: one swizzle row
constexpr int kW_B = 128 * kRowB;                // a CTA's weight rows of a stage
constexpr int kSlice = 16;                       // sorted rows an epilogue group takes at a time
constexpr int kMaxTurn = 16;                      // slices a unit at most
constexpr int kStage = 8;                        // ... and stages at once, where it stages in f32
constexpr int kEpiLd = 128 + 4;                  // f32 a staged row, padded
constexpr int kTab = 128;                        // a CTA's units held in a shared table (more: looked up)
constexpr int kStatic = 3 * 1024;                // the static shared arrays, up to the ring's alignment
constexpr int kMaxExpert = 2048;
constexpr int kMaxSplit = 4;                     // CTAs a unit at most (SPLIT)
constexpr int kMaxSt = 10;                       // stages at most

// What the host works out of a launch, so that no CTA divides for it.
struct Shape {
    Exl3bDiv n_mb, stride;   // weight-row blocks (PAIR: pairs) an output row; CTAs (PAIR, SPLIT: clusters) of the grid
    Exl3bDiv nt;            // sorted rows a unit at most
    int32_t nck, st, split; // stages of a unit's k, of the ring; CTAs a unit (SPLIT)
};

struct Unit {
    int32_t r0;          // first sorted row
    int32_t e, blk;      // expert, first 128-row block
    int32_t nr;          // sorted rows
};

// The sorted rows of expert e, and into how many groups of at most nt they fall.
struct Run {
    int32_t r0, rows;
};
__device__ __forceinline__ Run run_of(const Exl3bGmmOp& p, int e) {
    if (!p.expert_offset) return Run{ 0, (int32_t)p.n_rows };
    const int32_t a = max(p.expert_offset[e], 0), b = min(p.expert_offset[e + 1], (int32_t)p.n_rows);
    return Run{ a, max(b - a, 0) };
}
__device__ __forceinline__ uint32_t groups(const Run& r, const Exl3bDiv& nt) {
    return exl3b_div_of((uint32_t)r.rows + nt.d - 1, nt);
}

// Unit `local` of expert e: block by block, then group by group. An expert's rows are split evenly over its groups, in
// steps of the MMA's N, so that no group is left with a sliver.
template <int MB>
__device__ __forceinline__ Unit make_unit(int e, const Run& r, uint32_t local, const Shape& sh) {
    const Exl3bDiv& n_mb = sh.n_mb;
    const uint32_t g = exl3b_div_of(local, n_mb), ng = groups(r, sh.nt), step = 16 * MB;
    const uint32_t even = ng > 1 ? ((uint32_t)r.rows + ng - 1) / ng : (uint32_t)r.rows, per = (even + step - 1) / step * step;
    Unit u;
    u.e = e;
    u.blk = (int32_t)(local - g * n_mb.d) * MB;
    u.r0 = r.r0 + (int32_t)(g * per);
    u.nr = min((int32_t)per, r.rows - (int32_t)(g * per));
    return u;
}
// ... found by its number among all units.
template <int MB>
__device__ __forceinline__ Unit find_unit(const Exl3bGmmOp& p, const uint32_t* prefix, uint32_t unit, const Shape& sh) {
    int lo = 0, hi = p.n_expert;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= unit) lo = mid; else hi = mid;
    }
    return make_unit<MB>(lo, run_of(p, lo), unit - prefix[lo], sh);
}

// prefix[e]: the first unit of expert e (block-wide exclusive scan, a thread a run of experts); this CTA's units (first, first +
// stride, ...) go into the table by the threads that pass over their experts. wsum: a word a warp. A barrier is to follow.
template <int THREADS, int MB>
__device__ __forceinline__ void scan_units(const Exl3bGmmOp& p, const Shape& sh, uint32_t first, uint32_t* prefix, Unit* utab,
                                           uint32_t* wsum) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int per = (p.n_expert + THREADS - 1) / THREADS, e0 = tid * per, e1 = min(e0 + per, p.n_expert);
    const uint32_t n_mb = sh.n_mb.d, stride = sh.stride.d;
    const Run run0 = e0 < e1 ? run_of(p, e0) : Run{ 0, 0 };
    uint32_t sum = groups(run0, sh.nt) * n_mb;
#pragma unroll 1
    for (int e = e0 + 1; e < e1; ++e) sum += groups(run_of(p, e), sh.nt) * n_mb;
    uint32_t incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, incl, d);
        if (lane >= d) incl += v;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    uint32_t acc = incl - sum;
    for (int w = 0; w < warp; ++w) acc += wsum[w];
#pragma unroll 1
    for (int e = e0; e < e1; ++e) {
        const Run r = e == e0 ? run0 : run_of(p, e);
        const uint32_t n = groups(r, sh.nt) * n_mb;
        prefix[e] = acc;
        if (n) {
            uint32_t i = acc > first ? exl3b_div_of(acc - first + stride - 1, sh.stride) : 0u;
#pragma unroll 1
            for (; i < kTab && first + i * stride < acc + n; ++i)
                utab[i] = make_unit<MB>(e, r, first + i * stride - acc, sh);
        }
        acc += n;
    }
    if (tid == THREADS - 1) prefix[p.n_expert] = acc;
}

struct Pipe {
    uint32_t s = 0, ph = 0;
    __device__ __forceinline__ void next(uint32_t n) {
        if (++s == n) { s = 0; ph ^= 1u; }
    }
};

__device__ __forceinline__ uint64_t desc_sw128(uint32_t a) {      // K-major rows of 128 bytes, 8-row atoms
    return (uint64_t)((a & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}

// Four MMAs over 128 bytes of k: one stage, of K = 16 (KIND f16: f16, bf16) or 32 (f8f6f4: e4m3) each. The first accumulates
// when acc != 0.
#define EXL3B_MMA4(G, KIND)                                                                                                 \
    asm volatile(                                                                                                          \
        "{\n .reg .pred p, e, t;\n .reg .b64 a, b;\n"                                                                      \
        " setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, 0, 0;\n elect.sync _|e, 0xffffffff;\n"                                    \
        " @e tcgen05.mma.cta_group::" G ".kind::" KIND " [%0], %1, %2, %3, p;\n"                                           \
        " add.u64 a, %1, 2; add.u64 b, %2, 2;\n @e tcgen05.mma.cta_group::" G ".kind::" KIND " [%0], a, b, %3, t;\n"       \
        " add.u64 a, %1, 4; add.u64 b, %2, 4;\n @e tcgen05.mma.cta_group::" G ".kind::" KIND " [%0], a, b, %3, t;\n"       \
        " add.u64 a, %1, 6; add.u64 b, %2, 6;\n @e tcgen05.mma.cta_group::" G ".kind::" KIND " [%0], a, b, %3, t;\n"       \
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc))
template <bool PAIR>
__device__ __forceinline__ void mma4_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (PAIR) EXL3B_MMA4("2", "f16");
    else EXL3B_MMA4("1", "f16");
}
__device__ __forceinline__ void mma4_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
    const uint32_t acc = 0;
    EXL3B_MMA4("1", "f8f6f4");
}
// The MMAs issued so far done -> one arrival on bar (PAIR: on both CTAs' bar of that offset).
template <bool PAIR>
__device__ __forceinline__ void commit_el(uint64_t* bar) {
    if constexpr (PAIR)
        asm volatile("{\n .reg .pred e;\n .reg .b16 m;\n mov.b16 m, 3;\n elect.sync _|e, 0xffffffff;\n"
                     " @e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n}\n" ::
                         "r"(smem_u32(bar))
                     : "memory");
    else
        asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                     " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
                     : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
    if constexpr (PAIR) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <bool PAIR>
__device__ __forceinline__ void tmem_free(uint32_t t, uint32_t cols) {
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(cols) : "memory");
}
// 16 columns of this warp's 32 lanes; tmem_wait before the registers are read. tmem_ld16: lane l's 16 in thread l.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t r[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// ... and in 8 x 8 pieces: r[8 s + 4 h + 2 g + e] is lane 16 s + 8 g + t / 4, column 8 h + 2 (t % 4) + e in thread t, so
// that lanes 0..15 (silu_mul's gates) and 16..31 (its ups) meet in the same thread.
__device__ __forceinline__ void tmem_ld8x8(uint32_t taddr, uint32_t r[16]) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[8 * s]), "=r"(r[8 * s + 1]), "=r"(r[8 * s + 2]), "=r"(r[8 * s + 3]), "=r"(r[8 * s + 4]),
                       "=r"(r[8 * s + 5]), "=r"(r[8 * s + 6]), "=r"(r[8 * s + 7])
                     : "r"(taddr + ((16u * s) << 16)));
}
// Four 8 x 8 pieces of 16-bit pairs (columns 2 c and 2 c + 1 of lane t / 4 a word), transposed into shared memory: thread
// t's address is that of column t % 8 of piece t / 8, 16 bytes of eight lanes' values.
__device__ __forceinline__ void st8x8t(uint32_t dst, const uint32_t w[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w[0]), "r"(w[1]),
                 "r"(w[2]), "r"(w[3])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t r[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// A box of weight rows (x: k offset in elements, y: row, z: expert); elected lane of a whole warp.
__device__ __forceinline__ void tma_w_el(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n}\n" ::
                     "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}
// A block of silu_mul in one copy: box z = groups of 16 rows from `group` on, in each its gate rows and then its up rows.
__device__ __forceinline__ void tma_w5_el(void* dst, const CUtensorMap* map, int x, int group, int e, uint64_t* bar) {
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %3, %4, %5}], [%6];\n}\n" ::
                     "r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(0), "r"(group), "r"(e), "r"(smem_u32(bar))
                 : "memory");
}
// 16 bytes global -> shared; or 16 zero bytes, nothing read.
__device__ __forceinline__ void cp16(uint32_t dst, const uint8_t* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const uint8_t* src, bool read) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
// The calling thread's copies so far, landed -> one arrival on bar.
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Shared-memory writes this thread made or has been told of become visible to the asynchronous proxy (tcgen05's reads).
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// One arrival on the even CTA's barrier of the same offset. What it and the waits below order across the CTAs is tensor
// core work alone, which reads each SM's own shared and tensor memory: no thread reads what one of the other CTA wrote,
// so they keep the default (CTA) scope. Cluster scope costs a fence a stage: 805 against 356 us at 512 experts, 20480
// rows, 2048 -> 512 silu_mul.
__device__ __forceinline__ void arrive_even(uint64_t* bar) {
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, 0;\n"
                 " mbarrier.arrive.shared::cluster.b64 _, [a];\n}\n" ::"r"(smem_u32(bar))
                 : "memory");
}
// One arrival on the barrier of the same offset in the cluster's CTA `rank`, publishing what this thread has seen written.
__device__ __forceinline__ void arrive_at(uint64_t* bar, uint32_t rank) {
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n"
                 " mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n}\n" ::"r"(smem_u32(bar)), "r"(rank)
                 : "memory");
}
// Four floats at the same offset in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ void ld_cluster(const float* p, uint32_t rank, float v[4]) {
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %4, %5;\n ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n}\n"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                 : "r"(smem_u32(p)), "r"(rank)
                 : "memory");
}
// The x rows that a thread loads of a unit: rows first, first + step, ... of it. Their slots are fetched a unit ahead, so a
// unit's first copies do not wait for them. A dropped slot reads row 0 (its outputs are zeroed, not stored), a row past the
// unit's its last one; none lies past x's rows.
template <int N>
struct RowAhead {
    const Exl3bGmmOp& p;
    const int first, step;
    int32_t slot[N];
    __device__ __forceinline__ RowAhead(const Exl3bGmmOp& op, int f, int s) : p(op), first(f), step(s) {}
    __device__ __forceinline__ void fetch(const Unit& u) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = min(u.r0 + max(0, min(first + step * j, u.nr - 1)), (int)(p.n_rows - 1));
            slot[j] = p.top_k && p.sorted_tok ? p.sorted_tok[i] : i;
        }
    }
    __device__ __forceinline__ void rows(const uint8_t* base, int64_t pitch, const uint8_t* src[N]) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t t = exl3b_div_of((uint32_t)max(slot[j], 0), p.slots);
            src[j] = base + (int64_t)min(t, (uint32_t)p.x_rows - 1) * pitch;
        }
    }
};
// silu(z) * up = z / (1 + e^-z) * up, within 2^-19 of the value down to the bottom of f32's range. From -16 up the
// exponential is the special-function unit's, whose argument z log2(e) is then rounded by no more than 2^-20.
__device__ __forceinline__ float silu_up(float z, float up) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(z * -1.44269504f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + r));
    return z * r * up;
}
// ... below -16, rare enough for a branch (expf for every gate: 35.4 for 34.2 us at 64 experts, 20072 rows, 2048 -> 512,
// MXFP4). Below -60, where 1 + e^-z is e^-z to every bit, as z e^(z/2) up e^(z/2): each step is in range while the value is.
__device__ __forceinline__ float silu_up_low(float z, float up) {
    const bool far = z < -60.f;
    const float e = expf(far ? 0.5f * z : -z);
    const float v = z * (far ? e : 1.f / (1.f + e)) * up;
    return far ? v * e : v;
}
constexpr float kSiluLow = -16.f;
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if constexpr (DT == RAD_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Barrier over an epilogue group, and the same with a vote: whether any of its threads has `bad` set (they decide
// together whether to go on, since they meet at barriers).
__device__ __forceinline__ void epi_sync(int g) { asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory"); }
__device__ __forceinline__ bool epi_any(int g, bool bad) {
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(r)
                 : "r"((uint32_t)bad), "r"(1 + g)
                 : "memory");
    return r != 0;
}


// A slice's outputs: thread t's outputs t / 4 and t / 4 + 8 (act NONE: and 16 more) of four rows, from its sums as tmem_ld8x8
// gives them.
template <bool ACT>
__device__ __forceinline__ void act_slice(const uint32_t a[16], float (&v)[ACT ? 8 : 16]) {
    constexpr int NV = ACT ? 8 : 16;
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] = ACT ? silu_up(__uint_as_float(a[k]), __uint_as_float(a[(8 + k) & 15])) : __uint_as_float(a[k]);
    if constexpr (ACT) {
        float least = __uint_as_float(a[0]);
#pragma unroll
        for (int k = 1; k < NV; ++k) least = fminf(least, __uint_as_float(a[k]));
        if (least < kSiluLow) {
#pragma unroll
            for (int k = 0; k < NV; ++k)
                if (__uint_as_float(a[k]) < kSiluLow) v[k] = silu_up_low(__uint_as_float(a[k]), __uint_as_float(a[8 + k]));
        }
    }
}

// Rows outside the runs are zero: 512 bytes (MXFP4: 128 and their scales) of a row a warp, spread over the whole grid: this is
// warp w of `warps`. (A row a warp, 32 rows at a time, left the last rows to one pair: 172 us for 137 at 16 experts, 16067 of
// 16384 rows, 1536 -> 4096.)
template <int OUT>
__device__ __forceinline__ void clear_outside(const Exl3bGmmOp& p, uint32_t w, uint32_t warps, int lane) {
    if (!p.expert_offset) return;
    constexpr bool mx_out = OUT == (int)EXL3B_MX4;
    constexpr int es = OUT == RAD_F32 ? 4 : 2;
    uint8_t* const y = static_cast<uint8_t*>(p.y);
    const int64_t lo = min(max(p.expert_offset[0], 0), (int32_t)p.n_rows);
    const int64_t hi = max((int64_t)min(p.expert_offset[p.n_expert], (int32_t)p.n_rows), lo);
    const int64_t gone = lo + p.n_rows - hi;
    if (!gone) return;
    const int64_t bytes = mx_out ? p.n_out / 2 : p.n_out * es;
    const int64_t parts = (bytes + (mx_out ? 127 : 511)) / (mx_out ? 128 : 512);
    const uint32_t a = parts < warps ? (uint32_t)parts : warps, n_at = warps / a;
    const uint32_t at = w / a, part0 = w - at * a;
    if (at >= n_at) return;
    for (int64_t j = at; j < gone; j += n_at) {
        const int64_t r = j < lo ? j : j - lo + hi;
        for (int64_t c = part0; c < parts; c += a) {
            if (mx_out) {
                const int64_t o = c * 128 + lane * 4;
                if (o < bytes) *reinterpret_cast<uint32_t*>(y + r * p.y_pitch + o) = 0u;
                if (lane < 8 && c * 8 + lane < p.n_out / 32) p.y_scales[r * p.ys_pitch + c * 8 + lane] = 0;
            } else {
                const int64_t o = c * 512 + lane * 16;
                if (o < bytes) *reinterpret_cast<uint4*>(y + r * p.y_pitch * es + o) = make_uint4(0u, 0u, 0u, 0u);
            }
        }
    }
}

// A slice: v, a warp's outputs from n_warp on of up to 16 rows (`left` of them) at d. Thread t has outputs o = t / 4 and o + 8
// (act NONE: and 16 more) of four rows: 2 (t % 4), the next one, and 8 more each (tmem_ld8x8's), or with BY4 t % 4, 4 + t % 4,
// and 8 more each (tmem_ld4's). sw: 1 KB of shared memory of the warp's own.
template <int OUT, bool ACT, bool BY4 = false>
__device__ __forceinline__ void store_slice(const float (&v)[ACT ? 8 : 16], uint8_t* d, int64_t row_b, int64_t n_warp,
                                            int64_t n_out, int left, uint8_t* sw, int lane) {
    constexpr int NV = ACT ? 8 : 16;
    if constexpr (OUT == RAD_F32) {
        // straight from the registers: a warp's store is 32 bytes each of four rows
        const int o = lane >> 2, c2 = (BY4 ? 1 : 2) * (lane & 3);
        const int64_t n = n_warp + o;
        d += c2 * row_b + n * 4;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int j = 8 * (k >> 2 & 1) + (BY4 ? 4 : 1) * (k & 1), m = 16 * (k >> 3) + 8 * (k >> 1 & 1);
            if (c2 + j < left && n + m < n_out) *reinterpret_cast<float*>(d + j * row_b + 4 * m) = v[k];
        }
    } else {
        // Transposed through shared memory -- a row's outputs, 16-byte pieces swizzled against bank conflicts -- then 16 bytes
        // a thread: whole 32-byte sectors, and no warp waits for another. (Two-byte stores straight from the registers: 218
        // against 177 us at 16 experts, 16067 rows, 1536 -> 4096.)
        constexpr int P = NV / 4, SH = ACT ? 2 : 1;                   // 16-byte pieces a row; rows that share banks
        auto at = [](int row, int piece) { return (row * P + (piece ^ (row >> SH & (P - 1)))) * 16; };
        const int col = BY4 ? (lane >> 1 & 3) + 4 * (lane & 1) : lane & 7;
#pragma unroll
        for (int s = 0; s < NV / 8; ++s) {
            uint32_t w[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) w[m] = pack2<OUT>(v[8 * s + 2 * m], v[8 * s + 2 * m + 1]);
            st8x8t(smem_u32(sw) + at(8 * (lane >> 4) + col, 2 * s + (lane >> 3 & 1)), w);
        }
        __syncwarp();
#pragma unroll
        for (int s = 0; s < NV / 8; ++s) {
            const int row = (32 * s + lane) / P, piece = lane % P;
            const uint4 w = *reinterpret_cast<const uint4*>(sw + at(row, piece));
            const int64_t n = n_warp + 8 * piece;
            if (row < left && n < n_out) *reinterpret_cast<uint4*>(d + row * row_b + n * 2) = w;
        }
        __syncwarp();
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static inline EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    }
    return fn;
}

// Weights, boxes of 128 bytes of k: [expert][row][k] and a block's 128 rows; for silu_mul [expert][group of 16 rows]
// [gate, up][16][k] and a block's four groups, in one box (eight boxes of 16 rows a stage kept the issuing warp busy, 550
// cycles a stage) unless the last group is half a one and the box would leave the weight: then a box a half group.
// box_rows: plain boxes [1][box_rows][k] instead, whatever the act.
static inline int make_map(const Exl3bGmmOp* p, CUtensorMap* map, int box_rows = 0) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return -6;
    const CUtensorMapDataType dt = p->mx4 || p->f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                          : p->bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t k = (cuuint64_t)(p->mx4 ? p->n_in / 2 : p->n_in), pitch = (cuuint64_t)p->w_pitch_bytes;
    const cuuint32_t kb = p->mx4 || p->f8 ? 128u : 64u, one[5] = { 1, 1, 1, 1, 1 };
    const bool whole = !box_rows && p->act && p->n_out % 16 == 0;
    const cuuint64_t dims3[3] = { k, (cuuint64_t)p->w_rows, (cuuint64_t)p->n_expert };
    const cuuint64_t strides3[2] = { pitch, (cuuint64_t)p->w_expert_bytes };
    const cuuint32_t box3[3] = { kb, box_rows ? (cuuint32_t)box_rows : p->act ? 16u : 128u, 1u };
    const cuuint64_t dims5[5] = { k, 16, 2, (cuuint64_t)(p->n_out / 16), (cuuint64_t)p->n_expert };
    const cuuint64_t strides5[4] = { pitch, (cuuint64_t)p->n_out * pitch, 16 * pitch, (cuuint64_t)p->w_expert_bytes };
    const cuuint32_t box5[5] = { kb, 16, 2, 4, 1 };
    return fn(map, dt, whole ? 5 : 3, const_cast<void*>(p->w), whole ? dims5 : dims3, whole ? strides5 : strides3,
              whole ? box5 : box3, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0 : -6;
}

// An upper bound of the units: a group a live expert and one more each NT rows, times the blocks.
static inline int64_t most_units(const Exl3bGmmOp* p, int nt, int mb) {
    const int64_t blk = (p->act ? 64 : 128) * mb;
    const int64_t live = p->n_expert < p->n_rows ? p->n_expert : p->n_rows;
    return (live + p->n_rows / nt) * ((p->n_out + blk - 1) / blk);
}

// Sorted rows a unit of the pair form: where units of `most` leave pairs of SMs without one, as few as still give every
// pair at most one (one expert of 1024 rows, 2048 -> 2048, bf16: 16.3 us with units of 256 rows, 12.3 with these).
static inline int pair_rows(const Exl3bGmmOp* p, int most, int sm_count) {
    int nt = most;
    while (nt > 64 && most_units(p, nt - 32, 2) <= sm_count / 2) nt -= 32;
    return nt;
}

}  // namespace exl3b
