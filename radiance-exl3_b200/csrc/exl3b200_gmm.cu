// exl3b200_gmm.cu -- grouped_mm: matrix products grouped by expert with ragged sizes, over f16, bf16 or MXFP4 operands,
// on the 5th-generation tensor cores. sm_100a only.
//
//   z[n] = sum over k of x[t(i)][k] * w[e][n][k]  for every sorted row i of expert e (f32 accumulators), then
//   y[i][n] = z[n], or silu(z[n]) * z[n_out + n] (act silu_mul: w[e] holds n_out gate rows, then n_out up rows).
//
// The WEIGHT rows are the MMA's M (128 a block) and the sorted rows its N: experts hold a few to a few hundred rows, N
// goes in steps of 16, so a group of 40 rows costs 48 columns where rows as M would cost 128. A block of silu_mul is 64
// gate rows and their 64 up rows, so the epilogue has both halves of every output.
//
// One persistent CTA an SM walks the units (expert, up to NT of its sorted rows, MT blocks), expert-major, so that the
// CTAs working at one time share an expert's rows and weights in L2. Warps:
//   0      weights: cp.async.bulk.tensor of the unit's rows, 128 bytes of k a stage (64 f16 / bf16, 256 MXFP4 codes),
//          128-byte swizzled; MXFP4 scales by one bulk copy a block from their tiled form
//   1      input rows: tile::gather4 copies (a lane four rows), so x is read through sorted_tok in place
//   2      MMA issuer (and the TMEM allocation): tcgen05.mma kind::f16 (K 16) or kind::mxf4.block_scale (K 64), four a
//          block and stage; for MXFP4 tcgen05.cp moves the stage's scales into tensor memory before them
//   3      MXFP4: the input rows' scales, through registers into the layout tcgen05.cp reads
//   4..7   epilogue: tcgen05.ld, transposed through shared memory so that a row's outputs are stored contiguously;
//          silu_mul, and the rounding to y's type (MXFP4: with its blocks' scales), happen there
// Two accumulator buffers in tensor memory: one unit's epilogue runs under the next one's MMAs. Every wait is bounded;
// one that gives up sets the error word, and every role then drains and leaves.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "exl3b200_decode.cuh"
#include "exl3b200_dense.h"
#include "exl3b200_mx4.cuh"

using namespace exl3b;

namespace {

constexpr int kThreads = 256;
constexpr int kEpiWarp0 = 4, kEpiWarps = 4;
constexpr int kRowB = 128;                       // bytes of k a stage: one swizzle row
constexpr int kSlice = 16;                       // sorted rows the epilogue stages at a time
constexpr int kTab = 128;                        // a CTA's units held in a shared table (more: looked up)
constexpr int kMaxExpert = 2048;

template <bool MX, int MT, int NT>
struct Cfg {
    static constexpr int W_B = MT * 128 * kRowB;
    static constexpr int X_B = NT * kRowB;
    static constexpr int SFW_B = MX ? MT * 1024 : 0;             // two 128-k halves of 512 bytes a block
    static constexpr int SFX_B = MX ? 1024 : 0;
    static constexpr int STAGE_B = W_B + X_B + SFW_B + SFX_B;
    static constexpr int EPI_LD = MT * 128 + 4;                  // f32 a staged row, padded
    static constexpr int EPI_B = kSlice * EPI_LD * 4;
    static constexpr int ACC = MT * NT;                          // TMEM columns of one accumulator buffer
    static constexpr int SFC = MX ? 8 * MT + 8 : 0;              // TMEM columns of a stage's scales
    static constexpr int COLS = 2 * ACC + 2 * SFC;
    static constexpr int TMEM = COLS <= 32 ? 32 : COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static constexpr int PER_SM = TMEM <= 256 && MT == 1 ? 2 : 1;
    static constexpr int BUDGET = (PER_SM == 2 ? 112 : 225) * 1024 - 1024 - EPI_B - 512 - kTab * 16 - (kMaxExpert + 4) * 4;
    static constexpr int ST = BUDGET / STAGE_B > 8 ? 8 : BUDGET / STAGE_B;
    static constexpr int SMEM = 1024 + ST * STAGE_B + EPI_B + 512;   // the unit prefix follows
    static_assert(COLS <= 512 && ST >= 3, "tensor or shared memory");
    static_assert(NT <= 128 && (!MX || NT <= 128), "one gather4 a lane; one column group of scales");
};

struct Unit {
    int32_t r0;          // first sorted row
    int32_t e, blk;      // expert, first 128-row block
    int32_t nr;          // sorted rows
};

template <int NT>
__device__ __forceinline__ uint32_t groups(const Exl3bGmmOp& p, int e, int64_t* r0, int64_t* r1) {
    if (p.expert_offset) {
        *r0 = p.expert_offset[e];
        *r1 = p.expert_offset[e + 1];
        if (*r0 < 0) *r0 = 0;
        if (*r1 > p.n_rows) *r1 = p.n_rows;
    } else {
        *r0 = 0;
        *r1 = p.n_rows;
    }
    return *r1 > *r0 ? (uint32_t)((*r1 - *r0 + NT - 1) / NT) : 0u;
}

template <int NT>
__device__ __forceinline__ Unit find_unit(const Exl3bGmmOp& p, const uint32_t* prefix, uint32_t unit, uint32_t n_mb,
                                          int mt) {
    int lo = 0, hi = p.n_expert;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= unit) lo = mid; else hi = mid;
    }
    const uint32_t local = unit - prefix[lo], g = local / n_mb;
    int64_t r0, r1;
    const uint32_t ng = groups<NT>(p, lo, &r0, &r1);
    // the expert's rows split evenly over its groups, in steps of 16: no group is left with a sliver
    const int64_t per = ((r1 - r0 + ng - 1) / ng + 15) / 16 * 16;
    Unit u;
    u.e = lo;
    u.blk = (int32_t)(local % n_mb) * mt;
    const int64_t a = r0 + g * per, left = r1 - a;
    u.r0 = (int32_t)a;
    u.nr = (int32_t)(left < 0 ? 0 : left < per ? left : per);
    return u;
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
__device__ __forceinline__ uint64_t desc_plain(uint32_t a) {      // tcgen05.cp: rows of 16 bytes, 8-row cores of 128
    return (uint64_t)((a & 0x3FFFFu) >> 4) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}

// Four MMAs of K = 16 (f16 / bf16): a stage of one block. The first accumulates when acc != 0.
__device__ __forceinline__ void mma4_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, e, t;\n .reg .b64 a, b;\n"
        " setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, 0, 0;\n elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        " add.u64 a, %1, 2; add.u64 b, %2, 2;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
        " add.u64 a, %1, 4; add.u64 b, %2, 4;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
        " add.u64 a, %1, 6; add.u64 b, %2, 6;\n @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
// 512 bytes of scales (32 rows of 16) into four tensor-memory columns of all four lane quadrants.
__device__ __forceinline__ void cp_scales(uint32_t t, uint64_t desc) {
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n}\n" ::"r"(t), "l"(desc));
}
// Four MMAs of K = 64 (MXFP4): a stage of one block. Scales: two 128-k halves of four columns; within a half the first
// MMA takes bytes 0, 1 of each column and the second bytes 2, 3 (id2: the descriptor with both scale ids at 2).
__device__ __forceinline__ void mma4_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t id0, uint32_t id2, uint32_t sa,
                                         uint32_t sb, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p, e, t;\n .reg .b64 a, b;\n .reg .b32 u, v;\n"
        " setp.ne.b32 p, %7, 0;\n setp.eq.b32 t, 0, 0;\n elect.sync _|e, 0xffffffff;\n"
        " @e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n"
        " add.u64 a, %1, 2; add.u64 b, %2, 2;\n"
        " @e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %4, [%5], [%6], t;\n"
        " add.u64 a, %1, 4; add.u64 b, %2, 4; add.u32 u, %5, 4; add.u32 v, %6, 4;\n"
        " @e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [u], [v], t;\n"
        " add.u64 a, %1, 6; add.u64 b, %2, 6;\n"
        " @e tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %4, [u], [v], t;\n"
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(id0), "r"(id2), "r"(sa), "r"(sb), "r"(acc));
}
__device__ __forceinline__ void commit_el(uint64_t* bar) {
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float v[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
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
// Four rows of x (each 128 bytes from k offset x), by the calling lane.
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap* map, int x, const int r[4], uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], "
                 "[%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(smem_u32(bar))
                 : "memory");
}

// The x row of sorted row i (a dropped slot reads row 0: its outputs are zeroed, not stored), never past x's rows.
__device__ __forceinline__ int x_row(const Exl3bGmmOp& p, int64_t i) {
    if (p.top_k == 0) return (int)i;
    const int32_t f = p.sorted_tok ? p.sorted_tok[i] : (int32_t)i;
    const int32_t t = f < 0 ? 0 : f / p.top_k;
    return t < p.x_rows ? t : (int)(p.x_rows - 1);
}
// Whether any of the epilogue's threads has `bad` set (they decide together: they meet at barriers).
__device__ __forceinline__ bool epi_any(bool bad) {
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
                 : "=r"(r)
                 : "r"((uint32_t)bad), "n"(kEpiWarps * 32)
                 : "memory");
    return r != 0;
}

template <bool MX, int MT, int NT>
__global__ void __launch_bounds__(kThreads, Cfg<MX, MT, NT>::PER_SM)
    k_gmm(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Exl3bGmmOp p) {
    using C = Cfg<MX, MT, NT>;
    constexpr int ST = C::ST;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* w_ring = smem;                                   // [ST][MT][128 rows][128 B]
    uint8_t* x_ring = w_ring + ST * C::W_B;                   // [ST][NT rows][128 B]
    uint8_t* sfw_ring = x_ring + ST * C::X_B;                 // [ST][MT][2][512 B]
    uint8_t* sfx_ring = sfw_ring + ST * C::SFW_B;             // [ST][2][512 B]
    float* epi = reinterpret_cast<float*>(sfx_ring + ST * C::SFX_B);
    uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(epi) + C::EPI_B);
    uint64_t* full = bars;                                    // producers -> MMA (2, MXFP4 3 arrivals)
    uint64_t* empty = full + ST;                              // MMA commit -> producers
    uint64_t* acc_full = empty + ST;                          // MMA commit -> epilogue [2]
    uint64_t* acc_empty = acc_full + 2;                       // epilogue -> MMA [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    uint32_t* dead = tmem_slot + 1;                           // a wait gave up: everyone leaves
    uint32_t* prefix = reinterpret_cast<uint32_t*>(bars) + 128;   // [n_expert + 1]
    __shared__ Unit utab[kTab];
    static_assert((2 * ST + 4) * 8 + 8 <= 512, "barriers");

    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const int act = p.act;
    const int blk_out = act ? 64 : 128;                       // outputs a block
    const uint32_t n_mb = (uint32_t)((p.n_out + blk_out * MT - 1) / (blk_out * MT));
    if (tid == 0) {
        for (int s = 0; s < ST; ++s) { mbar_init(&full[s], MX ? 3 : 2); mbar_init(&empty[s], 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(&acc_full[s], 1); mbar_init(&acc_empty[s], kEpiWarps); }
        *dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(C::TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // prefix[e]: the first unit of expert e (block-wide exclusive scan, a thread a run of experts)
    {
        __shared__ uint32_t wsum[kThreads / 32];
        const int per = (p.n_expert + kThreads - 1) / kThreads;
        const int e0 = tid * per, e1 = min(e0 + per, p.n_expert);
        int64_t a, b;
        uint32_t sum = 0;
        for (int e = e0; e < e1; ++e) sum += groups<NT>(p, e, &a, &b) * n_mb;
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
        for (int e = e0; e < e1; ++e) {
            prefix[e] = acc;
            acc += groups<NT>(p, e, &a, &b) * n_mb;
        }
        if (tid == kThreads - 1) prefix[p.n_expert] = acc;
    }
    __syncthreads();
    const uint32_t n_units = prefix[p.n_expert];
    const uint32_t n_mine = n_units > blockIdx.x ? (n_units - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
    for (uint32_t i = tid; i < n_mine && i < kTab; i += kThreads)
        utab[i] = find_unit<NT>(p, prefix, blockIdx.x + i * gridDim.x, n_mb, MT);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
    auto unit_at = [&](uint32_t i) {
        return i < kTab ? utab[i] : find_unit<NT>(p, prefix, blockIdx.x + i * gridDim.x, n_mb, MT);
    };
    const int nck = (int)((p.n_in + (MX ? 255 : 63)) / (MX ? 256 : 64));
    volatile uint32_t* vdead = dead;
    // a bounded wait by a whole warp; false once any wait of the CTA has given up
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_wait_warp(bar, parity, p.err) && !*vdead) return true;
        *vdead = 1;
        return false;
    };
    uint32_t issued = 0;                                      // stages a producer filled
    Pipe pipe;

    if (warp == 0) {
        // ---------------------------------------------------------------- weights
        for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
            const Unit u = unit_at(i);
            for (int ck = 0; ck < nck; ++ck, pipe.next(ST), ++issued) {
                if (!wait(&empty[pipe.s], pipe.ph ^ 1)) break;
                mbar_expect_tx_el(&full[pipe.s], C::W_B + C::SFW_B);
                uint8_t* dst = w_ring + pipe.s * C::W_B;
                const int k = ck * (MX ? 128 : 64);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const int b = u.blk + m;
                    tma_w_el(dst + m * 16384, &wmap, k, b * blk_out, u.e, &full[pipe.s]);
                    tma_w_el(dst + m * 16384 + 8192, &wmap, k, act ? (int)p.n_out + b * 64 : b * 128 + 64, u.e, &full[pipe.s]);
                    if (MX)
                        tma_bulk_g2s_el(sfw_ring + pipe.s * C::SFW_B + m * 1024,
                                        p.w_scales + u.e * p.ws_expert_bytes + b * p.ws_blk_bytes + ck * 1024, 1024,
                                        &full[pipe.s]);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- input rows
        for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
            const Unit u = unit_at(i);
            const int n = (u.nr + 15) & ~15;
            int r[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = 4 * lane + j < u.nr ? x_row(p, u.r0 + 4 * lane + j) : 0;
            for (int ck = 0; ck < nck; ++ck, pipe.next(ST), ++issued) {
                if (!wait(&empty[pipe.s], pipe.ph ^ 1)) break;
                mbar_expect_tx_el(&full[pipe.s], n * kRowB);
                __syncwarp();
                if (4 * lane < n)
                    tma_gather4(smem_u32(x_ring + pipe.s * C::X_B) + lane * 512, &xmap, ck * (MX ? 128 : 64), r, &full[pipe.s]);
                __syncwarp();
            }
        }
    } else if (warp == 2) {
        // ---------------------------------------------------------------- MMA issuer
        const uint64_t wd0 = desc_sw128(smem_u32(w_ring)), xd0 = desc_sw128(smem_u32(x_ring));
        const uint64_t swd0 = desc_plain(smem_u32(sfw_ring)), sxd0 = desc_plain(smem_u32(sfx_ring));
        uint32_t ab = 0, sfp = 0;
        for (uint32_t i = 0; i < n_mine && !*vdead; ++i, ab ^= 1) {
            const Unit u = unit_at(i);
            const uint32_t n = (u.nr + 15) & ~15;
            // D f32, both operands K-major, M 128, N n; MXFP4: e2m1, E8M0 scales
            const uint32_t idesc = MX ? 1u << 7 | 1u << 10 | (n >> 3) << 17 | 1u << 23 | 8u << 24
                                      : 1u << 4 | (p.bf16 ? 1u << 7 | 1u << 10 : 0u) | (n >> 3) << 17 | 8u << 24;
            if (!wait(&acc_empty[ab], ((i >> 1) & 1) ^ 1)) break;
            fence_after();
            for (int ck = 0; ck < nck; ++ck, pipe.next(ST)) {
                if (!wait(&full[pipe.s], pipe.ph)) break;
                fence_after();
                const uint64_t xd = xd0 + (uint64_t)(pipe.s * C::X_B >> 4);
                const uint32_t sf = tmem + 2 * C::ACC + sfp * C::SFC;
                if (MX) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        cp_scales(sf + 8 * MT + 4 * h, sxd0 + (uint64_t)((pipe.s * C::SFX_B + h * 512) >> 4));
#pragma unroll
                        for (int m = 0; m < MT; ++m)
                            cp_scales(sf + 8 * m + 4 * h, swd0 + (uint64_t)((pipe.s * C::SFW_B + m * 1024 + h * 512) >> 4));
                    }
                }
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const uint32_t d = tmem + ab * C::ACC + m * NT;
                    const uint64_t wd = wd0 + (uint64_t)((pipe.s * C::W_B + m * 16384) >> 4);
                    if (MX) mma4_mx4(d, wd, xd, idesc, idesc | 2u << 4 | 2u << 29, sf + 8 * m, sf + 8 * MT, ck ? 1u : 0u);
                    else mma4_f16(d, wd, xd, idesc, ck ? 1u : 0u);
                }
                sfp ^= 1;
                commit_el(&empty[pipe.s]);
            }
            commit_el(&acc_full[ab]);
        }
    } else if (warp == 3) {
        // ---------------------------------------------------------------- MXFP4: the input rows' scales
        // Lane l holds rows l, l + 32, ... of the group, so that it writes 16 consecutive bytes of the layout (row r at
        // (r % 32) * 16 + (r / 32) * 4, four scales of 128 k). Chunks are fetched kAhead at a time, one batch ahead.
        if (MX) {
            constexpr int Q = (NT + 31) / 32, kAhead = 4;
            const int nsc = (int)(p.n_in / 32);
            const bool wide = (p.xs_pitch & 7) == 0 && (reinterpret_cast<uintptr_t>(p.x_scales) & 7) == 0;
            for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
                const Unit u = unit_at(i);
                const uint8_t* src[Q];
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    const int j = lane + 32 * q;
                    src[q] = j < u.nr ? p.x_scales + (int64_t)x_row(p, u.r0 + j) * p.xs_pitch : nullptr;
                }
                auto fetch = [&](int ck, uint2 v[Q]) {
#pragma unroll
                    for (int q = 0; q < Q; ++q) {
                        v[q] = make_uint2(0u, 0u);
                        if (!src[q] || ck >= nck) continue;
                        if (wide && ck * 8 + 8 <= nsc) {
                            v[q] = *reinterpret_cast<const uint2*>(src[q] + ck * 8);
                        } else {
                            for (int b = 0; b < 8; ++b)
                                if (ck * 8 + b < nsc) {
                                    const uint32_t w = (uint32_t)src[q][ck * 8 + b] << (8 * (b & 3));
                                    if (b < 4) v[q].x |= w; else v[q].y |= w;
                                }
                        }
                    }
                };
                uint2 cur[kAhead][Q], nxt[kAhead][Q];
#pragma unroll
                for (int a = 0; a < kAhead; ++a) fetch(a, cur[a]);
                bool go = true;
                for (int c0 = 0; c0 < nck && go; c0 += kAhead) {
#pragma unroll
                    for (int a = 0; a < kAhead; ++a) fetch(c0 + kAhead + a, nxt[a]);
#pragma unroll
                    for (int a = 0; a < kAhead; ++a) {
                        if (c0 + a >= nck || !go) continue;
                        if (!wait(&empty[pipe.s], pipe.ph ^ 1)) { go = false; continue; }
                        uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
                        lo.x = cur[a][0].x; hi.x = cur[a][0].y;
                        if (Q > 1) { lo.y = cur[a][Q > 1 ? 1 : 0].x; hi.y = cur[a][Q > 1 ? 1 : 0].y; }
                        if (Q > 2) { lo.z = cur[a][Q > 2 ? 2 : 0].x; hi.z = cur[a][Q > 2 ? 2 : 0].y; }
                        if (Q > 3) { lo.w = cur[a][Q > 3 ? 3 : 0].x; hi.w = cur[a][Q > 3 ? 3 : 0].y; }
                        uint4* dst = reinterpret_cast<uint4*>(sfx_ring + pipe.s * C::SFX_B) + lane;
                        dst[0] = lo;
                        dst[32] = hi;
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&full[pipe.s]);
                        pipe.next(ST);
                    }
#pragma unroll
                    for (int a = 0; a < kAhead; ++a)
#pragma unroll
                        for (int q = 0; q < Q; ++q) cur[a][q] = nxt[a][q];
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- epilogue
        const int q = warp & 3, ew = warp - kEpiWarp0;
        const int es = p.y_dtype == RAD_F32 ? 4 : 2;
        uint8_t* const y = static_cast<uint8_t*>(p.y);
        const bool mx_out = p.y_dtype == EXL3B_MX4;
        // rows no unit writes (outside the runs, dropped slots) are zero: a warp clears a row
        {
            int64_t lo = 0, hi = p.n_rows;
            if (p.expert_offset) {
                lo = p.expert_offset[0];
                hi = p.expert_offset[p.n_expert];
            }
            for (int64_t b = ((int64_t)blockIdx.x * kEpiWarps + ew) * 32; b < p.n_rows; b += (int64_t)gridDim.x * kEpiWarps * 32) {
                const int64_t i = b + lane;
                const bool gone = i < p.n_rows && (i < lo || i >= hi || (p.sorted_tok && p.sorted_tok[i] < 0));
                uint32_t mask = __ballot_sync(0xFFFFFFFFu, gone);
                while (mask) {
                    const int64_t r = b + __ffs(mask) - 1;
                    mask &= mask - 1;
                    if (mx_out) {
                        for (int64_t c = lane * 4; c < p.n_out / 2; c += 128) *reinterpret_cast<uint32_t*>(y + r * p.y_pitch + c) = 0u;
                        for (int64_t c = lane; c < p.n_out / 32; c += 32) p.y_scales[r * p.ys_pitch + c] = 0;
                    } else {
                        uint8_t* dst = y + r * p.y_pitch * es;
                        for (int64_t c = lane * 16; c < p.n_out * es; c += 512) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0u, 0u, 0u, 0u);
                    }
                }
            }
        }
        const int oc = MT * blk_out;                          // outputs a unit: 8 a lane
        const int lpt = oc / 8, tpw = 32 / lpt;               // lanes a row, rows a warp stores at a time
        const int c0 = (lane % lpt) * 8;                      // the lane's first output in the unit
        const int sc = act ? (c0 >> 6) * 128 + (c0 & 63) : c0;   // ... and its column in the staged row
        uint32_t ab = 0;
        for (uint32_t i = 0; i < n_mine; ++i, ab ^= 1) {
            const Unit u = unit_at(i);
            const int64_t n0 = (int64_t)u.blk * blk_out + c0;
            const bool col_ok = n0 < p.n_out;
            if (epi_any(!wait(&acc_full[ab], (i >> 1) & 1))) break;
            fence_after();
            for (int t0 = 0; t0 < u.nr; t0 += kSlice) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    float v[16];
                    tmem_ld16(tmem + ((uint32_t)(32 * q) << 16) + ab * C::ACC + m * NT + t0, v);
#pragma unroll
                    for (int j = 0; j < 16; ++j) epi[j * C::EPI_LD + m * 128 + 32 * q + lane] = v[j];
                }
                asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
                for (int j = ew * tpw + lane / lpt; j < kSlice; j += kEpiWarps * tpw) {
                    const int64_t r = u.r0 + t0 + j;
                    const bool row_ok = t0 + j < u.nr && !(p.sorted_tok && p.sorted_tok[r] < 0);
                    float v[8];
                    {
                        const float4* s = reinterpret_cast<const float4*>(&epi[j * C::EPI_LD + sc]);
                        const float4 a = s[0], b = s[1];
                        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
                        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
                    }
                    if (act) {
                        const float4* s = reinterpret_cast<const float4*>(&epi[j * C::EPI_LD + sc + 64]);
                        const float4 a = s[0], b = s[1];
                        const float up[8] = { a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w };
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = v[e] / (1.f + __expf(-v[e])) * up[e];
                    }
                    if (mx_out) {
                        const uint32_t code = mx4_quad_code(v);          // four lanes: 32 outputs of one row
                        if (row_ok && col_ok) {
                            *reinterpret_cast<uint32_t*>(y + r * p.y_pitch + n0 / 2) = mx4_pack8(v, code);
                            if ((lane & 3) == 0) p.y_scales[r * p.ys_pitch + n0 / 32] = (uint8_t)code;
                        }
                    } else if (row_ok && col_ok) {
                        uint8_t* dst = y + (r * p.y_pitch + n0) * es;
                        if (p.y_dtype == RAD_F32) st8<1>(dst, v);
                        else if (p.y_dtype == RAD_F16) st8<2>(dst, v);
                        else st8<3>(dst, v);
                    }
                }
                asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
            }
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[ab]);
        }
    }
    // after a wait that gave up: a producer's copies still in flight land before the CTA's memory goes
    if (*vdead && (warp == 0 || warp == 1)) {
        for (uint32_t j = 0; j < ST && j < issued; ++j) {
            const uint32_t at = issued - 1 - j;
            mbar_wait_warp(&full[at % ST], (at / ST) & 1, nullptr);
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 2) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM) : "memory");
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
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

// Weights: [expert][row][k], boxes of 64 rows; input rows: [row][k], boxes of one row (gather4). 128 bytes of k a box.
int make_maps(const Exl3bGmmOp* p, CUtensorMap* wmap, CUtensorMap* xmap) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return -6;
    const CUtensorMapDataType dt = p->mx4 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                          : p->bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t k = (cuuint64_t)(p->mx4 ? p->n_in / 2 : p->n_in);
    const cuuint32_t kb = p->mx4 ? 128 : 64, one[3] = { 1, 1, 1 };
    const cuuint64_t wd[3] = { k, (cuuint64_t)p->w_rows, (cuuint64_t)p->n_expert };
    const cuuint64_t ws[2] = { (cuuint64_t)p->w_pitch_bytes, (cuuint64_t)p->w_expert_bytes };
    const cuuint32_t wb[3] = { kb, 64, 1 };
    if (fn(wmap, dt, 3, const_cast<void*>(p->w), wd, ws, wb, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return -6;
    const cuuint64_t xd[2] = { k, (cuuint64_t)p->x_rows };
    const cuuint64_t xs[1] = { (cuuint64_t)p->x_pitch_bytes };
    const cuuint32_t xb[2] = { kb, 1 };
    if (fn(xmap, dt, 2, const_cast<void*>(p->x), xd, xs, xb, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return -6;
    return 0;
}

template <bool MX, int MT, int NT>
int launch(const Exl3bGmmOp* p, int sm_count, cudaStream_t st) {
    using C = Cfg<MX, MT, NT>;
    CUtensorMap wmap, xmap;
    const int rc = make_maps(p, &wmap, &xmap);
    if (rc) return rc;
    const int smem = C::SMEM + (p->n_expert + 4) * 4;
    auto kern = k_gmm<MX, MT, NT>;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -6;
    // at most this many units: a group a live expert, and one more each NT rows
    const int64_t blk = (p->act ? 64 : 128) * MT, n_mb = (p->n_out + blk - 1) / blk;
    const int64_t live = p->n_expert < p->n_rows ? p->n_expert : p->n_rows;
    const int64_t most = (live + p->n_rows / NT) * n_mb;
    int64_t grid = (int64_t)sm_count * C::PER_SM;
    if (most < grid) grid = most;
    kern<<<(unsigned)grid, kThreads, smem, st>>>(wmap, xmap, *p);
    return cudaGetLastError() == cudaSuccess ? 0 : -6;
}

}  // namespace

extern "C" int exl3b_cuda_gmm(const Exl3bGmmOp* p, int sm_count, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // narrow units (128 weight rows, 32 sorted rows, two CTAs an SM) while the experts hold few rows on average: more
    // units to spread a few experts' weights over the SMs; wide ones (256 weight rows) read each input row half as often
    const bool narrow = p->n_rows <= 16 * (int64_t)p->n_expert;
    if (p->mx4) return narrow ? launch<true, 1, 32>(p, sm_count, st) : launch<true, 2, 112>(p, sm_count, st);
    return narrow ? launch<false, 1, 32>(p, sm_count, st) : launch<false, 2, 128>(p, sm_count, st);
}

extern "C" int exl3b_gmm_max_expert(void) { return kMaxExpert; }
