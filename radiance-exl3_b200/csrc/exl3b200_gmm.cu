// exl3b200_gmm.cu -- grouped_mm: matrix products grouped by expert with ragged sizes, over f16, bf16 or MXFP4 operands,
// on the 5th-generation tensor cores. sm_100a only.
//
//   z[n] = sum over k of x[t(i)][k] * w[e][n][k]  for every sorted row i of expert e (f32 accumulators), then
//   y[i][n] = z[n], or silu(z[n]) * z[n_out + n] (act silu_mul: w[e] holds n_out gate rows, then n_out up rows).
//
// The WEIGHT rows are the MMA's M (128 a CTA) and the sorted rows its N: experts hold a few to a few hundred rows, N
// goes in steps of 16 (PAIR: 32), so a group of 40 rows costs 48 (64) columns where rows as M would cost 128. A block of
// silu_mul is 64 gate rows and their 64 up rows, 16 of each in turn: an epilogue warp, which can read 32 lanes of tensor
// memory, has both halves of its 16 outputs.
//
// Three forms of one kernel, all persistent over units (expert, a group of its sorted rows, a block of weight rows),
// expert-major, so that the CTAs working at one time share an expert's rows and weights in L2:
//   narrow  a CTA a unit of 128 weight rows and up to 32 sorted rows, two CTAs an SM: a few rows an expert, where the
//           weights' bytes count and units are needed to spread them over the SMs
//   SPLIT   the narrow form with few units: a cluster for each of them, every CTA a part of its k, the parts summed
//           through distributed shared memory in the CTAs' order
//   PAIR    two CTAs (a cluster) a unit of 256 weight rows and up to 256 sorted rows (MXFP4: 224, the scales take
//           tensor memory), tcgen05 cta_group::2: each CTA brings its 128 weight rows and HALF of the sorted rows, and
//           both multiply by all of them: 64 KB brought in a stage of 256 x 256 where two CTAs alone would bring 96 KB
// Warps of a CTA:
//   0       weights: cp.async.bulk.tensor of its 128 rows, 128 bytes of k a stage (64 f16 / bf16, 256 MXFP4 codes),
//           128-byte swizzled; MXFP4 scales by one bulk copy from their tiled form
//   1       MMA issuer (PAIR: of the even CTA; the odd one's reports its filled stages there): four tcgen05.mma a stage,
//           kind::f16 (K 16) or kind::mxf4.block_scale (K 64, tcgen05.cp moving the stage's scales before them)
//   2, 3    MXFP4: the sorted rows' scales, 128 rows a warp, through registers into the layout tcgen05.cp reads
//   4..7    sorted rows: 16-byte cp.async through sorted_tok into the same swizzle (tile::gather4 copies took ~80 cycles
//           for four rows: 444 against 205 us at 16 experts, 16067 rows, 1536 -> 4096)
//   8..     epilogue, groups of four warps: tcgen05.ld, silu_mul, the rounding to y's type, and the transposition through
//           shared memory by which whole 32-byte sectors of a row are stored (MXFP4: with their blocks' scales)
// Two accumulator buffers in tensor memory: one unit's epilogue runs under the next one's MMAs. Every wait is bounded;
// one that gives up sets the error word, and every role then drains and leaves.
//
// Measured on one B200 that copies 6539 GB/s and reaches 1650 TFLOP/s of bf16 in its library product; a launch's time in a
// CUDA graph, and what bounds it:
//   512 experts, 191 live of 624 rows, 640 -> 2560, bf16 (narrow)           95 us  6.6 TB/s: the weights' bytes
//   512 experts, 418 live of 20072 rows, 2048 -> 512 silu_mul, f16 (PAIR)  279 us  6.4 TB/s: the weights' bytes
//   16 experts of 16060 rows, 1536 -> 4096, bf16 (PAIR)                    151 us  1338 TFLOP/s: a stage of 256 x 256 x 64 in
//     about 510 cycles, the MMAs' own time at full rate, at a clock that power brings down to 1.2 .. 1.5 GHz
//   16 experts of 16060 rows, 4096 -> 1536, MXFP4 (PAIR)                    54 us  3743 TFLOP/s: a stage of 33 KB a CTA in
//     ~650 cycles where its MMAs take ~450: 51 bytes a cycle into an SM, in both MXFP4 cases, while L2 is at 29 % of its
//     peak (64 experts): the way into the SM, by inference, no counter; seven units a pair at most where 6.5 would do
//   64 experts of 20072 rows, 2048 -> 512 silu_mul, MXFP4 (PAIR)            31 us  2735 TFLOP/s: the same, 29 KB in ~560
//     cycles, and five of the 31 us before the first stage is there (launch, set-up, the first loads)
//   one token's ten experts, 2048 -> 512 silu_mul, f16 (narrow)             13 us  42 MB, 6.4 us at the copy rate; the rest
//     is the launch, the set-up and the first stage's latency. The same in MXFP4 (narrow): 8 us, of them 1.7 for bytes
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "exl3b200_chain.cuh"
#include "exl3b200_decode.cuh"
#include "exl3b200_dense.h"
#include "exl3b200_mx4.cuh"

using namespace exl3b;

namespace {

constexpr int kXWarp0 = 4, kXWarps = 4, kEpiWarp0 = 8;
constexpr int kRowB = 128;                       // bytes of k a stage: one swizzle row
constexpr int kW_B = 128 * kRowB;                // a CTA's weight rows of a stage
constexpr int kSlice = 16;                       // sorted rows an epilogue group takes at a time
constexpr int kMaxTurn = 16;                      // slices a unit at most
constexpr int kStage = 8;                        // ... and stages at once, where it stages in f32
constexpr int kEpiLd = 128 + 4;                  // f32 a staged row, padded
constexpr int kTab = 128;                        // a CTA's units held in a shared table (more: looked up)
constexpr int kStatic = 3072;                    // the static shared arrays, up to the ring's alignment
constexpr int kMaxExpert = 2048;
constexpr int kMaxSplit = 4;                     // CTAs a unit at most (SPLIT)
constexpr int kMaxSt = 10;                       // stages at most

template <bool MX, bool PAIR, bool SPLIT>
struct Cfg {
    static constexpr int NT = !PAIR ? 32 : MX ? 224 : 256;       // sorted rows a unit at most
    static constexpr int NL = PAIR ? NT / 2 : NT;                // ... of which this CTA brings
    // epilogue groups of four warps; PAIR: the third counts where the epilogue is the longer part, 16 experts of 16060 rows,
    // bf16 256 -> 1024 silu_mul in 28 us with two and 26 with three, and costs nothing elsewhere
    static constexpr int EPI_G = PAIR ? 3 : 1;
    static constexpr int THREADS = (kEpiWarp0 + 4 * EPI_G) * 32;
    static constexpr int X_B = NL * kRowB;
    static constexpr int SFW_B = MX ? 1024 : 0;                  // two 128-k halves of 512 bytes
    static constexpr int SFX_G = MX ? (NT + 127) / 128 : 0;      // 128-row groups of the sorted rows' scales
    static constexpr int SFX_B = SFX_G * 1024;
    static constexpr int STAGE_B = kW_B + X_B + SFW_B + SFX_B;
    static constexpr int EPI_B = (SPLIT ? NT : EPI_G * kStage) * kEpiLd * 4;
    static constexpr int SFC = MX ? 8 + 8 * SFX_G : 0;           // TMEM columns of a stage's scales
    static constexpr int COLS = 2 * NT + 2 * SFC;
    static constexpr int TMEM = COLS <= 64 ? 64 : COLS <= 128 ? 128 : 512;
    static constexpr int PER_SM = PAIR ? 1 : 2;
    // shared memory: alignment, staging, barriers, the unit prefix, and as many stages as fit beside the static arrays (the
    // narrow form: twice an SM)
    static constexpr int fixed(int n_expert) { return 1024 + EPI_B + 512 + (n_expert + 4) * 4; }
    static constexpr int stages(int n_expert, int per_sm) {
        const int n = ((per_sm == 1 ? 227 : 113) * 1024 - kStatic - fixed(n_expert)) / STAGE_B;
        return n < kMaxSt ? n : kMaxSt;
    }
    static_assert(COLS <= 512 && stages(kMaxExpert, PER_SM) >= (SPLIT ? 3 : 4), "tensor or shared memory");
    static_assert((2 * kMaxSt + 5) * 8 + 8 <= 512, "barriers");
};

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

// Four MMAs of K = 16 (f16 / bf16): one stage. The first accumulates when acc != 0.
#define EXL3B_MMA4_F16(G)                                                                                          \
    asm volatile(                                                                                                  \
        "{\n .reg .pred p, e, t;\n .reg .b64 a, b;\n"                                                              \
        " setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, 0, 0;\n elect.sync _|e, 0xffffffff;\n"                            \
        " @e tcgen05.mma.cta_group::" G ".kind::f16 [%0], %1, %2, %3, p;\n"                                        \
        " add.u64 a, %1, 2; add.u64 b, %2, 2;\n @e tcgen05.mma.cta_group::" G ".kind::f16 [%0], a, b, %3, t;\n"    \
        " add.u64 a, %1, 4; add.u64 b, %2, 4;\n @e tcgen05.mma.cta_group::" G ".kind::f16 [%0], a, b, %3, t;\n"    \
        " add.u64 a, %1, 6; add.u64 b, %2, 6;\n @e tcgen05.mma.cta_group::" G ".kind::f16 [%0], a, b, %3, t;\n"    \
        "}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc))
template <bool PAIR>
__device__ __forceinline__ void mma4_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (PAIR) EXL3B_MMA4_F16("2");
    else EXL3B_MMA4_F16("1");
}
// One MXFP4 stage: its scales into tensor memory (512 bytes, 32 rows of 16, into four columns of all four lane quadrants;
// PAIR: of both CTAs, each from its own shared memory), then four MMAs of K = 64. Scales: two 128-k halves; the weight
// rows' 4 columns a half from t on, the sorted rows' 4 G columns a half behind them. Within a half the first MMA takes
// bytes 0, 1 of each column and the second bytes 2, 3 (id2: the descriptor with both scale ids at 2). sw, sx: the
// descriptors of the weight rows' and the sorted rows' scales, [half][group][512 B].
#define EXL3B_CP(G, T, D) " @e tcgen05.cp.cta_group::" G ".32x128b.warpx4 [" T "], " D ";\n"
#define EXL3B_MX(G, A, B, I, SA, SB, P) \
    " @e tcgen05.mma.cta_group::" G ".kind::mxf4.block_scale.scale_vec::2X [%0], " A ", " B ", " I ", [" SA "], [" SB "], " P ";\n"
#define EXL3B_STAGE_HEAD                                                                                            \
    "{\n .reg .pred p, e, t;\n .reg .b64 a, b, w1, x1, x2, x3;\n .reg .b32 u, sb, v, x;\n"                          \
    " setp.ne.b32 p, %6, 0;\n setp.eq.b32 t, 0, 0;\n elect.sync _|e, 0xffffffff;\n"                                  \
    " add.u64 w1, %7, 32; add.u64 x1, %8, 32; add.u64 x2, %8, 64; add.u64 x3, %8, 96;\n"                             \
    " add.u32 u, %5, 4; add.u32 sb, %5, 8; add.u32 x, %5, 12; add.u32 v, sb, %9;\n"
#define EXL3B_STAGE_MMA(G)                                                                    \
    EXL3B_MX(G, "%1", "%2", "%3", "%5", "sb", "p")                                            \
    " add.u64 a, %1, 2; add.u64 b, %2, 2;\n" EXL3B_MX(G, "a", "b", "%4", "%5", "sb", "t")    \
    " add.u64 a, %1, 4; add.u64 b, %2, 4;\n" EXL3B_MX(G, "a", "b", "%3", "u", "v", "t")      \
    " add.u64 a, %1, 6; add.u64 b, %2, 6;\n" EXL3B_MX(G, "a", "b", "%4", "u", "v", "t") "}\n"
template <bool PAIR, int G>
__device__ __forceinline__ void stage_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t id0, uint32_t id2, uint32_t t,
                                          uint32_t acc, uint64_t sw, uint64_t sx) {
    if constexpr (PAIR)
        asm volatile(EXL3B_STAGE_HEAD EXL3B_CP("2", "%5", "%7") EXL3B_CP("2", "u", "w1") EXL3B_CP("2", "sb", "%8")
                         EXL3B_CP("2", "x", "x1") EXL3B_CP("2", "v", "x2") " add.u32 x, v, 4;\n" EXL3B_CP("2", "x", "x3")
                             EXL3B_STAGE_MMA("2") ::"r"(d), "l"(a), "l"(b), "r"(id0), "r"(id2), "r"(t), "r"(acc), "l"(sw),
                     "l"(sx), "n"(4 * G));
    else
        asm volatile(EXL3B_STAGE_HEAD EXL3B_CP("1", "%5", "%7") EXL3B_CP("1", "u", "w1") EXL3B_CP("1", "sb", "%8")
                         EXL3B_CP("1", "v", "x1") EXL3B_STAGE_MMA("1") ::"r"(d), "l"(a), "l"(b), "r"(id0), "r"(id2), "r"(t),
                     "r"(acc), "l"(sw), "l"(sx), "n"(4 * G));
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
// 16 scales of an x row from byte `off` on; what lies past the row's end is some byte or other. Rows on 16-byte boundaries
// are one load (`whole`; of the last row only where the row has them). Else the five words that hold them, shifted when they
// are used, not when they are loaded (85 and 55 us at 174 experts of 118 rows, 3808 -> 320); and byte by byte a word that
// would leave the scales' memory.
struct RowScales {
    const uint8_t *lo, *hi, *last;
    bool whole;
    __device__ __forceinline__ RowScales(const Exl3bGmmOp& p)
        : lo(p.x_scales), hi(p.x_scales + (p.x_rows - 1) * p.xs_pitch + p.n_in / 32), last(hi - p.n_in / 32),
          whole(((reinterpret_cast<uintptr_t>(p.x_scales) | (uintptr_t)p.xs_pitch) & 15) == 0) {}
    template <int U>
    __device__ __forceinline__ uint32_t word(const uint8_t* b) const {
        if (b >= lo && b + 4 <= hi) return *reinterpret_cast<const uint32_t*>(b);
        uint32_t w = 0;
#pragma unroll U
        for (int j = 0; j < 4; ++j)
            if (b + j >= lo && b + j < hi) w |= (uint32_t)b[j] << (8 * j);
        return w;
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

// OUT: y_dtype; ACT: silu_mul.
template <bool MX, bool PAIR, bool SPLIT, int OUT, bool ACT>
__global__ void __launch_bounds__(Cfg<MX, PAIR, SPLIT>::THREADS, Cfg<MX, PAIR, SPLIT>::PER_SM)
    k_gmm(const __grid_constant__ CUtensorMap wmap, const Exl3bGmmOp p, const Shape sh) {
    const int ST = sh.st, split = sh.split;
    using C = Cfg<MX, PAIR, SPLIT>;
    constexpr int NT = C::NT, THREADS = C::THREADS;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* w_ring = smem;                                   // [ST][128 rows][128 B]
    uint8_t* x_ring = w_ring + ST * kW_B;                     // [ST][NL rows][128 B]
    uint8_t* sfw_ring = x_ring + ST * C::X_B;                 // [ST][2 halves][512 B]
    uint8_t* sfx_ring = sfw_ring + ST * C::SFW_B;             // [ST][2 halves][SFX_G][512 B]
    float* epi = reinterpret_cast<float*>(sfx_ring + ST * C::SFX_B);
    uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(epi) + C::EPI_B);
    uint64_t* full = bars;                                    // producers (PAIR: and the odd CTA's MMA warp) -> MMA warp
    uint64_t* empty = full + ST;                              // MMA commit -> producers
    uint64_t* acc_full = empty + ST;                          // MMA commit -> epilogue [2]
    uint64_t* acc_empty = acc_full + 2;                       // epilogue (PAIR: of both CTAs) -> MMA [2]
    uint64_t* part_full = acc_empty + 2;                      // SPLIT: every CTA's partial sums are in its shared memory
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(part_full + 1);
    uint32_t* dead = tmem_slot + 1;                           // a wait gave up: everyone leaves
    uint32_t* prefix = reinterpret_cast<uint32_t*>(bars) + 128;   // [n_expert + 1]
    __shared__ Unit utab[kTab];

    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const uint32_t rank = PAIR ? blockIdx.x & 1u : 0u;        // which half of the unit's weight rows
    const uint32_t part = SPLIT ? blockIdx.x % split : 0u;    // which part of its k
    const uint32_t first = PAIR ? blockIdx.x >> 1 : SPLIT ? blockIdx.x / split : blockIdx.x;
    const uint32_t stride = sh.stride.d;
    constexpr bool act = ACT;
    const int blk_out = act ? 64 : 128;                       // outputs a block (a CTA's part of a unit)
    constexpr int MB = PAIR ? 2 : 1;
    const uint32_t n_mb = sh.n_mb.d;
    const int per = (p.n_expert + THREADS - 1) / THREADS, e0 = tid * per, e1 = min(e0 + per, p.n_expert);
    if (tid < ST) {
        mbar_init(&full[tid], 1 + 32 * kXWarps + C::SFX_G + (PAIR && rank == 0 ? 1 : 0));
        mbar_init(&empty[tid], 1);
    } else if (tid < ST + 2) {
        mbar_init(&acc_full[tid - ST], 1);
        mbar_init(&acc_empty[tid - ST], 4 * C::EPI_G * MB);
    } else if (tid == ST + 2) {
        *dead = 0;
        if (SPLIT) mbar_init(part_full, 4 * split);
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&wmap)) : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    if (warp == 1) tmem_alloc<PAIR>(tmem_slot, C::TMEM);
    if (PAIR || SPLIT) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    chain_wait();                                             // all above needs no memory but the CTA's own
    const Run run0 = e0 < e1 ? run_of(p, e0) : Run{ 0, 0 };
    // prefix[e]: the first unit of expert e (block-wide exclusive scan, a thread a run of experts); this CTA's units
    // (first, first + stride, ...) go into the table by the threads that pass over their experts
    {
        __shared__ uint32_t wsum[THREADS / 32];
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
    fence_before();
    __syncthreads();
    if (PAIR || SPLIT) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // all CTAs' barriers and tensor memory are set up
    fence_after();
    chain_next();                                             // every CTA has its tensor memory: a later kernel may ask for its own
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
    const uint32_t n_units = prefix[p.n_expert];
    // SPLIT: the grid has a cluster for every unit that offsets in ascending order can make, so one at most
    const uint32_t n_mine = n_units > first ? SPLIT ? 1u : exl3b_div_of(n_units - first + stride - 1, sh.stride) : 0u;
    auto unit_at = [&](uint32_t i) {
        return i < kTab ? utab[i] : find_unit<MB>(p, prefix, first + i * stride, sh);
    };
    const int nck = sh.nck;
    // this CTA's stages of a unit
    static_assert(!(MX && SPLIT), "scales are read from even stages on");
    const int k0 = SPLIT ? (int)(part * (uint32_t)nck / (uint32_t)split) : 0;
    const int k1 = SPLIT ? (int)((part + 1) * (uint32_t)nck / (uint32_t)split) : nck;
    volatile uint32_t* vdead = dead;
    // A bounded wait by a whole warp, which reports nothing: one that gives up marks the CTA dead, every other wait of the
    // CTA then gives up at its next try, and the roles leave at their next unit. (A result tested each stage cost up to
    // a seventh: 205 against 192 us at 16 experts, 16067 rows, 1536 -> 4096; 92 against 79 in MXFP4.)
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        const uint32_t a = smem_u32(bar);
        uint64_t t0 = 0;
        for (;;) {
            uint32_t done;
            asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
                         " selp.u32 %0, 1, 0, p;\n}\n"
                         : "=r"(done)
                         : "r"(a), "r"(parity), "r"(kSuspendNs)
                         : "memory");
            if (done || *vdead) break;
            const uint64_t now = globaltimer_ns();
            if (!t0) t0 = now;
            else if (now - t0 > kWaitLimitNs) {
                *vdead = 1;
                atomicOr(p.err, 1);
                break;
            }
        }
        __syncwarp();
    };
    Pipe pipe;

    if (warp == 0) {
        // ---------------------------------------------------------------- weights
        for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
            const Unit u = unit_at(i);
            const int b = u.blk + (int)rank;
            for (int ck = k0; ck < k1; ++ck, pipe.next(ST)) {
                wait(&empty[pipe.s], pipe.ph ^ 1);
                mbar_expect_tx_el(&full[pipe.s], kW_B + C::SFW_B);
                uint8_t* dst = w_ring + pipe.s * kW_B;
                const int k = ck * (MX ? 128 : 64);
                if (!act) {
                    tma_w_el(dst, &wmap, k, b * 128, u.e, &full[pipe.s]);
                } else if (p.n_out % 16 == 0) {
                    tma_w5_el(dst, &wmap, k, b * 4, u.e, &full[pipe.s]);
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        tma_w_el(dst + q * 4096, &wmap, k, b * 64 + 16 * q, u.e, &full[pipe.s]);
                        tma_w_el(dst + q * 4096 + 2048, &wmap, k, (int)p.n_out + b * 64 + 16 * q, u.e, &full[pipe.s]);
                    }
                }
                if (MX)
                    tma_bulk_g2s_el(sfw_ring + pipe.s * C::SFW_B,
                                    p.w_scales + u.e * p.ws_expert_bytes + b * p.ws_blk_bytes + ck * 1024, 1024,
                                    &full[pipe.s]);
            }
        }
        // after a wait that gave up: a millisecond for the copies still in flight, before the CTA's memory goes
        if (*vdead)
            for (int j = 0; j < 50; ++j) __nanosleep(20000);
    } else if (warp == 1 && rank == 1) {
        // ---------------------------------------------------------------- PAIR, odd CTA: its filled stages, reported
        for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
            for (int ck = k0; ck < k1; ++ck, pipe.next(ST)) {
                wait(&full[pipe.s], pipe.ph);
                proxy_fence();
                if (lane == 0) arrive_even(&full[pipe.s]);
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        const uint64_t wd0 = desc_sw128(smem_u32(w_ring)), xd0 = desc_sw128(smem_u32(x_ring));
        const uint64_t swd0 = desc_plain(smem_u32(sfw_ring)), sxd0 = desc_plain(smem_u32(sfx_ring));
        uint32_t ab = 0, sfp = 0;
        for (uint32_t i = 0; i < n_mine && !*vdead; ++i, ab ^= 1) {
            const Unit u = unit_at(i);
            const uint32_t n = (u.nr + 16 * MB - 1) & ~(16 * MB - 1);
            // D f32, both operands K-major, M 128 (PAIR: 256), N n; MXFP4: e2m1, E8M0 scales
            const uint32_t idesc = (n >> 3) << 17 | (8u * MB) << 24 |
                                   (MX ? 1u << 7 | 1u << 10 | 1u << 23 : 1u << 4 | (p.bf16 ? 1u << 7 | 1u << 10 : 0u));
            wait(&acc_empty[ab], ((i >> 1) & 1) ^ 1);
            fence_after();
            const uint32_t d = tmem + ab * NT;
            for (int ck = k0; ck < k1; ++ck, pipe.next(ST)) {
                wait(&full[pipe.s], pipe.ph);
                proxy_fence();
                fence_after();
                const uint64_t wd = wd0 + (uint64_t)(pipe.s * kW_B >> 4), xd = xd0 + (uint64_t)(pipe.s * C::X_B >> 4);
                if constexpr (MX) {
                    stage_mx4<PAIR, C::SFX_G>(d, wd, xd, idesc, idesc | 2u << 4 | 2u << 29, tmem + 2 * NT + sfp * C::SFC,
                                              ck > k0 ? 1u : 0u, swd0 + (uint64_t)(pipe.s * C::SFW_B >> 4),
                                              sxd0 + (uint64_t)(pipe.s * C::SFX_B >> 4));
                    sfp ^= 1;
                } else {
                    mma4_f16<PAIR>(d, wd, xd, idesc, ck > k0 ? 1u : 0u);
                }
                commit_el<PAIR>(&empty[pipe.s]);
            }
            commit_el<PAIR>(&acc_full[ab]);
        }
    } else if (warp < kXWarp0) {
        // ---------------------------------------------------------------- MXFP4: the sorted rows' scales
        // Warp 2 the unit's rows 0..127, warp 3 (PAIR) the others; both CTAs of a pair need them all. Row r's four scales of
        // 128 k go to (r % 32) * 16 + (r / 32) * 4: lane l holds rows l, l + 32, ... and writes 16 consecutive bytes. A lane
        // reads 16 bytes of each of its rows at a time, two stages' worth (each row is a line of its own: 4-byte copies a
        // stage kept the L1 busy), into two register sets in turn, one on its way while the other is used, across units.
        const int g = warp - 2;
        auto run = [&](auto whole, const RowScales& rs) {                          // whole: RowScales'
            constexpr bool WHOLE = decltype(whole)::value;
            constexpr int Q = NT < 128 ? NT / 32 : 4;
            struct Set {
                uint32_t w[Q][WHOLE ? 4 : 5], sh;
            };
            const int nsc = (int)(p.n_in / 32);
            RowAhead<Q> ahead(p, lane + g * 128, 32);
            const uint8_t* src[Q];
            uint32_t lu = 0, cu = 0;                          // units of the next load and of the next batch used
            int lc = k0, cc = k0;                             // ... and their first stages
            bool edge;                                        // one of the warp's rows is x's last
            auto rows = [&]() {
                ahead.rows(p.x_scales, p.xs_pitch, src);
                bool mine = false;
#pragma unroll
                for (int q = 0; q < Q; ++q) mine |= src[q] == rs.last;
                edge = __any_sync(0xFFFFFFFFu, mine);
            };
            ahead.fetch(unit_at(0));
            rows();
            if (n_mine > 1) ahead.fetch(unit_at(1));
            // nothing here touches what it loads: it is waited for where it is used. x.sh: each row's shift, a byte a row
            auto load = [&](Set& x) {
                const int off = 8 * lc;
                if (lc >= k1) return;
                x.sh = 0;
                if (WHOLE && (off + 16 <= nsc || !edge)) {
#pragma unroll
                    for (int q = 0; q < Q; ++q) {
                        const uint4 t = *reinterpret_cast<const uint4*>(src[q] + off);
                        x.w[q][0] = t.x; x.w[q][1] = t.y; x.w[q][2] = t.z; x.w[q][3] = t.w;
                    }
                } else {
                    const uint8_t* b[Q];
                    bool in = true;
#pragma unroll
                    for (int q = 0; q < Q; ++q) {
                        const uint32_t by = (uint32_t)(reinterpret_cast<uintptr_t>(src[q] + off) & 3);
                        b[q] = src[q] + off - by;
                        x.sh |= by << (8 * q + 3);
                        in = in && b[q] >= rs.lo && b[q] + 20 <= rs.hi;
                    }
                    constexpr int W = WHOLE ? 4 : 5;
                    if (!WHOLE && __all_sync(0xFFFFFFFFu, in)) {
#pragma unroll
                        for (int q = 0; q < Q; ++q)
#pragma unroll
                            for (int i = 0; i < W; ++i) x.w[q][i] = *reinterpret_cast<const uint32_t*>(b[q] + 4 * i);
                    } else {
#pragma unroll
                        for (int q = 0; q < Q; ++q)
#pragma unroll
                            for (int i = 0; i < W; ++i) x.w[q][i] = rs.word<WHOLE ? 4 : 1>(b[q] + 4 * i);
                    }
                }
                if ((lc += 2) >= k1 && ++lu < n_mine) {
                    lc = k0;
                    rows();
                    if (lu + 1 < n_mine) ahead.fetch(unit_at(lu + 1));
                }
            };
            auto use = [&](const Set& x) {
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    if (cc + a >= k1) break;
                    wait(&empty[pipe.s], pipe.ph ^ 1);
                    uint4* dst = reinterpret_cast<uint4*>(sfx_ring + pipe.s * C::SFX_B + g * 512) + lane;
                    auto put = [&](uint32_t m0, uint32_t m1) {
                        auto word = [&](int q, int h) {
                            const int r = q < Q ? q : 0, i = 2 * a + h;
                            return q >= Q ? 0u : WHOLE ? x.w[r][i] : __funnelshift_r(x.w[r][i], x.w[r][(i + 1) % 5], x.sh >> (8 * r));
                        };
                        dst[0] = make_uint4(word(0, 0) & m0, word(1, 0) & m0, word(2, 0) & m0, word(3, 0) & m0);
                        dst[C::SFX_G * 32] = make_uint4(word(0, 1) & m1, word(1, 1) & m1, word(2, 1) & m1, word(3, 1) & m1);
                    };
                    const int left = nsc - 8 * (cc + a);
                    if (left >= 8) {
                        put(~0u, ~0u);
                    } else {                                   // past the row's end the scales of zero codes: any but a NaN
                        put(left >= 4 ? ~0u : (1u << (8 * left)) - 1, left > 4 ? (1u << (8 * (left - 4))) - 1 : 0u);
                    }
                    __syncwarp();                              // the MMA warp's fence covers these writes too
                    if (lane == 0) mbar_arrive(&full[pipe.s]);
                    pipe.next(ST);
                }
                if ((cc += 2) >= k1) {
                    cc = k0;
                    ++cu;
                }
            };
            Set even = {}, odd = {};
            load(even);
            load(odd);
            while (cu < n_mine && !*vdead) {
                use(even);
                load(even);
                if (cu >= n_mine) break;
                use(odd);
                load(odd);
            }
        };
        if constexpr (MX) {
            const RowScales rs(p);
            if (g < C::SFX_G && n_mine) {
                if (rs.whole) run(std::true_type(), rs);
                else run(std::false_type(), rs);
            }
        }
    } else if (warp < kEpiWarp0) {
        // ---------------------------------------------------------------- sorted rows
        // Eight lanes a row of a stage, 16 rows a pass of the four warps; each thread's copies arrive on the stage's barrier
        // when they have landed. The MMA warp, which sees that, makes them visible to the asynchronous proxy (a fence by
        // the loaders would wait for every copy they have in flight).
        constexpr int RP = (C::NL + 15) / 16, kStep = 4;      // passes a stage; stages a step of the row pointers
        const int xt = tid - kXWarp0 * 32, c = xt & 7, rr = xt >> 3;
        const int kb = (int)(MX ? p.n_in / 2 : p.n_in * 2);
        const uint32_t dst0 = smem_u32(x_ring) + rr * kRowB + ((c ^ (rr & 7)) << 4);
        RowAhead<RP> ahead(p, rr, 16);
        auto mine = [&](uint32_t i) {                         // this CTA's rows of its i-th unit; blk: rows of its tile
            Unit u = unit_at(i);
            const int nl = ((u.nr + 16 * MB - 1) & ~(16 * MB - 1)) / MB;
            u.r0 += (int)rank * nl;
            u.nr = min(u.nr - (int)rank * nl, nl);
            u.blk = nl;
            return u;
        };
        Unit u = n_mine ? mine(0) : Unit{};
        if (n_mine) ahead.fetch(u);
        for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
            const int nl = u.blk;
            const uint8_t* src[RP];
            ahead.rows(static_cast<const uint8_t*>(p.x) + k0 * kRowB + c * 16, p.x_pitch_bytes, src);
            if (i + 1 < n_mine) {
                u = mine(i + 1);
                ahead.fetch(u);
            }
            for (int c0 = k0; c0 < k1; c0 += kStep) {
#pragma unroll
                for (int a = 0; a < kStep; ++a) {
                    if (c0 + a >= k1) break;
                    wait(&empty[pipe.s], pipe.ph ^ 1);
                    const uint32_t dst = dst0 + pipe.s * C::X_B;
                    if ((c0 + a + 1) * kRowB <= kb) {
#pragma unroll
                        for (int j = 0; j < RP; ++j)
                            if (16 * j < nl) cp16(dst + j * 16 * kRowB, src[j] + a * kRowB);
                    } else {                                  // the row ends in this stage: zeros behind it
                        const bool in = (c0 + a) * kRowB + c * 16 < kb;
#pragma unroll
                        for (int j = 0; j < RP; ++j)
                            if (16 * j < nl) cp16_or_zero(dst + j * 16 * kRowB, in ? src[j] + a * kRowB : src[j], in);
                    }
                    cp_arrive(&full[pipe.s]);
                    pipe.next(ST);
                }
#pragma unroll
                for (int j = 0; j < RP; ++j) src[j] += kStep * kRowB;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        // ---------------------------------------------------------------- epilogue
        const int q = warp & 3, g = (warp - kEpiWarp0) >> 2, ew = warp - kEpiWarp0;
        constexpr int es = OUT == RAD_F32 ? 4 : 2;
        uint8_t* const y = static_cast<uint8_t*>(p.y);
        constexpr bool mx_out = OUT == (int)EXL3B_MX4;
        // Rows outside the runs are zero: 512 bytes (MXFP4: 128 and their scales) of a row a warp, spread over the whole grid.
        // (A row a warp, 32 rows at a time, left the last rows to one pair: 172 us for 137 at 16 experts, 16067 of 16384
        // rows, 1536 -> 4096.)
        if (p.expert_offset) {
            const int64_t lo = min(max(p.expert_offset[0], 0), (int32_t)p.n_rows);
            const int64_t hi = max((int64_t)min(p.expert_offset[p.n_expert], (int32_t)p.n_rows), lo);
            const int64_t gone = lo + p.n_rows - hi;
            if (gone) {
                const int64_t bytes = mx_out ? p.n_out / 2 : p.n_out * es;
                const int64_t parts = (bytes + (mx_out ? 127 : 511)) / (mx_out ? 128 : 512);
                const uint32_t warps = gridDim.x * 4 * C::EPI_G, w = blockIdx.x * 4 * C::EPI_G + ew;
                const uint32_t a = parts < warps ? (uint32_t)parts : warps, n_at = warps / a;
                const uint32_t at = w / a, part0 = w - at * a;
                if (at < n_at) {
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
            }
        }
        float* const st = epi + g * kStage * kEpiLd;
        const int64_t row_b = p.y_pitch * es;
        // a unit's slots, row 32 b + lane in slot[b]: fetched a unit ahead
        constexpr int LB = (NT + 31) / 32;
        int32_t slot[LB];
        auto fetch = [&](const Unit& n) {
#pragma unroll
            for (int b = 0; b < LB; ++b) slot[b] = p.sorted_tok && 32 * b + lane < n.nr ? p.sorted_tok[n.r0 + 32 * b + lane] : 0;
        };
        uint32_t ab = 0, turn = g;                            // turn: this group's first slice of the unit
        Unit u = n_mine ? unit_at(0) : Unit{};
        if (n_mine) fetch(u);
        for (uint32_t i = 0; i < n_mine; ++i, ab ^= 1) {
            const int64_t b0 = (int64_t)(u.blk + rank) * blk_out;           // the block's first output
            uint32_t live = 0;                                               // which of its rows are, 32 a lane
#pragma unroll
            for (int b = 0; b < LB; ++b) {
                const uint32_t m = __ballot_sync(0xFFFFFFFFu, slot[b] >= 0);
                if (lane == b) live = m;
            }
            const Unit now = u;
            if (i + 1 < n_mine) {
                u = unit_at(i + 1);
                fetch(u);
            }
            wait(&acc_full[ab], (i >> 1) & 1);
            if (mx_out && !SPLIT ? epi_any(g, *vdead) : __any_sync(0xFFFFFFFFu, *vdead)) break;
            fence_after();
            if constexpr (SPLIT) {
                // The parts' sums meet through distributed shared memory: every CTA puts its own into its shared memory,
                // then sums every split-th row over the CTAs, in their order, and stores it.
                for (int t0 = 0; t0 < now.nr; t0 += kSlice) {
                    uint32_t a[16];
                    tmem_ld16(tmem + ((uint32_t)(32 * q) << 16) + ab * NT + t0, a);
                    tmem_wait(a);
#pragma unroll
                    for (int j = 0; j < 16; ++j) st[(t0 + j) * kEpiLd + 32 * q + lane] = __uint_as_float(a[j]);
                }
                fence_before();
                __syncwarp();                                  // the arrivals publish the whole warp's sums
                if (lane < split) arrive_at(part_full, lane);
                __syncwarp();
                wait(part_full, 0);
                asm volatile("fence.acq_rel.cluster;" ::: "memory");
                const bool out_lane = !act || !(lane & 4);    // silu_mul: 16 gate columns, then their 16 up columns
                const int64_t n0 = b0 + (act ? 16 * (lane >> 3) + 4 * (lane & 3) : 4 * lane);
                const uint32_t rows_live = __shfl_sync(0xFFFFFFFFu, live, 0);
                for (int j = part + split * q; j < now.nr; j += split * 4) {
                    float f[kMaxSplit][4], v[4];
#pragma unroll
                    for (int s = 0; s < kMaxSplit; ++s)       // all on their way before the first is added
                        if (s < split) ld_cluster(&st[j * kEpiLd + 4 * lane], s, f[s]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = f[0][e];
#pragma unroll
                        for (int s = 1; s < kMaxSplit; ++s)
                            if (s < split) v[e] += f[s][e];
                    }
                    if (act) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float up = __shfl_xor_sync(0xFFFFFFFFu, v[e], 4);
                            v[e] = v[e] < kSiluLow ? silu_up_low(v[e], up) : silu_up(v[e], up);
                        }
                    }
                    const int64_t r = now.r0 + j;
                    const bool ok = out_lane && n0 < p.n_out;
                    if (!(rows_live >> j & 1)) v[0] = v[1] = v[2] = v[3] = 0.f;        // a dropped slot
                    if (mx_out) {
                        uint32_t m = max(max(mx4_mag(v[0]), mx4_mag(v[1])), max(mx4_mag(v[2]), mx4_mag(v[3])));
                        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
                        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
                        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, act ? 8 : 4));      // the eight lanes of a block of 32
                        const uint32_t code = mx4_scale_code(m);
                        const float f[8] = { v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f };
                        if (ok) {
                            *reinterpret_cast<uint16_t*>(y + r * p.y_pitch + n0 / 2) = (uint16_t)mx4_pack8(f, code);
                            if ((n0 & 31) == 0) p.y_scales[r * p.ys_pitch + n0 / 32] = (uint8_t)code;
                        }
                    } else if (ok) {
                        uint8_t* d = y + r * row_b + n0 * es;
                        if constexpr (OUT == RAD_F32) *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
                        else *reinterpret_cast<uint2*>(d) = make_uint2(pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3]));
                    }
                }
                break;
            }
            // Thread t has outputs o and o + 8 (act NONE: and 16 more) of rows c2, c2 + 1, 8 + c2, 9 + c2 of a slice
            constexpr int NV = ACT ? 8 : 16;
            const int o = lane >> 2, c2 = 2 * (lane & 3);
            const int64_t n_warp = b0 + (act ? 16 : 32) * q;                 // the warp's first output
            const uint32_t acc = tmem + ((uint32_t)(32 * q) << 16) + ab * NT;
            uint32_t a[16];
            // the groups take turns at slices, on from where the last unit's ended
            const int t1 = (int)turn * kSlice;
            if (t1 < now.nr) tmem_ld8x8(acc + t1, a);
            turn = (turn + C::EPI_G * kMaxTurn - (uint32_t)(now.nr + kSlice - 1) / kSlice) % C::EPI_G;
            for (int t0 = t1; t0 < now.nr; t0 += C::EPI_G * kSlice) {
                tmem_wait(a);
                float v[NV];
#pragma unroll
                for (int k = 0; k < NV; ++k) v[k] = act ? silu_up(__uint_as_float(a[k]), __uint_as_float(a[(8 + k) & 15])) : __uint_as_float(a[k]);
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
                if (t0 + C::EPI_G * kSlice < now.nr) tmem_ld8x8(acc + t0 + C::EPI_G * kSlice, a);   // the next slice, meanwhile
                const int left = now.nr - t0;                                     // rows of the slice, if less than 16
                const uint32_t here = __shfl_sync(0xFFFFFFFFu, live, t0 >> 5) >> (t0 & 31);
                if ((here & 0xFFFFu) != 0xFFFFu) {                                // dropped slots are zero
#pragma unroll
                    for (int k = 0; k < NV; ++k)
                        if (!(here >> (8 * (k >> 2 & 1) + c2 + (k & 1)) & 1)) v[k] = 0.f;
                }
                if constexpr (OUT == RAD_F32) {
                    // straight from the registers: a warp's store is 32 bytes each of four rows
                    const int64_t n = n_warp + o;
                    uint8_t* d = y + (now.r0 + t0 + c2) * row_b + n * 4;
#pragma unroll
                    for (int k = 0; k < NV; ++k) {
                        const int j = 8 * (k >> 2 & 1) + (k & 1), m = 16 * (k >> 3) + 8 * (k >> 1 & 1);
                        if (c2 + j < left && n + m < p.n_out) *reinterpret_cast<float*>(d + j * row_b + 4 * m) = v[k];
                    }
                } else if constexpr (!mx_out) {
                    // Transposed through the warp's own 1 KB of shared memory -- a row's outputs, 16-byte pieces swizzled
                    // against bank conflicts -- then 16 bytes a thread: whole 32-byte sectors, and no warp waits for another.
                    // (Two-byte stores straight from the registers: 218 against 177 us at 16 experts, 16067 rows, 1536 ->
                    // 4096.)
                    constexpr int P = NV / 4, SH = ACT ? 2 : 1;                   // 16-byte pieces a row; rows that share banks
                    uint8_t* const sw = reinterpret_cast<uint8_t*>(epi) + ew * 1024;
                    auto at = [](int row, int piece) { return (row * P + (piece ^ (row >> SH & (P - 1)))) * 16; };
#pragma unroll
                    for (int s = 0; s < NV / 8; ++s) {
                        uint32_t w[4];
#pragma unroll
                        for (int m = 0; m < 4; ++m) w[m] = pack2<OUT>(v[8 * s + 2 * m], v[8 * s + 2 * m + 1]);
                        st8x8t(smem_u32(sw) + at(8 * (lane >> 4) + (lane & 7), 2 * s + (lane >> 3 & 1)), w);
                    }
                    __syncwarp();
#pragma unroll
                    for (int s = 0; s < NV / 8; ++s) {
                        const int row = (32 * s + lane) / P, piece = lane % P;
                        const uint4 w = *reinterpret_cast<const uint4*>(sw + at(row, piece));
                        const int64_t n = n_warp + 8 * piece;
                        if (row < left && n < p.n_out) *reinterpret_cast<uint4*>(y + (now.r0 + t0 + row) * row_b + n * 2) = w;
                    }
                    __syncwarp();
                } else {
                    // MXFP4: staged in f32, since a block's 32 outputs lie in two warps (silu_mul); eight of a row a thread
                    const int lpt = blk_out / 8, tpw = 32 / lpt, c0 = (lane % lpt) * 8;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int k = 0; k < NV; ++k)
                            if ((k >> 2 & 1) == h)
                                st[(c2 + (k & 1)) * kEpiLd + (act ? 16 : 32) * q + 16 * (k >> 3) + 8 * (k >> 1 & 1) + o] = v[k];
                        epi_sync(g);
                        if (q * tpw < kStage) {                                  // whole warps: the quads vote
                            const int j = q * tpw + lane / lpt;
                            const int64_t r = now.r0 + t0 + 8 * h + j, n0 = b0 + c0;
                            float f[8];
                            ld8(&st[j * kEpiLd + c0], f);
                            const uint32_t code = mx4_quad_code(f);              // four lanes: 32 outputs of one row
                            if (8 * h + j < left && n0 < p.n_out) {
                                *reinterpret_cast<uint32_t*>(y + r * p.y_pitch + n0 / 2) = mx4_pack8(f, code);
                                if ((lane & 3) == 0) p.y_scales[r * p.ys_pitch + n0 / 32] = (uint8_t)code;
                            }
                        }
                        epi_sync(g);
                    }
                }
            }
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) arrive_even(&acc_empty[ab]);
                else mbar_arrive(&acc_empty[ab]);
            }
        }
    }
    fence_before();
    __syncthreads();
    if (PAIR || SPLIT) cluster_sync_all();                    // no CTA's memory goes while another uses it
    if (warp == 1) {
        fence_after();
        tmem_free<PAIR>(tmem, C::TMEM);
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

// Weights, boxes of 128 bytes of k: [expert][row][k] and a block's 128 rows; for silu_mul [expert][group of 16 rows]
// [gate, up][16][k] and a block's four groups, in one box (eight boxes of 16 rows a stage kept the issuing warp busy, 550
// cycles a stage) unless the last group is half a one and the box would leave the weight: then a box a half group.
int make_map(const Exl3bGmmOp* p, CUtensorMap* map) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return -6;
    const CUtensorMapDataType dt = p->mx4 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                          : p->bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t k = (cuuint64_t)(p->mx4 ? p->n_in / 2 : p->n_in), pitch = (cuuint64_t)p->w_pitch_bytes;
    const cuuint32_t kb = p->mx4 ? 128u : 64u, one[5] = { 1, 1, 1, 1, 1 };
    const bool whole = p->act && p->n_out % 16 == 0;
    const cuuint64_t dims3[3] = { k, (cuuint64_t)p->w_rows, (cuuint64_t)p->n_expert };
    const cuuint64_t strides3[2] = { pitch, (cuuint64_t)p->w_expert_bytes };
    const cuuint32_t box3[3] = { kb, p->act ? 16u : 128u, 1u };
    const cuuint64_t dims5[5] = { k, 16, 2, (cuuint64_t)(p->n_out / 16), (cuuint64_t)p->n_expert };
    const cuuint64_t strides5[4] = { pitch, (cuuint64_t)p->n_out * pitch, 16 * pitch, (cuuint64_t)p->w_expert_bytes };
    const cuuint32_t box5[5] = { kb, 16, 2, 4, 1 };
    return fn(map, dt, whole ? 5 : 3, const_cast<void*>(p->w), whole ? dims5 : dims3, whole ? strides5 : strides3,
              whole ? box5 : box3, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0 : -6;
}

// An upper bound of the units: a group a live expert and one more each NT rows, times the blocks.
int64_t most_units(const Exl3bGmmOp* p, int nt, int mb) {
    const int64_t blk = (p->act ? 64 : 128) * mb;
    const int64_t live = p->n_expert < p->n_rows ? p->n_expert : p->n_rows;
    return (live + p->n_rows / nt) * ((p->n_out + blk - 1) / blk);
}

// Sorted rows a unit of the pair form: where units of `most` leave pairs of SMs without one, as few as still give every
// pair at most one (one expert of 1024 rows, 2048 -> 2048, bf16: 16.3 us with units of 256 rows, 12.3 with these).
int pair_rows(const Exl3bGmmOp* p, int most, int sm_count) {
    int nt = most;
    while (nt > 64 && most_units(p, nt - 32, 2) <= sm_count / 2) nt -= 32;
    return nt;
}

typedef void (*Kern)(CUtensorMap, Exl3bGmmOp, Shape);
int out_kind(int dt) { return dt == RAD_F32 ? 0 : dt == RAD_F16 ? 1 : dt == RAD_BF16 ? 2 : 3; }

// split: CTAs a unit, each a part of its k (SPLIT); PAIR: two CTAs a unit all the same.
template <bool MX, bool PAIR, bool SPLIT>
int launch(const Exl3bGmmOp* p, int sm_count, int split, cudaStream_t st) {
    using C = Cfg<MX, PAIR, SPLIT>;
    CUtensorMap map;
    const int rc = make_map(p, &map);
    if (rc) return rc;
    static const Kern kerns[8] = { k_gmm<MX, PAIR, SPLIT, RAD_F32, false>, k_gmm<MX, PAIR, SPLIT, RAD_F16, false>,
                                    k_gmm<MX, PAIR, SPLIT, RAD_BF16, false>, k_gmm<MX, PAIR, SPLIT, EXL3B_MX4, false>,
                                    k_gmm<MX, PAIR, SPLIT, RAD_F32, true>, k_gmm<MX, PAIR, SPLIT, RAD_F16, true>,
                                    k_gmm<MX, PAIR, SPLIT, RAD_BF16, true>, k_gmm<MX, PAIR, SPLIT, EXL3B_MX4, true> };
    static bool allowed[64][8];                               // the most shared memory, once a device
    const int which = out_kind(p->y_dtype) + (p->act ? 4 : 0);
    const Kern kern = kerns[which];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -6;
    if (!allowed[dev][which]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - kStatic) != cudaSuccess) return -6;
        allowed[dev][which] = true;
    }
    const int ctas = PAIR ? 2 : split;                        // of a cluster
    const int nt = PAIR ? pair_rows(p, C::NT, sm_count) : C::NT;
    const int64_t most = most_units(p, nt, PAIR ? 2 : 1);
    // few units: one CTA an SM, with the whole of its shared memory for stages in flight; clusters of three or four do not
    // fill the SMs of every processing cluster, and such that found no room would wait for the others (48 units in three
    // parts: 15.8 us with one CTA an SM, 9.7 with two)
    const int64_t alone = ctas > 2 ? sm_count - sm_count / 8 : sm_count;
    const int per_sm = !PAIR && most * ctas <= alone ? 1 : C::PER_SM;
    const int64_t room = (int64_t)sm_count * per_sm / ctas;
    const int stages = C::stages(p->n_expert, per_sm);
    const int64_t units = most < room ? most : room, blk = (p->act ? 64 : 128) * (PAIR ? 2 : 1);
    const Shape sh = { exl3b_div((uint32_t)((p->n_out + blk - 1) / blk)), exl3b_div((uint32_t)units), exl3b_div((uint32_t)nt),
                       (int32_t)((p->n_in + (MX ? 255 : 63)) / (MX ? 256 : 64)), stages, split };
    return chain_launch(kern, dim3((unsigned)(units * ctas)), dim3(C::THREADS), C::fixed(p->n_expert) + stages * C::STAGE_B,
                        ctas, st, map, *p, sh);
}

template <bool MX>
int launch_form(const Exl3bGmmOp* p, int sm_count, cudaStream_t st) {
    // The pair form from 16 rows an expert on average (512 -> 2240 over 479 experts of 15 rows, MXFP4: narrow 39 us, pair
    // 43; 792 -> 1648 over 112 experts of 33 rows, bf16: 68 and 50), or 96 where a weight has so few rows that its last pair
    // of blocks is mostly empty (448 -> 320 over 298 experts of 84 rows, MXFP4: 17 and 24); and where its units, as short as
    // 96 rows, keep half the pairs busy (one expert, bf16: 4096 rows, 2048 -> 512: 18.7 and 12.6; 306 rows, 3064 -> 328: 8.9
    // and 16.5).
    const int64_t few = p->w_rows < 512 ? 96 : 16;
    if (p->n_rows > few * (int64_t)p->n_expert && most_units(p, 96, 2) >= sm_count / 4) {
        return launch<MX, true, false>(p, sm_count, 1, st);
    }
    // Few narrow units over a long k: up to four CTAs a unit while each has an SM, four stages a part at least (one token,
    // two experts, 2048 -> 512 silu_mul: 8.2 us, in four parts 5.7; 16 rows, 4096 -> 4096: 13.8 and 9.5; ten experts make
    // 80 units: in three parts, more CTAs than SMs, 13.7 and 15.1; clusters of eight do not always fit at once: 15.1 for
    // 8.9). MXFP4 has a quarter of the stages and gains nothing (two experts 8.9 and 10.3).
    if (!MX) {
        const int64_t most = most_units(p, 32, 1), nck = (p->n_in + 63) / 64;
        int64_t split = sm_count / most;                      // so the grid has room for a cluster a unit: the kernel counts on it
        if (split > nck / 4) split = nck / 4;
        if (split > kMaxSplit) split = kMaxSplit;
        if (split >= 2) return launch<false, false, true>(p, sm_count, (int)split, st);
    }
    return launch<MX, false, false>(p, sm_count, 1, st);
}

}  // namespace

extern "C" int exl3b_cuda_gmm(const Exl3bGmmOp* p, int sm_count, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return p->mx4 ? launch_form<true>(p, sm_count, st) : launch_form<false>(p, sm_count, st);
}

extern "C" int exl3b_gmm_max_expert(void) { return kMaxExpert; }
