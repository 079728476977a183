// exl3b200_gmm8w.cuh -- grouped_mm over FP8 operands where experts have many rows: the SORTED rows are the MMA's M (128) and the
// weight rows its N, the other way round than in exl3b200_gmm8.cu. A thread of the summing warps then has one sorted row and 128
// of its columns, so that a block's scale is one number a thread (sx of its row times sw of its columns' block): the sums cost
// an FMA a value and no shared memory. (With the weight rows as M every column has a scale of its own, which a thread reads from
// shared memory, four bytes a lane a cycle: 174 against 138 us at 16 experts, 16060 rows, 4096 -> 1536, and 253 against 182 at
// 418 experts of 20072 rows, 2048 -> 512 silu_mul.)
//
// Persistent over units (expert, a group of up to 128 of its sorted rows, a block of 256 weight rows; silu_mul: 128 gate rows
// and their 128 up rows), one CTA an SM. A unit's weight rows are two groups of 128 columns of the accumulator, four summing
// warps each: act NONE in order; silu_mul 64 gate rows and their 64 up rows, and the next 64 of each, so that a thread has
// both of its 64 outputs.
// Warps of a CTA:
//   0       weights: cp.async.bulk.tensor, 128-byte swizzled
//   1       MMA issuer: four tcgen05.mma (kind::f8f6f4, M 128, N 256, K 32) a stage of 128 k, into one of two accumulators in
//           tensor memory (one of 128 columns a group instead, two each: 128.4 against 126.1 us at 16 experts)
//   2, 3    nothing: they leave their registers to the summing warps
//   4..7    sorted rows: 16-byte cp.async through sorted_tok
//   8..15   sums: 32 sorted rows and a group's 128 columns each, then their outputs
// A stage's MMAs take 512 cycles, a stage 920 (16 experts; 64 experts 820) once a unit's first four are over, a unit 34700
// (18700): 5200 (5500) besides its stages, for its outputs and the accumulators' refilling after them. What is left is not
// the sums' instructions: with the sums left out 128 us became 121, with the outputs too 112, with most of the loads as well
// 103. It is the round trip of an accumulator, of which tensor memory holds two: the MMAs' completion, its barrier, the
// reads, their barrier and the next issue; then a unit's outputs, which wait for its last stage; then the last round, which
// a third of the CTAs or fewer take part in (16 and 64 experts: five or six units a CTA).
// 20 runs in a graph, the SMs at 1.6 to 1.75 GHz by the kernel's own clock: 177 us at 410 live experts of 20075 rows, 2048 ->
// 512 silu_mul (0.88 GB, 5.0 TB/s); 75 at 64 experts of them (with the rows' f8_quantize); 130 at 16 experts, 16066 rows,
// 4096 -> 1536 (202 GFLOP, 1560 TFLOP/s). Run on end, at the power limit's 1.3 to 1.5 GHz: 207, 83 and 148 us (1365 TFLOP/s).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "exl3b200_chain.cuh"
#include "exl3b200_decode.cuh"
#include "exl3b200_dense.h"
#include "exl3b200_gmm.cuh"

namespace exl3b {
namespace wide {

constexpr int kGroups = 2;                                   // of four summing warps, each for 128 weight rows
constexpr int kThreads = (kEpiWarp0 + 4 * kGroups) * 32;
constexpr int kRows = 128;                                   // sorted rows a unit at most: the MMA's lanes
constexpr int kCols = 128;                                   // of a group: its weight rows
constexpr int kDb = 2;                                       // accumulators in turn, of both groups' columns
constexpr int kWideW_B = kGroups * kW_B, kX_B = kRows * kRowB, kStageB = kWideW_B + kX_B;
constexpr int fixed_bytes(int n_expert) { return 1024 + 512 + (n_expert + 4) * 4; }
constexpr int stages_of(int n_expert) {
    const int n = (227 * 1024 - kStatic - fixed_bytes(n_expert)) / kStageB;
    return n < kMaxSt ? n : kMaxSt;
}
constexpr int kPolls = 64;                                   // of a barrier, before a suspended wait
static_assert(stages_of(kMaxExpert) >= 4 && (2 * kMaxSt + 2 * kDb) * 8 + 8 <= 512, "shared memory");

// One arrival, by one lane of a whole warp.
__device__ __forceinline__ void arrive_el(uint32_t bar) {
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n @e mbarrier.arrive.shared::cta.b64 _, [%0];\n}\n" ::"r"(bar)
                 : "memory");
}
// 32 or 16 columns of this warp's 32 lanes, lane l's in thread l; tmem_got before they are read.
__device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_got(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_got(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
// A number from global memory if `ok`, else v as it was. In place: a value that met another one on the way would be waited for
// where they meet.
__device__ __forceinline__ void ld_if(float& v, const float* p, bool ok) {
    asm volatile("{\n .reg .pred p;\n setp.ne.u32 p, %2, 0;\n @p ld.global.f32 %0, [%1];\n}\n" : "+f"(v) : "l"(p), "r"((uint32_t)ok));
}

// OUT: y_dtype; ACT: silu_mul.
template <int OUT, bool ACT>
__global__ void __launch_bounds__(kThreads, 1) k_gmm8w(const __grid_constant__ CUtensorMap wmap, const Exl3bGmmOp p, const Shape sh) {
    const int ST = sh.st;
    constexpr int blk_out = ACT ? 128 : 256;                  // outputs of a unit
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* w_ring = smem;                                   // [ST][256 rows][128 B]
    uint8_t* x_ring = w_ring + ST * kWideW_B;                 // [ST][128 rows][128 B]
    uint64_t* bars = reinterpret_cast<uint64_t*>(x_ring + ST * kX_B);
    uint64_t* full = bars;                                    // producers -> MMA warp
    uint64_t* empty = full + ST;                              // MMA commit -> producers
    uint64_t* d_full = empty + ST;                            // MMA commit -> sums [kDb]
    uint64_t* d_empty = d_full + kDb;                         // sums -> MMA [kDb]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_empty + kDb);
    uint32_t* dead = tmem_slot + 1;                           // a wait gave up: everyone leaves
    uint32_t* prefix = reinterpret_cast<uint32_t*>(bars) + 128;   // [n_expert + 1]
    __shared__ Unit utab[kTab];
    __shared__ uint32_t wsum[kThreads / 32];

    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const uint32_t first = blockIdx.x, stride = sh.stride.d;
    if (tid < ST) {
        mbar_init(&full[tid], 1 + 32 * kXWarps);
        mbar_init(&empty[tid], 1);
    } else if (tid >= 32 && tid < 32 + kDb) {
        mbar_init(&d_full[tid - 32], 1);
        mbar_init(&d_empty[tid - 32], 4 * kGroups);
    } else if (tid == 64) {
        *dead = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&wmap)) : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    if (warp == 1) tmem_alloc<false>(tmem_slot, kDb * kGroups * kCols);
    chain_wait();                                             // all above needs no memory but the CTA's own
    scan_units<kThreads, 1>(p, sh, first, prefix, utab, wsum);
    fence_before();
    __syncthreads();
    fence_after();
    chain_next();                                             // every CTA has its tensor memory: a later kernel may ask for its own
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
    const uint32_t n_units = prefix[p.n_expert];
    const uint32_t n_mine = n_units > first ? exl3b_div_of(n_units - first + stride - 1, sh.stride) : 0u;
    auto unit_at = [&](uint32_t i) {
        return i < kTab ? utab[i] : find_unit<1>(p, prefix, first + i * stride, sh);
    };
    const int nck = sh.nck;
    volatile uint32_t* vdead = dead;
    // A bounded wait by a whole warp, which reports nothing: one that gives up marks the CTA dead, every other wait of the
    // CTA then gives up at its next try, and the roles leave at their next unit. It asks a few times before it lets itself be
    // suspended, which takes longer to wake from (132 against 128 us at 16 experts).
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        const uint32_t a = smem_u32(bar);
#pragma unroll 1
        for (int j = 0; j < kPolls; ++j) {
            uint32_t done;
            asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
                         " selp.u32 %0, 1, 0, p;\n}\n"
                         : "=r"(done)
                         : "r"(a), "r"(parity)
                         : "memory");
            if (done) {
                __syncwarp();
                return;
            }
        }
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
    Pipe pipe;                                                // of the stages

    // The summing warps' sums need more than the 128 registers a thread that 512 threads start with: 256 x 208 + 256 x 48 are
    // the 512 x 128 of the launch.
    if (warp < kEpiWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
        if (warp == 0) {
            // ------------------------------------------------------------ weights
            for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
                const Unit u = unit_at(i);
                for (int ck = 0; ck < nck; ++ck, pipe.next(ST)) {
                    wait(&empty[pipe.s], pipe.ph ^ 1);
                    mbar_expect_tx_el(&full[pipe.s], kWideW_B);
                    uint8_t* dst = w_ring + pipe.s * kWideW_B;
                    const int k = ck * 128;
#pragma unroll
                    for (int h = 0; h < 4; ++h) {                // 64 rows a box, two boxes a group
                        const int row = ACT ? u.blk * 128 + 64 * (h >> 1) + (h & 1 ? (int)p.n_out : 0) : u.blk * 256 + 64 * h;
                        tma_w_el(dst + h * (64 * kRowB), &wmap, k, row, u.e, &full[pipe.s]);
                    }
                }
            }
            // after a wait that gave up: a millisecond for the copies still in flight, before the CTA's memory goes
            if (*vdead)
                for (int j = 0; j < 50; ++j) __nanosleep(20000);
        } else if (warp == 1) {
            // ------------------------------------------------------------ MMA issuer
            const uint64_t wd0 = desc_sw128(smem_u32(w_ring)), xd0 = desc_sw128(smem_u32(x_ring));
            // D f32, e4m3 both, both operands K-major, M 128, N 256
            constexpr uint32_t idesc = (uint32_t)(kGroups * kCols) >> 3 << 17 | 8u << 24 | 1u << 4;
            Pipe db;
            for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
                for (int ck = 0; ck < nck; ++ck, pipe.next(ST)) {
                    wait(&full[pipe.s], pipe.ph);
                    proxy_fence();
                    wait(&d_empty[db.s], db.ph ^ 1);
                    fence_after();
                    mma4_f8(tmem + db.s * kGroups * kCols, xd0 + (uint64_t)(pipe.s * kX_B >> 4),
                            wd0 + (uint64_t)(pipe.s * kWideW_B >> 4), idesc);
                    commit_el<false>(&d_full[db.s]);
                    db.next(kDb);
                    commit_el<false>(&empty[pipe.s]);
                }
            }
        } else if (warp >= kXWarp0) {
            // ------------------------------------------------------------ sorted rows
            // Eight lanes a row of a stage, 16 rows a pass of the four warps; each thread's copies arrive on the stage's
            // barrier when they have landed, and the MMA warp, which sees that, makes them visible to the asynchronous proxy.
            // Rows past the unit's are left as they were: their sums are nobody's.
            constexpr int RP = kRows / 16, kStep = 4;             // passes a stage; stages a step of the row pointers
            const int xt = tid - kXWarp0 * 32, c = xt & 7, rr = xt >> 3;
            const int kb = (int)p.n_in;
            const uint32_t dst0 = smem_u32(x_ring) + rr * kRowB + ((c ^ (rr & 7)) << 4);
            RowAhead<RP> ahead(p, rr, 16);
            Unit u = n_mine ? unit_at(0) : Unit{};
            if (n_mine) ahead.fetch(u);
            for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
                const int nl = u.nr;
                const uint8_t* src[RP];
                ahead.rows(static_cast<const uint8_t*>(p.x) + c * 16, p.x_pitch_bytes, src);
                if (i + 1 < n_mine) {
                    u = unit_at(i + 1);
                    ahead.fetch(u);
                }
                for (int c0 = 0; c0 < nck; c0 += kStep) {
#pragma unroll
                    for (int a = 0; a < kStep; ++a) {
                        if (c0 + a >= nck) break;
                        wait(&empty[pipe.s], pipe.ph ^ 1);
                        const uint32_t dst = dst0 + pipe.s * kX_B;
                        if ((c0 + a + 1) * kRowB <= kb) {
#pragma unroll
                            for (int j = 0; j < RP; ++j)
                                if (16 * j < nl) cp16(dst + j * 16 * kRowB, src[j] + a * kRowB);
                        } else {                              // the row ends in this stage: zeros behind it
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
        }
    } else {
        // ---------------------------------------------------------------- sums
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int q = warp & 3, g = (warp - kEpiWarp0) >> 2, ew = warp - kEpiWarp0;
        constexpr int es = OUT == RAD_F32 ? 4 : 2;
        clear_outside<OUT>(p, blockIdx.x * 4 * kGroups + ew, gridDim.x * 4 * kGroups, lane);
        const bool sectors = ((reinterpret_cast<uintptr_t>(p.y) | (uintptr_t)(p.y_pitch * es)) & 31) == 0;
        RowAhead<1> ahead(p, 32 * q + lane, 1);
        // four blocks' scales: of the thread's row, and of its columns' block of the weight (silu_mul: of gate's and of up's)
        struct Scales {
            float x[4], w[ACT ? 8 : 4];
        };
        const float *xs = nullptr, *ws = nullptr;
        const int64_t ws_up = p.ws_blocks * p.ws_blk_bytes / 4;
        auto load = [&](Scales& s, int ck) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                ld_if(s.x[j], xs + ck + j, ck + j < nck);
                ld_if(s.w[j], ws + ck + j, ck + j < nck);
                if (ACT) ld_if(s.w[(4 + j) % (ACT ? 8 : 4)], ws + ws_up + ck + j, ck + j < nck);
            }
        };
        Scales next = {};
        bool live_next = false;
        auto begin = [&](uint32_t i) {                        // unit i's rows and first scales; its slots are there
            const Unit u = unit_at(i);
            const uint8_t* at[1];
            ahead.rows(p.x_scales, p.xs_pitch, at);
            xs = reinterpret_cast<const float*>(at[0]);
            const int b = ACT ? u.blk : min(2 * u.blk + g, p.ws_blocks - 1);
            ws = reinterpret_cast<const float*>(p.w_scales + u.e * p.ws_expert_bytes + b * p.ws_blk_bytes);
            load(next, 0);
        };
        auto fetch = [&](uint32_t i) {                        // ... are asked for
            const Unit u = unit_at(i);
            ahead.fetch(u);
            live_next = 32 * q + lane < u.nr && (!p.sorted_tok || p.sorted_tok[u.r0 + 32 * q + lane] >= 0);
        };
        if (n_mine) {
            fetch(0);
            begin(0);
        }
        // the accumulators' barriers' addresses held, not worked out each stage (86 against 79 us at 64 experts of 20072 rows,
        // 2048 -> 512 silu_mul)
        uint32_t d_free[kDb];
#pragma unroll
        for (int b = 0; b < kDb; ++b) {
            d_free[b] = smem_u32(&d_empty[b]);
            asm volatile("" : "+r"(d_free[b]));
        }
        Pipe db;
        for (uint32_t i = 0; i < n_mine; ++i) {
            const Unit u = unit_at(i);
            const bool any = 32 * q < u.nr, live = live_next;
            if (i + 1 < n_mine) fetch(i + 1);
            uint64_t acc[8][8];                               // 128 columns, two a word
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) acc[c][k] = 0;
            float f[ACT ? 8 : 4];                             // of the next four stages: for columns 0 .. 63, silu_mul: 64 .. 127
#pragma unroll 1
            for (int ck = 0; ck < nck; ++ck) {
                if ((ck & 3) == 0) {
#pragma unroll
                    for (int j = 0; j < (ACT ? 8 : 4); ++j) f[j] = next.x[j & 3] * next.w[j];
                    if (ck + 4 < nck) load(next, ck + 4);
                }
                const uint64_t f0 = f2pk(f[0], f[0]), f1 = ACT ? f2pk(f[ACT ? 4 : 0], f[ACT ? 4 : 0]) : f0;
#pragma unroll
                for (int j = 0; j < (ACT ? 8 : 4); ++j)
                    if ((j & 3) < 3) f[j] = f[j + 1];
                wait(&d_full[db.s], db.ph);
                fence_after();
                const uint32_t d = tmem + ((uint32_t)(32 * q) << 16) + (kGroups * db.s + g) * kCols;
                const uint32_t done = d_free[db.s];
                db.next(kDb);
                if (any) {
                    // 32 and 16 columns in turn, the next ones' load in flight under the FMAs
                    uint32_t a[32], b[16];
                    auto sum = [&](const uint32_t* v, int c0, int n) {
#pragma unroll
                        for (int k = 0; k < n; k += 2)
                            acc[(c0 + k) >> 4][(c0 + k) >> 1 & 7] =
                                fma2(f2pk(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), c0 + k < 64 ? f0 : f1,
                                     acc[(c0 + k) >> 4][(c0 + k) >> 1 & 7]);
                    };
                    tmem_get(d, a);
#pragma unroll
                    for (int c = 0; c < 96; c += 48) {
                        tmem_got(a);
                        tmem_get(d + c + 32, b);
                        sum(a, c, 32);
                        tmem_got(b);
                        tmem_get(d + c + 48, a);
                        sum(b, c + 32, 16);
                    }
                    tmem_got(a);
                    fence_before();
                    arrive_el(done);
                    sum(a, 96, 32);
                } else {
                    arrive_el(done);
                }
            }
            if (__any_sync(0xFFFFFFFFu, *vdead)) break;
            if (i + 1 < n_mine) begin(i + 1);                 // its first scales, on their way under the epilogue
            const int row = 32 * q + lane;
            if (row < u.nr) {
                constexpr int NV = ACT ? 64 : 128;
                const int64_t n0 = (int64_t)u.blk * blk_out + NV * g;            // the thread's first output
                uint8_t* d = static_cast<uint8_t*>(p.y) + (u.r0 + row) * (p.y_pitch * es) + n0 * es;
                const int left = (int)min((int64_t)NV, p.n_out - n0);
                // 32 bytes a store, whole sectors, where they are aligned
                constexpr int VS = 32 / es;
#pragma unroll
                for (int j = 0; j < NV / VS; ++j) {
                    if (VS * j >= left) break;
                    float v[VS];
                    auto two = [&](int k, float& a, float& b) { f2upk(acc[k >> 4][k >> 1 & 7], a, b); };   // columns k, k + 1
#pragma unroll
                    for (int k = 0; k < VS; k += 2) two(VS * j + k, v[k], v[k + 1]);
                    if constexpr (ACT) {
                        float up[VS], least = v[0];
#pragma unroll
                        for (int k = 0; k < VS; k += 2) two((64 + VS * j + k) & 127, up[k], up[k + 1]);
#pragma unroll
                        for (int k = 1; k < VS; ++k) least = fminf(least, v[k]);
                        if (least < kSiluLow) {
#pragma unroll
                            for (int k = 0; k < VS; ++k) v[k] = v[k] < kSiluLow ? silu_up_low(v[k], up[k]) : silu_up(v[k], up[k]);
                        } else {
#pragma unroll
                            for (int k = 0; k < VS; ++k) v[k] = silu_up(v[k], up[k]);
                        }
                    }
                    if (!live) {                                                  // a dropped slot
#pragma unroll
                        for (int k = 0; k < VS; ++k) v[k] = 0.f;
                    }
                    uint32_t w[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        if constexpr (OUT == RAD_F32) w[k] = __float_as_uint(v[k]);
                        else w[k] = pack2<OUT>(v[(2 * k) % VS], v[(2 * k + 1) % VS]);
                    }
                    if (sectors && VS * (j + 1) <= left) {
                        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(d + 32 * j), "r"(w[0]), "r"(w[1]),
                                     "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                                     : "memory");
                    } else {
                        *reinterpret_cast<uint4*>(d + 32 * j) = make_uint4(w[0], w[1], w[2], w[3]);
                        if (VS * j + VS / 2 < left) *reinterpret_cast<uint4*>(d + 32 * j + 16) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
            }
            __syncwarp();
        }
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        tmem_free<false>(tmem, kDb * kGroups * kCols);
    }
}

template <bool ACT>
int launch(const Exl3bGmmOp* p, int sm_count, cudaStream_t st) {
    typedef void (*Kern)(CUtensorMap, Exl3bGmmOp, Shape);
    CUtensorMap map;
    const int rc = make_map(p, &map, 64);
    if (rc) return rc;
    static const Kern kerns[3] = { k_gmm8w<RAD_F32, ACT>, k_gmm8w<RAD_F16, ACT>, k_gmm8w<RAD_BF16, ACT> };
    static bool allowed[64][3];                               // the most shared memory, once a device
    const int which = p->y_dtype == RAD_F32 ? 0 : p->y_dtype == RAD_F16 ? 1 : 2;
    const Kern kern = kerns[which];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -6;
    if (!allowed[dev][which]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - kStatic) != cudaSuccess) return -6;
        allowed[dev][which] = true;
    }
    const int64_t blk = ACT ? 128 : 256, n_mb = (p->n_out + blk - 1) / blk;
    const int64_t live = p->n_expert < p->n_rows ? p->n_expert : p->n_rows;
    const int64_t most = (live + p->n_rows / kRows) * n_mb;
    const int64_t units = most < sm_count ? most : sm_count;
    const int stages = stages_of(p->n_expert);
    const Shape sh = { exl3b_div((uint32_t)n_mb), exl3b_div((uint32_t)units), exl3b_div((uint32_t)kRows),
                       (int32_t)((p->n_in + 127) / 128), stages, 1 };
    return chain_launch(kern, dim3((unsigned)units), dim3(kThreads), fixed_bytes(p->n_expert) + stages * kStageB, 1, st, map,
                        *p, sh);
}

}  // namespace wide
}  // namespace exl3b
