// exl3b200_gmm8w.cuh -- grouped_mm over FP8 operands where experts have many rows: the SORTED rows are the MMA's M and the
// weight rows its N, the other way round than in exl3b200_gmm8.cu's narrow form. A thread of the summing warps then has one
// sorted row and 128 of its outputs, so that a block's scale is one number a thread (sx of its row times sw of its columns'
// block): the sums cost an LDTM and half an FFMA2 a value and no shared memory. (With the weight rows as M every column has a
// scale of its own, read from shared memory four bytes a lane: 215 against X us at 16 experts, 16060 rows, 4096 -> 1536.)
//
// Two forms, persistent over units (expert, a group of its sorted rows, a block of 256 weight rows; silu_mul: 128 gate rows and
// their 128 up rows):
//   SOLO   one CTA, up to 128 sorted rows: experts of few rows, where the weights' bytes count
//   PAIR   two CTAs (a cluster), up to 256 sorted rows, tcgen05 cta_group::2: each CTA brings half of the sorted rows and half
//          of the weight rows, and both multiply by all of them
// Columns: act NONE: the block's weight rows in order. silu_mul: 64 gate rows, their 64 up rows, and the next 64 of each, so
// that a thread has both of its 64 outputs.
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

template <bool PAIR>
struct Cfg {
    static constexpr int NL = 128;                               // sorted rows a CTA at most: the MMA's lanes
    static constexpr int NT = PAIR ? 2 * NL : NL;                // ... and a unit
    static constexpr int WR = PAIR ? 128 : 256;                  // weight rows that a CTA brings
    static constexpr int COLS = 256;                             // of an accumulator: a unit's weight rows
    static constexpr int DB = 2;                                 // accumulators in turn
    static constexpr int SUM_G = 2;                              // groups of four summing warps, 128 columns each
    static constexpr int THREADS = (kEpiWarp0 + 4 * SUM_G) * 32;
    static constexpr int W_B = WR * kRowB, X_B = NL * kRowB, STAGE_B = W_B + X_B;
    static constexpr int BARS = 2 * kMaxSt + 2 * DB;
    static constexpr int fixed(int n_expert) { return 1024 + 512 + (n_expert + 4) * 4; }
    static constexpr int stages(int n_expert) {
        const int n = (227 * 1024 - kStatic - fixed(n_expert)) / STAGE_B;
        return n < kMaxSt ? n : kMaxSt;
    }
    static_assert(stages(kMaxExpert) >= 4 && BARS * 8 + 8 <= 512, "shared memory");
};

// 32 columns of this warp's 32 lanes, lane l's in thread l; tmem_wait32 before the registers are read.
__device__ __forceinline__ void tmem_ld32(uint32_t t, uint32_t r[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(t));
}
__device__ __forceinline__ void tmem_wait32(uint32_t r[32]) {
    tmem_wait(r);
    tmem_wait(r + 16);
}

// The sorted rows of a unit that CTA `rank` brings: `nl` from `first` on, in tiles alike (PAIR: halves in steps of 16).
struct Rows {
    int first, n;
};
template <bool PAIR>
__device__ __forceinline__ Rows rows_of(const Unit& u, uint32_t rank) {
    if (!PAIR) return Rows{ u.r0, u.nr };
    const int nl = (u.nr + 31) / 32 * 16;
    return Rows{ u.r0 + (int)rank * nl, rank ? max(u.nr - nl, 0) : min(u.nr, nl) };
}

// OUT: y_dtype; ACT: silu_mul.
template <bool PAIR, int OUT, bool ACT>
__global__ void __launch_bounds__(Cfg<PAIR>::THREADS, 1)
    k_gmm8w(const __grid_constant__ CUtensorMap wmap, const Exl3bGmmOp p, const Shape sh) {
    const int ST = sh.st;
    using C = Cfg<PAIR>;
    constexpr int THREADS = C::THREADS, MB = PAIR ? 2 : 1, DB = C::DB;
    constexpr int blk_out = ACT ? 128 : 256;                  // outputs of a unit
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* w_ring = smem;                                   // [ST][WR rows][128 B]
    uint8_t* x_ring = w_ring + ST * C::W_B;                   // [ST][NL rows][128 B]
    uint64_t* bars = reinterpret_cast<uint64_t*>(x_ring + ST * C::X_B);
    uint64_t* full = bars;                                    // producers (PAIR: and the odd CTA's MMA warp) -> MMA warp
    uint64_t* empty = full + ST;                              // MMA commit -> producers
    uint64_t* d_full = empty + ST;                            // MMA commit -> sums [DB]
    uint64_t* d_empty = d_full + DB;                          // sums (PAIR: of both CTAs) -> MMA [DB]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(d_empty + DB);
    uint32_t* dead = tmem_slot + 1;                           // a wait gave up: everyone leaves
    uint32_t* prefix = reinterpret_cast<uint32_t*>(bars) + 128;   // [n_expert + 1]
    __shared__ Unit utab[kTab];
    __shared__ uint32_t wsum[THREADS / 32];

    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const uint32_t rank = PAIR ? blockIdx.x & 1u : 0u;
    const uint32_t first = PAIR ? blockIdx.x >> 1 : blockIdx.x;
    const uint32_t stride = sh.stride.d;
    if (tid < ST) {
        mbar_init(&full[tid], 1 + 32 * kXWarps + (PAIR && rank == 0 ? 1 : 0));
        mbar_init(&empty[tid], 1);
    } else if (tid >= 32 && tid < 32 + DB) {
        mbar_init(&d_full[tid - 32], 1);
        mbar_init(&d_empty[tid - 32], 4 * C::SUM_G * MB);
    } else if (tid == 64) {
        *dead = 0;
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&wmap)) : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    if (warp == 1) tmem_alloc<PAIR>(tmem_slot, DB * C::COLS);
    if (PAIR) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    chain_wait();                                             // all above needs no memory but the CTA's own
    scan_units<THREADS, 1>(p, sh, first, prefix, utab, wsum);
    fence_before();
    __syncthreads();
    if (PAIR) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // both CTAs' barriers and tensor memory are set up
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
    // CTA then gives up at its next try, and the roles leave at their next unit.
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
    Pipe pipe;                                                // of the stages

    // The summing warps' sums need more than the 128 registers a thread that 512 threads start with: 256 x 192 + 256 x 64 are
    // the 512 x 128 of the launch.
    if (warp < kEpiWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 0) {
            // ------------------------------------------------------------ weights
            for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
                const Unit u = unit_at(i);
                for (int ck = 0; ck < nck; ++ck, pipe.next(ST)) {
                    wait(&empty[pipe.s], pipe.ph ^ 1);
                    mbar_expect_tx_el(&full[pipe.s], C::W_B);
                    uint8_t* dst = w_ring + pipe.s * C::W_B;
                    const int k = ck * 128;
#pragma unroll
                    for (int h = 0; h < C::WR / 128; ++h) {      // 128 columns at a time
                        const int at = h + (int)rank;
                        if (!ACT) {
                            tma_w_el(dst + h * kW_B, &wmap, k, u.blk * 256 + 128 * at, u.e, &full[pipe.s]);
                        } else {
                            const int o = u.blk * 128 + 64 * at;
                            tma_w_el(dst + h * kW_B, &wmap, k, o, u.e, &full[pipe.s]);
                            tma_w_el(dst + h * kW_B + kW_B / 2, &wmap, k, (int)p.n_out + o, u.e, &full[pipe.s]);
                        }
                    }
                }
            }
            // after a wait that gave up: a millisecond for the copies still in flight, before the CTA's memory goes
            if (*vdead)
                for (int j = 0; j < 50; ++j) __nanosleep(20000);
        } else if (warp == 1 && rank == 1) {
            // ------------------------------------------------------------ PAIR, odd CTA: its filled stages, reported
            for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
                for (int ck = 0; ck < nck; ++ck, pipe.next(ST)) {
                    wait(&full[pipe.s], pipe.ph);
                    proxy_fence();
                    if (lane == 0) arrive_even(&full[pipe.s]);
                    __syncwarp();
                }
            }
        } else if (warp == 1) {
            // ------------------------------------------------------------ MMA issuer
            const uint64_t wd0 = desc_sw128(smem_u32(w_ring)), xd0 = desc_sw128(smem_u32(x_ring));
            // D f32, e4m3 both, both operands K-major, M 128 (PAIR: 256), N 256
            const uint32_t idesc = (uint32_t)C::COLS >> 3 << 17 | (8u * MB) << 24 | 1u << 4;
            Pipe db;
            for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
                for (int ck = 0; ck < nck; ++ck, pipe.next(ST), db.next(DB)) {
                    wait(&full[pipe.s], pipe.ph);
                    proxy_fence();
                    wait(&d_empty[db.s], db.ph ^ 1);
                    fence_after();
                    mma4_f8<PAIR>(tmem + db.s * C::COLS, xd0 + (uint64_t)(pipe.s * C::X_B >> 4), wd0 + (uint64_t)(pipe.s * C::W_B >> 4),
                                  idesc, 0u);
                    commit_el<PAIR>(&d_full[db.s]);
                    commit_el<PAIR>(&empty[pipe.s]);
                }
            }
        } else if (warp >= kXWarp0) {
            // ------------------------------------------------------------ sorted rows
            // Eight lanes a row of a stage, 16 rows a pass of the four warps; each thread's copies arrive on the stage's
            // barrier when they have landed, and the MMA warp, which sees that, makes them visible to the asynchronous proxy.
            // Rows past the unit's are left as they were: their sums are nobody's.
            constexpr int RP = C::NL / 16, kStep = 4;             // passes a stage; stages a step of the row pointers
            const int xt = tid - kXWarp0 * 32, c = xt & 7, rr = xt >> 3;
            const int kb = (int)p.n_in;
            const uint32_t dst0 = smem_u32(x_ring) + rr * kRowB + ((c ^ (rr & 7)) << 4);
            RowAhead<RP> ahead(p, rr, 16);
            auto mine = [&](uint32_t i) {
                Unit u = unit_at(i);
                const Rows r = rows_of<PAIR>(u, rank);
                u.r0 = r.first;
                u.nr = r.n;
                return u;
            };
            Unit u = n_mine ? mine(0) : Unit{};
            if (n_mine) ahead.fetch(u);
            for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
                const int nl = u.nr;
                const uint8_t* src[RP];
                ahead.rows(static_cast<const uint8_t*>(p.x) + c * 16, p.x_pitch_bytes, src);
                if (i + 1 < n_mine) {
                    u = mine(i + 1);
                    ahead.fetch(u);
                }
                for (int c0 = 0; c0 < nck; c0 += kStep) {
#pragma unroll
                    for (int a = 0; a < kStep; ++a) {
                        if (c0 + a >= nck) break;
                        wait(&empty[pipe.s], pipe.ph ^ 1);
                        const uint32_t dst = dst0 + pipe.s * C::X_B;
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
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        const int q = warp & 3, g = (warp - kEpiWarp0) >> 2, ew = warp - kEpiWarp0;
        constexpr int es = OUT == RAD_F32 ? 4 : 2;
        clear_outside<OUT>(p, blockIdx.x * 4 * C::SUM_G + ew, gridDim.x * 4 * C::SUM_G, lane);
        const bool whole = ((reinterpret_cast<uintptr_t>(p.x_scales) | (uintptr_t)p.xs_pitch) & 15) == 0;
        RowAhead<1> ahead(p, 32 * q + lane, 1);
        // four blocks' scales: of the thread's row, and of the weight, one a lane (lanes 4 .. 7: silu_mul's up rows)
        struct Scales {
            float x[4], w;
        };
        const float *xs = nullptr, *ws = nullptr;
        auto load = [&](Scales& s, int ck) {
            if (whole && ck + 4 <= nck) {
                const float4 t = *reinterpret_cast<const float4*>(xs + ck);
                s.x[0] = t.x; s.x[1] = t.y; s.x[2] = t.z; s.x[3] = t.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) s.x[j] = ck + j < nck ? xs[ck + j] : 0.f;
            }
            s.w = ck + (lane & 3) < nck ? ws[ck + (lane & 3)] : 0.f;
        };
        Scales next;
        bool live_next = false;
        auto begin = [&](uint32_t i) {                        // unit i's rows and first scales; its slots are there
            const Unit u = unit_at(i);
            const uint8_t* at[1];
            ahead.rows(p.x_scales, p.xs_pitch, at);
            xs = reinterpret_cast<const float*>(at[0]);
            const int b = ACT ? u.blk + (lane & 4 ? p.ws_blocks : 0) : min(2 * u.blk + g, p.ws_blocks - 1);
            ws = reinterpret_cast<const float*>(p.w_scales + u.e * p.ws_expert_bytes + b * p.ws_blk_bytes);
            load(next, 0);
        };
        auto fetch = [&](uint32_t i) {                        // ... are asked for
            Unit u = unit_at(i);
            const Rows r = rows_of<PAIR>(u, rank);
            u.r0 = r.first;
            u.nr = r.n;
            ahead.fetch(u);
            const int at = r.first + 32 * q + lane;
            live_next = 32 * q + lane < r.n && (!p.sorted_tok || p.sorted_tok[at] >= 0);
        };
        if (n_mine) {
            fetch(0);
            begin(0);
        }
        Pipe db;
        for (uint32_t i = 0; i < n_mine; ++i) {
            const Unit u = unit_at(i);
            const Rows r = rows_of<PAIR>(u, rank);
            const bool any = 32 * q < r.n, live = live_next;
            if (i + 1 < n_mine) fetch(i + 1);
            uint64_t acc[4][16];                              // 128 columns, two a word
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
                for (int k = 0; k < 16; ++k) acc[c][k] = 0;
            Scales s = next;
#pragma unroll 1
            for (int ck = 0; ck < nck; ++ck, db.next(DB)) {
                if ((ck & 3) == 0) {
                    s = next;
                    if (ck + 4 < nck) load(next, ck + 4);
                }
                float f[2];
                f[0] = s.x[0] * __shfl_sync(0xFFFFFFFFu, s.w, ck & 3);
                f[1] = ACT ? s.x[0] * __shfl_sync(0xFFFFFFFFu, s.w, 4 + (ck & 3)) : f[0];
                s.x[0] = s.x[1]; s.x[1] = s.x[2]; s.x[2] = s.x[3];
                wait(&d_full[db.s], db.ph);
                fence_after();
                const uint32_t d = tmem + ((uint32_t)(32 * q) << 16) + db.s * C::COLS + 128 * g;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t a[32];
                    if (any) {
                        tmem_ld32(d + 32 * c, a);
                        tmem_wait32(a);
                    }
                    if (c == 3) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if (PAIR) arrive_even(&d_empty[db.s]);
                            else mbar_arrive(&d_empty[db.s]);
                        }
                    }
                    if (any) {
                        const uint64_t ff = f2pk(f[c >> 1], f[c >> 1]);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            acc[c][k] = fma2(f2pk(__uint_as_float(a[2 * k]), __uint_as_float(a[2 * k + 1])), ff, acc[c][k]);
                    }
                }
            }
            if (__any_sync(0xFFFFFFFFu, *vdead)) break;
            if (i + 1 < n_mine) begin(i + 1);                 // its first scales, on their way under the epilogue
            const int row = 32 * q + lane;
            if (row < r.n) {
                constexpr int NV = ACT ? 64 : 128;
                const int64_t n0 = (int64_t)u.blk * blk_out + NV * g;            // the thread's first output
                uint8_t* d = static_cast<uint8_t*>(p.y) + (r.first + row) * (p.y_pitch * es) + n0 * es;
                const int left = (int)min((int64_t)NV, p.n_out - n0);
#pragma unroll
                for (int j = 0; j < NV / 8; ++j) {
                    if (8 * j >= left) break;
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) f2upk(acc[j >> 2][4 * (j & 3) + k], v[2 * k], v[2 * k + 1]);
                    if constexpr (ACT) {
                        float up[8];
#pragma unroll
                        for (int k = 0; k < 4; ++k) f2upk(acc[2 + (j >> 2)][4 * (j & 3) + k], up[2 * k], up[2 * k + 1]);
                        float least = v[0];
#pragma unroll
                        for (int k = 1; k < 8; ++k) least = fminf(least, v[k]);
                        if (least < kSiluLow) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) v[k] = v[k] < kSiluLow ? silu_up_low(v[k], up[k]) : silu_up(v[k], up[k]);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k) v[k] = silu_up(v[k], up[k]);
                        }
                    }
                    if (!live) {                                                  // a dropped slot
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[k] = 0.f;
                    }
                    if constexpr (OUT == RAD_F32) {
                        *reinterpret_cast<float4*>(d + 32 * j) = make_float4(v[0], v[1], v[2], v[3]);
                        *reinterpret_cast<float4*>(d + 32 * j + 16) = make_float4(v[4], v[5], v[6], v[7]);
                    } else {
                        *reinterpret_cast<uint4*>(d + 16 * j) = make_uint4(pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3]),
                                                                            pack2<OUT>(v[4], v[5]), pack2<OUT>(v[6], v[7]));
                    }
                }
            }
            __syncwarp();
        }
    }
    fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();                             // no CTA's memory goes while another uses it
    if (warp == 1) {
        fence_after();
        tmem_free<PAIR>(tmem, DB * C::COLS);
    }
}

template <bool PAIR, bool ACT>
int launch(const Exl3bGmmOp* p, int sm_count, cudaStream_t st) {
    using C = Cfg<PAIR>;
    typedef void (*Kern)(CUtensorMap, Exl3bGmmOp, Shape);
    CUtensorMap map;
    const int rc = make_map(p, &map, ACT ? 64 : 128);
    if (rc) return rc;
    static const Kern kerns[3] = { k_gmm8w<PAIR, RAD_F32, ACT>, k_gmm8w<PAIR, RAD_F16, ACT>, k_gmm8w<PAIR, RAD_BF16, ACT> };
    static bool allowed[64][3];                               // the most shared memory, once a device
    const int which = p->y_dtype == RAD_F32 ? 0 : p->y_dtype == RAD_F16 ? 1 : 2;
    const Kern kern = kerns[which];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -6;
    if (!allowed[dev][which]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - kStatic) != cudaSuccess) return -6;
        allowed[dev][which] = true;
    }
    const int ctas = PAIR ? 2 : 1;
    const int64_t blk = ACT ? 128 : 256, n_mb = (p->n_out + blk - 1) / blk;
    const int64_t live = p->n_expert < p->n_rows ? p->n_expert : p->n_rows;
    const int64_t most = (live + p->n_rows / C::NT) * n_mb, room = sm_count / ctas, units = most < room ? most : room;
    const int stages = C::stages(p->n_expert);
    const Shape sh = { exl3b_div((uint32_t)n_mb), exl3b_div((uint32_t)units), exl3b_div((uint32_t)C::NT),
                       (int32_t)((p->n_in + 127) / 128), stages, 1 };
    return chain_launch(kern, dim3((unsigned)(units * ctas)), dim3(C::THREADS), C::fixed(p->n_expert) + stages * C::STAGE_B,
                        ctas, st, map, *p, sh);
}

}  // namespace wide
}  // namespace exl3b
