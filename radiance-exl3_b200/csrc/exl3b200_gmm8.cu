// exl3b200_gmm8.cu -- grouped_mm over FP8 operands: e4m3 codes with an f32 scale for each 128 values of a row of x and each
// 128 x 128 of a weight, on the 5th-generation tensor cores. sm_100a only.
//
//   z[n] = sum over blocks b of 128 k:  sx[t(i)][b] * sw[e][n / 128][b] * sum over k of b of x[t(i)][k] * w[e][n][k]
//   y[i][n] = z[n], or silu(z[n]) * z[n_out + n] (act silu_mul), for every sorted row i of expert e
//
// The units of work, the operands' way into shared memory and the roles of the warps are grouped_mm's for 16-bit operands
// (exl3b200_gmm.cu; exl3b200_gmm.cuh); a stage is 128 bytes of k, here one block of 128. What differs is the sum over k. The
// scales are any f32 numbers, so the tensor cores' sums of one block cannot run on into the next one's: each stage's four MMAs
// (kind::f8f6f4, K 32) start a fresh accumulator in tensor memory, one of several in turn, and the summing warps, which hold the
// unit's sums in registers, add it times its scales:
//   sum[n] = fma(d[n], sx * sw, sum[n])    in f32, one rounding a block of 128 and one for the scales' product
// Where experts have many rows, exl3b200_gmm8w.cuh's kernel does it; here, where they have few, the WEIGHT rows are the MMA's M
// (128) and up to 32 sorted rows its N, in steps of 16, two CTAs an SM. With few units (SPLIT) a cluster for each of them, every
// CTA a part of its k, the parts summed through distributed shared memory in the CTAs' order.
// Warps of a CTA:
//   0       weights: cp.async.bulk.tensor, 128-byte swizzled
//   1       MMA issuer
//   2       scales: sx * sw of the sorted rows into a ring of stages; silu_mul: for gate rows and for up rows
//   4..7    sorted rows: 16-byte cp.async through sorted_tok
//   8..11   sums: each warp 32 weight rows, then its outputs
// Every wait is bounded; one that gives up sets the error word, and every role then drains and leaves.
// Few rows an expert are bounded by the weights' way from HBM: 173 live experts, 629 rows, 640 -> 2560, 286 MB in 50 us (5.7
// TB/s); one token's ten experts, 2048 -> 512 silu_mul, 21 MB, in 10 us with its f8_quantize, by the launches, the set-up and
// the first loads.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "exl3b200_chain.cuh"
#include "exl3b200_decode.cuh"
#include "exl3b200_dense.h"
#include "exl3b200_gmm.cuh"
#include "exl3b200_gmm8w.cuh"

using namespace exl3b;

namespace {

constexpr int kScaleSt = 4;                      // stages of scales at once

template <bool SPLIT, bool ACT>
struct Cfg {
    static constexpr int NT = 32;                                // sorted rows a unit at most
    static constexpr int THREADS = (kEpiWarp0 + 4) * 32;
    static constexpr int X_B = NT * kRowB;
    static constexpr int STAGE_B = kW_B + X_B;
    static constexpr int HALVES = ACT ? 2 : 1;                   // scales a sorted row: gate's, up's
    static constexpr int SC_ROWS = NT * 2;                       // floats of a half's scales: each twice
    static constexpr int SC_B = kScaleSt * HALVES * SC_ROWS * 4;
    static constexpr int EPI_B = SPLIT ? NT * kEpiLd * 4 : 4 * 1024;
    static constexpr int DB = 4;                                 // accumulators in turn, of NT columns
    static constexpr int PER_SM = 2;
    static constexpr int BARS = 2 * kMaxSt + 2 * DB + 2 * kScaleSt + 1;
    static constexpr int fixed(int n_expert) { return 1024 + EPI_B + SC_B + 512 + (n_expert + 4) * 4; }
    static constexpr int stages(int n_expert, int per_sm) {
        const int n = ((per_sm == 1 ? 227 : 113) * 1024 - kStatic - fixed(n_expert)) / STAGE_B;
        return n < kMaxSt ? n : kMaxSt;
    }
    static_assert(stages(kMaxExpert, PER_SM) >= (SPLIT ? 3 : 4) && BARS * 8 + 8 <= 512, "shared memory");
};

// Where row r's scale lies in the ring, twice: with those of row r + 4, when r % 8 < 4, 16 bytes that a thread of tmem_ld4's
// rows loads at once.
__device__ __forceinline__ int scale_at(int r) { return (r >> 3) * 16 + (r & 3) * 4 + (r & 4) / 2; }

// 32 columns of 16 lanes: r[2 i + v] is lane t / 4 + 8 v, column 4 i + t % 4 in thread t. (Of the ways to read 16 lanes at a time
// this moves 128 bytes a cycle, tmem_ld8x8's 64.)
__device__ __forceinline__ void tmem_ld4(uint32_t taddr, uint32_t r[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x128b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// OUT: y_dtype; ACT: silu_mul.
template <bool SPLIT, int OUT, bool ACT>
__global__ void __launch_bounds__(Cfg<SPLIT, ACT>::THREADS, Cfg<SPLIT, ACT>::PER_SM)
    k_gmm8(const __grid_constant__ CUtensorMap wmap, const Exl3bGmmOp p, const Shape sh) {
    const int ST = sh.st, split = sh.split;
    using C = Cfg<SPLIT, ACT>;
    constexpr int NT = C::NT, THREADS = C::THREADS, DB = C::DB;
    constexpr int blk_out = ACT ? 64 : 128;                   // outputs a block (a CTA's part of a unit)
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* w_ring = smem;                                   // [ST][128 rows][128 B]
    uint8_t* x_ring = w_ring + ST * kW_B;                     // [ST][32 rows][128 B]
    float* sc_ring = reinterpret_cast<float*>(x_ring + ST * C::X_B);   // [kScaleSt][HALVES][SC_ROWS]
    float* epi = sc_ring + C::SC_B / 4;
    uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(epi) + C::EPI_B);
    uint64_t* full = bars;                                    // producers -> MMA warp
    uint64_t* empty = full + ST;                              // MMA commit -> producers
    uint64_t* d_full = empty + ST;                            // MMA commit -> sums [DB]
    uint64_t* d_empty = d_full + DB;                          // sums -> MMA [DB]
    uint64_t* sc_full = d_empty + DB;                         // scales -> sums [kScaleSt]
    uint64_t* sc_empty = sc_full + kScaleSt;                  // sums -> scales [kScaleSt]
    uint64_t* part_full = sc_empty + kScaleSt;                // SPLIT: every CTA's partial sums are in its shared memory
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(part_full + 1);
    uint32_t* dead = tmem_slot + 1;                           // a wait gave up: everyone leaves
    uint32_t* prefix = reinterpret_cast<uint32_t*>(bars) + 128;   // [n_expert + 1]
    __shared__ Unit utab[kTab];
    __shared__ uint32_t wsum[THREADS / 32];

    const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0), lane = tid & 31;
    const uint32_t part = SPLIT ? blockIdx.x % split : 0u;    // which part of its k
    const uint32_t first = SPLIT ? blockIdx.x / split : blockIdx.x;
    const uint32_t stride = sh.stride.d;
    if (tid < ST) {
        mbar_init(&full[tid], 1 + 32 * kXWarps);
        mbar_init(&empty[tid], 1);
    } else if (tid >= 32 && tid < 32 + DB) {
        mbar_init(&d_full[tid - 32], 1);
        mbar_init(&d_empty[tid - 32], 4);
    } else if (tid >= 64 && tid < 64 + kScaleSt) {
        mbar_init(&sc_full[tid - 64], 1);
        mbar_init(&sc_empty[tid - 64], 4);
    } else if (tid == 96) {
        *dead = 0;
        if (SPLIT) mbar_init(part_full, 4 * split);
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&wmap)) : "memory");
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    if (warp == 1) tmem_alloc<false>(tmem_slot, DB * NT);
    if (SPLIT) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    chain_wait();                                             // all above needs no memory but the CTA's own
    scan_units<THREADS, 1>(p, sh, first, prefix, utab, wsum);
    fence_before();
    __syncthreads();
    if (SPLIT) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // all CTAs' barriers and tensor memory are set up
    fence_after();
    chain_next();                                             // every CTA has its tensor memory: a later kernel may ask for its own
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, *tmem_slot, 0);
    const uint32_t n_units = prefix[p.n_expert];
    // SPLIT: the grid has a cluster for every unit that offsets in ascending order can make, so one at most
    const uint32_t n_mine = n_units > first ? SPLIT ? 1u : exl3b_div_of(n_units - first + stride - 1, sh.stride) : 0u;
    auto unit_at = [&](uint32_t i) {
        return i < kTab ? utab[i] : find_unit<1>(p, prefix, first + i * stride, sh);
    };
    const int nck = sh.nck;
    // this CTA's stages of a unit
    const int k0 = SPLIT ? (int)(part * (uint32_t)nck / (uint32_t)split) : 0;
    const int k1 = SPLIT ? (int)((part + 1) * (uint32_t)nck / (uint32_t)split) : nck;
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
    if (warp == 0) {
        // ---------------------------------------------------------------- weights
        for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
            const Unit u = unit_at(i);
            for (int ck = k0; ck < k1; ++ck, pipe.next(ST)) {
                wait(&empty[pipe.s], pipe.ph ^ 1);
                mbar_expect_tx_el(&full[pipe.s], kW_B);
                uint8_t* dst = w_ring + pipe.s * kW_B;
                const int k = ck * 128;
                if (!ACT) {
                    tma_w_el(dst, &wmap, k, u.blk * 128, u.e, &full[pipe.s]);
                } else if (p.n_out % 16 == 0) {
                    tma_w5_el(dst, &wmap, k, u.blk * 4, u.e, &full[pipe.s]);
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        tma_w_el(dst + q * 4096, &wmap, k, u.blk * 64 + 16 * q, u.e, &full[pipe.s]);
                        tma_w_el(dst + q * 4096 + 2048, &wmap, k, (int)p.n_out + u.blk * 64 + 16 * q, u.e, &full[pipe.s]);
                    }
                }
            }
        }
        // after a wait that gave up: a millisecond for the copies still in flight, before the CTA's memory goes
        if (*vdead)
            for (int j = 0; j < 50; ++j) __nanosleep(20000);
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer
        const uint64_t wd0 = desc_sw128(smem_u32(w_ring)), xd0 = desc_sw128(smem_u32(x_ring));
        Pipe db;
        for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
            // D f32, e4m3 both, both operands K-major, M 128, N the rows in steps of 16
            const uint32_t idesc = ((uint32_t)unit_at(i).nr + 15) / 16 << 18 | 8u << 24 | 1u << 4;
            for (int ck = k0; ck < k1; ++ck, pipe.next(ST), db.next(DB)) {
                wait(&full[pipe.s], pipe.ph);
                proxy_fence();
                wait(&d_empty[db.s], db.ph ^ 1);
                fence_after();
                mma4_f8(tmem + db.s * NT, wd0 + (uint64_t)(pipe.s * kW_B >> 4), xd0 + (uint64_t)(pipe.s * C::X_B >> 4), idesc);
                commit_el<false>(&d_full[db.s]);
                commit_el<false>(&empty[pipe.s]);
            }
        }
    } else if (warp == 2) {
        // ---------------------------------------------------------------- scales
        // A lane has a sorted row and loads four blocks' scales of it at a time, into two register sets in turn, one on its way
        // while the other is used, across units; the weight's scales of a batch are one a lane (lanes 4 .. 7: up's).
        struct Set {
            float x[4], w;
        };
        RowAhead<1> ahead(p, lane, 1);
        const uint8_t* src[1];
        const float* wsrc = nullptr;
        const bool whole = ((reinterpret_cast<uintptr_t>(p.x_scales) | (uintptr_t)p.xs_pitch) & 15) == 0;
        uint32_t lu = 0, cu = 0;                              // units of the next load and of the next batch used
        int lc = k0, cc = k0;                                 // ... and their first stages
        auto rows = [&](const Unit& u) {
            ahead.rows(p.x_scales, p.xs_pitch, src);
            const int b = u.blk * blk_out / 128 + (lane & 4 ? p.ws_blocks * (C::HALVES - 1) : 0);
            wsrc = reinterpret_cast<const float*>(p.w_scales + u.e * p.ws_expert_bytes + b * p.ws_blk_bytes);
        };
        if (n_mine) {
            const Unit u = unit_at(0);
            ahead.fetch(u);
            rows(u);
            if (n_mine > 1) ahead.fetch(unit_at(1));
        }
        auto load = [&](Set& s) {
            if (lu >= n_mine) return;
            const float* at = reinterpret_cast<const float*>(src[0]) + lc;
            if (whole && lc + 4 <= k1 && (lc & 3) == 0) {     // SPLIT: a part may start inside four blocks
                const float4 t = *reinterpret_cast<const float4*>(at);
                s.x[0] = t.x; s.x[1] = t.y; s.x[2] = t.z; s.x[3] = t.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) s.x[j] = lc + j < k1 ? at[j] : 0.f;
            }
            s.w = lc + (lane & 3) < k1 ? wsrc[lc + (lane & 3)] : 0.f;
            if ((lc += 4) >= k1) {
                lc = k0;
                if (++lu < n_mine) {
                    rows(unit_at(lu));
                    if (lu + 1 < n_mine) ahead.fetch(unit_at(lu + 1));
                }
            }
        };
        auto use = [&](const Set& s) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (cc + j >= k1) break;
                wait(&sc_empty[pipe.s], pipe.ph ^ 1);
#pragma unroll
                for (int h = 0; h < C::HALVES; ++h) {
                    const float f = s.x[j] * __shfl_sync(0xFFFFFFFFu, s.w, 4 * h + j);
                    *reinterpret_cast<float2*>(sc_ring + (pipe.s * C::HALVES + h) * C::SC_ROWS + scale_at(lane)) = make_float2(f, f);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sc_full[pipe.s]);
                pipe.next(kScaleSt);
            }
            if ((cc += 4) >= k1) {
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
    } else if (warp >= kXWarp0 && warp < kEpiWarp0) {
        // ---------------------------------------------------------------- sorted rows
        // Eight lanes a row of a stage, 16 rows a pass of the four warps; each thread's copies arrive on the stage's barrier
        // when they have landed, and the MMA warp, which sees that, makes them visible to the asynchronous proxy.
        constexpr int RP = NT / 16, kStep = 4;                // passes a stage; stages a step of the row pointers
        const int xt = tid - kXWarp0 * 32, c = xt & 7, rr = xt >> 3;
        const int kb = (int)p.n_in;
        const uint32_t dst0 = smem_u32(x_ring) + rr * kRowB + ((c ^ (rr & 7)) << 4);
        RowAhead<RP> ahead(p, rr, 16);
        Unit u = n_mine ? unit_at(0) : Unit{};
        if (n_mine) ahead.fetch(u);
        for (uint32_t i = 0; i < n_mine && !*vdead; ++i) {
            const int nl = u.nr;
            const uint8_t* src[RP];
            ahead.rows(static_cast<const uint8_t*>(p.x) + k0 * kRowB + c * 16, p.x_pitch_bytes, src);
            if (i + 1 < n_mine) {
                u = unit_at(i + 1);
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
    } else if (warp >= kEpiWarp0) {
        // ---------------------------------------------------------------- sums
        const int q = warp & 3;
        constexpr int es = OUT == RAD_F32 ? 4 : 2;
        uint8_t* const y = static_cast<uint8_t*>(p.y);
        clear_outside<OUT>(p, blockIdx.x * 4 + q, gridDim.x * 4, lane);
        const int64_t row_b = p.y_pitch * es;
        // which of a unit's rows are live: its slots are fetched a unit ahead
        int32_t slot = 0;
        auto fetch = [&](const Unit& n) { slot = p.sorted_tok && lane < n.nr ? p.sorted_tok[n.r0 + lane] : 0; };
        if (n_mine) fetch(unit_at(0));
        Pipe db;
        for (uint32_t i = 0; i < n_mine; ++i) {
            const Unit u = unit_at(i);
            const uint32_t live = __ballot_sync(0xFFFFFFFFu, slot >= 0);
            if (i + 1 < n_mine) fetch(unit_at(i + 1));
            uint64_t acc[2][8];                               // sums of each half of the lanes as tmem_ld4 has them, two a word
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[k >> 3][k & 7] = 0;
            for (int ck = k0; ck < k1; ++ck, pipe.next(kScaleSt), db.next(DB)) {
                wait(&sc_full[pipe.s], pipe.ph);
                wait(&d_full[db.s], db.ph);
                fence_after();
                const float* sc = sc_ring + pipe.s * C::HALVES * C::SC_ROWS + 4 * (lane & 3);
                const uint32_t d = tmem + ((uint32_t)(32 * q) << 16) + db.s * NT;
                // one half's 16 registers at a time: with both, the pairs did not fit (13.8 against 10.7 us at one token)
                uint32_t a[16];
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    tmem_ld4(d + ((16u * s) << 16), a);
                    tmem_wait(a);
                    if (s == 1) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&d_empty[db.s]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {             // eight rows: two of them this thread's
                        const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(sc + (ACT ? s * C::SC_ROWS : 0) + 16 * e);
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            uint64_t& t = acc[s][2 * e + v];
                            const int k = 4 * e + 2 * v;
                            t = fma2(f2pk(__uint_as_float(a[k]), __uint_as_float(a[k + 1])), v ? f.y : f.x, t);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sc_empty[pipe.s]);
            }
            if (__any_sync(0xFFFFFFFFu, *vdead)) break;
            const int64_t b0 = (int64_t)u.blk * blk_out;           // the block's first output
            if constexpr (SPLIT) {
                // The parts' sums meet through distributed shared memory: every CTA puts its own into its shared memory,
                // then sums every split-th row over the CTAs, in their order, and stores it.
                float* const st = epi;
#pragma unroll
                for (int k = 0; k < 32; ++k)
                    st[(4 * (k >> 1 & 7) + (lane & 3)) * kEpiLd + 32 * q + 16 * (k >> 4) + 8 * (k & 1) + (lane >> 2)] =
                        __uint_as_float((uint32_t)(acc[k >> 4][k >> 1 & 7] >> (32 * (k & 1))));
                __syncwarp();                                  // the arrivals publish the whole warp's sums
                if (lane < split) arrive_at(part_full, lane);
                __syncwarp();
                wait(part_full, 0);
                asm volatile("fence.acq_rel.cluster;" ::: "memory");
                const bool out_lane = !ACT || !(lane & 4);    // silu_mul: 16 gate columns, then their 16 up columns
                const int64_t n0 = b0 + (ACT ? 16 * (lane >> 3) + 4 * (lane & 3) : 4 * lane);
                for (int j = part + split * q; j < u.nr; j += split * 4) {
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
                    if (ACT) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float up = __shfl_xor_sync(0xFFFFFFFFu, v[e], 4);
                            v[e] = v[e] < kSiluLow ? silu_up_low(v[e], up) : silu_up(v[e], up);
                        }
                    }
                    if (!(live >> j & 1)) v[0] = v[1] = v[2] = v[3] = 0.f;        // a dropped slot
                    if (out_lane && n0 < p.n_out) {
                        uint8_t* d = y + (u.r0 + j) * row_b + n0 * es;
                        if constexpr (OUT == RAD_F32) *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
                        else *reinterpret_cast<uint2*>(d) = make_uint2(pack2<OUT>(v[0], v[1]), pack2<OUT>(v[2], v[3]));
                    }
                }
                break;
            }
            const int64_t n_warp = b0 + (ACT ? 16 : 32) * q;                 // the warp's first output
#pragma unroll
            for (int sl = 0; sl < NT / kSlice; ++sl) {
                const int t0 = kSlice * sl;
                if (t0 >= u.nr) break;
                uint32_t a[16];                                               // as act_slice takes them
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    a[k] = (uint32_t)(acc[k >> 3][4 * sl + 2 * (k >> 2 & 1) + (k & 1)] >> (32 * (k >> 1 & 1)));
                constexpr int NV = ACT ? 8 : 16;
                float v[NV];
                act_slice<ACT>(a, v);
                const uint32_t here = live >> t0;
                if ((here & 0xFFFFu) != 0xFFFFu) {                            // dropped slots are zero
#pragma unroll
                    for (int k = 0; k < NV; ++k)
                        if (!(here >> (8 * (k >> 2 & 1) + 4 * (k & 1) + (lane & 3)) & 1)) v[k] = 0.f;
                }
                store_slice<OUT, ACT, true>(v, y + (u.r0 + t0) * row_b, row_b, n_warp, p.n_out, u.nr - t0,
                                            reinterpret_cast<uint8_t*>(epi) + q * 1024, lane);
            }
        }
    }
    fence_before();
    __syncthreads();
    if (SPLIT) cluster_sync_all();                            // no CTA's memory goes while another uses it
    if (warp == 1) {
        fence_after();
        tmem_free<false>(tmem, DB * NT);
    }
}

typedef void (*Kern)(CUtensorMap, Exl3bGmmOp, Shape);

// split: CTAs a unit, each a part of its k (SPLIT).
template <bool SPLIT, bool ACT>
int launch(const Exl3bGmmOp* p, int sm_count, int split, cudaStream_t st) {
    using C = Cfg<SPLIT, ACT>;
    CUtensorMap map;
    const int rc = make_map(p, &map);
    if (rc) return rc;
    static const Kern kerns[3] = { k_gmm8<SPLIT, RAD_F32, ACT>, k_gmm8<SPLIT, RAD_F16, ACT>, k_gmm8<SPLIT, RAD_BF16, ACT> };
    static bool allowed[64][3];                               // the most shared memory, once a device
    const int which = p->y_dtype == RAD_F32 ? 0 : p->y_dtype == RAD_F16 ? 1 : 2;
    const Kern kern = kerns[which];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -6;
    if (!allowed[dev][which]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - kStatic) != cudaSuccess) return -6;
        allowed[dev][which] = true;
    }
    const int64_t most = most_units(p, C::NT, 1);
    // few units: one CTA an SM, with the whole of its shared memory for stages in flight; clusters of three or four do not
    // fill the SMs of every processing cluster
    const int64_t alone = split > 2 ? sm_count - sm_count / 8 : sm_count;
    const int per_sm = most * split <= alone ? 1 : C::PER_SM;
    const int64_t room = (int64_t)sm_count * per_sm / split, units = most < room ? most : room;
    const int stages = C::stages(p->n_expert, per_sm);
    const int64_t blk = ACT ? 64 : 128;
    const Shape sh = { exl3b_div((uint32_t)((p->n_out + blk - 1) / blk)), exl3b_div((uint32_t)units), exl3b_div((uint32_t)C::NT),
                       (int32_t)((p->n_in + 127) / 128), stages, split };
    return chain_launch(kern, dim3((unsigned)(units * split)), dim3(C::THREADS), C::fixed(p->n_expert) + stages * C::STAGE_B, split, st,
                        map, *p, sh);
}

// About how many units there will be: groups of nt rows, half a one more an expert for its remainder, one an expert at least.
int64_t likely_units(const Exl3bGmmOp* p, int nt, int64_t blk) {
    const int64_t live = p->n_expert < p->n_rows ? p->n_expert : p->n_rows, some = p->n_rows / nt + live / 2;
    return (some > live ? some : live) * ((p->n_out + blk - 1) / blk);
}

// 0: the wide form; otherwise the narrow one, with as many CTAs a unit, each a part of its k.
int form_of(const Exl3bGmmOp* p, int sm_count) {
    // The wide form where its units cost less: a unit's stage there takes 3.1 times as long as a narrow one's (2 times where the
    // SMs have a unit each at most), and its start and end as long as five of those; narrow units run two an SM. Narrow and wide,
    // us: 64 experts, 2048 -> 512 silu_mul, 28 rows each 28.3 and 29.1, 40 rows 32.9 and 29.9, 130 rows 62.4 and 40.7; 640 ->
    // 2560, 40 rows 27.5 and 27.8, 96 rows 47.4 and 36.9; 300 experts of 96 rows, 448 -> 160 silu_mul 30.9 and 32.1; one expert,
    // 4096 -> 1536, 512 rows 17.8 and 22.3, 1024 rows 30.2 and 22.7.
    const int64_t nck = (p->n_in + 127) / 128, sm = sm_count;
    const int64_t wide_units = likely_units(p, 128, p->act ? 128 : 256), narrow_units = likely_units(p, 32, p->act ? 64 : 128);
    const int64_t wide_cost = wide_units > sm ? wide_units * (31 * nck + 50) : sm * (20 * nck + 50);
    if (wide_cost < 10 * nck * (narrow_units > 2 * sm ? narrow_units : 2 * sm)) return 0;
    int64_t split = sm / most_units(p, 32, 1);                // so the grid has room for a cluster a unit: the kernel counts on it
    if (split > nck / 4) split = nck / 4;
    if (split > kMaxSplit) split = kMaxSplit;
    return split >= 2 ? (int)split : 1;
}

template <bool ACT>
int launch_form(const Exl3bGmmOp* p, int sm_count, cudaStream_t st) {
    const int form = form_of(p, sm_count);
    if (form == 0) return wide::launch<ACT>(p, sm_count, st);
    if (form > 1) return launch<true, ACT>(p, sm_count, form, st);
    return launch<false, ACT>(p, sm_count, 1, st);
}

}  // namespace

extern "C" {

int exl3b_gmm8_form(int64_t n_expert, int64_t n_rows, int64_t n_out, int64_t n_in, int act, int sm_count) {
    Exl3bGmmOp p = {};
    p.n_expert = (int32_t)n_expert;
    p.n_rows = n_rows;
    p.n_out = n_out;
    p.n_in = n_in;
    p.act = act;
    return form_of(&p, sm_count);
}

int exl3b_cuda_gmm8(const Exl3bGmmOp* p, int sm_count, void* stream) {
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return p->act ? launch_form<true>(p, sm_count, st) : launch_form<false>(p, sm_count, st);
}

}  // extern "C"
