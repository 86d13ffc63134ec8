// Products of the linear-head cross-entropy on the 5th-generation tensor cores (tcgen05 / TMEM / TMA), sm_100a only: 16-bit operands,
// fp32 accumulators.  linear_ce.cu has the mathematics and the pass over the rows that stands between the two kernels.
//
//   LOGITS   z = x w^T, a tile of 256 rows x 256 columns at a time (128 x 256 up to 128 rows); the epilogue leaves reference, sum and u of each row and
//            half tile (see linear_ce.cu): the logits never reach memory
//   GRADS    dx = d w and dw = d^T x in one launch.  dx has few tiles with a long sum (the vocabulary), dw many with a short one; the long
//            ones start first and are cut along the sum when one alone would take longer than everything spread over the SMs.  d, w and x are
//            read where they are, in whichever order their rows run (K-major or MN-major descriptors).
//
// Two SMs work on a tile of 256 rows x 256 columns (cta_group::2): each loads its 128 rows of A and half of B's 256, one thread of the
// first issues the products of both, and each holds its own rows' accumulators.  A step of 64 then costs an SM 32 KB from L2 and 512
// clocks of products; a CTA alone (128 x 256) needs 48 KB for the same time, more than L2 gives every SM at once.  Eight warps of each CTA
// read accumulators (two per 32 rows, 128 columns each), one loads.  The accumulator is double-buffered in tensor memory, so an epilogue
// runs under the next tile's products; a running pair takes over the tiles of pairs that have not started (cluster launch control), so
// long and short tiles balance without a counter in memory.  Up to 128 rows a CTA works alone (PAIR = false, 128 x 256): the pair's second
// half of A would be empty (13 rows x 32,000 x 2,048: a pass without gradients 54 us in pairs, 50 alone, the gradients' products 71 and 67).
// 4,096 rows: without gradients 334 us in pairs, 364 alone; the products 674 and 736.  Loads and products are issued by one lane of a warp that
// stays together, products from descriptors in two words: with lanes that ran by themselves these took 357 and 748 us in pairs.
#include "sg_native.h"
#include "tc_half.cuh"
#include "per_device.h"
#include "launch_early.cuh"
#include "linear_ce.h"
#include <cfloat>

namespace sg {
namespace {
using namespace tc;

constexpr int BN = 256, BK = 64, THREADS = 352;
constexpr uint32_t A_BYTES = 128 * BK * 2, OUT_BYTES = 32 * 128;
// a tile (of the pair, or of a CTA alone) and what one CTA holds of its operands
template <bool PAIR> struct Shape {
    static constexpr int CTAS = PAIR ? 2 : 1, BM = 128 * CTAS, B_ROWS = BN / CTAS, STAGES = PAIR ? 6 : 4;
    static constexpr uint32_t B_BYTES = B_ROWS * BK * 2, STAGE = A_BYTES + B_BYTES;
};
constexpr int GROUP_M = 16;                                               // tile rows that sweep over the columns together

struct alignas(16) LItem {
    int m0, n0, kb0, nkb, kind, split, unused[2];                         // kind: 0 end of the work, 1 logits or dx, 2 dw
};
// full, acc_empty, item_empty and clc are used in the first CTA of the pair
struct LBars {
    uint64_t full[6], empty[6], acc_full[2], acc_empty[2], item_full[2], item_empty[2], clc;
    uint4 answer;
    LItem item[2];
    uint32_t tmem_slot;
};

struct LArgs {
    // LOGITS
    const int64_t* target;
    float2* stats;
    float* z_target;
    int store_u;
    // GRADS
    const float *dw_prev, *row_scale;
    const float *gout, *inv;
    int splits, f32_w;                                                    // dx is left as fp32 sums of its splits; f32_w: dw is fp32
    int items_x;                                                          // items below this are dx
    const int* count;                                                     // rows there are: *count - first, `rows` at most
    int first, rows, V, D;
    int* err;
};

// tile of the logits: m fastest inside a group of GROUP_M tile rows, so that w is streamed once per group
__device__ __forceinline__ void logits_tile(int i, int tm, int tn, int& m, int& n) {
    const int per = GROUP_M * tn, first = (i / per) * GROUP_M, g = tm - first < GROUP_M ? tm - first : GROUP_M, r = i % per;
    m = first + r % g;
    n = r / g;
}

__device__ __forceinline__ uint32_t cta_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
// the address of a shared variable of CTA `rank` of the cluster
__device__ __forceinline__ uint32_t in_cta(const void* p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
    return r;
}
// Arrivals at barriers of the other CTA carry no data through generic memory (operands and accumulators are ordered by the asynchronous
// units' own completions), so they are plain arrivals: cluster-scope releases and acquires cost each waiting warp a fence.
__device__ __forceinline__ void cluster_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void cluster_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// 16 bytes into a CTA's shared memory, counted by a barrier there
__device__ __forceinline__ void cluster_store(uint32_t addr, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// a load whose arrival is counted by a barrier of the (pair's first) CTA
template <bool PAIR> __device__ __forceinline__ void tile_load(void* dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    if constexpr (PAIR)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tile_mma(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\tsetp.ne.b32 p, %6, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n\t}"
                     ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
    else tc_mma_ss(d, a_lo, a_hi, b_lo, b_hi, idesc, accumulate);
}
// arrives at the barrier (of both CTAs) when the products issued so far are done
template <bool PAIR> __device__ __forceinline__ void tile_commit(uint64_t* bar) {
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else tc_commit(bar);
}

template <typename T, bool GRADS, bool PAIR>
__global__ void __launch_bounds__(THREADS, 1) lce_sm100_kernel(const __grid_constant__ CUtensorMap map_a1, const __grid_constant__ CUtensorMap map_b1,
                                                               const __grid_constant__ CUtensorMap map_c1, const __grid_constant__ CUtensorMap map_a2,
                                                               const __grid_constant__ CUtensorMap map_b2, const __grid_constant__ CUtensorMap map_c2,
                                                               const __grid_constant__ LArgs a) {
    using S = Shape<PAIR>;
    constexpr int BM = S::BM, STAGES = S::STAGES;
    constexpr uint32_t STAGE = S::STAGE;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    // the same offset in both CTAs: the dynamic part starts at the same address in every CTA of a kernel
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* s_out = smem + STAGES * STAGE;                               // [8 warps][OUT_BYTES]
    LBars* b = reinterpret_cast<LBars*>(s_out + 8 * OUT_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cta_rank() : 0u;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(&b->full[s], 1); mbar_init(&b->empty[s], 1); }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b->acc_full[i], 1); mbar_init(&b->acc_empty[i], 8 * S::CTAS);
            mbar_init(&b->item_full[i], 1); mbar_init(&b->item_empty[i], 9 * S::CTAS + 1);     // per CTA a loading and eight reading warps, and the issuing one
        }
        mbar_init(&b->clc, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&b->tmem_slot)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&b->tmem_slot)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();
    tc_fence_after();
    const uint32_t tmem = b->tmem_slot;
    after_previous();
    const int live = min(max(*a.count - a.first, 0), a.rows);       // rows of this piece
    // the item that every warp of both CTAs works on next
    auto take = [&](uint32_t n, LItem& w) {
        const uint32_t s = n & 1;
        if (!mbar_wait(&b->item_full[s], (n >> 1) & 1)) return false;
        w = b->item[s];
        return true;
    };
    auto arrive_first = [&](uint64_t* bar) { if (rank == 0) mbar_arrive(bar); else cluster_arrive(in_cta(bar, 0)); };
    auto release = [&](uint32_t n) { arrive_first(&b->item_empty[n & 1]); };

    if (warp == 10) {
        // the scheduler, one thread of the first CTA: writes the items of both
        if (rank == 0 && lane == 0) {
            int i = (int)blockIdx.x / S::CTAS;
            uint32_t n_item = 0, n_clc = 0;
            bool more = true;
            while (true) {
                LItem w{};
                bool empty = false;                                       // a tile past the last row: nothing to do
                if (more) {
                    mbar_expect_tx(&b->clc, 16);
                    clc_ask(&b->answer, &b->clc);
                    w.kind = 1;
                    if constexpr (!GRADS) {
                        int m, n;
                        logits_tile(i, (a.rows + BM - 1) / BM, (a.V + BN - 1) / BN, m, n);
                        w.m0 = m * BM; w.n0 = n * BN; w.nkb = (a.D + BK - 1) / BK;
                        empty = w.m0 >= live;
                    } else {
                        const int tn = (a.D + BN - 1) / BN;
                        if (i < a.items_x) {
                            const int tm = (a.rows + BM - 1) / BM, kb = (a.V + BK - 1) / BK, per = (kb + a.splits - 1) / a.splits;
                            w.split = i / (tm * tn);
                            const int r = i % (tm * tn);
                            w.m0 = r % tm * BM; w.n0 = r / tm * BN;
                            w.kb0 = w.split * per;
                            w.nkb = kb - w.kb0 < per ? kb - w.kb0 : per;
                            if (w.nkb < 0) w.nkb = 0;                     // a split past the end: all zeros
                            empty = w.m0 >= live;
                        } else {
                            const int r = i - a.items_x;
                            w.kind = 2;
                            w.m0 = r / tn * BM; w.n0 = r % tn * BN; w.nkb = (live + BK - 1) / BK;
                        }
                    }
                }
                if (!empty) {
                    const uint32_t s = n_item & 1;
                    if (n_item >= 2 && !mbar_wait(&b->item_empty[s], ((n_item >> 1) & 1) ^ 1)) { atomicExch(a.err, 101); break; }
                    ++n_item;
                    if constexpr (PAIR) {
                        for (uint32_t r = 0; r < 2; ++r) {
                            const uint32_t bar = in_cta(&b->item_full[s], r), to = in_cta(&b->item[s], r);
                            cluster_expect(bar, 32);
                            cluster_store(to, w.m0, w.n0, w.kb0, w.nkb, bar);
                            cluster_store(to + 16, w.kind, w.split, 0, 0, bar);
                        }
                    } else {
                        b->item[s] = w;
                        mbar_arrive(&b->item_full[s]);
                    }
                }
                if (!more) break;
                if (!mbar_wait(&b->clc, n_clc & 1)) { atomicExch(a.err, 103); break; }
                ++n_clc;
                more = clc_answer(&b->answer, i);
                i /= S::CTAS;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
        }
    } else if (warp == 8) {
        uint32_t n_item = 0, it = 0;
        bool ok = true;
        while (ok) {
            LItem w;
            if (!__all_sync(0xffffffffu, take(n_item, w))) { if (lane == 0) atomicExch(a.err, 100); break; }
            __syncwarp();
            if (lane == 0) release(n_item);
            ++n_item;
            if (w.kind == 0) break;
            const int m0 = w.m0 + 128 * (int)rank, n0 = w.n0 + S::B_ROWS * (int)rank;       // this CTA's rows of A, of B
            auto steps = [&](auto load) {
                for (int k = 0; k < w.nkb; ++k, ++it) {                   // what lies past the end of an operand is filled with zeros
                    const uint32_t st = it % STAGES;
                    if (it >= STAGES && !warp_wait(&b->empty[st], ((it / STAGES) & 1) ^ 1)) { if (lane == 0) atomicExch(a.err, 102); ok = false; break; }
                    if (elect_one()) {
                        const uint32_t bar = in_cta(&b->full[st], 0);
                        if (rank == 0) mbar_expect_tx(&b->full[st], S::CTAS * STAGE);       // what both CTAs load
                        load(smem + st * STAGE, (w.kb0 + k) * BK, bar);
                    }
                    __syncwarp();
                }
            };
            if constexpr (!GRADS) {
                steps([&](uint8_t* dst, int kc, uint32_t bar) {
                    tile_load<PAIR>(dst, &map_a1, kc, m0, bar);
                    tile_load<PAIR>(dst + A_BYTES, &map_b1, kc, n0, bar);
                });
            } else if (w.kind == 1) {
                steps([&](uint8_t* dst, int kc, uint32_t bar) {
                    tile_load<PAIR>(dst, &map_a1, kc, m0, bar);
#pragma unroll
                    for (int c = 0; c < S::B_ROWS / 64; ++c) tile_load<PAIR>(dst + A_BYTES + c * (BK * 128), &map_b1, n0 + 64 * c, kc, bar);
                });
            } else {
                steps([&](uint8_t* dst, int kc, uint32_t bar) {
                    tile_load<PAIR>(dst, &map_a2, m0, kc, bar);
                    tile_load<PAIR>(dst + BK * 128, &map_a2, m0 + 64, kc, bar);
#pragma unroll
                    for (int c = 0; c < S::B_ROWS / 64; ++c) tile_load<PAIR>(dst + A_BYTES + c * (BK * 128), &map_b2, n0 + 64 * c, kc, bar);
                });
            }
        }
    } else if (warp == 9) {
        if (rank == 0) {
            uint32_t n_item = 0, it = 0;
            bool ok = true;
            const uint32_t ring = smem_u32(smem);
            while (ok) {
                LItem w;
                if (!__all_sync(0xffffffffu, take(n_item, w))) { if (lane == 0) atomicExch(a.err, 104); break; }
                __syncwarp();
                if (lane == 0) release(n_item);
                if (w.kind == 0) break;
                const uint32_t s = n_item & 1;
                if (n_item >= 2 && !warp_wait(&b->acc_empty[s], ((n_item >> 1) & 1) ^ 1)) { if (lane == 0) atomicExch(a.err, 105); break; }
                ++n_item;
                tc_fence_after();
                const bool a_mn = GRADS && w.kind == 2, b_mn = GRADS;
                const uint32_t idesc = idesc_f16(Half2<T>::FMT, BM, BN, b_mn) | ((uint32_t)a_mn << 15), d = tmem + s * BN;
                // descriptors of the ring's first stage; a stage is STAGE >> 4 further
                const Desc da = desc_of(a_mn ? make_desc_sw128_mn(ring, BK * 128, 1024) : make_desc_sw128(ring));
                const Desc db = desc_of(b_mn ? make_desc_sw128_mn(ring + A_BYTES, BK * 128, 1024) : make_desc_sw128(ring + A_BYTES));
                const uint32_t a_step = a_mn ? 128 : 2;
                for (int k = 0; k < w.nkb; ++k, ++it) {
                    const uint32_t st = it % STAGES;
                    if (!warp_wait(&b->full[st], (it / STAGES) & 1)) { if (lane == 0) atomicExch(a.err, 106); ok = false; break; }
                    tc_fence_after();
                    const uint32_t al = da.lo + st * (STAGE >> 4), bl = db.lo + st * (STAGE >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int k4 = 0; k4 < BK / 16; ++k4)
                            tile_mma<PAIR>(d, al + a_step * k4, da.hi, bl + (b_mn ? 128 : 2) * k4, db.hi, idesc, (k > 0 || k4 > 0) ? 1u : 0u);
                        tile_commit<PAIR>(&b->empty[st]);
                    }
                    __syncwarp();
                }
                if (elect_one()) tile_commit<PAIR>(&b->acc_full[s]);
                __syncwarp();
            }
        }
    } else if (warp < 8) {
        const int q = warp & 3, half = warp >> 2;
        const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
        uint8_t* stg = s_out + warp * OUT_BYTES;
        const float f = GRADS && a.gout ? a.gout[0] * a.inv[0] / LceUnit<T>::value : 1.f;
        uint32_t n_item = 0;
        // a box of 128 bytes x 32 rows leaves through shared memory (16-byte piece k of row r at piece k ^ (r & 7))
        auto store_box = [&](const CUtensorMap* map, int col, int row) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                tma_store_2d(map, stg, col, row);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
            __syncwarp();
        };
        auto put = [&](int piece, uint4 v) { *reinterpret_cast<uint4*>(stg + lane * 128 + ((piece ^ (lane & 7)) << 4)) = v; };
        while (true) {
            const uint32_t s = n_item & 1;
            LItem w;
            if (!__all_sync(0xffffffffu, take(n_item, w))) { atomicExch(a.err, 107); break; }
            __syncwarp();
            if (lane == 0) release(n_item);
            if (w.kind == 0) break;
            if (!__all_sync(0xffffffffu, mbar_wait(&b->acc_full[s], (n_item >> 1) & 1))) { atomicExch(a.err, 108); break; }
            ++n_item;
            tc_fence_after();
            w.m0 += 128 * (int)rank;                                      // this CTA's rows
            const uint32_t acc = tmem + s * BN + half * 128 + lane_addr;
            const int row = w.m0 + q * 32 + lane, n0 = w.n0 + half * 128;
            if constexpr (!GRADS) {
                uint32_t r[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tc_ld32(acc + c * 32, r[c]);
                tc_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_first(&b->acc_empty[s]);             // everything is in registers
                if (n0 < a.V) {
                    const int64_t t = row < live ? a.target[row] : -1;
                    const int tc = t >= n0 && t < n0 + 128 && t < a.V ? (int)(t - n0) : -1;        // the target's column, if it is here
                    if (n0 + 128 > a.V) {                                 // columns past the vocabulary
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int i = 0; i < 32; ++i) if (n0 + c * 32 + i >= a.V) r[c][i] = __float_as_uint(-INFINITY);
                    }
                    float mx = -1e30f;                                    // finite, so that a row of -inf gives zeros, not NaN
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; i += 2) mx = max3f(mx, __uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1]));
                    // the reference: the maximum (fp16), or a multiple of 64 powers of two that most tiles share (bf16)
                    float ref = mx * LOG2E;
                    if constexpr (Half2<T>::FMT == 1) ref = fabsf(ref) <= 64.f ? 0.f : 64.f * rintf(ref * (1.f / 64.f));
                    const float mc = -ref;
                    float sum0 = 0.f, sum1 = 0.f;
                    auto chunk = [&](uint32_t (&rc)[32], int c) {         // 32 columns
                        uint32_t zt = 0u;
                        float et = 0.f;
                        const bool here = (tc >> 5) == c;
                        if (__any_sync(0xffffffffu, here)) {              // one tile in a few per row block: the target's logit, kept out of the sum
#pragma unroll
                            for (int i = 0; i < 32; ++i)                  // written as a selection in C++ this becomes an index into r[], which then lives in memory
                                asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, %2;\n\t@p mov.b32 %0, %3;\n\t}" : "+r"(zt) : "r"(tc & 31), "r"(i), "r"(rc[i]));
                            if (here) a.z_target[row] = __uint_as_float(zt);
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            float e0, e1;
                            fma2(__uint_as_float(rc[i]), __uint_as_float(rc[i + 1]), LOG2E, LOG2E, mc, mc, e0, e1);
                            rc[i] = __float_as_uint(ex2f(e0)); rc[i + 1] = __float_as_uint(ex2f(e1));
                        }
                        if (__any_sync(0xffffffffu, here)) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) if (!here || (tc & 31) != i) et += __uint_as_float(rc[i]);
                            sum0 += et;
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i += 2) { sum0 += __uint_as_float(rc[i]); sum1 += __uint_as_float(rc[i + 1]); }
                        }
                        if (a.store_u) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                uint32_t pk[4];
#pragma unroll
                                for (int v = 0; v < 4; ++v)
                                    pk[v] = Half2<T>::pack(__uint_as_float(rc[8 * k + 2 * v]) * LceUnit<T>::value, __uint_as_float(rc[8 * k + 2 * v + 1]) * LceUnit<T>::value);
                                put((c & 1) * 4 + k, make_uint4(pk[0], pk[1], pk[2], pk[3]));
                            }
                            if ((c & 1) && n0 + (c - 1) * 32 < a.V && w.m0 + q * 32 < a.rows) store_box(&map_c1, n0 + (c - 1) * 32, w.m0 + q * 32);
                        }
                    };
                    chunk(r[0], 0); chunk(r[1], 1); chunk(r[2], 2); chunk(r[3], 3);
                    if (row < live) a.stats[(int64_t)row * ((a.V + LCE_COLUMNS - 1) / LCE_COLUMNS) + n0 / LCE_COLUMNS] = make_float2(ref, sum0 + sum1);
                }
            } else {
                const bool is_x = w.kind == 1, f32 = is_x || a.f32_w;
                const CUtensorMap* map = is_x ? &map_c1 : &map_c2;
                const int tm = (a.rows + BM - 1) / BM, mrow = w.m0 + q * 32 + (is_x ? w.split * tm * BM : 0);      // partial sums of dx: [split][rows]
                const float fr = is_x && a.row_scale && row < live ? f * a.row_scale[row] : f;
                const float* prev = !is_x && a.dw_prev && row < a.V ? a.dw_prev + (int64_t)row * a.D : nullptr;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const int col = n0 + c * 32;
                    if (col >= a.D || w.m0 + q * 32 >= (is_x ? a.rows : a.V)) break;
                    uint32_t r[32];
                    if (w.nkb > 0) { tc_ld32(acc + c * 32, r); tc_wait_ld(); }
                    else
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[i] = 0u;
                    if (prev) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            if (col + i < a.D) {                          // D is a multiple of 8
                                const float4 p = *reinterpret_cast<const float4*>(prev + col + i);
                                r[i] = __float_as_uint(__uint_as_float(r[i]) + p.x); r[i + 1] = __float_as_uint(__uint_as_float(r[i + 1]) + p.y);
                                r[i + 2] = __float_as_uint(__uint_as_float(r[i + 2]) + p.z); r[i + 3] = __float_as_uint(__uint_as_float(r[i + 3]) + p.w);
                            }
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * fr);
                    if (f32) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) put(k, make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]));
                        store_box(map, col, mrow);
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t pk[4];
#pragma unroll
                            for (int v = 0; v < 4; ++v) pk[v] = Half2<T>::pack(__uint_as_float(r[8 * k + 2 * v]), __uint_as_float(r[8 * k + 2 * v + 1]));
                            put((c & 1) * 4 + k, make_uint4(pk[0], pk[1], pk[2], pk[3]));
                        }
                        if ((c & 1) || col + 32 >= a.D) store_box(map, col - (c & 1) * 32, mrow);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_first(&b->acc_empty[s]);
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    __syncwarp();
    if (PAIR) cluster_sync();                                             // neither CTA leaves while the other may still signal it
    if (warp == 9) {
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <typename T, bool GRADS, bool PAIR>
int launch(unsigned items, const CUtensorMap& a1, const CUtensorMap& b1, const CUtensorMap& c1, const CUtensorMap& a2, const CUtensorMap& b2, const CUtensorMap& c2,
           const LArgs& k, cudaStream_t st) {
    using S = Shape<PAIR>;
    constexpr size_t smem = S::STAGES * S::STAGE + 8 * OUT_BYTES + sizeof(LBars) + 1024;
    static std::atomic<uint64_t> done{0};
    if (!once_per_device(done, current_device(), [&] {
            return cudaFuncSetAttribute(lce_sm100_kernel<T, GRADS, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess;
        })) return 11;
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = S::CTAS; at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(items * S::CTAS); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st; cfg.attrs = at; cfg.numAttrs = 2;
    count_launch();
    return cudaLaunchKernelEx(&cfg, lce_sm100_kernel<T, GRADS, PAIR>, a1, b1, c1, a2, b2, c2, k) == cudaSuccess ? 0 : 12;
}

template <typename T, bool PAIR> int logits(const LceArgs& a, int* err, cudaStream_t st) {
    using S = Shape<PAIR>;
    CUtensorMap mx, mw, mu;
    if (!make_map(&mx, a.x, a.rows, a.D, a.ldx, 128, BK, true) || !make_map(&mw, a.w, a.V, a.D, a.ldw, S::B_ROWS, BK, true)) return 10;
    if (a.u && !make_map(&mu, a.u, a.rows, a.ldu, a.ldu, 32, 64, true)) return 10;
    LArgs k{};
    k.target = a.target; k.stats = a.stats; k.z_target = a.z_target; k.count = a.count; k.first = a.first;
    k.store_u = a.u != nullptr; k.rows = a.rows; k.V = a.V; k.D = a.D; k.err = err;
    const CUtensorMap& c = a.u ? mu : mx;                                 // without u no map of it is used
    return launch<T, false, PAIR>((unsigned)((a.rows + S::BM - 1) / S::BM) * (unsigned)((a.V + BN - 1) / BN), mx, mw, c, mx, mw, c, k, st);
}

bool in_pairs(int rows) { return rows > 128; }

// Pieces that a tile of dx is cut into along the vocabulary: so many that one takes about half of what a CTA (or pair) does on average
// (769 x 50,021 x 1,000: all of it 177 us, a half 138, a quarter 142, an eighth 153; 1,536 x 50,048 x 1,024: 304, 210, 216, 230).  A tile costs
// its 64-deep steps and about six more for its epilogue.
int dx_splits(int rows, int V, int D, bool with_dw) {
    const int64_t bm = in_pairs(rows) ? 256 : 128, teams = device_sms() / (bm / 128);
    const int64_t tn = (D + BN - 1) / BN, tx = (rows + bm - 1) / bm * tn, kx = (V + BK - 1) / BK, tw = with_dw ? (V + bm - 1) / bm * tn : 0, kw = (rows + BK - 1) / BK;
    const int64_t share = (tx * (kx + 6) + tw * (kw + 6)) / (teams > 0 ? teams : 1) + 1;
    int64_t s = (2 * kx + share / 2) / share;
    if (s > kx / 8) s = kx / 8;                                           // eight steps at least, or the partial sums cost more than the products
    if (s > 64) s = 64;
    return s < 1 ? 1 : (int)s;
}

template <typename T, bool PAIR> int grads(const LceArgs& a, const LceGrads& g, int* err, cudaStream_t st) {
    using S = Shape<PAIR>;
    CUtensorMap ua, wb, cx, um, xb, cw;
    const int tm = (a.rows + S::BM - 1) / S::BM, tn = (a.D + BN - 1) / BN;
    if (!make_map(&ua, a.u, a.rows, a.V, a.ldu, 128, BK, true) || !make_map(&um, a.u, a.rows, a.V, a.ldu, BK, 64, true) ||
        !make_map(&wb, a.w, a.V, a.D, a.ldw, BK, 64, true) || !make_map(&xb, a.x, a.rows, a.D, a.ldx, BK, 64, true)) return 10;
    cx = ua; cw = ua;
    if (g.dx_part && !make_map(&cx, g.dx_part, g.parts * g.row_pitch, a.D, a.D, 32, 32, false)) return 10;
    if (g.dw && !make_map(&cw, g.dw, a.V, a.D, a.D, 32, g.f32_dw ? 32 : 64, !g.f32_dw)) return 10;
    LArgs k{};
    k.dw_prev = g.dw_prev; k.row_scale = a.row_scale; k.splits = g.parts; k.f32_w = g.f32_dw; k.rows = a.rows; k.V = a.V; k.D = a.D; k.err = err; k.count = a.count; k.first = a.first;
    k.gout = g.gout; k.inv = g.inv_count;
    k.items_x = g.dx_part ? g.parts * tm * tn : 0;
    const unsigned items = (unsigned)k.items_x + (g.dw ? (unsigned)((a.V + S::BM - 1) / S::BM) * (unsigned)tn : 0u);
    return launch<T, true, PAIR>(items, ua, wb, cx, um, xb, cw, k, st);
}

}  // namespace

bool lce_sm100_takes(int dtype, const LceArgs& a) {
    const auto ok = [](const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld > 0 && ld % 8 == 0; };
    return dtype != F32 && a.D % 8 == 0 && ok(a.x, a.ldx) && ok(a.w, a.ldw);
}
int lce_sm100_dx_parts(int rows, int V, int D, bool with_dw, int64_t* row_pitch) {
    const int bm = in_pairs(rows) ? 256 : 128;
    *row_pitch = (int64_t)((rows + bm - 1) / bm) * bm;
    return dx_splits(rows, V, D, with_dw);
}
int lce_sm100_logits(int dtype, const LceArgs& a, int* err, cudaStream_t st) {
    if (in_pairs(a.rows)) return dtype == BF16 ? logits<__nv_bfloat16, true>(a, err, st) : logits<__half, true>(a, err, st);
    return dtype == BF16 ? logits<__nv_bfloat16, false>(a, err, st) : logits<__half, false>(a, err, st);
}
int lce_sm100_grads(int dtype, const LceArgs& a, const LceGrads& g, int* err, cudaStream_t st) {
    if (in_pairs(a.rows)) return dtype == BF16 ? grads<__nv_bfloat16, true>(a, g, err, st) : grads<__half, true>(a, g, err, st);
    return dtype == BF16 ? grads<__nv_bfloat16, false>(a, g, err, st) : grads<__half, false>(a, g, err, st);
}

}  // namespace sg
