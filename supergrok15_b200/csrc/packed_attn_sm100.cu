// Attention over packed sequences with grouped heads on the 5th-generation tensor cores (tcgen05 / TMEM / TMA), sm_100a only.  16-bit
// operands (bf16, fp16), head sizes that are multiples of 8 up to 128, fp32 scores, sums and accumulators.
//
//   o_i = sum_j p_ij v_j,  p_ij = softmax_j(scale q_i . k_j),  j over the rows of i's sequence (causal: j <= i)
//
// q, k, v are read where they are ([rows, heads, hd] views with any row and head pitch that TMA takes): a map of three dimensions
// (hd, heads, rows), boxes of 64 columns x 128 rows of one head, columns past hd filled with zeros, so a head of 80 runs as two boxes.
//
// Work is handed out by the hardware: the grid has one CTA per item, one CTA fits an SM, and a running CTA takes over the items of CTAs
// that have not started (cluster launch control).  Lengths are known on the device only, so no static split balances them; the barriers,
// the tensor memory and the loads of the next item carry over from item to item without a counter in memory to be zeroed.
//
// Rows behind a sequence's end belong to the next sequence or to nobody.  As keys they are masked in the scores by selection, and as rows of
// an operand that is multiplied by a zero probability they are zeroed in shared memory, because zero times NaN or infinity is NaN.
#include "sg_native.h"
#include "tc_half.cuh"
#include "per_device.h"
#include "launch_early.cuh"
#include "packed_attn.h"
#include <cfloat>

namespace sg {
namespace {
using namespace tc;

constexpr uint32_t HALF_TILE = 128 * 128;                                // [128 rows x 64 elements of 2 bytes] = 16 KB
constexpr int STAGE_PITCH = 80;                                          // 64 bytes of a row and a pad: conflict-free 16-byte accesses
template <uint32_t V> struct Const { static constexpr uint32_t v = V; };
// descriptor step of the kk-th 16 columns of a K-major tile: 32 bytes inside a box of 64 columns, then the next box
__device__ __forceinline__ constexpr uint32_t KSTEP(int kk) { return (uint32_t)(kk / 4) * (HALF_TILE >> 4) + 2u * (kk % 4); }

// What the scheduling warp tells the others about an item.
struct Item {
    int lo, hi, row0, head, kind;                                        // kind: 0 end of the work, 1 rows of a sequence, 2 rows of none
};

// rows [first, 128) of a tile (HALVES boxes of 64 columns) become zero; called by a whole warp between the arrival of the tile and its use
template <int HALVES> __device__ __forceinline__ void zero_rows(uint8_t* tile, int first) {
    const int lane = (int)(threadIdx.x & 31);
    const int n16 = (128 - first) * 8;                                    // a row of a box is 128 consecutive bytes, however swizzled
#pragma unroll
    for (int hf = 0; hf < HALVES; ++hf) {
        uint4* p = reinterpret_cast<uint4*>(tile + hf * HALF_TILE + first * 128);
        for (int i = lane; i < n16; i += 32) p[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
}

// ---------------------------------------------------------------------------------------------------------------------------
// Forward.  An item is 256 query rows of one head: two tiles A and B of 128 rows that share every key tile, each with its own score
// buffer and accumulator in tensor memory and its own group of 128 softmax threads (one row per thread).  The tensor cores alternate
//     O_A += P_A(j) V_j,  S_A(j+1) = Q_A K_{j+1}^T,  O_B += P_B(j) V_j,  S_B(j+1)
// so a group's softmax runs under the other tile's products.  P overwrites S in place (the first 64 columns of its buffer) and is read
// from tensor memory; O stays there, and a row is rescaled only when its maximum has grown by more than 2^8.  P is at most 2^8 then, and in fp16
// is multiplied by 2^7 besides, so that it has all its bits down to 2^-21 of the largest; the sum carries the factor too.
//   warps 0-3, 4-7   softmax and epilogue of tile A, of tile B
//   warp 8           takes items, loads Q and the rings of two K and two V tiles      warp 9   issues the products
// A row of 128 scores is held in registers: the softmax warpgroups take 208 per thread and leave 88 to the third (256 x 208 + 128 x 88 =
// 384 x 168, the registers of the launch).
// Bound by the chain S -> softmax -> P V of the two tiles: 8,192 rows, 16 heads of 128, causal, bf16: 276 us, tensor pipe 51 % busy, 34 % of
// the issue slots, 0.19 GB of DRAM traffic.  Key halves of 64 (349 us against 291 at that step), twice the softmax warps (398), P handed over
// in halves (295 against 278) and exponentials by polynomial (295 against 279) were all slower.
constexpr int FWD_THREADS = 384;
constexpr int REGS_SOFTMAX = 208, REGS_OTHERS = 88;
struct FwdBars {
    uint64_t item_full[2], item_empty[2], clc, q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], v_tail;
    uint64_t s_full[2], p_full[2], o_done[2], o_empty[2];
    uint4 answer;
    Item item[2];
    uint32_t tmem_slot;
};

struct FwdArgs {
    void *out, *out_lo;
    float* lse;
    PackedSeqs seqs;
    int heads, group, hd, causal, slots;
    float scale;
    int* err;
};

template <typename T, int HD>
__global__ void __launch_bounds__(FWD_THREADS, 1) packed_fwd_sm100_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                          const __grid_constant__ CUtensorMap map_v, const __grid_constant__ FwdArgs a) {
    constexpr int HALVES = HD / 64;
    constexpr bool FP16 = Half2<T>::FMT == 0;
    constexpr uint32_t TILE = HALVES * HALF_TILE;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sQ = smem;                                                   // [2 tiles]
    uint8_t* sK = sQ + 2 * TILE;                                          // [2]
    uint8_t* sV = sK + 2 * TILE;                                          // [2]
    uint8_t* s_stage = sV + 2 * TILE;                                     // [8 warps][32 rows][STAGE_PITCH]
    FwdBars* b = reinterpret_cast<FwdBars*>(s_stage + 8 * 32 * STAGE_PITCH);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b->item_full[i], 1); mbar_init(&b->item_empty[i], 9);
            mbar_init(&b->k_full[i], 1); mbar_init(&b->k_empty[i], 1); mbar_init(&b->v_full[i], 1); mbar_init(&b->v_empty[i], 1);
            mbar_init(&b->s_full[i], 1); mbar_init(&b->p_full[i], 4); mbar_init(&b->o_done[i], 1); mbar_init(&b->o_empty[i], 4);
        }
        mbar_init(&b->clc, 1); mbar_init(&b->q_full, 1); mbar_init(&b->q_empty, 1); mbar_init(&b->v_tail, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&b->tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // all 512 columns are allocated, so they start at 0: a constant keeps address arithmetic out of the loops.  Tile t: S / P at 128 t, O at 256 + 128 t
    constexpr uint32_t tmem = 0;

    // key tiles that tile t of an item meets
    auto blocks = [&](const Item& w, int t) {
        const int r = w.row0 + 128 * t;
        if (r >= w.hi) return 0;
        const int last = a.causal && r + 128 < w.hi ? r + 128 : w.hi;
        return (last - w.lo + 127) / 128;
    };

    if (warp < 8) {
        reg_inc<REGS_SOFTMAX>();
        const int t = warp >> 2, q = warp & 3, row = q * 32 + lane;  // tile of the group, TMEM lane quarter of the warp, row of the thread
        const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
        const uint32_t ts = tmem + t * 128 + lane_addr, to = tmem + 256 + t * 128 + lane_addr;
        const float c2 = a.scale * LOG2E;
        uint8_t* stg = s_stage + warp * 32 * STAGE_PITCH;
        uint32_t n_item = 0, n_s = 0, n_o = 0;
        bool ok = true;
        while (ok) {
            const uint32_t si = n_item & 1;
            if (!warp_wait(&b->item_full[si], (n_item >> 1) & 1)) { atomicExch(a.err, 74); break; }
            const Item w = b->item[si];
            __syncwarp();
            if (lane == 0) mbar_arrive(&b->item_empty[si]);
            ++n_item;
            if (w.kind == 0) break;
            const int row0 = w.row0 + 128 * t + q * 32;                   // first row of this warp
            const int n = w.kind == 1 ? blocks(w, t) : 0;
            float m_ref = -FLT_MAX, l = 0.f;
            for (int j = 0; j < n && ok; ++j, ++n_s) {
                if (!warp_wait(&b->s_full[t], n_s & 1)) { atomicExch(a.err, 75); ok = false; break; }
                tc_fence_after();
                uint32_t r[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tc_ld32(ts + c * 32, r[c]);
                tc_wait_ld();
                // columns that this row sees: up to the diagonal in the last tile of a causal row block (it holds the sequence's end too),
                // up to the sequence's end in the last tile otherwise.  Masked scores are -inf: no score is smaller.
                if (j + 1 == n) {
                    const int see = a.causal ? row + 1 : w.hi - (w.lo + j * 128);
                    if (a.causal || see < 128) {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
#pragma unroll
                            for (int i = 0; i < 32; ++i) if (c * 32 + i >= see) r[c][i] = __float_as_uint(-INFINITY);
                    }
                }
                float top[4] = {-FLT_MAX, -FLT_MAX, -FLT_MAX, -FLT_MAX};  // finite, so that a tile of -inf scores gives zeros, not NaN; four chains
#pragma unroll
                for (int i = 0; i < 32; i += 2)
#pragma unroll
                    for (int c = 0; c < 4; ++c) top[c] = max3f(top[c], __uint_as_float(r[c][i]), __uint_as_float(r[c][i + 1]));
                const float mx = fmaxf(max3f(top[0], top[1], top[2]), top[3]);
                float alpha = 1.f;
                bool move = false;
                if (j == 0) m_ref = mx;
                else if ((mx - m_ref) * c2 > 8.f) { alpha = ex2f((m_ref - mx) * c2); m_ref = mx; move = true; }
                // S_j was issued behind P_{j-1} V_{j-1}: O is complete up to there
                if (j > 0 && __any_sync(0xffffffffu, move)) {
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        uint32_t u[32];
                        tc_ld32(to + c * 32, u);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * alpha);
                        tc_st32(to + c * 32, u);
                    }
                }
                const float mc = FP16 ? fmaf(-m_ref, c2, 7.f) : -m_ref * c2;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t pk[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int k0 = c * 64 + 2 * i;
                        float e0, e1;
                        fma2(__uint_as_float(r[k0 >> 5][k0 & 31]), __uint_as_float(r[(k0 + 1) >> 5][(k0 + 1) & 31]), c2, c2, mc, mc, e0, e1);
                        const float p0 = ex2f(e0), p1 = ex2f(e1);
                        sum[2 * (i & 1)] += p0; sum[2 * (i & 1) + 1] += p1;
                        pk[i] = Half2<T>::pack(p0, p1);
                    }
                    tc_st32(ts + c * 32, pk);
                }
                tc_wait_st();
                tc_fence_before();
                warp_arrive(&b->p_full[t]);
                l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
            }
            if (!ok) break;
            float inv = 0.f;
            if (n > 0) {
                ok = warp_wait(&b->o_done[t], n_o & 1);
                if (!ok) { atomicExch(a.err, 76); break; }
                ++n_o;
                tc_fence_after();
                inv = 1.f / l;
            }
            if (row0 < w.hi) {                                            // rows of no sequence: n = 0, zeros
                const int live = w.hi - row0;                             // rows of this warp that belong to the item
                const int64_t ld = (int64_t)a.heads * a.hd;
#pragma unroll 1
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t u[32];
                    if (n > 0) {
                        tc_ld32(to + c * 32, u);
                        tc_wait_ld();
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) u[i] = n > 0 ? __float_as_uint(__uint_as_float(u[i]) * inv) : 0u;
#pragma unroll
                    for (int pass = 0; pass < 2; ++pass) {                 // the rounded output, then what the rounding took
                        T* base = (T*)(pass ? a.out_lo : a.out);
                        if (base == nullptr) break;
                        base += (int64_t)row0 * ld + (int64_t)w.head * a.hd + c * 32;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t pk[4];
#pragma unroll
                            for (int v = 0; v < 4; ++v) {
                                const float x = __uint_as_float(u[8 * k + 2 * v]), y = __uint_as_float(u[8 * k + 2 * v + 1]);
                                pk[v] = Half2<T>::pack(x, y);
                                if (pass) { const float2 f = Half2<T>::unpack(pk[v]); pk[v] = Half2<T>::pack(x - f.x, y - f.y); }
                            }
                            *reinterpret_cast<uint4*>(stg + lane * STAGE_PITCH + k * 16) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                        }
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 4; ++k) {                      // four lanes store 64 consecutive bytes of a row
                            const int rr = k * 8 + (lane >> 2), piece = lane & 3;
                            if (rr < live && c * 32 + piece * 8 < a.hd)
                                *reinterpret_cast<uint4*>(base + rr * ld + piece * 8) = *reinterpret_cast<const uint4*>(stg + rr * STAGE_PITCH + piece * 16);
                        }
                        __syncwarp();
                    }
                }
                if (a.lse && lane < live) a.lse[(int64_t)w.head * a.seqs.total + row0 + lane] = n > 0 ? m_ref * a.scale + logf(FP16 ? l * 0x1p-7f : l) : 0.f;
            }
            if (n > 0) { tc_fence_before(); warp_arrive(&b->o_empty[t]); }
        }
    } else {
        reg_dec<REGS_OTHERS>();
        if (warp == 8) {
            int item = (int)blockIdx.x;
            uint32_t n_item = 0, n_clc = 0, n_q = 0, n_k = 0, n_tail = 0;
            bool ok = true, more = true;
            while (ok && more) {
                if (lane == 0) {
                    mbar_expect_tx(&b->clc, 16);
                    clc_ask(&b->answer, &b->clc);
                }
                const PackedTile t = packed_tile<256>(a.seqs, a.slots - 1 - item / a.heads);    // late tiles see most keys: they start first
                if (t.live) {
                    const Item w{t.lo, t.hi, t.row0, item % a.heads, t.pad ? 2 : 1};
                    const uint32_t s = n_item & 1;
                    if (n_item >= 2) ok = warp_wait(&b->item_empty[s], ((n_item >> 1) & 1) ^ 1);
                    if (!ok) { if (lane == 0) atomicExch(a.err, 61); break; }
                    if (lane == 0) { b->item[s] = w; mbar_arrive(&b->item_full[s]); }
                    ++n_item;
                    if (!t.pad) {
                        const int hk = w.head / a.group, live_b = t.row0 + 128 < t.hi ? 1 : 0;
                        int n = blocks(w, 0);
                        if (live_b) n = blocks(w, 1);
                        if (n_q > 0) ok = warp_wait(&b->q_empty, (n_q - 1) & 1);
                        if (!ok) { if (lane == 0) atomicExch(a.err, 62); break; }
                        ++n_q;
                        if (lane == 0) {
                            mbar_expect_tx(&b->q_full, (1 + live_b) * TILE);
                            for (int q = 0; q <= live_b; ++q)
                                for (int hf = 0; hf < HALVES; ++hf) tma_load_3d(sQ + q * TILE + hf * HALF_TILE, &map_q, hf * 64, w.head, t.row0 + q * 128, &b->q_full);
                        }
                        for (int j = 0; j < n && ok; ++j, ++n_k) {
                            const uint32_t r = n_k & 1, par = ((n_k >> 1) & 1) ^ 1;
                            const int row = t.lo + j * 128, have = t.hi - row;
                            if (n_k >= 2) ok = warp_wait(&b->k_empty[r], par);
                            if (!ok) { if (lane == 0) atomicExch(a.err, 63); break; }
                            if (lane == 0) {
                                mbar_expect_tx(&b->k_full[r], TILE);
                                for (int hf = 0; hf < HALVES; ++hf) tma_load_3d(sK + r * TILE + hf * HALF_TILE, &map_k, hf * 64, hk, row, &b->k_full[r]);
                            }
                            if (n_k >= 2) ok = warp_wait(&b->v_empty[r], par);
                            if (!ok) { if (lane == 0) atomicExch(a.err, 64); break; }
                            uint64_t* bar = have < 128 ? &b->v_tail : &b->v_full[r];
                            if (lane == 0) {
                                mbar_expect_tx(bar, TILE);
                                for (int hf = 0; hf < HALVES; ++hf) tma_load_3d(sV + r * TILE + hf * HALF_TILE, &map_v, hf * 64, hk, row, bar);
                            }
                            if (have < 128) {
                                ok = warp_wait(&b->v_tail, n_tail & 1);
                                if (!ok) { if (lane == 0) atomicExch(a.err, 65); break; }
                                ++n_tail;
                                zero_rows<HALVES>(sV + r * TILE, have);
                                if (lane == 0) mbar_arrive(&b->v_full[r]);
                            }
                        }
                    }
                }
                if (!warp_wait(&b->clc, n_clc & 1)) { if (lane == 0) atomicExch(a.err, 66); ok = false; break; }
                ++n_clc;
                more = clc_answer(&b->answer, item);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the answer has been read before the next one is written over it
                __syncwarp();
            }
            if (ok && (n_item < 2 || warp_wait(&b->item_empty[n_item & 1], ((n_item >> 1) & 1) ^ 1)) && lane == 0) {
                b->item[n_item & 1].kind = 0;
                mbar_arrive(&b->item_full[n_item & 1]);
            }
        } else if (warp == 9) {
            {
                const uint32_t idesc_qk = idesc_f16(Half2<T>::FMT, 128, 128, 0), idesc_pv = idesc_f16(Half2<T>::FMT, 128, (a.hd + 15) / 16 * 16, 1);
                const int ksteps = (a.hd + 15) / 16;
                const Desc dq = desc_of(make_desc_sw128(smem_u32(sQ))), dk = desc_of(make_desc_sw128(smem_u32(sK))),
                           dv = desc_of(make_desc_sw128_mn(smem_u32(sV), HALF_TILE, 1024));
                uint32_t n_item = 0, n_q = 0, n_k = 0, n_p[2] = {0, 0}, n_o[2] = {0, 0};
                bool ok = true;
                while (ok) {
                    const uint32_t si = n_item & 1;
                    if (!warp_wait(&b->item_full[si], (n_item >> 1) & 1)) { if (lane == 0) atomicExch(a.err, 67); break; }
                    const Item w = b->item[si];
                    warp_arrive(&b->item_empty[si]);
                    ++n_item;
                    if (w.kind == 0) break;
                    if (w.kind == 2) continue;
                    const int nA = blocks(w, 0), nB = blocks(w, 1), n = nB > 0 ? nB : nA, lastt = nB > 0 ? 1 : 0;
                    if (!warp_wait(&b->q_full, n_q & 1)) { if (lane == 0) atomicExch(a.err, 68); ok = false; break; }
                    ++n_q;
                    // a product of 128 rows by 128 keys, issued by one lane; the ring slot is a constant in each of the two copies
                auto qk = [&](int t, auto slot) {
                    const uint32_t qa = dq.lo + t * (TILE >> 4), kb = dk.lo + slot.v * (TILE >> 4);
                    if (ksteps == HD / 16) {
#pragma unroll
                        for (int kk = 0; kk < HD / 16; ++kk) tc_mma_ss(tmem + t * 128, qa + KSTEP(kk), dq.hi, kb + KSTEP(kk), dk.hi, idesc_qk, kk > 0 ? 1u : 0u);
                    } else
#pragma unroll 1
                        for (int kk = 0; kk < ksteps; ++kk) tc_mma_ss(tmem + t * 128, qa + KSTEP(kk), dq.hi, kb + KSTEP(kk), dk.hi, idesc_qk, kk > 0 ? 1u : 0u);
                };
                auto pv = [&](int t, auto slot, bool add) {
                    const uint32_t vb = dv.lo + slot.v * (TILE >> 4), o = tmem + 256 + t * 128, pa = tmem + t * 128;
#pragma unroll
                    for (int kk = 0; kk < 8; ++kk) tc_mma_ts(o, pa + kk * 8, vb + kk * (2048 >> 4), dv.hi, idesc_pv, (kk > 0 || add) ? 1u : 0u);
                };
                auto issue_qk = [&](int t, int j) {
                    const uint32_t r = (n_k + j) & 1;
                    if (elect_one()) {
                        if (t == 0) { if (r == 0) qk(0, Const<0>{}); else qk(0, Const<1>{}); }
                        else { if (r == 0) qk(1, Const<0>{}); else qk(1, Const<1>{}); }
                        if (t == lastt) { tc_commit(&b->k_empty[r]); if (j + 1 == n) tc_commit(&b->q_empty); }
                        tc_commit(&b->s_full[t]);
                    }
                    __syncwarp();
                };
                auto issue_pv = [&](int t, int j, int nt) {
                    const uint32_t r = (n_k + j) & 1;
                    if (elect_one()) {
                        if (t == 0) { if (r == 0) pv(0, Const<0>{}, j > 0); else pv(0, Const<1>{}, j > 0); }
                        else { if (r == 0) pv(1, Const<0>{}, j > 0); else pv(1, Const<1>{}, j > 0); }
                        if (t == lastt) tc_commit(&b->v_empty[r]);
                        if (j + 1 == nt) tc_commit(&b->o_done[t]);
                    }
                    __syncwarp();
                };
                if (!warp_wait(&b->k_full[n_k & 1], (n_k >> 1) & 1)) { if (lane == 0) atomicExch(a.err, 69); ok = false; break; }
                    tc_fence_after();
                    issue_qk(0, 0);
                    if (nB > 0) issue_qk(1, 0);
                    for (int j = 0; j < n && ok; ++j) {
                        const uint32_t g = n_k + j;
                        if (!warp_wait(&b->v_full[g & 1], (g >> 1) & 1)) { if (lane == 0) atomicExch(a.err, 70); ok = false; break; }
                        if (j + 1 < n && !warp_wait(&b->k_full[(g + 1) & 1], ((g + 1) >> 1) & 1)) { if (lane == 0) atomicExch(a.err, 71); ok = false; break; }
                        for (int t = 0; t < 2 && ok; ++t) {
                            const int nt = t == 0 ? nA : nB;
                            if (j >= nt) continue;
                            if (j == 0 && n_o[t] > 0 && !warp_wait(&b->o_empty[t], (n_o[t] - 1) & 1)) { if (lane == 0) atomicExch(a.err, 72); ok = false; break; }
                            if (!warp_wait(&b->p_full[t], n_p[t] & 1)) { if (lane == 0) atomicExch(a.err, 73); ok = false; break; }
                            ++n_p[t];
                            tc_fence_after();
                            issue_pv(t, j, nt);
                            if (j + 1 < nt) issue_qk(t, j + 1);
                        }
                    }
                    n_k += n;
                    ++n_o[0];
                    if (nB > 0) ++n_o[1];
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---------------------------------------------------------------------------------------------------------------------------
// Backward, without atomics: delta = rowsum(dO (O + rest)), then two kernels of one form, X = R0 T0^T and Y = R1 T1^T with R resident
// and T streamed:
//   KV = true:  an item is 128 keys of a key head (R = K, V); over the query tiles of all heads of its group (T = Q, dO)
//               X = S^T, Y = dP^T,  dV += P^T dO,  dK += dS^T Q
//   KV = false: an item is 128 queries of a head (R = Q, dO); over its key tiles (T = K, V)
//               X = S, Y = dP,  dQ += dS K
// with P = exp(scale S - lse), dS = P (dP - delta); the factor scale of dS is applied once at the end.  The second operand of every
// accumulating product is the tile that served as K-major operand of the first, read again through an MN-major descriptor.  Four groups of
// 128 threads share a tile, a thread has one row and 32 columns; P and dS go back to tensor memory as 16-bit A operands, each group's into
// columns that it alone has read.  The next tile's X is issued as soon as this tile's scores have been taken out, its Y as soon as dS is
// stored, so the tensor cores work on dV and X while the threads form dS, on dK and Y while they form the next P.
// Bound by the chain X -> P -> dS -> product of each tile, which the look-ahead hides in part, and by the rate at which one thread issues
// products (tc_half.cuh).  8,192 rows, 16 heads of 128, causal, bf16: dK/dV 505 us with the tensor pipe 57 % busy, dQ 407 us and 52 %,
// delta 19 us (bandwidth).
// The two kernels do not depend on each other: dQ's CTAs start as those of dK/dV leave their SMs, knowing that delta is complete because every
// CTA of dK/dV has seen that, and wait for the whole of dK/dV at their end, for what comes behind both (14 documents in 8,192 rows, 16 heads of 128,
// forward and backward: 409 -> 395 us).
// P and dS are rounded to 16 bits to be operands (half a step of each value); everything they come from and are added to is fp32.  bf16 has the
// exponents of fp32.  In fp16 a value below 2^-14 has fewer bits than that (8,192 flat keys and dO of 2^-10: dS near 2^-20, dq 0.8 % off), and one
// above 65,504 is infinite, so dS carries a power of two of its accumulator's row, which the epilogue takes back: a row of dK or dQ is a
// row of dS times Q or K.  |dS_ij| <= |dO_i| |v_j| + |delta_i| as P <= 1; the pass that forms delta leaves the norms and the largest of each 32 rows,
// and the threads of an item look for the largest of the rows that it meets while its predecessor ends.  The bound times the row's unit lies
// between 2^14 and 2^15, so dS keeps all its bits down to 2^-29 of the bound.  Rows with NaN or infinity do not count: what they meet is NaN anyhow.
// P as operand of dV carries 2^15, which the exponent takes up for nothing.  The 14 documents in fp16: backward 308 -> 336 us, 15 of it the pass that
// reads v for its norms, 8 the look-up in dK/dV and 2 in dQ.
constexpr int BWD_THREADS = 640;
constexpr int BWD_REGS = 104, BWD_REGS_OTHERS = 64;                       // 512 x 104 + 128 x 64 = 640 x 96, the registers of the launch
constexpr int BWD_PITCH = 48;                                             // 32 bytes of a row and a pad
struct BwdBars {
    uint64_t item_full[2], item_empty[2], clc, res_full, res_empty, ring_full[2], ring_empty[2], tail, a_full, b_full, pa_full, pb_full, done;
    // Two, because a warp that has parked the values of tile n + 1 can be done with tile n before another warp has looked whether those of tile n
    // are there: on one barrier that warp would miss its phase and wait for good.  Those of tile n + 2 need every warp's part of tile n.
    uint64_t vec_full[2];
    uint64_t unit_full[2];                                                // the warps' shares of an item's largest norms (fp16)
    float2 peak[2][16];
    uint4 answer;
    Item item[2];
    uint32_t tmem_slot;
};

constexpr float P_UNIT_LOG2 = 15.f, P_UNIT = 32768.f;                     // fp16: dK/dV's probabilities are multiplied by this (P <= 1)
constexpr int UNIT_ROWS = 32;                                             // rows of a block of PackedAttn::units
// a power of two u with 2^14 <= bound * u < 2^15 (bounds from 2^-60 to 2^63)
__device__ __forceinline__ float unit_for(float bound) {
    const int e = min(max(__float_as_int(bound) >> 23, 127 - 60), 127 + 63);
    return __int_as_float((2 * 127 + 14 - e) << 23);
}
__device__ __forceinline__ float inverse_of_power(float u) { return __int_as_float((254 << 23) - __float_as_int(u)); }

struct BwdArgs {
    const float *lse, *delta;
    const float2* peak;                                                   // fp16: [heads, then key heads][blocks] largest |dO| and |delta|, largest |v|
    const float* norm;                                                    // fp16: [heads, then key heads][total] |dO|, |v|
    int blocks;
    void *out0, *out1;                                                    // dV, dK, or dQ
    PackedSeqs seqs;
    int heads, group, hd, causal, slots;
    int split;                                                            // KV: parts of a group of heads, each an item of its own with fp32 results
    float scale;
    int* err;
};

template <typename T, int HD, bool KV>
__global__ void __launch_bounds__(BWD_THREADS, 1) packed_bwd_sm100_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                          const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                                                                          const __grid_constant__ BwdArgs a) {
    constexpr int HALVES = HD / 64;
    constexpr uint32_t TILE = HALVES * HALF_TILE;
    constexpr bool UNIT = Half2<T>::FMT == 0;                             // fp16: dS carries a power of two
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sR0 = smem;
    uint8_t* sR1 = sR0 + TILE;
    uint8_t* sT0 = sR1 + TILE;                                            // [2]
    uint8_t* sT1 = sT0 + 2 * TILE;                                        // [2]
    float* s_lse = reinterpret_cast<float*>(sT1 + 2 * TILE);              // [2][128]  -lse * log2(e)
    float* s_del = s_lse + 256;                                           // [2][128]
    uint8_t* s_stage = reinterpret_cast<uint8_t*>(s_del + 256);
    BwdBars* b = reinterpret_cast<BwdBars*>(s_stage + 16 * 32 * BWD_PITCH);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_heads = KV ? a.heads / a.group : a.heads, n_parts = KV ? n_heads * a.split : n_heads;      // heads, and items of a tile
    const int group = KV ? a.group / a.split : a.group;                   // KV: query heads of an item (item `head` is key head * split + part)
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b->item_full[i], 1); mbar_init(&b->item_empty[i], 17); mbar_init(&b->ring_full[i], 1); mbar_init(&b->ring_empty[i], 1);
            mbar_init(&b->vec_full[i], 8); mbar_init(&b->unit_full[i], 16);
        }
        mbar_init(&b->clc, 1); mbar_init(&b->res_full, 1); mbar_init(&b->res_empty, 1); mbar_init(&b->tail, 1); mbar_init(&b->a_full, 1); mbar_init(&b->b_full, 1);
        mbar_init(&b->pa_full, 16); mbar_init(&b->pb_full, 16); mbar_init(&b->done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 17) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&b->tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0, tm_x = 0, tm_y = 128, tm_acc0 = 256, tm_acc1 = 384;       // all 512 columns are allocated, so they start at 0
    if (KV) {
        after_previous();
        let_next_start();
    }

    // tiles of the other axis that one head of an item meets: [first, first + count) in tiles of 128 rows from the sequence's begin
    auto first_tile = [&](const Item& w) { return KV && a.causal ? (w.row0 - w.lo) / 128 : 0; };
    auto tiles = [&](const Item& w) {
        if (!KV && a.causal) return (w.row0 - w.lo) / 128 + 1;
        return (w.hi - w.lo + 127) / 128 - first_tile(w);
    };

    if (warp < 16) {
        reg_inc<BWD_REGS>();
        const int q = warp & 3, g = warp >> 2, row = q * 32 + lane, tl = (int)threadIdx.x;
        const uint32_t lane_addr = (uint32_t)(q * 32) << 16;
        const uint32_t my_x = tm_x + lane_addr + g * 32, my_y = tm_y + lane_addr + g * 32;
        const float c2 = a.scale * LOG2E;
        uint8_t* stg = s_stage + warp * 32 * BWD_PITCH;
        uint32_t n_item = 0, n = 0, n_done = 0;
        bool ok = true;
        auto take = [&](Item& w) {
            const uint32_t si = n_item & 1;
            if (!warp_wait(&b->item_full[si], (n_item >> 1) & 1)) { atomicExch(a.err, 81); return false; }
            w = b->item[si];
            __syncwarp();
            if (lane == 0) mbar_arrive(&b->item_empty[si]);
            ++n_item;
            return true;
        };
        // KV: the per-query vectors of a tile, one value per thread (threads 0..127 -lse log2 e, 128..255 delta); queries past the end get
        // probability zero.  Else: both values of the thread's own query.
        const bool carries = KV && tl < 256;
        auto fetch = [&](const Item& w, int h, int i) {
            const int r = w.lo + i * 128 + (tl & 127);
            if (r >= w.hi) return tl < 128 ? INFINITY : 0.f;
            return __ldcg((tl < 128 ? a.lse : a.delta) + (int64_t)h * a.seqs.total + r);      // scaled when it is parked: nothing here waits for the load
        };
        const float vmul = tl < 128 ? -LOG2E : 1.f, vadd = UNIT && tl < 128 ? P_UNIT_LOG2 : 0.f;        // -lse log2 e, with the unit of P; delta
        float v0 = 0.f, v1 = 0.f, own = 0.f, unit = 1.f;                  // own: |v| or |dO| of the thread's row
        uint32_t n_unit = 0;                                              // items with a unit so far
        // This warp's share of the largest norms that the item's rows meet: whole blocks from their table, the rows at both ends one by one.  Two
        // buffers are enough: a warp that parks for item n + 2 has seen every warp store the last dS of item n.
        auto park_peaks = [&](const Item& w) {
            const int r0 = w.lo + first_tile(w) * 128, r1 = !KV && a.causal && w.row0 + 128 < w.hi ? w.row0 + 128 : w.hi;
            const int h0 = KV ? w.head * group : a.heads + w.head / a.group, heads = KV ? group : 1;
            int b0 = (r0 + UNIT_ROWS - 1) / UNIT_ROWS, b1 = r1 / UNIT_ROWS;
            if (b1 <= b0) { b0 = (r1 + UNIT_ROWS - 1) / UNIT_ROWS; b1 = b0; }             // no whole block: all rows stand before b0
            const int before = min(b0 * UNIT_ROWS, r1) - r0, behind = max(r1 - b1 * UNIT_ROWS, 0), each = (b1 - b0) + before + behind;
            float x = 0.f, y = 0.f;
#pragma unroll 4
            for (int i = tl; i < heads * each; i += 512) {
                const int64_t h = h0 + i / each;
                const int k = i % each;
                if (k < b1 - b0) {
                    const float2 p = __ldcg(a.peak + h * a.blocks + b0 + k);
                    x = fmaxf(x, p.x); y = fmaxf(y, p.y);
                } else {
                    const int e = k - (b1 - b0), r = e < before ? r0 + e : b1 * UNIT_ROWS + (e - before);
                    x = fmaxf(x, __ldcg(a.norm + h * a.seqs.total + r));
                    if (KV) { const float d = fabsf(__ldcg(a.delta + h * a.seqs.total + r)); if (d < INFINITY) y = fmaxf(y, d); }
                }
            }
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) { x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off)); y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, off)); }
            if (lane == 0) b->peak[n_unit & 1][warp] = make_float2(x, y);
            warp_arrive(&b->unit_full[n_unit & 1]);
            own = w.row0 + row < w.hi ? __ldcg(a.norm + (int64_t)(KV ? a.heads + w.head / a.split : w.head) * a.seqs.total + w.row0 + row) : 0.f;
        };
        auto fetch_first = [&](const Item& w) {
            if (w.kind != 1) return;
            if constexpr (UNIT) park_peaks(w);
            if (KV) { if (carries) v0 = fetch(w, w.head * group, first_tile(w)); }
            else if (w.row0 + row < w.hi) {
                const int64_t at = (int64_t)w.head * a.seqs.total + w.row0 + row;
                v0 = __ldcg(a.lse + at); v1 = __ldcg(a.delta + at);
            }
        };
        Item w;
        ok = take(w);
        if (ok) fetch_first(w);
        while (ok && w.kind != 0) {
            const int per_head = w.kind == 1 ? tiles(w) : 0, n_it = KV ? per_head * group : per_head;
            const float lse_row = v0 * LOG2E, del_row = v1;
            if (carries && n_it > 0) {
                (tl < 128 ? s_lse : s_del)[(n & 1) * 128 + (tl & 127)] = fmaf(v0, vmul, vadd);    // buffer n & 1: every thread has left iteration n - 2
                warp_arrive(&b->vec_full[n & 1]);
            }
            if (UNIT && n_it > 0) {
                if (!warp_wait(&b->unit_full[n_unit & 1], (n_unit >> 1) & 1)) { atomicExch(a.err, 96); ok = false; break; }
                const float2 p = b->peak[n_unit & 1][lane & 15];
                float x = p.x, y = p.y;
#pragma unroll
                for (int off = 8; off > 0; off >>= 1) { x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off)); y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, off)); }
                unit = unit_for(x * own + (KV ? y : fabsf(del_row)));
                if (KV) unit *= 1.f / P_UNIT;                             // the probabilities carry theirs already
                ++n_unit;
            }
            int h = KV ? w.head * group : w.head, i = first_tile(w);
            const int i0 = i, i1 = i + per_head;
            for (int it = 0; it < n_it; ++it, ++n) {
                const int bs = n & 1;
                // the vectors of the NEXT tile are fetched now and parked in the other buffer at the end of this iteration
                float nx = 0.f;
                const bool diag = a.causal && i == (KV ? i0 : i1 - 1);
                const int see = KV ? 128 : w.hi - (w.lo + i * 128);      // keys of this tile that exist
                if (++i == i1 && KV) { i = i0; ++h; }
                if (carries && it + 1 < n_it) nx = fetch(w, h, i);
                if (KV && !warp_wait(&b->vec_full[bs], (n >> 1) & 1)) { atomicExch(a.err, 82); ok = false; break; }
                if (!warp_wait(&b->a_full, n & 1)) { atomicExch(a.err, 83); ok = false; break; }
                tc_fence_after();
                uint32_t r[32];
                tc_ld32(my_x, r);
                tc_wait_ld();
                if (!KV) { tc_fence_before(); warp_arrive(&b->pa_full); }         // P stays in registers: X is free
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    float4 nl = make_float4(-lse_row, -lse_row, -lse_row, -lse_row);
                    if (KV) nl = *reinterpret_cast<const float4*>(s_lse + bs * 128 + g * 32 + k);
                    float e0, e1, e2, e3;
                    fma2(__uint_as_float(r[k]), __uint_as_float(r[k + 1]), c2, c2, nl.x, nl.y, e0, e1);
                    fma2(__uint_as_float(r[k + 2]), __uint_as_float(r[k + 3]), c2, c2, nl.z, nl.w, e2, e3);
                    r[k] = __float_as_uint(ex2f(e0)); r[k + 1] = __float_as_uint(ex2f(e1));
                    r[k + 2] = __float_as_uint(ex2f(e2)); r[k + 3] = __float_as_uint(ex2f(e3));
                }
                if (diag || see < 128) {
                    // KV: key `row` is seen by the queries (columns) from the diagonal on; else query `row` sees the keys up to it, and those
                    // that exist
                    const int from = KV ? row - g * 32 : 0, to = KV ? 32 : (diag ? row + 1 : see) - g * 32;
#pragma unroll
                    for (int k = 0; k < 32; ++k) if (k < from || k >= to) r[k] = 0u;
                }
                uint32_t d[32];                                          // dP; its first half also takes the packed operands, in place
                if (KV) {
                    uint32_t pk[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) pk[k] = Half2<T>::pack(__uint_as_float(r[2 * k]), __uint_as_float(r[2 * k + 1]));
                    tc_st16(my_x, pk);
                    tc_wait_st();
                    tc_fence_before();
                    warp_arrive(&b->pa_full);
                }
                if (!warp_wait(&b->b_full, n & 1)) { atomicExch(a.err, 84); ok = false; break; }
                tc_fence_after();
                tc_ld32(my_y, d);
                tc_wait_ld();
                uint32_t pk[16];
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    float4 de = make_float4(del_row, del_row, del_row, del_row);
                    if (KV) de = *reinterpret_cast<const float4*>(s_del + bs * 128 + g * 32 + k);
                    float t0, t1, t2, t3;
                    fma2(de.x, de.y, -1.f, -1.f, __uint_as_float(d[k]), __uint_as_float(d[k + 1]), t0, t1);               // dP - delta
                    fma2(de.z, de.w, -1.f, -1.f, __uint_as_float(d[k + 2]), __uint_as_float(d[k + 3]), t2, t3);
                    fma2(__uint_as_float(r[k]), __uint_as_float(r[k + 1]), t0, t1, 0.f, 0.f, t0, t1);
                    fma2(__uint_as_float(r[k + 2]), __uint_as_float(r[k + 3]), t2, t3, 0.f, 0.f, t2, t3);
                    if constexpr (UNIT) { fma2(t0, t1, unit, unit, 0.f, 0.f, t0, t1); fma2(t2, t3, unit, unit, 0.f, 0.f, t2, t3); }
                    pk[k / 2] = Half2<T>::pack(t0, t1);
                    pk[k / 2 + 1] = Half2<T>::pack(t2, t3);
                }
                tc_st16(my_y, pk);                                        // this group alone has read these columns
                tc_wait_st();
                tc_fence_before();
                warp_arrive(&b->pb_full);
                if (carries && it + 1 < n_it) { (tl < 128 ? s_lse : s_del)[(bs ^ 1) * 128 + (tl & 127)] = fmaf(nx, vmul, vadd); warp_arrive(&b->vec_full[bs ^ 1]); }
            }
            if (!ok) break;
            const Item cur = w;
            ok = take(w);
            if (!ok) break;
            fetch_first(w);
            if (n_it > 0) {
                if (!warp_wait(&b->done, n_done & 1)) { atomicExch(a.err, 85); ok = false; break; }
                ++n_done;
                tc_fence_after();
            }
            // KV: groups 0 and 1 write dV, 2 and 3 dK, each half of the columns; else each group writes a quarter of dQ (HD = 64: two of them
            // half).  Rows of no sequence: zeros
            const int row0 = cur.row0 + q * 32, live = cur.hi - row0;
            if (live > 0) {
                const int64_t ld = (int64_t)n_heads * a.hd;
                const bool second = KV && g >= 2;
                const int head = KV ? cur.head / a.split : cur.head;
                const int64_t at = (int64_t)row0 * ld + (int64_t)head * a.hd;
                T* base = (T*)(second ? a.out1 : a.out0) + at;
                float* part = KV && a.split > 1 ? (float*)(second ? a.out1 : a.out0) + (int64_t)(cur.head % a.split) * a.seqs.total * ld + at + lane * ld : nullptr;
                constexpr float p_inv = UNIT && KV ? 1.f / P_UNIT : 1.f;
                const float f = KV && !second ? p_inv : (UNIT ? a.scale * inverse_of_power(unit) * p_inv : a.scale);
                const uint32_t acc = (second ? tm_acc1 : tm_acc0) + lane_addr;
                const int c0 = KV ? (g & 1) * (HD / 64) : g, c1 = KV ? c0 + HD / 64 : (g < HD / 32 ? g + 1 : g);
#pragma unroll 1
                for (int c = c0; c < c1; ++c) {
                    uint32_t t[32];
                    if (n_it > 0) {
                        tc_ld32(acc + c * 32, t);
                        tc_wait_ld();
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k) t[k] = 0u;
                    }
                    if (KV && part) {                                     // a part of a sum: fp32, added up by packed_join_kernel
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            if (lane < live && c * 32 + k < a.hd)
                                *reinterpret_cast<float4*>(part + c * 32 + k) = make_float4(__uint_as_float(t[k]) * f, __uint_as_float(t[k + 1]) * f,
                                                                                           __uint_as_float(t[k + 2]) * f, __uint_as_float(t[k + 3]) * f);
                        continue;
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {                // 16 columns at a time, two lanes store 32 consecutive bytes of a row
#pragma unroll
                        for (int u = 2 * half; u < 2 * half + 2; ++u) {
                            uint32_t pk[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) pk[e] = Half2<T>::pack(__uint_as_float(t[8 * u + 2 * e]) * f, __uint_as_float(t[8 * u + 2 * e + 1]) * f);
                            *reinterpret_cast<uint4*>(stg + lane * BWD_PITCH + (u & 1) * 16) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
                        }
                        __syncwarp();
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const int rr = u * 16 + (lane >> 1), col = c * 32 + half * 16 + (lane & 1) * 8;
                            if (rr < live && col < a.hd)
                                *reinterpret_cast<uint4*>(base + rr * ld + col) = *reinterpret_cast<const uint4*>(stg + rr * BWD_PITCH + (lane & 1) * 16);
                        }
                        __syncwarp();
                    }
                }
            }
            tc_fence_before();                                            // the accumulators have been read: the next item's products wait for this
        }                                                                 // group's pa_full / pb_full
    } else {
        reg_dec<BWD_REGS_OTHERS>();
        if (warp == 16) {
            int item = (int)blockIdx.x;
            uint32_t n_item = 0, n_clc = 0, n_res = 0, n = 0, n_tail = 0;
            bool ok = true, more = true;
            while (ok && more) {
                if (lane == 0) {
                    mbar_expect_tx(&b->clc, 16);
                    clc_ask(&b->answer, &b->clc);
                }
                // the tiles with the most work start first: early keys are seen by most queries, late queries see most keys
                const int ord = item / n_parts;
                const PackedTile t = packed_tile<128>(a.seqs, KV ? ord : a.slots - 1 - ord);
                if (t.live) {
                    const Item w{t.lo, t.hi, t.row0, item % n_parts, t.pad ? 2 : 1};
                    const uint32_t s = n_item & 1;
                    if (n_item >= 2) ok = warp_wait(&b->item_empty[s], ((n_item >> 1) & 1) ^ 1);
                    if (!ok) { if (lane == 0) atomicExch(a.err, 86); break; }
                    if (lane == 0) { b->item[s] = w; mbar_arrive(&b->item_full[s]); }
                    ++n_item;
                    const int per_head = t.pad ? 0 : tiles(w), n_it = KV ? per_head * group : per_head, i0 = first_tile(w);
                    const int hk = KV ? w.head / a.split : w.head / a.group;
                    int h = KV ? w.head * group : w.head, i = i0;
                    for (int it = 0; it < n_it; ++it, ++n) {
                        const uint32_t r = n & 1;
                        const int row = t.lo + i * 128, have = t.hi - row;
                        if (n >= 2) ok = warp_wait(&b->ring_empty[r], ((n >> 1) & 1) ^ 1);
                        if (!ok) { if (lane == 0) atomicExch(a.err, 87); break; }
                        uint64_t* bar = have < 128 ? &b->tail : &b->ring_full[r];
                        if (lane == 0) {
                            mbar_expect_tx(bar, 2 * TILE);
                            for (int hf = 0; hf < HALVES; ++hf) {
                                tma_load_3d(sT0 + r * TILE + hf * HALF_TILE, KV ? &map_q : &map_k, hf * 64, KV ? h : hk, row, bar);
                                tma_load_3d(sT1 + r * TILE + hf * HALF_TILE, KV ? &map_do : &map_v, hf * 64, KV ? h : hk, row, bar);
                            }
                        }
                        if (it == 0) {
                            if (n_res > 0) ok = warp_wait(&b->res_empty, (n_res - 1) & 1);
                            if (!ok) { if (lane == 0) atomicExch(a.err, 88); break; }
                            ++n_res;
                            if (lane == 0) {
                                mbar_expect_tx(&b->res_full, 2 * TILE);
                                for (int hf = 0; hf < HALVES; ++hf) {
                                    tma_load_3d(sR0 + hf * HALF_TILE, KV ? &map_k : &map_q, hf * 64, KV ? hk : w.head, t.row0, &b->res_full);
                                    tma_load_3d(sR1 + hf * HALF_TILE, KV ? &map_v : &map_do, hf * 64, KV ? hk : w.head, t.row0, &b->res_full);
                                }
                            }
                        }
                        if (have < 128) {
                            ok = warp_wait(&b->tail, n_tail & 1);
                            if (!ok) { if (lane == 0) atomicExch(a.err, 89); break; }
                            ++n_tail;
                            zero_rows<HALVES>(sT0 + r * TILE, have);
                            zero_rows<HALVES>(sT1 + r * TILE, have);
                            if (lane == 0) mbar_arrive(&b->ring_full[r]);
                        }
                        if (++i == i0 + per_head) { i = i0; ++h; }
                    }
                    if (!ok) break;
                }
                if (!warp_wait(&b->clc, n_clc & 1)) { if (lane == 0) atomicExch(a.err, 90); ok = false; break; }
                ++n_clc;
                more = clc_answer(&b->answer, item);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the answer has been read before the next one is written over it
                __syncwarp();
            }
            if (ok && (n_item < 2 || warp_wait(&b->item_empty[n_item & 1], ((n_item >> 1) & 1) ^ 1)) && lane == 0) {
                b->item[n_item & 1].kind = 0;
                mbar_arrive(&b->item_full[n_item & 1]);
            }
        } else if (warp == 17) {
            const uint32_t idesc_first = idesc_f16(Half2<T>::FMT, 128, 128, 0), idesc_acc = idesc_f16(Half2<T>::FMT, 128, (a.hd + 15) / 16 * 16, 1);
            const int ksteps = (a.hd + 15) / 16;
            uint32_t n_item = 0, n_res = 0;
            // iterations of the next item; 0 at the end of the work, -1 when a wait ran out, -2 for rows of no sequence
            auto take = [&]() {
                const uint32_t si = n_item & 1;
                if (!warp_wait(&b->item_full[si], (n_item >> 1) & 1)) { if (lane == 0) atomicExch(a.err, 91); return -1; }
                const Item w = b->item[si];
                warp_arrive(&b->item_empty[si]);
                ++n_item;
                if (w.kind != 1) return w.kind == 0 ? 0 : -2;
                return KV ? tiles(w) * group : tiles(w);
            };
            const Desc r0 = desc_of(make_desc_sw128(smem_u32(sR0))), r1 = desc_of(make_desc_sw128(smem_u32(sR1))), t0 = desc_of(make_desc_sw128(smem_u32(sT0))),
                       t1 = desc_of(make_desc_sw128(smem_u32(sT1))), m0 = desc_of(make_desc_sw128_mn(smem_u32(sT0), HALF_TILE, 1024)),
                       m1 = desc_of(make_desc_sw128_mn(smem_u32(sT1), HALF_TILE, 1024));
            // X or Y = R T^T of ring slot `slot` (a constant in each of its two copies)
            auto first_copy = [&](uint32_t tm, const Desc& res, const Desc& ring, auto slot) {
                const uint32_t rb = ring.lo + slot.v * (TILE >> 4);
                if (ksteps == HD / 16) {
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk) tc_mma_ss(tm, res.lo + KSTEP(kk), res.hi, rb + KSTEP(kk), ring.hi, idesc_first, kk > 0 ? 1u : 0u);
                } else
#pragma unroll 1
                    for (int kk = 0; kk < ksteps; ++kk) tc_mma_ss(tm, res.lo + KSTEP(kk), res.hi, rb + KSTEP(kk), ring.hi, idesc_first, kk > 0 ? 1u : 0u);
            };
            auto first_product = [&](uint32_t tm, const Desc& res, const Desc& ring, uint32_t slot) {
                if (slot == 0) first_copy(tm, res, ring, Const<0>{}); else first_copy(tm, res, ring, Const<1>{});
            };
            // acc += A T, A the 16-bit operand in the columns of X or Y (32 of its columns in the first half of 32), T a ring tile read MN-major
            auto acc_copy = [&](uint32_t acc, uint32_t tm, const Desc& ring, auto slot, bool add) {
                const uint32_t rb = ring.lo + slot.v * (TILE >> 4);
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                    tc_mma_ts(acc, tm + (kk >> 1) * 32 + (kk & 1) * 8, rb + kk * (2048 >> 4), ring.hi, idesc_acc, (kk > 0 || add) ? 1u : 0u);
            };
            auto acc_product = [&](uint32_t acc, uint32_t tm, const Desc& ring, uint32_t slot, bool add) {
                if (slot == 0) acc_copy(acc, tm, ring, Const<0>{}, add); else acc_copy(acc, tm, ring, Const<1>{}, add);
            };
            auto tiles_ready = [&](uint32_t n, bool first_it) {
                if (first_it) {
                    if (!warp_wait(&b->res_full, n_res & 1)) { if (lane == 0) atomicExch(a.err, 92); return false; }
                    ++n_res;
                }
                if (!warp_wait(&b->ring_full[n & 1], (n >> 1) & 1)) { if (lane == 0) atomicExch(a.err, 93); return false; }
                tc_fence_after();
                return true;
            };
            bool ok = true;
            int n_it = -2;
            for (uint32_t n = 0; ok && n_it != 0;) {
                if (n_it < 0) {                                           // no item's first products are on their way
                    do n_it = take(); while (n_it == -2);
                    if (n_it <= 0) break;
                    if (!tiles_ready(n, true)) break;
                    if (elect_one()) {
                        first_product(tm_x, r0, t0, n & 1);
                        tc_commit(&b->a_full);
                        first_product(tm_y, r1, t1, n & 1);
                        tc_commit(&b->b_full);
                        if (n_it == 1) tc_commit(&b->res_empty);
                    }
                    __syncwarp();
                }
                int n_next = 0;
                for (int it = 0; it < n_it; ++it, ++n) {
                    const int s = n & 1, ns = s ^ 1;
                    const bool last = it + 1 == n_it;
                    // one item ahead, no further: the other warps take the item behind it only when this one is done
                    if (last) { n_next = take(); if (n_next == -1) { ok = false; break; } }
                    const bool next = !last || n_next > 0;
                    if (!warp_wait(&b->pa_full, n & 1)) { if (lane == 0) atomicExch(a.err, 94); ok = false; break; }
                    tc_fence_after();
                    if (KV && elect_one()) acc_product(tm_acc0, tm_x, m1, s, it > 0);                    // dV += P^T dO
                    __syncwarp();
                    if (next) {
                        if (!tiles_ready(n + 1, last)) { ok = false; break; }
                        if (elect_one()) {
                            first_product(tm_x, r0, t0, ns);
                            tc_commit(&b->a_full);
                        }
                        __syncwarp();
                    }
                    if (!warp_wait(&b->pb_full, n & 1)) { if (lane == 0) atomicExch(a.err, 95); ok = false; break; }
                    tc_fence_after();
                    if (elect_one()) {
                        acc_product(KV ? tm_acc1 : tm_acc0, tm_y, m0, s, it > 0);                        // dK += dS^T Q / dQ += dS K
                        tc_commit(&b->ring_empty[s]);
                        if (last) tc_commit(&b->done);
                        if (next) {
                            first_product(tm_y, r1, t1, ns);
                            tc_commit(&b->b_full);
                            if (last ? n_next == 1 : it + 2 == n_it) tc_commit(&b->res_empty);           // the last first products of their item
                        }
                    }
                    __syncwarp();
                }
                n_it = n_next;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 17) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (!KV) after_previous();
}

// out0 / out1 = the sums of their parts, in order, n elements each (a multiple of 8)
template <typename T>
__global__ void __launch_bounds__(256) packed_join_kernel(const float* p0, const float* p1, int split, int64_t n, T* o0, T* o1) {
    after_previous();
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (i >= n) return;
    const float* p = (blockIdx.y ? p1 : p0) + i;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < split; ++s) {
        const float4 x = *reinterpret_cast<const float4*>(p + s * n), y = *reinterpret_cast<const float4*>(p + s * n + 4);
        v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
    }
    *reinterpret_cast<uint4*>((blockIdx.y ? o1 : o0) + i) = make_uint4(Half2<T>::pack(v[0], v[1]), Half2<T>::pack(v[2], v[3]), Half2<T>::pack(v[4], v[5]), Half2<T>::pack(v[6], v[7]));
}

// delta[head][row] = dO . (O + rest): 16 bytes of each per lane, 8 or 16 lanes per (row, head)
template <typename T, int LANES>
__global__ void __launch_bounds__(256) packed_delta_sm100_kernel(PackedAttn p) {
    let_next_start();
    const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
    const int part = (int)(threadIdx.x % LANES);
    const bool live = item < (int64_t)p.seqs.total * p.heads;
    float acc = 0.f;
    if (live && part * 8 < p.hd) {
        const int64_t at = item * p.hd + part * 8;
        const uint4 o = *reinterpret_cast<const uint4*>((const T*)p.out + at), e = *reinterpret_cast<const uint4*>((const T*)p.out_lo + at),
                    d = *reinterpret_cast<const uint4*>((const T*)p.dout + at);
        const uint32_t ov[4] = {o.x, o.y, o.z, o.w}, ev[4] = {e.x, e.y, e.z, e.w}, dv[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 x = Half2<T>::unpack(ov[k]), y = Half2<T>::unpack(ev[k]), z = Half2<T>::unpack(dv[k]);
            acc = fmaf(x.x + y.x, z.x, fmaf(x.y + y.y, z.y, acc));
        }
    }
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    if (live && part == 0) p.delta[(item % p.heads) * p.seqs.total + item / p.heads] = acc;
}

// The same for fp16, with what the units need: a CTA takes 32 rows of one head of dO (delta and |dO|) or of v (|v|), and leaves the largest
// finite norm and |delta| among them.
template <int LANES>
__global__ void __launch_bounds__(256) packed_norms_sm100_kernel(PackedAttn p, float2* peak, float* norm, int blocks) {
    let_next_start();
    __shared__ float2 sh[8];
    const int hk = p.heads / p.group, all = p.heads + hk, h = (int)(blockIdx.x % (unsigned)all), blk = (int)(blockIdx.x / (unsigned)all);
    const int part = (int)(threadIdx.x % LANES);
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int r = 0; r < UNIT_ROWS; r += 256 / LANES) {
        const int row = blk * UNIT_ROWS + r + (int)threadIdx.x / LANES;
        const bool live = row < p.seqs.total;
        float acc = 0.f, sq = 0.f;
        if (live && part * 8 < p.hd) {
            const int64_t at = ((int64_t)row * p.heads + h) * p.hd + part * 8;
            const uint4 d = h < p.heads ? *reinterpret_cast<const uint4*>((const __half*)p.dout + at)
                                        : *reinterpret_cast<const uint4*>((const __half*)p.v + row * p.v_ld + (h - p.heads) * p.v_hs + part * 8);
            uint4 o = make_uint4(0u, 0u, 0u, 0u), e = o;
            if (h < p.heads) { o = *reinterpret_cast<const uint4*>((const __half*)p.out + at); e = *reinterpret_cast<const uint4*>((const __half*)p.out_lo + at); }
            const uint32_t ov[4] = {o.x, o.y, o.z, o.w}, ev[4] = {e.x, e.y, e.z, e.w}, dv[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 a = Half2<__half>::unpack(ov[k]), b = Half2<__half>::unpack(ev[k]), z = Half2<__half>::unpack(dv[k]);
                acc = fmaf(a.x + b.x, z.x, fmaf(a.y + b.y, z.y, acc));
                sq = fmaf(z.x, z.x, fmaf(z.y, z.y, sq));
            }
        }
#pragma unroll
        for (int off = LANES / 2; off > 0; off >>= 1) { acc += __shfl_xor_sync(0xffffffffu, acc, off); sq += __shfl_xor_sync(0xffffffffu, sq, off); }
        const float n = sq < INFINITY ? sqrtf(sq) : 0.f;                  // false for NaN too
        if (live && part == 0) {
            norm[(int64_t)h * p.seqs.total + row] = n;
            if (h < p.heads) p.delta[(int64_t)h * p.seqs.total + row] = acc;
        }
        x = fmaxf(x, n);
        if (fabsf(acc) < INFINITY) y = fmaxf(y, fabsf(acc));
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) { x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off)); y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, off)); }
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = make_float2(x, y);
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int i = 1; i < 8; ++i) { x = fmaxf(x, sh[i].x); y = fmaxf(y, sh[i].y); }
        peak[(int64_t)h * blocks + blk] = make_float2(x, y);
    }
}

bool head_map(CUtensorMap* m, const void* base, const PackedAttn& p, int heads, int64_t ld, int64_t hs) {
    return make_map_heads(m, base, p.seqs.total, heads, p.hd, ld, hs, 128);
}

template <typename T, int HD> int fwd(const PackedAttn& p, int* err, cudaStream_t st) {
    CUtensorMap mq, mk, mv;
    const int hk = p.heads / p.group;
    if (!head_map(&mq, p.q, p, p.heads, p.q_ld, p.q_hs) || !head_map(&mk, p.k, p, hk, p.k_ld, p.k_hs) || !head_map(&mv, p.v, p, hk, p.v_ld, p.v_hs)) return 10;
    constexpr size_t smem = 6 * (HD / 64) * HALF_TILE + 8 * 32 * STAGE_PITCH + sizeof(FwdBars) + 1024;
    static std::atomic<uint64_t> done{0};
    if (!once_per_device(done, current_device(), [&] {
            return cudaFuncSetAttribute(packed_fwd_sm100_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess;
        })) return 11;
    const FwdArgs a{p.out, p.out_lo, p.lse, p.seqs, p.heads, p.group, p.hd, p.causal, packed_slots(p.seqs.n, p.seqs.total, 256), p.scale, err};
    count_launch();
    packed_fwd_sm100_kernel<T, HD><<<(unsigned)a.slots * (unsigned)p.heads, FWD_THREADS, smem, st>>>(mq, mk, mv, a);
    return cudaGetLastError() == cudaSuccess ? 0 : 12;
}

template <typename T, int HD> int bwd(const PackedAttn& p, int* err, cudaStream_t st) {
    CUtensorMap mq, mk, mv, md;
    const int hk = p.heads / p.group;
    if (!head_map(&mq, p.q, p, p.heads, p.q_ld, p.q_hs) || !head_map(&mk, p.k, p, hk, p.k_ld, p.k_hs) || !head_map(&mv, p.v, p, hk, p.v_ld, p.v_hs) ||
        !head_map(&md, p.dout, p, p.heads, (int64_t)p.heads * p.hd, p.hd)) return 10;
    constexpr size_t smem = 6 * (HD / 64) * HALF_TILE + 2048 + 16 * 32 * BWD_PITCH + sizeof(BwdBars) + 1024;
    static std::atomic<uint64_t> done{0};
    if (!once_per_device(done, current_device(), [&] {
            return cudaFuncSetAttribute(packed_bwd_sm100_kernel<T, HD, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess &&
                   cudaFuncSetAttribute(packed_bwd_sm100_kernel<T, HD, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess;
        })) return 11;
    constexpr int LANES = HD / 8;
    const int slots = packed_slots(p.seqs.n, p.seqs.total, 128);
    const int split = p.kv_parts ? packed_attn_sm100_split(p) : 1;
    const int64_t n_kv = (int64_t)p.seqs.total * hk * p.hd;
    const int blocks = (p.seqs.total + UNIT_ROWS - 1) / UNIT_ROWS;
    float2* peak = reinterpret_cast<float2*>(p.units);
    float* norm = p.units ? p.units + (int64_t)2 * (p.heads + hk) * blocks : nullptr;
    BwdArgs a{p.lse, p.delta, peak, norm, blocks, split > 1 ? (void*)p.kv_parts : p.dv, split > 1 ? (void*)(p.kv_parts + split * n_kv) : p.dk, p.seqs, p.heads, p.group, p.hd, p.causal, slots,
              split, p.scale, err};
    count_launch(split > 1 ? 4 : 3);
    if constexpr (Half2<T>::FMT == 0) packed_norms_sm100_kernel<LANES><<<(unsigned)blocks * (unsigned)(p.heads + hk), 256, 0, st>>>(p, peak, norm, blocks);
    else packed_delta_sm100_kernel<T, LANES><<<(unsigned)(((int64_t)p.seqs.total * p.heads * LANES + 255) / 256), 256, 0, st>>>(p);
    if (cudaGetLastError() != cudaSuccess ||
        launch_early(packed_bwd_sm100_kernel<T, HD, true>, dim3((unsigned)slots * (unsigned)(hk * split)), BWD_THREADS, smem, st, mq, mk, mv, md, a) != cudaSuccess) return 12;
    a.out0 = p.dq; a.out1 = nullptr;
    if (launch_early(packed_bwd_sm100_kernel<T, HD, false>, dim3((unsigned)slots * (unsigned)p.heads), BWD_THREADS, smem, st, mq, mk, mv, md, a) != cudaSuccess) return 12;
    if (split > 1 && launch_early(packed_join_kernel<T>, dim3((unsigned)((n_kv / 8 + 255) / 256), 2), 256, 0, st, p.kv_parts, p.kv_parts + split * n_kv, split, n_kv, (T*)p.dv,
                                  (T*)p.dk) != cudaSuccess) return 12;
    return 0;
}

}  // namespace

// Scores are compared before they are scaled, so the scale has to be positive.
bool packed_attn_sm100_takes(int dtype, const PackedAttn& p) {
    const int hk = p.heads / p.group;
    return dtype != F32 && p.hd % 8 == 0 && p.hd <= 128 && p.scale > 0.f && p.scale < 1e30f && packed_tma_view(p.q, p.q_ld, p.q_hs, p.seqs.total, p.heads) &&
           packed_tma_view(p.k, p.k_ld, p.k_hs, p.seqs.total, hk) && packed_tma_view(p.v, p.v_ld, p.v_hs, p.seqs.total, hk) &&
           (int64_t)packed_slots(p.seqs.n, p.seqs.total, 128) * p.heads < ((int64_t)1 << 31);
}

// Parts that the query heads of a key head are cut into for dK and dV.  An item of that kernel visits every query tile of all its heads; with
// few key heads there are few items and SMs stay without one, but parts are fp32 sums to be written and added up, and what long items leave
// idle at the end, dQ fills.  So: an item for each SM, two where a head has up to 64 columns (half the sums); below 256 rows a sequence all
// items are short.  Backward pass of 16 query heads, us whole / in two / four / eight parts: 14 documents in 8,192 rows, 4 key heads of 128 295 /
// 294 / 334, 2 key heads 336 / 312 / 293 / 332, 4 key heads of 64 264 / 220 / 242; 14,354 + 2,030 rows, 2 key heads of 128 2,512 / 2,542 / 2,577.
// Documents of very different lengths would want more parts than the number of items says (2 key heads of 128 get two here, four take 6 % less):
// how different they are is known on the device only.
int packed_attn_sm100_split(const PackedAttn& p) {
    const int64_t hk = p.heads / p.group, tiles = p.seqs.total / 128, each = p.seqs.n > 0 ? p.seqs.total / p.seqs.n : 0;
    if (p.group == 1 || each < 256 || tiles == 0) return 1;
    const int64_t want = ((p.hd > 64 ? 1 : 2) * (int64_t)device_sms() + hk * tiles - 1) / (hk * tiles);
    for (int s = 1; s < p.group; ++s) if (p.group % s == 0 && s >= want) return s;
    return p.group;
}
int64_t packed_attn_sm100_units(int dtype, const PackedAttn& p) {
    if (dtype != F16) return 0;
    return (int64_t)(p.heads + p.heads / p.group) * (2 * (int64_t)((p.seqs.total + UNIT_ROWS - 1) / UNIT_ROWS) + p.seqs.total);
}
int packed_attn_sm100_fwd(int dtype, const PackedAttn& p, int* err, cudaStream_t st) {
    if (p.hd > 64) return dtype == BF16 ? fwd<__nv_bfloat16, 128>(p, err, st) : fwd<__half, 128>(p, err, st);
    return dtype == BF16 ? fwd<__nv_bfloat16, 64>(p, err, st) : fwd<__half, 64>(p, err, st);
}
int packed_attn_sm100_bwd(int dtype, const PackedAttn& p, int* err, cudaStream_t st) {
    if (p.hd > 64) return dtype == BF16 ? bwd<__nv_bfloat16, 128>(p, err, st) : bwd<__half, 128>(p, err, st);
    return dtype == BF16 ? bwd<__nv_bfloat16, 64>(p, err, st) : bwd<__half, 64>(p, err, st);
}

}  // namespace sg
