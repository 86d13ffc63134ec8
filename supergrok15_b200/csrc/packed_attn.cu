// Attention over packed sequences on the CUDA cores: every type, every head size up to 128, any strides.  It takes what the tensor-core
// kernels of packed_attn_sm100.cu do not: fp32 operands (a product of two 24-bit mantissas does not fit their 16-bit operands) and rows
// that TMA cannot address.
//
//   o_i = sum_j p_ij v_j,  p_ij = softmax_j(scale q_i . k_j),  j over the rows of i's sequence (causal: j <= i)
//   backward, with delta_i = do_i . o_i:  ds_ij = p_ij (do_i . v_j - delta_i),  dq_i = scale sum_j ds_ij k_j,
//                                         dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i  (i over the query heads of the group)
//
// An error e in delta_i shifts every ds_ij by p_ij e, and with it dq_i by e times the mean key that row i sees: a common shift of the keys,
// which the exact gradient does not feel, scales it.  The rounding of a 16-bit o_i is such an error (2.2 % of dq's norm with keys six
// standard deviations from zero), so a training forward also stores what the rounding took and delta is formed from the sum of the two.
//
// A CTA of 256 threads takes a 64-row tile against 64-row tiles of the other axis, all of them in shared memory as fp32 rows of DP + 4
// words (DP + 4 = 4 mod 32: sixteen lanes reading sixteen rows, four words each, touch every bank once).  A thread owns 4 x 4 scores (rows
// ty + 16 i, columns tx + 16 j) and, of an accumulator, 4 rows x DP / 64 pieces of four columns.  One pass over the keys with the running
// maximum and sum; dk / dv and dq come from two kernels, so that nothing is added by atomics.  They do not depend on each other: dq's CTAs start
// when every CTA of dk / dv has seen the end of the delta pass (read from L2), and wait for all of dk / dv at their end (1,023 rows in five
// sequences, 4 heads of 80, fp32, forward and backward: 219 -> 154 us, as one of them alone does not fill the SMs).  Bound by the FMA pipe and the shared memory
// that feeds it (8 loads of 16 bytes per 64 FMAs of the scores).
#include "sg_native.h"
#include "optim_math.cuh"
#include "packed_attn.h"
#include "per_device.h"
#include "launch_early.cuh"

namespace sg {
namespace {

constexpr int PT = 64, PTHREADS = 256;

// rows [row0, row0 + 64) of a head, zero where row >= hi or column >= hd: four columns of DP / 16 rows per thread, all loads in flight at once
template <typename T, int DP>
__device__ __forceinline__ void load_tile(float* dst, const T* base, int64_t ld, int row0, int hi, int hd) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const bool vec = sizeof(T) == 4 && ((reinterpret_cast<uintptr_t>(base) & 15) | (ld & 3) | (hd & 3)) == 0;
    float4 v[4][DP / 64];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < DP / 64; ++m) {
            const int row = row0 + ty + 16 * i, c = 4 * (tx + 16 * m);
            const T* src = base + (int64_t)row * ld + c;
            if (vec) v[i][m] = row < hi && c < hd ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
            else {
                float e[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) e[u] = row < hi && c + u < hd ? Cvt<T>::to(src[u]) : 0.f;
                v[i][m] = make_float4(e[0], e[1], e[2], e[3]);
            }
        }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m = 0; m < DP / 64; ++m) *reinterpret_cast<float4*>(dst + (ty + 16 * i) * (DP + 4) + 4 * (tx + 16 * m)) = v[i][m];
}

// s[i][j] = a[ty + 16 i] . b[tx + 16 j]
template <int DP> __device__ __forceinline__ void dot4x4(const float* a, const float* b, int hd, int ty, int tx, float (&s)[4][4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < hd; d += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = *reinterpret_cast<const float4*>(a + (ty + 16 * i) * (DP + 4) + d);
            y[i] = *reinterpret_cast<const float4*>(b + (tx + 16 * i) * (DP + 4) + d);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = fmaf(x[i].x, y[j].x, fmaf(x[i].y, y[j].y, fmaf(x[i].z, y[j].z, fmaf(x[i].w, y[j].w, s[i][j]))));
    }
}

// acc[i][m] += sum_r w[r][ty + 16 i] * t[r][4 (tx + 16 m) ..]   (w: [64][68], TRANS reads w[ty + 16 i][r] instead)
template <int DP, bool TRANS>
__device__ __forceinline__ void acc_rows(const float* w, const float* t, int ty, int tx, float4 (&acc)[4][DP / 64]) {
#pragma unroll 4
    for (int r = 0; r < PT; ++r) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = TRANS ? w[(ty + 16 * i) * 68 + r] : w[r * 68 + ty + 16 * i];
#pragma unroll
        for (int m = 0; m < DP / 64; ++m) {
            const float4 v = *reinterpret_cast<const float4*>(t + r * (DP + 4) + 4 * (tx + 16 * m));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[i][m].x = fmaf(f[i], v.x, acc[i][m].x); acc[i][m].y = fmaf(f[i], v.y, acc[i][m].y);
                acc[i][m].z = fmaf(f[i], v.z, acc[i][m].z); acc[i][m].w = fmaf(f[i], v.w, acc[i][m].w);
            }
        }
    }
}

template <typename T, int DP>
__device__ __forceinline__ void store_row(T* dst, int tx, int hd, const float4 (&v)[DP / 64], float f) {
#pragma unroll
    for (int m = 0; m < DP / 64; ++m) {
        const int c = 4 * (tx + 16 * m);
        const float e[4] = {v[m].x, v[m].y, v[m].z, v[m].w};
#pragma unroll
        for (int u = 0; u < 4; ++u) if (c + u < hd) dst[c + u] = Cvt<T>::from(e[u] * f);
    }
}

template <typename T, int DP>
__device__ __forceinline__ void store_row_rest(T* dst, int tx, int hd, const float4 (&v)[DP / 64], float f) {
#pragma unroll
    for (int m = 0; m < DP / 64; ++m) {
        const int c = 4 * (tx + 16 * m);
        const float e[4] = {v[m].x, v[m].y, v[m].z, v[m].w};
#pragma unroll
        for (int u = 0; u < 4; ++u) if (c + u < hd) dst[c + u] = Cvt<T>::from(e[u] * f - Cvt<T>::to(Cvt<T>::from(e[u] * f)));
    }
}

__device__ __forceinline__ PackedTile block_tile(const PackedSeqs& ps, PackedTile* sh) {
    if (threadIdx.x < 32) {
        const PackedTile t = packed_tile<PT>(ps, (int)gridDim.x - 1 - (int)blockIdx.x);     // late tiles see most keys: they start first
        if (threadIdx.x == 0) *sh = t;
    }
    __syncthreads();
    return *sh;
}

template <typename T, int DP>
__global__ void __launch_bounds__(PTHREADS) packed_fwd_kernel(PackedAttn p) {
    extern __shared__ __align__(16) float sm[];
    __shared__ PackedTile sh;
    float* sQ = sm;
    float* sK = sQ + PT * (DP + 4);
    float* sV = sK + PT * (DP + 4);
    float* sP = sV + PT * (DP + 4);                                       // [64 rows][68]
    const PackedTile t = block_tile(p.seqs, &sh);
    if (!t.live) return;
    const int h = blockIdx.y, hk = h / p.group, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    T* out = (T*)p.out + (int64_t)h * p.hd;
    const int64_t ldo = (int64_t)p.heads * p.hd;
    if (t.pad) {
        const float4 z[DP / 64] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = t.row0 + ty + 16 * i;
            if (row < t.hi) {
                store_row<T, DP>(out + row * ldo, tx, p.hd, z, 0.f);
                if (p.out_lo) store_row<T, DP>((T*)p.out_lo + (int64_t)h * p.hd + row * ldo, tx, p.hd, z, 0.f);
                if (p.lse && tx == 0) p.lse[(int64_t)h * p.seqs.total + row] = 0.f;
            }
        }
        return;
    }
    load_tile<T, DP>(sQ, (const T*)p.q + h * p.q_hs, p.q_ld, t.row0, t.hi, p.hd);
    float m[4], l[4];
    float4 o[4][DP / 64] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) { m[i] = -INFINITY; l[i] = 0.f; }
    const int last = p.causal ? (t.row0 + PT < t.hi ? t.row0 + PT : t.hi) : t.hi;          // keys that any row of the tile sees
    for (int k0 = t.lo; k0 < last; k0 += PT) {
        __syncthreads();
        load_tile<T, DP>(sK, (const T*)p.k + hk * p.k_hs, p.k_ld, k0, t.hi, p.hd);
        load_tile<T, DP>(sV, (const T*)p.v + hk * p.v_hs, p.v_ld, k0, t.hi, p.hd);
        __syncthreads();
        float s[4][4];
        dot4x4<DP>(sQ, sK, p.hd, ty, tx, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = t.row0 + ty + 16 * i;
            float mx = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = k0 + tx + 16 * j;
                s[i][j] = key < t.hi && (!p.causal || key <= row) ? s[i][j] * p.scale : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
            // -inf only while the row has met nothing but -inf scores: any finite reference then gives exp(-inf) = 0
            const float ref = mx == -INFINITY ? 0.f : mx, a = expf(m[i] - ref);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float e = expf(s[i][j] - ref);
                sum += e;
                sP[(ty + 16 * i) * 68 + tx + 16 * j] = e;
            }
#pragma unroll
            for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            l[i] = l[i] * a + sum;
            m[i] = mx;
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) { o[i][c].x *= a; o[i][c].y *= a; o[i][c].z *= a; o[i][c].w *= a; }
        }
        __syncwarp();                                                      // a row's sixteen lanes share a warp: they alone read its probabilities
        acc_rows<DP, true>(sP, sV, ty, tx, o);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = t.row0 + ty + 16 * i;
        if (row < t.hi) {
            store_row<T, DP>(out + row * ldo, tx, p.hd, o[i], 1.f / l[i]);
            if (p.out_lo) store_row_rest<T, DP>((T*)p.out_lo + (int64_t)h * p.hd + row * ldo, tx, p.hd, o[i], 1.f / l[i]);
            if (p.lse && tx == 0) p.lse[(int64_t)h * p.seqs.total + row] = m[i] + logf(l[i]);
        }
    }
}

// The tile's probabilities and ds for the query rows [q0, q0 + 64) x keys [k0, k0 + 64), written as [query][key]
template <int DP>
__device__ __forceinline__ void bwd_scores(const PackedAttn& p, const float* sQ, const float* sK, const float* sDO, const float* sV, float* sP, float* sS, int h,
                                           int q0, int k0, int hi, int ty, int tx) {
    float s[4][4], d[4][4];
    dot4x4<DP>(sQ, sK, p.hd, ty, tx, s);
    dot4x4<DP>(sDO, sV, p.hd, ty, tx, d);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = q0 + ty + 16 * i;
        const int64_t at = (int64_t)h * p.seqs.total + row;
        const float lse = row < hi ? __ldcg(p.lse + at) : 0.f, de = row < hi ? __ldcg(p.delta + at) : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int key = k0 + tx + 16 * j;
            const bool on = row < hi && key < hi && (!p.causal || key <= row);
            const float e = on ? expf(s[i][j] * p.scale - lse) : 0.f;
            if (sP) sP[(ty + 16 * i) * 68 + tx + 16 * j] = e;
            sS[(ty + 16 * i) * 68 + tx + 16 * j] = on ? e * (d[i][j] - de) : 0.f;
        }
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(PTHREADS) packed_bwd_kv_kernel(PackedAttn p) {
    after_previous();
    let_next_start();
    extern __shared__ __align__(16) float sm[];
    __shared__ PackedTile sh;
    float* sK = sm;
    float* sV = sK + PT * (DP + 4);
    float* sQ = sV + PT * (DP + 4);
    float* sD = sQ + PT * (DP + 4);
    float* sP = sD + PT * (DP + 4);
    float* sS = sP + PT * 68;
    const PackedTile t = block_tile(p.seqs, &sh);
    if (!t.live) return;
    const int hk = blockIdx.y, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    float4 dk[4][DP / 64] = {}, dv[4][DP / 64] = {};
    if (!t.pad) {
        load_tile<T, DP>(sK, (const T*)p.k + hk * p.k_hs, p.k_ld, t.row0, t.hi, p.hd);
        load_tile<T, DP>(sV, (const T*)p.v + hk * p.v_hs, p.v_ld, t.row0, t.hi, p.hd);
        for (int h = hk * p.group; h < (hk + 1) * p.group; ++h)
            for (int q0 = p.causal ? t.row0 : t.lo; q0 < t.hi; q0 += PT) {
                __syncthreads();
                load_tile<T, DP>(sQ, (const T*)p.q + h * p.q_hs, p.q_ld, q0, t.hi, p.hd);
                load_tile<T, DP>(sD, (const T*)p.dout + (int64_t)h * p.hd, (int64_t)p.heads * p.hd, q0, t.hi, p.hd);
                __syncthreads();
                bwd_scores<DP>(p, sQ, sK, sD, sV, sP, sS, h, q0, t.row0, t.hi, ty, tx);
                __syncthreads();
                acc_rows<DP, false>(sP, sD, ty, tx, dv);
                acc_rows<DP, false>(sS, sQ, ty, tx, dk);
            }
    }
    const int64_t ld = (int64_t)(p.heads / p.group) * p.hd;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = t.row0 + ty + 16 * i;
        if (row < t.hi) {
            store_row<T, DP>((T*)p.dk + row * ld + (int64_t)hk * p.hd, tx, p.hd, dk[i], p.scale);
            store_row<T, DP>((T*)p.dv + row * ld + (int64_t)hk * p.hd, tx, p.hd, dv[i], 1.f);
        }
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(PTHREADS) packed_bwd_q_kernel(PackedAttn p) {
    extern __shared__ __align__(16) float sm[];
    __shared__ PackedTile sh;
    float* sQ = sm;
    float* sD = sQ + PT * (DP + 4);
    float* sK = sD + PT * (DP + 4);
    float* sV = sK + PT * (DP + 4);
    float* sS = sV + PT * (DP + 4);
    const PackedTile t = block_tile(p.seqs, &sh);
    if (!t.live) {
        after_previous();
        return;
    }
    const int h = blockIdx.y, hk = h / p.group, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    float4 dq[4][DP / 64] = {};
    if (!t.pad) {
        load_tile<T, DP>(sQ, (const T*)p.q + h * p.q_hs, p.q_ld, t.row0, t.hi, p.hd);
        load_tile<T, DP>(sD, (const T*)p.dout + (int64_t)h * p.hd, (int64_t)p.heads * p.hd, t.row0, t.hi, p.hd);
        const int last = p.causal ? (t.row0 + PT < t.hi ? t.row0 + PT : t.hi) : t.hi;
        for (int k0 = t.lo; k0 < last; k0 += PT) {
            __syncthreads();
            load_tile<T, DP>(sK, (const T*)p.k + hk * p.k_hs, p.k_ld, k0, t.hi, p.hd);
            load_tile<T, DP>(sV, (const T*)p.v + hk * p.v_hs, p.v_ld, k0, t.hi, p.hd);
            __syncthreads();
            bwd_scores<DP>(p, sQ, sK, sD, sV, nullptr, sS, h, t.row0, k0, t.hi, ty, tx);
            __syncwarp();
            acc_rows<DP, true>(sS, sK, ty, tx, dq);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = t.row0 + ty + 16 * i;
        if (row < t.hi) store_row<T, DP>((T*)p.dq + row * (int64_t)p.heads * p.hd + (int64_t)h * p.hd, tx, p.hd, dq[i], p.scale);
    }
    after_previous();
}

// delta[h][row] = do . o, a warp per (row, head)
template <typename T>
__global__ void __launch_bounds__(256) packed_delta_kernel(PackedAttn p) {
    let_next_start();
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= (int64_t)p.seqs.total * p.heads) return;
    const int lane = threadIdx.x & 31;
    const T* o = (const T*)p.out + item * p.hd;
    const T* lo = p.out_lo ? (const T*)p.out_lo + item * p.hd : nullptr;
    const T* d = (const T*)p.dout + item * p.hd;
    float s = 0.f;
    for (int c = lane; c < p.hd; c += 32) s = fmaf(Cvt<T>::to(o[c]) + (lo ? Cvt<T>::to(lo[c]) : 0.f), Cvt<T>::to(d[c]), s);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (lane == 0) p.delta[(item % p.heads) * p.seqs.total + item / p.heads] = s;
}

template <typename K> bool allow_smem(std::atomic<uint64_t>& done, K kernel, size_t bytes) {
    return once_per_device(done, current_device(), [&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess; });
}

template <typename T, int DP> int fwd(const PackedAttn& p, cudaStream_t st) {
    constexpr size_t smem = (3 * PT * (DP + 4) + PT * 68) * sizeof(float);
    static std::atomic<uint64_t> done{0};
    if (!allow_smem(done, packed_fwd_kernel<T, DP>, smem)) return 2;
    count_launch();
    packed_fwd_kernel<T, DP><<<dim3(packed_slots(p.seqs.n, p.seqs.total, PT), p.heads), PTHREADS, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? 0 : 3;
}
template <typename T, int DP> int bwd(const PackedAttn& p, cudaStream_t st) {
    constexpr size_t smem_kv = (4 * PT * (DP + 4) + 2 * PT * 68) * sizeof(float), smem_q = (4 * PT * (DP + 4) + PT * 68) * sizeof(float);
    static std::atomic<uint64_t> done_kv{0}, done_q{0};
    if (!allow_smem(done_kv, packed_bwd_kv_kernel<T, DP>, smem_kv) || !allow_smem(done_q, packed_bwd_q_kernel<T, DP>, smem_q)) return 2;
    count_launch(3);
    const int slots = packed_slots(p.seqs.n, p.seqs.total, PT);
    packed_delta_kernel<T><<<(unsigned)(((int64_t)p.seqs.total * p.heads + 7) / 8), 256, 0, st>>>(p);
    if (cudaGetLastError() != cudaSuccess || launch_early(packed_bwd_kv_kernel<T, DP>, dim3(slots, p.heads / p.group), PTHREADS, smem_kv, st, p) != cudaSuccess) return 3;
    return launch_early(packed_bwd_q_kernel<T, DP>, dim3(slots, p.heads), PTHREADS, smem_q, st, p) == cudaSuccess ? 0 : 3;
}

}  // namespace

#define SG_PACKED_GO(fn) \
    if (p.hd > 64) { if (dtype == F32) return fn<float, 128>(p, st); if (dtype == BF16) return fn<__nv_bfloat16, 128>(p, st); return fn<__half, 128>(p, st); } \
    if (dtype == F32) return fn<float, 64>(p, st); \
    if (dtype == BF16) return fn<__nv_bfloat16, 64>(p, st); \
    return fn<__half, 64>(p, st);
int packed_attn_fwd(int dtype, const PackedAttn& p, cudaStream_t st) { SG_PACKED_GO(fwd) }
int packed_attn_bwd(int dtype, const PackedAttn& p, cudaStream_t st) { SG_PACKED_GO(bwd) }
#undef SG_PACKED_GO

}  // namespace sg
