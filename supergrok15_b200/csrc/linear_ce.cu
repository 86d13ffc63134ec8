// Softmax cross-entropy of a linear head, z = x w^T, that never holds the logits:
//
//   loss = mean over counted rows of lse_r - z_{r,t_r},  lse_r = log sum_v exp z_rv
//   d_rv = p_rv - [v = t_r],  p_rv = exp(z_rv - lse_r);   dx = f d w,  dw = f d^T x,  f = gout / count
//
// Rows go through in pieces.  (1) lce_logits: the product, tile by tile; a tile's epilogue leaves, per row, the maximum m and the sum of
// u = exp(z - m), and, for a training pass, u itself in the type of x: the logits have been consumed when the tile's accumulators are
// free.  (2) lce_rows: one pass over the statistics gives lse and the loss, one over u in place gives d = u exp(m - lse).  The sums leave
// out the target's column: with s' the sum of the others and e_t = exp(z_t - max), 1 - p_t = s' / (s' + e_t) and the loss of a likely
// target is log1p(s' / e_t), both to full precision however certain the target is (p_t - 1 from a rounded p_t, or lse - z_t, would be
// rounding noise).  (3) lce_grads: both products with d.  Two roundings to 16 bits stand between z and a product, of u and of d, each at most half a
// step of the value itself.
//
// Against a pass that recomputes z for the gradient this saves a fourth of all products (6 N V D operations instead of 8) and costs
// reading and writing u once more.
//
// This file: the pass over the rows, and products on the CUDA cores for fp32 operands and for 16-bit ones that TMA cannot address.  Their
// 64 x 64 tiles take 4 x 4 outputs per thread from shared memory in steps of 16, bound by the FMA pipe and its operand loads.
#include "sg_native.h"
#include "optim_math.cuh"
#include "linear_ce.h"
#include "per_device.h"
#include <cfloat>

namespace sg {
namespace {

constexpr int CT = 64, CK = 16, CTHREADS = 256;

// s[i][j] += sum_k A(m0 + ty*4 + i, k) B(n0 + tx*4 + j, k).  AM / BN: the operand's m / n index is the contiguous one, else its k index.
template <typename T, bool AM, bool BN>
__device__ __forceinline__ void tile_product(const T* A, int64_t lda, const T* B, int64_t ldb, int M, int N, int K, int m0, int n0, float (&s)[4][4]) {
    __shared__ __align__(16) float sa[CK][CT + 4], sb[CK][CT + 4];
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    for (int k0 = 0; k0 < K; k0 += CK) {
        __syncthreads();
#pragma unroll
        for (int i = threadIdx.x; i < CT * CK; i += CTHREADS) {
            const int ma = AM ? i % CT : i / CK, ka = AM ? i / CT : i % CK;
            sa[ka][ma] = m0 + ma < M && k0 + ka < K ? Cvt<T>::to(AM ? A[(int64_t)(k0 + ka) * lda + m0 + ma] : A[(int64_t)(m0 + ma) * lda + k0 + ka]) : 0.f;
            const int nb = BN ? i % CT : i / CK, kb = BN ? i / CT : i % CK;
            sb[kb][nb] = n0 + nb < N && k0 + kb < K ? Cvt<T>::to(BN ? B[(int64_t)(k0 + kb) * ldb + n0 + nb] : B[(int64_t)(n0 + nb) * ldb + k0 + kb]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < CK; ++k) {
            const float4 a = *reinterpret_cast<const float4*>(&sa[k][ty * 4]), b = *reinterpret_cast<const float4*>(&sb[k][tx * 4]);
            const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) s[i][j] = fmaf(av[i], bv[j], s[i][j]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(CTHREADS) lce_logits_kernel(LceArgs a) {
    const int m0 = blockIdx.y * CT, n0 = blockIdx.x * CT, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    float s[4][4] = {};
    tile_product<T, false, false>((const T*)a.x, a.ldx, (const T*)a.w, a.ldw, a.rows, a.V, a.D, m0, n0, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = m0 + ty * 4 + i;
        const int64_t t = row < a.rows ? a.target[row] : -1;
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int v = n0 + tx * 4 + j;
            if (v >= a.V) s[i][j] = -INFINITY;
            else if (v == t) a.z_target[row] = s[i][j];
            mx = fmaxf(mx, s[i][j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float ref = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int v = n0 + tx * 4 + j;
            const float e = expf(s[i][j] - ref);
            if (v != t) sum += e;
            if (a.u && row < a.rows && v < a.V) ((T*)a.u)[(int64_t)row * a.ldu + v] = Cvt<T>::from(e * LceUnit<T>::value);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (tx == 0 && row < a.rows) {
            a.tile_max[(int64_t)blockIdx.x * a.rows + row] = mx;
            a.tile_sum[(int64_t)blockIdx.x * a.rows + row] = sum;
        }
    }
}

template <typename T, typename TO, bool AM>
__global__ void __launch_bounds__(CTHREADS) lce_grad_kernel(const T* A, int64_t lda, const T* B, int64_t ldb, int M, int N, int K, const float* prev, TO* out,
                                                            const float* gout, const float* inv) {
    const int m0 = blockIdx.y * CT, n0 = blockIdx.x * CT, ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    float s[4][4] = {};
    tile_product<T, AM, true>(A, lda, B, ldb, M, N, K, m0, n0, s);
    const float f = gout ? gout[0] * inv[0] / LceUnit<T>::value : 1.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m < M && n < N) out[(int64_t)m * N + n] = Cvt<TO>::from(f * (prev ? s[i][j] + prev[(int64_t)m * N + n] : s[i][j]));
        }
}

// One CTA per row: the loss from the tiles' statistics, then u -> d in place (16 bytes per thread and step).
constexpr int ROW_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) lce_rows_kernel(LceArgs a, int tiles, int tile_cols) {
    extern __shared__ float fac[];                                        // [tiles] factor of a tile's columns
    __shared__ float red[ROW_THREADS / 32];
    constexpr int PER = 16 / sizeof(T);
    const int row = blockIdx.x;
    float mx = -INFINITY;
    for (int i = threadIdx.x; i < tiles; i += ROW_THREADS) mx = fmaxf(mx, a.tile_max[(int64_t)i * a.rows + row]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROW_THREADS / 32; ++i) mx = fmaxf(mx, red[i]);
    __syncthreads();
    const float ref = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    for (int i = threadIdx.x; i < tiles; i += ROW_THREADS) sum += a.tile_sum[(int64_t)i * a.rows + row] * expf(a.tile_max[(int64_t)i * a.rows + row] - ref);
    sum = block_sum(sum, red);                                            // in the first warp
    if (threadIdx.x == 0) red[0] = sum;
    __syncthreads();
    const float others = red[0];                                          // sum of exp(z - max) over all columns but the target's
    const int64_t t = a.target[row];
    const bool counted = t != a.ignore_index && t >= 0 && t < a.V;
    const float zt = counted ? a.z_target[row] : 0.f, et = counted ? expf(zt - ref) : 0.f, total = others + et;
    // far below the maximum e_t loses digits and then vanishes, and the plain difference is exact enough
    if (threadIdx.x == 0) a.loss[row] = !counted ? 0.f : (et > 1e-6f ? log1pf(others / et) : (ref - zt) + logf(total));
    if (!a.u) return;
    const float inv = 1.f / total;
    for (int i = threadIdx.x; i < tiles; i += ROW_THREADS) fac[i] = expf(a.tile_max[(int64_t)i * a.rows + row] - ref) * inv;
    __syncthreads();
    T* u = (T*)a.u + (int64_t)row * a.ldu;
    for (int c = threadIdx.x * PER; c < a.ldu; c += ROW_THREADS * PER) {
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if (counted) {
            raw = *reinterpret_cast<const uint4*>(u + c);
            T* e = reinterpret_cast<T*>(&raw);
            const float f = fac[c / tile_cols];                            // PER divides the tile's width
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                float d = Cvt<T>::to(e[k]) * f;
                if (c + k == t) d = -others * inv * LceUnit<T>::value;
                if (c + k >= a.V) d = 0.f;                                 // columns between V and the pitch meet zeros of w
                e[k] = Cvt<T>::from(d);
            }
        }
        *reinterpret_cast<uint4*>(u + c) = raw;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) lce_finish_kernel(const float* __restrict__ in, T* __restrict__ out, int64_t n, const float* gout, const float* inv) {
    const float f = gout[0] * inv[0] / LceUnit<T>::value;
    const int64_t step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n / 4; i += step) {
        const float4 v = reinterpret_cast<const float4*>(in)[i];
        const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) out[4 * i + k] = Cvt<T>::from(e[k] * f);
    }
    for (int64_t i = n / 4 * 4 + (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) out[i] = Cvt<T>::from(in[i] * f);
}

template <typename T> int logits(const LceArgs& a, cudaStream_t st) {
    count_launch();
    lce_logits_kernel<T><<<dim3((a.V + CT - 1) / CT, (a.rows + CT - 1) / CT), CTHREADS, 0, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? 0 : 3;
}

template <typename T> int rows(const LceArgs& a, int tile_cols, cudaStream_t st) {
    const int tiles = (a.V + tile_cols - 1) / tile_cols;
    const size_t smem = tiles * sizeof(float);
    static std::atomic<uint64_t> done{0};
    if (!once_per_device(done, current_device(), [] { return cudaFuncSetAttribute(lce_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) == cudaSuccess; }))
        return 2;
    if (smem > 200 * 1024) return 4;
    count_launch();
    lce_rows_kernel<T><<<a.rows, ROW_THREADS, smem, st>>>(a, tiles, tile_cols);
    return cudaGetLastError() == cudaSuccess ? 0 : 3;
}

template <typename T, typename TO> int grads(const LceArgs& a, const LceGrads& g, cudaStream_t st) {
    const T *d = (const T*)a.u, *x = (const T*)a.x, *w = (const T*)a.w;
    if (g.dx) {
        count_launch();
        lce_grad_kernel<T, TO, false><<<dim3((a.D + CT - 1) / CT, (a.rows + CT - 1) / CT), CTHREADS, 0, st>>>(d, a.ldu, w, a.ldw, a.rows, a.D, a.V, nullptr,
                                                                                                           (TO*)g.dx, g.gout, g.inv_count);
    }
    if (g.dw) {
        count_launch();
        lce_grad_kernel<T, TO, true><<<dim3((a.D + CT - 1) / CT, (a.V + CT - 1) / CT), CTHREADS, 0, st>>>(d, a.ldu, x, a.ldx, a.V, a.D, a.rows, g.dw_prev,
                                                                                                       (TO*)g.dw, g.gout, g.inv_count);
    }
    return cudaGetLastError() == cudaSuccess ? 0 : 3;
}

}  // namespace

#define SG_LCE_GO(fn, ...) { if (dtype == F32) return fn<float>(__VA_ARGS__); if (dtype == BF16) return fn<__nv_bfloat16>(__VA_ARGS__); return fn<__half>(__VA_ARGS__); }
int lce_tile_columns(int dtype, const LceArgs& a) { return lce_sm100_takes(dtype, a) ? LCE_SM100_COLUMNS : CT; }
int64_t lce_scratch(int dtype, const LceArgs& a, bool dx, bool dw) { return dx && lce_sm100_takes(dtype, a) ? lce_sm100_scratch(a.rows, a.V, a.D, dw) : 0; }
int lce_logits(int dtype, const LceArgs& a, int* err, cudaStream_t st) {
    if (lce_sm100_takes(dtype, a)) return lce_sm100_logits(dtype, a, err, st);
    SG_LCE_GO(logits, a, st)
}
int lce_rows(int dtype, const LceArgs& a, cudaStream_t st) SG_LCE_GO(rows, a, lce_tile_columns(dtype, a), st)
int lce_grads(int dtype, const LceArgs& a, const LceGrads& g, float* scratch, int* err, cudaStream_t st) {
    if (lce_sm100_takes(dtype, a)) return lce_sm100_grads(dtype, a, g, scratch, err, st);
    if (dtype == F32) return grads<float, float>(a, g, st);
    if (dtype == BF16) return g.f32_out ? grads<__nv_bfloat16, float>(a, g, st) : grads<__nv_bfloat16, __nv_bfloat16>(a, g, st);
    return g.f32_out ? grads<__half, float>(a, g, st) : grads<__half, __half>(a, g, st);
}
#undef SG_LCE_GO
int lce_finish(int dtype, const float* in, void* out, int64_t n, const float* gout, const float* inv, cudaStream_t st) {
    if (n == 0) return 0;
    const int64_t want = (n / 4 + 255) / 256 + 1;
    const int grid = (int)(want < 148 * 8 ? want : 148 * 8);
    count_launch();
    if (dtype == F32) lce_finish_kernel<float><<<grid, 256, 0, st>>>(in, (float*)out, n, gout, inv);
    else if (dtype == BF16) lce_finish_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(in, (__nv_bfloat16*)out, n, gout, inv);
    else lce_finish_kernel<__half><<<grid, 256, 0, st>>>(in, (__half*)out, n, gout, inv);
    return cudaGetLastError() == cudaSuccess ? 0 : 3;
}

}  // namespace sg
