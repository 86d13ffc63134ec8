// Softmax cross-entropy of a linear head, z = x w^T, that never holds the logits:
//
//   loss = mean over counted rows of lse_r - z_{r,t_r},  lse_r = log sum_v exp z_rv
//   d_rv = p_rv - [v = t_r],  p_rv = exp(z_rv - lse_r);   dx = f d w,  dw = f d^T x,  f = gout / count
//
// Rows without a counted target are left out first (lce_gather copies the others together): half of a fine-tuning batch is prompt, and what
// stands there (padding, NaN) cannot reach a product.  The rows go through in pieces.  (1) lce_logits: the product, tile by tile; a tile's
// epilogue leaves, per row, a reference r and the sum of u = 2^(z log2 e - r), and, for a training pass, u itself in the type of x: the
// logits have been consumed when the tile's accumulators are free.  (2) lce_rows: the statistics give the loss and the row's scale s, with
// which d = s u 2^(r - r_row).  The sums leave out the target's column: with s' the sum of the others and e_t the target's term,
// 1 - p_t = s' / (s' + e_t) and the loss of a likely target is log1p(s' / e_t), both to full precision however certain the target is
// (p_t - 1 from a rounded p_t, or lse - z_t, would be rounding noise).  (3) lce_grads: both products with d; (4) lce_scatter puts the rows
// of dx back.
//
// fp16 and fp32: r is the tile's maximum and lce_rows turns u into d in place.  bf16 has the exponents of fp32, so r need not follow the
// maximum: it is 0 while the tile's largest |z| stays below 64 log 2 = 44, else the nearest multiple of 64 powers of two.  All tiles of nearly
// every row then share one reference, u needs no second pass, and s moves into the products: dx = s (u w) in the epilogue, dw = u^T (s x)
// with the rows of x scaled in place (tiles with another reference are rescaled, by a power of two, exactly).  8,188 x 32,000: 256 us of
// reading and writing u become 29.  Between z and a product stand at most two roundings to 16 bits (u and d, or u and s x), each at
// most half a step of the value itself.
//
// Against a pass that recomputes z for the gradient this saves a fourth of all products (6 N V D operations instead of 8) and costs
// reading and writing u once more.
//
// Every kernel behind lce_gather is launched early; the passes over rows let the next one in at once, the tensor-core products, which leave no
// room for another CTA, when they end (13 rows x 32,000 x 2,048: 108 -> 100 us).
//
// This file: the passes over the rows, and products on the CUDA cores for fp32 operands and for 16-bit ones that TMA cannot address.  Their
// 128 x 128 tiles take 8 x 8 outputs per thread in steps of 16, the next step's operands on their way to registers under this one's
// products; two fused multiply-adds per instruction (packed pairs), four 16-byte loads from shared memory for 64 of them.
#include "sg_native.h"
#include "optim_math.cuh"
#include "linear_ce.h"
#include "per_device.h"
#include "launch_early.cuh"
#include <cfloat>

namespace sg {
namespace {

constexpr int CT = 128, CK = 16, CTHREADS = 256;
using Pair = unsigned long long;                                          // two fp32 values

__device__ __forceinline__ Pair twice(float a) {
    Pair p;
    asm("mov.b64 %0, {%1, %1};" : "=l"(p) : "f"(a));
    return p;
}
__device__ __forceinline__ float2 both(Pair p) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ void fma_pair(Pair& acc, Pair a, Pair b) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b)); }

// A step's operand, 128 indices x 16 of k: two vectors of four per thread, from memory in which the index (IM) or k is contiguous
template <typename T, bool IM> struct StepLoad {
    float v[2][4];
    // vec: rows start on 16 bytes and the contiguous extent is whole fours (fp32)
    __device__ __forceinline__ void load(const T* p, int64_t ld, bool vec, int i0, int I, int k0, int K) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int q = threadIdx.x + u * CTHREADS;
            const int i = i0 + (IM ? (q & 31) * 4 : q >> 2), k = k0 + (IM ? q >> 5 : (q & 3) * 4);
            const T* src = IM ? p + (int64_t)k * ld + i : p + (int64_t)i * ld + k;
            const bool row = IM ? k < K : i < I;
            if (sizeof(T) == 4 && vec) {
                const float4 f = row && (IM ? i < I : k < K) ? __ldcg(reinterpret_cast<const float4*>(src)) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[u][0] = f.x; v[u][1] = f.y; v[u][2] = f.z; v[u][3] = f.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[u][e] = row && (IM ? i + e < I : k + e < K) ? Cvt<T>::to(__ldcg(src + e)) : 0.f;
            }
        }
    }
    __device__ __forceinline__ void store(float (*s)[CT + 4]) const {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int q = threadIdx.x + u * CTHREADS;
            if (IM) *reinterpret_cast<float4*>(&s[q >> 5][(q & 31) * 4]) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) s[(q & 3) * 4 + e][q >> 2] = v[u][e];
        }
    }
};

// Whether an operand's rows can be read four at a time; n: its contiguous extent
__device__ __forceinline__ bool fours(const void* p, int64_t ld, int n) { return ((reinterpret_cast<uintptr_t>(p) & 15) | (ld & 3) | (n & 3)) == 0; }

// M, KA: extents of A (u is zero from V to its pitch, so that its rows can be read to whole fours); N: of B, whose k ends with k1.
// acc[i][j] += sum over [k0, k1) of A(m, k) B(n, k), m = m0 + row(i), n = n0 + 4 tx + 64 (j / 2) + 2 (j % 2) and the next; row(i) = 4 ty + i % 4 + 64 (i / 4)
template <typename T, bool AM, bool BN>
__device__ __forceinline__ void tile_product(const T* A, int64_t lda, const T* B, int64_t ldb, int M, int KA, int N, int k0, int k1, int m0, int n0, Pair (&acc)[8][4]) {
    __shared__ __align__(16) float sa[2][CK][CT + 4], sb[2][CK][CT + 4];
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const bool va = fours(A, lda, AM ? M : KA), vb = fours(B, ldb, BN ? N : k1);
    StepLoad<T, AM> la;
    StepLoad<T, BN> lb;
    la.load(A, lda, va, m0, M, k0, KA); lb.load(B, ldb, vb, n0, N, k0, k1);
    la.store(sa[0]); lb.store(sb[0]);
    __syncthreads();
    int cur = 0;
    for (int k = k0; k < k1; k += CK, cur ^= 1) {
        const bool more = k + CK < k1;
        if (more) { la.load(A, lda, va, m0, M, k + CK, KA); lb.load(B, ldb, vb, n0, N, k + CK, k1); }
#pragma unroll
        for (int kk = 0; kk < CK; ++kk) {
            const float4 a0 = *reinterpret_cast<const float4*>(&sa[cur][kk][ty * 4]), a1 = *reinterpret_cast<const float4*>(&sa[cur][kk][64 + ty * 4]);
            const ulonglong2 b0 = *reinterpret_cast<const ulonglong2*>(&sb[cur][kk][tx * 4]), b1 = *reinterpret_cast<const ulonglong2*>(&sb[cur][kk][64 + tx * 4]);
            const float av[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const Pair aa = twice(av[i]);
                fma_pair(acc[i][0], aa, b0.x); fma_pair(acc[i][1], aa, b0.y); fma_pair(acc[i][2], aa, b1.x); fma_pair(acc[i][3], aa, b1.y);
            }
        }
        if (more) { la.store(sa[cur ^ 1]); lb.store(sb[cur ^ 1]); }
        __syncthreads();
    }
}
__device__ __forceinline__ int tile_row(int i) { return (int)(threadIdx.x >> 4) * 4 + (i & 3) + 64 * (i >> 2); }
__device__ __forceinline__ int tile_col(int j) { return (int)(threadIdx.x & 15) * 4 + (j & 3) + 64 * (j >> 2); }
__device__ __forceinline__ void row_of(const Pair (&acc)[4], float (&s)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) { const float2 v = both(acc[j]); s[2 * j] = v.x; s[2 * j + 1] = v.y; }
}

template <typename T>
__global__ void __launch_bounds__(CTHREADS, 2) lce_logits_kernel(LceArgs a) {
    after_previous();
    const int m0 = blockIdx.y * CT, n0 = blockIdx.x * CT, tx = threadIdx.x & 15, rows = lce_active(a);
    if (m0 >= rows) return;
    Pair acc[8][4] = {};
    tile_product<T, false, false>((const T*)a.x, a.ldx, (const T*)a.w, a.ldw, rows, a.D, a.V, 0, a.D, m0, n0, acc);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = m0 + tile_row(i);
        const int64_t t = row < rows ? a.target[row] : -1;
        float s[8], mx = -INFINITY;
        row_of(acc[i], s);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int v = n0 + tile_col(j);
            if (v >= a.V) s[j] = -INFINITY;
            else if (v == t) a.z_target[row] = s[j];
            s[j] *= 1.4426950408889634f;                                  // from here on in powers of two
            mx = fmaxf(mx, s[j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float ref = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int v = n0 + tile_col(j);
            const float e = exp2f(s[j] - ref);
            if (v != t) sum += e;
            if (a.u && row < rows && v < a.V) ((T*)a.u)[(int64_t)row * a.ldu + v] = Cvt<T>::from(e * LceUnit<T>::value);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (tx == 0 && row < rows) a.stats[(int64_t)row * gridDim.x + blockIdx.x] = make_float2(mx, sum);
    }
}

// dx (AM = false: d [rows, V] times w [V, D], part blockIdx.z of the sum) or dw (AM = true: d^T times x [rows, D]).  Behind dx, dw starts as dx's
// CTAs leave their SMs: every one of them has seen the end of the row pass, and what that wrote is read from L2.  It waits for the whole of dx
// at its end, for what comes behind both.
template <typename T, typename TO, bool AM>
__global__ void __launch_bounds__(CTHREADS, 2) lce_grad_kernel(LceArgs a, const float* prev, TO* out, int64_t row_pitch, const float* gout, const float* inv, bool behind_dx) {
    if (!behind_dx) after_previous();
    if (!AM) let_next_start();
    const int m0 = blockIdx.y * CT, n0 = blockIdx.x * CT, rows = lce_active(a);
    const int M = AM ? a.V : rows;
    if (m0 >= M) return;                                                  // never all CTAs of dw
    Pair acc[8][4] = {};
    if (AM) tile_product<T, true, true>((const T*)a.u, a.ldu, (const T*)a.x, a.ldx, (int)a.ldu, rows, a.D, 0, rows, m0, n0, acc);
    else {
        const int per = ((a.V + (int)gridDim.z - 1) / (int)gridDim.z + CK - 1) / CK * CK, k0 = per * (int)blockIdx.z;
        out += (int64_t)blockIdx.z * row_pitch * a.D;
        if (k0 < a.V) tile_product<T, false, true>((const T*)a.u, a.ldu, (const T*)a.w, a.ldw, rows, min(k0 + per, (int)a.ldu), a.D, k0, min(k0 + per, a.V), m0, n0, acc);
    }
    const float f = gout ? gout[0] * inv[0] / LceUnit<T>::value : 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int m = m0 + tile_row(i);
        float s[8];
        row_of(acc[i], s);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int n = n0 + tile_col(j);
            if (m < M && n < a.D) out[(int64_t)m * a.D + n] = Cvt<TO>::from(f * (prev ? s[j] + prev[(int64_t)m * a.D + n] : s[j]));
        }
    }
    if (behind_dx) after_previous();
}

constexpr int ROW_THREADS = 256;
__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROW_THREADS / 32; ++i) v = fmaxf(v, red[i]);
    return v;
}
// the sum in every thread, added in a fixed order
__device__ __forceinline__ float block_total(float v, float* red) {
    v = block_sum(v, red);                                                // in the first warp
    __syncthreads();
    if (threadIdx.x == 0) red[0] = v;
    __syncthreads();
    return red[0];
}

// A row from its reference, the sum of the other columns' terms 2^(z log2 e - top) and the target's logit
struct RowTerms {
    float et, loss;
};
__device__ __forceinline__ RowTerms row_terms(float top, float others, float zt) {
    const float below = zt * 1.4426950408889634f - top, et = exp2f(below);
    // far below the others e_t loses digits and then vanishes, and the plain difference is exact enough
    return {et, et > 1e-6f * others ? log1pf(others / et) : logf(others + et) - below * 0.6931471805599453f};
}

// The CTA that finishes last adds up the losses of all pieces, in a fixed order.
__device__ __forceinline__ void last_adds(const LceArgs& a, float* red) {
    __shared__ bool is_last;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        is_last = atomicAdd(a.done, 1u) + 1 == gridDim.x * gridDim.y;
    }
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    const int n = *a.count;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = threadIdx.x; i < n; i += 4 * ROW_THREADS)
#pragma unroll
        for (int k = 0; k < 4; ++k) if (i + k * ROW_THREADS < n) s[k] += __ldcg(a.loss_all + i + k * ROW_THREADS);
    const float total = block_total((s[0] + s[1]) + (s[2] + s[3]), red), inv = 1.f / (n > 0 ? n : 1);
    if (threadIdx.x == 0) { *a.out_loss = total * inv; *a.inv_count = inv; }
}

// Training: the loss of a row from its tiles' statistics, then u -> d in place, two pieces of 16 bytes in flight per thread (4,096 rows of
// 32,000 columns, one in flight: 110 us, 4.7 TB/s).  A row is cut over gridDim.y CTAs when there are few (13 rows: 11.6 us by one CTA each);
// every one of them adds up the statistics, which are a hundredth of the row.
template <typename T> __device__ __forceinline__ uint4 scaled(uint4 raw, float f) {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int k = 0; k < 16 / (int)sizeof(T); ++k) e[k] = Cvt<T>::from(Cvt<T>::to(e[k]) * f);
    return raw;
}
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) lce_rows_kernel(LceArgs a, int tiles, bool last) {
    let_next_start();
    after_previous();
    extern __shared__ float fac[];                                        // [tiles] factor of a tile's columns
    __shared__ float red[32];
    constexpr int PER = 16 / sizeof(T), STEP = ROW_THREADS * PER;
    const int row = blockIdx.x, rows = lce_active(a);
    const int slice = (int)((a.ldu / PER + gridDim.y - 1) / gridDim.y) * PER, c0 = blockIdx.y * slice, c1 = min((int64_t)(c0 + slice), a.ldu);
    T* u = (T*)a.u + (int64_t)row * a.ldu;
    if (row < rows) {
        const float2* st = a.stats + (int64_t)row * tiles;
        float mx = -INFINITY;
        for (int i = threadIdx.x; i < tiles; i += ROW_THREADS) { fac[i] = st[i].x; mx = fmaxf(mx, fac[i]); }
        mx = block_max(mx, red);
        const float top = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f;
        for (int i = threadIdx.x; i < tiles; i += ROW_THREADS) { fac[i] = exp2f(fac[i] - top); sum += st[i].y * fac[i]; }
        const float others = block_total(sum, red);                       // without the target's column
        const int t = (int)a.target[row];
        const RowTerms rt = row_terms(top, others, a.z_target[row]);
        const float inv = 1.f / (others + rt.et), at_target = -others * inv * LceUnit<T>::value;
        if (threadIdx.x == 0 && blockIdx.y == 0) a.loss[row] = rt.loss;
        for (int c = c0 + threadIdx.x * PER; c < c1; c += 2 * STEP) {     // PER divides a tile's columns
            const int c2 = c + STEP;
            const uint4 x = *reinterpret_cast<const uint4*>(u + c), y = c2 < c1 ? *reinterpret_cast<const uint4*>(u + c2) : make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(u + c) = scaled<T>(x, fac[min(c / LCE_COLUMNS, tiles - 1)] * inv);
            if (c2 < c1) *reinterpret_cast<uint4*>(u + c2) = scaled<T>(y, fac[min(c2 / LCE_COLUMNS, tiles - 1)] * inv);
        }
        __syncthreads();
        if (threadIdx.x == 0 && t >= c0 && t < c1) u[t] = Cvt<T>::from(at_target);
        if (c1 > a.V) for (int c = max(c0, a.V) + (int)threadIdx.x; c < c1; c += ROW_THREADS) u[c] = Cvt<T>::from(0.f);      // columns between V and the pitch meet zeros of w
    } else if (row < (rows + 63) / 64 * 64) {                              // the products take rows in steps of 64
        for (int c = c0 + threadIdx.x * PER; c < c1; c += STEP) *reinterpret_cast<uint4*>(u + c) = make_uint4(0u, 0u, 0u, 0u);
    }
    if (last) last_adds(a, red);
}

// Evaluation: a warp per row.
__global__ void __launch_bounds__(ROW_THREADS) lce_row_losses_kernel(LceArgs a, int tiles, bool last) {
    let_next_start();
    after_previous();
    __shared__ float red[32];
    const int row = blockIdx.x * (ROW_THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row < lce_active(a)) {
        const float2* st = a.stats + (int64_t)row * tiles;
        float mx = -INFINITY, sum = 0.f;
        for (int i = lane; i < tiles; i += 32) mx = fmaxf(mx, st[i].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float top = mx == -INFINITY ? 0.f : mx;
        for (int i = lane; i < tiles; i += 32) sum += st[i].y * exp2f(st[i].x - top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) a.loss[row] = row_terms(top, sum, a.z_target[row]).loss;
    }
    if (last) last_adds(a, red);
}

// Training in bf16: a warp per row.  The loss and the row's scale; the target's entry of u; the tiles with another reference than the row's;
// the row of x times the scale, in place (nothing else reads it any more).
__global__ void __launch_bounds__(ROW_THREADS) lce_scale_rows_kernel(LceArgs a, int tiles, bool last) {
    let_next_start();
    after_previous();
    constexpr int XV = 4;
    __shared__ float red[32];
    const int row = blockIdx.x * (ROW_THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row < lce_active(a)) {
        const float2* st = a.stats + (int64_t)row * tiles;
        uint4* x = reinterpret_cast<uint4*>((__nv_bfloat16*)a.x + (int64_t)row * a.ldx);      // D is a multiple of 8 here
        uint4 v[XV];                                                      // the first pieces are on their way while the scale is found
#pragma unroll
        for (int k = 0; k < XV; ++k) if (lane + 32 * k < a.D / 8) v[k] = x[lane + 32 * k];
        float mx = -INFINITY, mn = INFINITY, sum = 0.f;
#pragma unroll 4
        for (int i = lane; i < tiles; i += 32) { const float r = st[i].x; mx = fmaxf(mx, r); mn = fminf(mn, r); }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o)); mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o)); }
#pragma unroll 4
        for (int i = lane; i < tiles; i += 32) sum += st[i].y * exp2f(st[i].x - mx);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const RowTerms rt = row_terms(mx, sum, a.z_target[row]);
        const float s = 1.f / (sum + rt.et);
        __nv_bfloat16* u = (__nv_bfloat16*)a.u + (int64_t)row * a.ldu;
        if (mn != mx)
            for (int i = 0; i < tiles; ++i) {
                const float r = st[i].x;
                if (r == mx) continue;
                const float f = exp2f(r - mx);
                for (int c = i * LCE_COLUMNS + lane; c < (i + 1) * LCE_COLUMNS && c < a.V; c += 32) u[c] = __float2bfloat16_rn(__bfloat162float(u[c]) * f);
            }
        __syncwarp();
        if (lane == 0) {
            a.loss[row] = rt.loss;
            a.row_scale[row] = s;
            u[a.target[row]] = __float2bfloat16_rn(-sum);
        }
#pragma unroll 1
        for (int c = lane; c < a.D / 8; c += 32 * XV) {
            if (c != lane)
#pragma unroll
                for (int k = 0; k < XV; ++k) if (c + 32 * k < a.D / 8) v[k] = x[c + 32 * k];
#pragma unroll
            for (int k = 0; k < XV; ++k) if (c + 32 * k < a.D / 8) x[c + 32 * k] = scaled<__nv_bfloat16>(v[k], s);
        }
    }
    if (last) last_adds(a, red);
}

// ---- the counted rows
constexpr int GATHER_ROWS = 16, COUNT_ROWS = 4096, GATHER_DIRECT = 16384;
__device__ __forceinline__ bool counted(int64_t t, int64_t ignore_index, int V) { return t != ignore_index && t >= 0 && t < V; }

// blocks[b] = counted rows among [4096 b, 4096 (b + 1))
__global__ void __launch_bounds__(256) lce_count_kernel(const int64_t* __restrict__ target, int64_t ignore_index, int rows, int V, int* __restrict__ blocks) {
    int n = 0;
    for (int i = threadIdx.x; i < COUNT_ROWS; i += 256) {
        const int r = blockIdx.x * COUNT_ROWS + i;
        if (r < rows && counted(target[r], ignore_index, V)) ++n;
    }
    n = __reduce_add_sync(0xffffffffu, n);
    __shared__ int sh[8];
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = n;
    __syncthreads();
    if (threadIdx.x == 0) { int s = 0; for (int i = 0; i < 8; ++i) s += sh[i]; blocks[blockIdx.x] = s; }
}

// A CTA moves the counted ones of 16 rows: it counts the rows before its own (all of them up to 16,384 rows, else those of the
// 4,096-row block it lies in, on top of the blocks' counts), so the order is kept and no CTA waits for another.
__global__ void __launch_bounds__(256) lce_gather_kernel(const uint8_t* __restrict__ x, int64_t pitch, const int64_t* __restrict__ target, int64_t ignore_index, int rows,
                                                         int V, int row_bytes, int row_pitch, int vec, int* __restrict__ place, uint8_t* __restrict__ xc, int64_t* __restrict__ tc,
                                                         int* __restrict__ count, unsigned* __restrict__ done, const int* __restrict__ blocks) {
    let_next_start();
    __shared__ int sh[8], base;
    __shared__ int to[GATHER_ROWS];
    const int r0 = blockIdx.x * GATHER_ROWS, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int n = 0, from = 0;
    if (blocks) {
        from = r0 / COUNT_ROWS * COUNT_ROWS;
        for (int i = threadIdx.x; i < r0 / COUNT_ROWS; i += 256) n += blocks[i];
    }
#pragma unroll 8
    for (int r = from + threadIdx.x; r < r0; r += 256) n += counted(target[r], ignore_index, V) ? 1 : 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) sh[warp] = n;
    __syncthreads();
    if (warp == 0) {
        int b = 0;
        for (int i = 0; i < 8; ++i) b += sh[i];
        const int r = r0 + lane;
        const int64_t t = r < rows ? target[r] : -1;
        const bool on = lane < GATHER_ROWS && r < rows && counted(t, ignore_index, V);
        const unsigned m = __ballot_sync(0xffffffffu, on);
        const int p = on ? b + __popc(m & ((1u << lane) - 1)) : -1;
        if (lane < GATHER_ROWS) {
            to[lane] = p;
            if (r < rows) place[r] = p;
        }
        if (on) tc[p] = t;
        if (lane == 0) base = b + __popc(m);
    }
    __syncthreads();
    for (int i = warp; i < GATHER_ROWS; i += 8) {
        const int p = to[i];
        if (p < 0) continue;
        const uint8_t* src = x + (int64_t)(r0 + i) * pitch;
        uint8_t* dst = xc + (int64_t)p * row_pitch;
        if (vec) {
            for (int c = lane * 16; c < row_bytes; c += 8 * 512) {
                uint4 v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) if (c + k * 512 < row_bytes) v[k] = *reinterpret_cast<const uint4*>(src + c + k * 512);
#pragma unroll
                for (int k = 0; k < 8; ++k) if (c + k * 512 < row_bytes) *reinterpret_cast<uint4*>(dst + c + k * 512) = v[k];
            }
        } else for (int c = lane * 2; c < row_bytes; c += 64) *reinterpret_cast<uint16_t*>(dst + c) = *reinterpret_cast<const uint16_t*>(src + c);
    }
    if (blockIdx.x == gridDim.x - 1) {
        const int end = (base + 63) / 64 * 64 < rows ? (base + 63) / 64 * 64 : rows;
        for (int64_t i = (int64_t)base * row_pitch + 2 * threadIdx.x; i < (int64_t)end * row_pitch; i += 512) *reinterpret_cast<uint16_t*>(xc + i) = 0;
        if (threadIdx.x == 0) { *count = base; *done = 0u; }
    }
}

__global__ void __launch_bounds__(256) lce_add_parts_kernel(const float* part, int parts, int64_t pitch, int64_t n, float* out) {
    let_next_start();
    after_previous();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = 0.f;
        for (int k = 0; k < parts; ++k) s += part[k * pitch + i];
        out[i] = s;
    }
}

// A warp per row and 32 x PER columns (PER = 8, or 1 where a row is not a whole number of eights), the parts eight at a time
template <typename T, int PER>
__global__ void __launch_bounds__(256) lce_scatter_kernel(const int* place, int rows, int D, int first, const float* early, const float* part, int parts, int64_t row_pitch,
                                                          const float* gout, const float* inv, T* dx) {
    after_previous();
    const int pieces = (D + 32 * PER - 1) / (32 * PER), lane = threadIdx.x & 31;
    const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int row = (int)(item / pieces), c = (int)(item % pieces) * 32 * PER + lane * PER;
    if (row >= rows || c >= D) return;
    const int p = place[row];
    float v[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) v[k] = 0.f;
    if (p >= 0) {
        const float* src = p < first ? early + (int64_t)p * D + c : part + (int64_t)(p - first) * D + c;
        const int n = p < first ? 1 : parts;
        const float f = p < first ? gout[0] * inv[0] / LceUnit<T>::value : 1.f;
#pragma unroll 8
        for (int s = 0; s < n; ++s) {
            const float* q = src + s * row_pitch * D;
            if constexpr (PER == 8) {
                const float4 x = reinterpret_cast<const float4*>(q)[0], y = reinterpret_cast<const float4*>(q)[1];
                v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w; v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
            } else v[0] += q[0];
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) v[k] *= f;
    }
    T o[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) o[k] = Cvt<T>::from(v[k]);
    T* dst = dx + (int64_t)row * D + c;
    if constexpr (PER == 8) {
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(dst)[k] = reinterpret_cast<const uint4*>(o)[k];
    } else dst[0] = o[0];
}

template <typename T> int logits(const LceArgs& a, cudaStream_t st) {
    count_launch();
    return launch_early(lce_logits_kernel<T>, dim3((a.V + CT - 1) / CT, (a.rows + CT - 1) / CT), CTHREADS, 0, st, a) == cudaSuccess ? 0 : 3;
}

template <typename T> int rows(const LceArgs& a, bool last, cudaStream_t st) {
    const int tiles = (a.V + LCE_COLUMNS - 1) / LCE_COLUMNS;
    count_launch();
    if (!a.u) {
        return launch_early(lce_row_losses_kernel, dim3((a.rows + 7) / 8), ROW_THREADS, 0, st, a, tiles, last) == cudaSuccess ? 0 : 3;
    }
    if (a.row_scale) {
        return launch_early(lce_scale_rows_kernel, dim3((a.rows + 7) / 8), ROW_THREADS, 0, st, a, tiles, last) == cudaSuccess ? 0 : 3;
    }
    const size_t smem = tiles * sizeof(float);
    static std::atomic<uint64_t> done{0};
    if (!once_per_device(done, current_device(), [] { return cudaFuncSetAttribute(lce_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) == cudaSuccess; }))
        return 2;
    if (smem > 200 * 1024) return 4;
    const int cut = a.rows >= 2 * device_sms() ? 1 : (2 * device_sms() + a.rows - 1) / a.rows;
    return launch_early(lce_rows_kernel<T>, dim3(a.rows, cut < 8 ? cut : 8), ROW_THREADS, smem, st, a, tiles, last) == cudaSuccess ? 0 : 3;
}

template <typename T, typename TO> int grads(const LceArgs& a, const LceGrads& g, cudaStream_t st) {
    if (g.dx_part) {
        count_launch();
        if (launch_early(lce_grad_kernel<T, float, false>, dim3((a.D + CT - 1) / CT, (a.rows + CT - 1) / CT, g.parts), CTHREADS, 0, st, a, nullptr, g.dx_part, g.row_pitch,
                         g.gout, g.inv_count, false) != cudaSuccess) return 3;
    }
    if (g.dw) {
        count_launch();
        if (launch_early(lce_grad_kernel<T, TO, true>, dim3((a.D + CT - 1) / CT, (a.V + CT - 1) / CT), CTHREADS, 0, st, a, g.dw_prev, (TO*)g.dw, 0, g.gout, g.inv_count,
                         g.dx_part != nullptr) !=
            cudaSuccess) return 3;
    }
    return 0;
}

template <typename T>
int scatter(const int* place, int rows, int D, int first, const float* early, const float* part, int parts, int64_t row_pitch, const float* gout, const float* inv,
            void* dx, cudaStream_t st) {
    count_launch();
    const int cols = D % 8 == 0 ? 256 : 32;
    const unsigned grid = (unsigned)(((int64_t)rows * ((D + cols - 1) / cols) + 7) / 8);
    return launch_early(D % 8 == 0 ? lce_scatter_kernel<T, 8> : lce_scatter_kernel<T, 1>, dim3(grid), 256, 0, st, place, rows, D, first, early, part, parts, row_pitch, gout, inv,
                        (T*)dx) == cudaSuccess ? 0 : 3;
}

}  // namespace

#define SG_LCE_GO(fn, ...) { if (dtype == F32) return fn<float>(__VA_ARGS__); if (dtype == BF16) return fn<__nv_bfloat16>(__VA_ARGS__); return fn<__half>(__VA_ARGS__); }
static_assert(CT == LCE_COLUMNS, "a tile of the logits is a tile of the statistics");
bool lce_scales_rows(int dtype, const LceArgs& a) { return dtype == BF16 && lce_sm100_takes(dtype, a); }
int lce_dx_parts(int dtype, const LceArgs& a, bool with_dw, int64_t* row_pitch) {
    if (lce_sm100_takes(dtype, a)) return lce_sm100_dx_parts(a.rows, a.V, a.D, with_dw, row_pitch);
    // Two tiles per SM at a time: the parts (each at least 256 columns of the vocabulary) that give the shortest rounds, a tile's start and
    // end counted as 128 columns (28 tiles x 5,003 columns: eleven parts are a round and twelve tiles more, ten are one round)
    *row_pitch = a.rows;
    const int64_t tiles = (int64_t)((a.rows + CT - 1) / CT) * ((a.D + CT - 1) / CT), most = a.V / 256 < 64 ? a.V / 256 : 64;
    int best = 1;
    int64_t least = INT64_MAX;
    for (int64_t n = 1; n <= (most < 1 ? 1 : most); ++n) {
        const int64_t cost = (tiles * n + 2 * device_sms() - 1) / (2 * device_sms()) * ((a.V + n - 1) / n + 128);
        if (cost < least) { least = cost; best = (int)n; }
    }
    return best;
}
int lce_gather_blocks(int rows) { return rows > GATHER_DIRECT ? (rows + COUNT_ROWS - 1) / COUNT_ROWS : 0; }
int lce_gather(int dtype, const void* x, int64_t ldx, const int64_t* target, int64_t ignore_index, int rows, int V, int D, int* place, void* xc, int64_t* tc,
               int* count, unsigned* done, int* blocks, cudaStream_t st) {
    const int es = dtype == F32 ? 4 : 2, nb = lce_gather_blocks(rows);
    const int vec = ((reinterpret_cast<uintptr_t>(x) | (uintptr_t)(ldx * es) | (uintptr_t)(D * es)) & 15) == 0;
    if (nb) {
        count_launch();
        lce_count_kernel<<<nb, 256, 0, st>>>(target, ignore_index, rows, V, blocks);
    }
    count_launch();
    lce_gather_kernel<<<(rows + GATHER_ROWS - 1) / GATHER_ROWS, 256, 0, st>>>((const uint8_t*)x, ldx * es, target, ignore_index, rows, V, D * es, (int)lce_pitch(D, es) * es, vec, place, (uint8_t*)xc, tc,
                                                                            count, done, nb ? blocks : nullptr);
    return cudaGetLastError() == cudaSuccess ? 0 : 3;
}
int lce_logits(int dtype, const LceArgs& a, int* err, cudaStream_t st) {
    if (lce_sm100_takes(dtype, a)) return lce_sm100_logits(dtype, a, err, st);
    SG_LCE_GO(logits, a, st)
}
int lce_rows(int dtype, const LceArgs& a, bool last, cudaStream_t st) SG_LCE_GO(rows, a, last, st)
int lce_grads(int dtype, const LceArgs& a, const LceGrads& g, int* err, cudaStream_t st) {
    if (lce_sm100_takes(dtype, a)) return lce_sm100_grads(dtype, a, g, err, st);
    if (dtype == F32) return grads<float, float>(a, g, st);
    if (dtype == BF16) return g.f32_dw ? grads<__nv_bfloat16, float>(a, g, st) : grads<__nv_bfloat16, __nv_bfloat16>(a, g, st);
    return g.f32_dw ? grads<__half, float>(a, g, st) : grads<__half, __half>(a, g, st);
}
int lce_add_parts(const float* part, int parts, int64_t pitch, int64_t n, float* out, cudaStream_t st) {
    count_launch();
    return launch_early(lce_add_parts_kernel, dim3((unsigned)((n + 255) / 256 < 148 * 8 ? (n + 255) / 256 : 148 * 8)), 256, 0, st, part, parts, pitch, n, out) == cudaSuccess ? 0 : 3;
}
int lce_scatter(int dtype, const int* place, int rows, int D, int first, const float* early, const float* part, int parts, int64_t row_pitch, const float* gout,
                const float* inv_count, void* dx, cudaStream_t st) SG_LCE_GO(scatter, place, rows, D, first, early, part, parts, row_pitch, gout, inv_count, dx, st)
#undef SG_LCE_GO

}  // namespace sg
