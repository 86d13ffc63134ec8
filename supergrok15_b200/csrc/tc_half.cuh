// Helpers of the tensor-core kernels whose 16-bit operands are bf16 or fp16 and whose work is handed out on the device.
#pragma once
#include "tc_sm100.cuh"
#include <cuda_fp16.h>

namespace sg {
namespace tc {

constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct Half2;
template <> struct Half2<__nv_bfloat16> {
    static constexpr uint32_t FMT = 1;                                    // operand format of the instruction descriptor
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }
};
template <> struct Half2<__half> {
    static constexpr uint32_t FMT = 0;
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    static __device__ __forceinline__ float2 unpack(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
};
// instruction descriptor of kind::f16: fp32 accumulator, both operands of format FMT, b_mn = 1 when B is MN-major
__device__ __forceinline__ uint32_t idesc_f16(uint32_t fmt, int M, int N, int b_mn) {
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void fma2(float x0, float x1, float a0, float a1, float b0, float b1, float& y0, float& y1) {
    asm("{\n\t.reg .b64 vx, va, vb, vy;\n\tmov.b64 vx, {%2, %3};\n\tmov.b64 va, {%4, %5};\n\tmov.b64 vb, {%6, %7};\n\t"
        "fma.rn.f32x2 vy, vx, va, vb;\n\tmov.b64 {%0, %1}, vy;\n\t}"
        : "=f"(y0), "=f"(y1) : "f"(x0), "f"(x1), "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <int N> __device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Cluster launch control: ask for a CTA of this grid that has not started; its index comes back as 16 bytes in shared memory.
__device__ __forceinline__ void clc_ask(uint4* answer, uint64_t* bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool clc_answer(const uint4* answer, int& item) {
    uint32_t got, x;
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b128 a;\n\tld.shared.b128 a, [%2];\n\t"
                 "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, a;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
                 "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, a;\n\t}"
                 : "=r"(got), "=r"(x) : "r"(smem_u32(answer)) : "memory");
    item = (int)x;
    return got != 0;
}

__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                   "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}

// Operand descriptors in two words: everything but the address is the same for every tile, and the address is the lowest field of the lower word,
// so the step from one product to the next is one addition.  One thread issues all products of a CTA, and what it computes between two of
// them delays the tensor cores: with descriptors put together for every product it needed 130 clocks per product of 64.
struct Desc {
    uint32_t lo, hi;
};
__device__ __forceinline__ Desc desc_of(uint64_t d) { return {(uint32_t)d, (uint32_t)(d >> 32)}; }
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\tsetp.ne.b32 p, %6, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}"
                 ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
                 ::"r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate) : "memory");
}

// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// One arrival for a whole warp (barriers count warps): 4 to 16 arrivals at a barrier instead of 128 to 512.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
// a wait of a whole warp that ends the same way for every lane
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); }

}  // namespace tc
}  // namespace sg
