// Kernels that are launched programmatically: such a kernel may be set up while the one before it in the stream still runs, and touches
// nothing in global memory before after_previous() has seen all of that kernel (and, since that one waited too, of what came before it).  A
// kernel that starts without the wait, because what it reads comes from an earlier one, says at its place why it may, and waits at its end
// instead, for what comes behind it.
// What an earlier kernel wrote is therefore not read through the read-only path (no __ldg, no const __restrict__), whose loads the compiler
// may move.  let_next_start() lets the next kernel's CTAs in as soon as every CTA of this one has called it or ended.
#pragma once
#include <cuda_runtime.h>

namespace sg {

__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, const A&... args) {
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = st; cfg.attrs = &at; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

}  // namespace sg
