// Launching the short kernels of a recording back to back.
#pragma once
#include <cuda_runtime.h>

#include <utility>

namespace nu {

// Small kernels are launched so that their blocks may be placed while the operator before them drains; each starts
// with griddepcontrol.wait, after which the earlier operator's writes are visible, so nothing else changes. Saves part
// of the launch latency between short dependent kernels.
template <typename... KArgs, typename... Args>
static void launch_after_previous_smem(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args &&...args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}
template <typename... KArgs, typename... Args>
static void launch_after_previous(void (*kernel)(KArgs...), dim3 grid, dim3 block, cudaStream_t s, Args &&...args) {
    launch_after_previous_smem(kernel, grid, block, 0, s, std::forward<Args>(args)...);
}
__device__ __forceinline__ void wait_for_previous_operator() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
}

}  // namespace nu
