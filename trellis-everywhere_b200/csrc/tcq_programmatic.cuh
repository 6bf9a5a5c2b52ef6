// Kernels that begin while the one before them in their stream ends: what they do before they wait for it costs no time.
//
// Every kernel launched this way waits (wait_for_kernel_before) before it reads or writes global memory that another kernel may have to do with, and only then lets the next one begin
// (launch_dependents): when a kernel begins, all but the one right before it have ended, and when its wait is over, that one too.
//
// Such a kernel lives while others still write what it reads, so nothing in it is read by read-only loads (`.nc`, which are defined for memory that nobody writes while the kernel runs): behind the
// wait loads are ordinary ones, or `asm volatile`, which the compiler keeps behind it, and before the wait, of what kernels have written that have ended, relaxed ones of the GPU's scope, which
// no first-level cache answers with what it held before.
#pragma once

#include <cuda_runtime.h>

namespace tcq {

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ int load_before_wait(const int* p) {
    int v;
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
// For threads whose bulk or tensor loads read what a kernel before has written with ordinary stores; behind the wait.
__device__ __forceinline__ void fence_for_bulk_loads() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ void wait_for_kernel_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... Params, typename... Args>
cudaError_t launch_programmatic(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2] = {};
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = unsigned(cluster);
    attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = cluster > 0 ? 2 : 1;                  // 0: a kernel that takes no clusters
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace tcq
