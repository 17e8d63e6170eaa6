// launch.cuh -- launches of the operators beside the DiT, chained by
// programmatic dependent launch.
//
// Every such kernel calls chain_begin() before it touches global memory: it
// lets the next kernel of the stream be set up (its CTAs take their places as
// these leave) and waits until the kernels before it have finished and their
// writes are visible.  A run of them saves the 2 us that a launch after a
// finished kernel costs; after a kernel that does not take part the wait is
// over at once.  What these kernels read was written by others while they were
// already running, so no load is a read-only one (__ldg, const __restrict__):
// those promise data that stays the same for the kernel's whole life.
#pragma once
#include <cuda_runtime.h>

namespace s2b {

__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void chain_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void chain_begin() {
    chain_release();
    chain_wait();
}

// 1 (kernel launched), or -1 - the CUDA error that refused it.  cluster: CTAs a
// cluster (0: none).
template <typename... P, typename... A>
int launch_chained(void (*f)(P...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, f, static_cast<P>(args)...);
    return e == cudaSuccess ? 1 : -1 - (int)e;
}

}  // namespace s2b
