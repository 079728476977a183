// exl3b200_chain.cuh -- kernels that follow one another on a stream: each may be launched while its predecessor ends, so
// that its launch and set-up run under the predecessor's last work. A kernel waits for the predecessor's end, and for all
// that it wrote, before it touches any memory but its own (every thread does, so that its own end implies the
// predecessor's); after a kernel that does not give way early, or an operation of another kind, the stream's usual order
// holds. sm_100a only.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace exl3b {

// The stream's earlier work is done and visible from here on.
__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// The next kernel's CTAs may be scheduled where there is room once every CTA of this grid has come here (or left).
__device__ __forceinline__ void chain_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// cluster: CTAs of a cluster along x.
template <typename... P, typename... A>
int chain_launch(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...) == cudaSuccess ? 0 : -6;
}

}  // namespace exl3b
