// pdl.cuh -- programmatic dependent launch of the decoder operators' kernels.
//
// Each kernel lets the next one start as soon as its own CTAs have started (pdl_trigger; one that
// uses tensor memory: as soon as they have allocated it) and touches global memory only after everything before it in the stream has finished (pdl_wait),
// so a launch's own latency overlaps the kernel before it and results are those of plain stream
// order.  Kernels launched without the attribute are unaffected.
#pragma once

#include "ql_common.cuh"

namespace ql {

__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// cluster > 1: that many CTAs along x form a cluster.
template <typename... P, typename... A>
static cudaError_t launch_pdl(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, unsigned cluster,
                              const A &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

}  // namespace ql
