// Launches of kernels that start while the kernel before them on the stream still runs (programmatic dependent launch): blocks
// set up their barriers and tensor memory meanwhile, and stop in `await_inputs` before they touch global memory, until
// everything launched before has ended and can be seen.  A chain of small products gains the gap between kernels, about 1 us
// each.  Every thread of such a kernel calls await_inputs, so that its end is also that of all before it.
#pragma once
#include <cuda_runtime.h>

#include "common.cuh"

namespace vi {

__device__ __forceinline__ void await_inputs() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// From here on (for the last block to get here) the next kernel may be set up beside this one.  Called when a block's loads
// are done: earlier, the next kernel's blocks would take the room that is free at the moment and lie unevenly on the SMs.
__device__ __forceinline__ void release_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// `cluster` blocks to a cluster; without `early` the kernel starts when those before it have ended.
template <typename... Params, typename... Args>
int launch_early(const char* what, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, int cluster, bool early, cudaStream_t st, Args... args) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = early ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {(unsigned)cluster, 1, 1};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
    return e == cudaSuccess ? VI_OK : fail(VI_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
}

}  // namespace vi
