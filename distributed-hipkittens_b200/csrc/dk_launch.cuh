// Launches that may begin while the kernel before them on the stream still runs (programmatic stream
// serialization). The rules that make this invisible to a caller:
//   - every thread that reads or writes global memory passes previous_done() first (or hangs, through a barrier in
//     shared memory, on a thread that has), and every CTA passes it: when it returns, all kernels before this one on
//     the stream are complete and what they wrote is visible;
//   - before it a kernel only sets itself up. A kernel whose predecessor is known (one of the same call) may also load
//     what that predecessor does not write, provided the predecessor says next_may_begin() after its own
//     previous_done(): said earlier, kernels before the predecessor may still be running;
//   - next_may_begin() says that the following kernel may set itself up too. A kernel that was not launched in this
//     way starts after the end of this one, as ever.
// After anything but a kernel (a copy, an event of another stream) the boundary is a full one.
#pragma once
#include <cuda_runtime.h>

#include "dk_host.h"

namespace dk {

__device__ __forceinline__ void next_may_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void previous_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
int launch_early(void (*kernel)(P...), dim3 grid, int threads, int smem, int cluster, cudaStream_t st, A&&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    DK_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
    return DK_OK;
}

}  // namespace dk
