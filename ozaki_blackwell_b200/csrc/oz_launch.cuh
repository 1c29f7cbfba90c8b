// oz_launch.cuh -- launches that may begin before the kernel in front of them in the stream has ended.
//
// A kernel launched by launch_behind() is set up while its predecessor runs out, and waits in behind_predecessors() -- which every
// thread calls before its first access to global memory -- until that has ended and its writes are visible. (Plain loads behind it: the
// read-only path is for data that does not change while the kernel is there.) Because every such kernel waits for its own
// predecessor, the end of one implies the end of all before it. Saves about 1 us a kernel in a chain of short ones.
#pragma once
#include <cuda_runtime.h>

namespace ozk {

__device__ __forceinline__ void behind_predecessors() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

inline int multiprocessors() {   // of the current device
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev)) cudaGetLastError();
    return n;
}

template <class... P, class... A>
cudaError_t launch_behind(void (*kernel)(P...), int grid, int block, size_t smem, int cluster, cudaStream_t st, A &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)block);
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
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

}  // namespace ozk
