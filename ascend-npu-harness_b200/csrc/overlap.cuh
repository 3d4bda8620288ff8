// Launches whose setup overlaps the end of the kernel before them in the stream (programmatic stream
// serialisation).
//
// A kernel launched by launch_overlapped() calls overlap_begin() in every thread before it touches
// global memory: that waits until the kernels before it have completed and their writes are visible,
// then lets the next kernel in the stream be set up in the same way.  Every CTA waits, so a kernel's
// completion still implies that of everything before it.  Kernels launched without the attribute,
// before or after, order as ever.  It takes one to three microseconds off each launch in a stream
// that runs one kernel after the other, which is what a layer does.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>

namespace hc {

__device__ __forceinline__ void overlap_begin() {
    cudaGridDependencySynchronize();
    cudaTriggerProgrammaticLaunchCompletion();
}

// cluster: CTAs per cluster along x, 0 for a kernel without clusters or with a compile-time size.
template <typename... Params, typename... Args>
void launch_overlapped(void (*kernel)(Params...), dim3 grid, unsigned block, size_t smem, unsigned cluster,
                       cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster;
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    cfg.attrs = attr;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
}

}  // namespace hc
