// Launches whose setup overlaps the end of the kernel before them in the stream (programmatic stream
// serialisation).
//
// A kernel launched by launch_overlapped() calls overlap_begin() in every thread before it touches
// global memory: that waits until the kernels before it have completed and their writes are visible,
// then lets the next kernel in the stream be set up in the same way.  Every CTA waits, so a kernel's
// completion still implies that of everything before it.  Kernels launched without the attribute,
// before or after, order as ever.  It takes one to three microseconds off each launch in a stream
// that runs one kernel after the other, which is what a layer does.
//
// Such a kernel exists while its inputs may still be written, so they are not constant for its lifetime:
// the read-only path (ld.global.nc, by __ldg or by const __restrict__ parameters) is closed to it.  It reads
// them with ld_input() and ld_input_once() below, with plain loads through pointers without __restrict__, or with
// cp.async and TMA; none of these can be moved in front of the wait.  Plain loads are for elements behind a
// condition, which the compiler can predicate then ([8192, 4001] bf16 GELU with its checkpoint 46 us, with
// ld_input 54).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace hc {

__device__ __forceinline__ void overlap_begin() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Loads of 1 to 16 bytes from global memory.  Volatile, so they stay behind the wait; without a memory clobber, so
// that they need not wait for the kernel's own stores, which never go to its inputs.
template <typename T>
__device__ __forceinline__ T ld_input(const T* p) {
    const size_t at = __cvta_generic_to_global(p);
    if constexpr (sizeof(T) == 16) {
        uint4 v;
        asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
        return *reinterpret_cast<const T*>(&v);
    } else if constexpr (sizeof(T) == 4) {
        uint32_t v;
        asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(at));
        return *reinterpret_cast<const T*>(&v);
    } else if constexpr (sizeof(T) == 2) {
        uint16_t v;
        asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(at));
        return *reinterpret_cast<const T*>(&v);
    } else {
        static_assert(sizeof(T) == 1, "1, 2, 4 or 16 bytes");
        uint32_t v;
        asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(at));
        const uint8_t b = static_cast<uint8_t>(v);
        return *reinterpret_cast<const T*>(&b);
    }
}
// The same for data that is read once (evicted first).
template <typename T>
__device__ __forceinline__ T ld_input_once(const T* p) {
    const size_t at = __cvta_generic_to_global(p);
    if constexpr (sizeof(T) == 16) {
        uint4 v;
        asm volatile("ld.global.cs.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
        return *reinterpret_cast<const T*>(&v);
    } else if constexpr (sizeof(T) == 8) {
        uint2 v;
        asm volatile("ld.global.cs.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(at));
        return *reinterpret_cast<const T*>(&v);
    } else {
        static_assert(sizeof(T) == 4, "4, 8 or 16 bytes");
        uint32_t v;
        asm volatile("ld.global.cs.u32 %0, [%1];" : "=r"(v) : "l"(at));
        return *reinterpret_cast<const T*>(&v);
    }
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
