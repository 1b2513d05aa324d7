// Launches of kernels that may begin while the kernel before them ends.
#pragma once

#include "device.cuh"

namespace b200fft {

namespace {

// Programmatic dependent launch: what comes before this may run while the kernel before it ends.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Every kernel of the sequence operators may start while the one before it in the stream ends, and waits for that before
// its first access to what a kernel may have written (wait_for_previous, by every CTA: otherwise a grid could end before
// the one it follows).  That takes 2 us off the gap between two of them, and a launch costs 3.0 instead of 3.9 us.
template <typename Kernel, typename... Args>
cudaError_t launch(Kernel *kernel, dim3 grid, int threads, int shared, cudaStream_t s, const Args &...args) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = s;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    if (shared) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shared);
        if (e != cudaSuccess) return e;
    }
    before_launch();
    return cudaLaunchKernelEx(&config, kernel, args...);
}


}  // namespace

}  // namespace b200fft
