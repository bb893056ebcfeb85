// fme_host.h - what the library's translation units share on the host side: the thread's error message.
#pragma once
#include <cuda_runtime.h>
#include <stdio.h>

#include "fme.h"

namespace fme {

// Records msg for fme_last_error on the calling thread and returns code (defined in fme.cu; never throws).
int host_fail(int code, const char* msg) noexcept;

// FME_OK, or FME_E_CUDA with the error of the launch just made.
inline int launch_status(const char* what) noexcept {
    const cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) return FME_OK;
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", what, cudaGetErrorString(e));
    return host_fail(FME_E_CUDA, msg);
}

// A kernel that may be launched while the one before it in the stream still runs: its CTAs take their places as those of the other
// leave theirs, and wait (await_previous) before they touch what it writes.
template <typename... P, typename... Args>
inline int launch_behind(const char* what, void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args) noexcept {
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = grid; c.blockDim = block; c.dynamicSmemBytes = smem; c.stream = st; c.attrs = &at; c.numAttrs = 1;
    cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
    return launch_status(what);
}
#ifdef __CUDACC__
__device__ __forceinline__ void await_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
#endif

}  // namespace fme
