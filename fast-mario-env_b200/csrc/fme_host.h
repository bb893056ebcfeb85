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

}  // namespace fme
