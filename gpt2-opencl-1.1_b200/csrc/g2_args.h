// g2_args.h -- host side of the single-kernel entry points that take many
// device pointers (g2k_matvec_q4, g2k_kv8_*, g2k_process_logits).
#pragma once
#include <cuda_runtime.h>

#include <cstdio>
#include <initializer_list>

#include "g2_internal.h"
#include "gpt2b200.h"

namespace g2 {

inline int arg_error(int code, const char *who, const char *what) {
    char buf[256];
    snprintf(buf, sizeof buf, "%s: %s", who, what);
    return set_error(code, buf);
}

inline bool aligned(const void *p, size_t n) { return (reinterpret_cast<size_t>(p) % n) == 0; }

// Every non-null pointer must be memory that the current device can use: host
// memory or another device's would fault inside the kernel, which ends the
// caller's context, so it is refused here.
inline int check_device_ptrs(const char *who, std::initializer_list<const void *> ptrs) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        return arg_error(G2_ERR_CUDA, who, "no current CUDA device");
    }
    for (const void *p : ptrs) {
        if (!p) continue;
        cudaPointerAttributes a;
        if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
            cudaGetLastError();
            return arg_error(G2_ERR_CUDA, who, "cannot query a pointer");
        }
        if (a.type == cudaMemoryTypeManaged) continue;
        if (a.type != cudaMemoryTypeDevice || a.device != dev)
            return arg_error(G2_ERR_ARG, who, "an array is not memory of the current device");
    }
    return G2_OK;
}

// A launch just made on the current device: its error, if any.
inline int launch_status(const char *who, cudaError_t r) {
    if (r != cudaSuccess) cudaGetLastError();
    return r == cudaSuccess ? G2_OK : arg_error(G2_ERR_CUDA, who, cudaGetErrorString(r));
}
inline int launch_status(const char *who) { return launch_status(who, cudaGetLastError()); }

// SMs of the current device (a B200's where there is none to ask).
inline int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
    }
    return n > 0 ? n : 148;
}

}  // namespace g2
