// host_util.h -- what the host sides of the device translation units share.
#pragma once

#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstdio>

#include "../../include/b200_decode.h"

namespace b200 {

constexpr int kMaxDevices = 64;

inline int current_device() {
    int d = 0;
    cudaGetDevice(&d);
    return d;
}

inline int cuda_status(cudaError_t e) {
    if (e != cudaSuccess) {
        fprintf(stderr, "b200_decode: CUDA error %s (%s)\n", cudaGetErrorName(e), cudaGetErrorString(e));
        return B200_ECUDA;
    }
    return B200_OK;
}

#define CR_(x)                        \
    do {                              \
        const int r_ = (x);           \
        if (r_ != B200_OK) return r_; \
    } while (0)

// Launch attribute for programmatic dependent launch (see b200i_gemv).
inline cudaLaunchAttribute pdl_attr() {
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    return at;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// cuTensorMapEncodeTiled through the runtime's driver entry point (no link
// against the driver library).
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

}  // namespace b200
