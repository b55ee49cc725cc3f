// Checks of the device pointers that callers of single kernels pass.
#pragma once
#include "internal.h"

#include <initializer_list>

namespace lumi {

// Every pointer that is not 0 has to be memory of the current device: a kernel that is given host memory or another device's would fault.
inline int32_t check_device_memory(const char* what, std::initializer_list<uint64_t> pointers) {
    int dev = 0;
    LUMI_CUDA(cudaGetDevice(&dev));
    for (const uint64_t p : pointers) {
        if (p == 0) continue;
        cudaPointerAttributes at;
        LUMI_CUDA(cudaPointerGetAttributes(&at, reinterpret_cast<const void*>(p)));
        if ((at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) || at.device != dev)
            return fail(LUMI_E_INVALID, "%s: a pointer is not memory of the current device (%d)", what, dev);
    }
    return LUMI_OK;
}

}  // namespace lumi
