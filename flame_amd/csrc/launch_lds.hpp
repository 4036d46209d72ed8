// A kernel's dynamic LDS size, told to the runtime once per kernel and device.
#pragma once
#include <hip/hip_runtime.h>

#include <atomic>

#include "../../include/flame_attn.h"

namespace fattn {

inline int set_lds_of_device(const void* kern, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return (int)hipErrorInvalidDevice;
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return FLAME_ATTN_OK;
    const hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return (int)e;
    done.fetch_or(bit, std::memory_order_relaxed);
    return FLAME_ATTN_OK;
}

}  // namespace fattn
