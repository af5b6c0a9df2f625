// Host-side helpers shared by the C-ABI launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "flaggems_vllm_amd.h"

namespace fgv {

// Records msg as this thread's last error and returns code.
int fail(int code, const char* msg);

inline bool aligned(const void* p, uintptr_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// Status of the launch just issued: 0, or the positive hipError_t.
inline int launch_status() {
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? FGV_OK : static_cast<int>(e);
}

// CUs of the current device (256 on MI355X), asked once per device.
inline int cu_count() {
    static std::atomic<int> known[64];
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess)
        return 256;
    const bool kept = dev >= 0 && dev < 64;
    if (kept && (cus = known[dev].load(std::memory_order_relaxed)) > 0)
        return cus;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0)
        return 256;
    if (kept)
        known[dev].store(cus, std::memory_order_relaxed);
    return cus;
}

}  // namespace fgv
