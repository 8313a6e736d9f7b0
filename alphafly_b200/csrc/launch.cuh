// What a launch needs to know of a kernel on the current device, asked of the runtime once.  Calls may come from several
// host threads at a time.
#pragma once

#include <mutex>

#include "common.cuh"

namespace afb {

constexpr int kMaxDevices = 64;

inline int current_device() {
    int dev = 0;
    AFB_CUDA(cudaGetDevice(&dev));
    AFB_CHECK(dev >= 0 && dev < kMaxDevices, "device index out of range");
    return dev;
}

// Lets the kernel take that much dynamic shared memory on the current device.  The limit is only ever raised, and set and
// noted together: a thread that asks for less must not lower it under another's launch.
template <auto kKernel>
void allow_shared(size_t bytes) {
    static std::mutex lock;
    static size_t allowed[kMaxDevices] = {0};
    if (bytes <= 32 * 1024) return;
    const int dev = current_device();
    const std::lock_guard<std::mutex> held(lock);
    if (allowed[dev] >= bytes) return;
    AFB_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    allowed[dev] = bytes;
}

// CTAs of a kernel that the current device holds at once (asked for again when the shared memory changes).
template <auto kKernel>
int64_t resident(int threads, size_t shared) {
    static std::mutex lock;
    static size_t of[kMaxDevices] = {0};
    static int64_t ctas[kMaxDevices] = {0};
    const int dev = current_device();
    const std::lock_guard<std::mutex> held(lock);
    if (ctas[dev] && of[dev] == shared) return ctas[dev];
    int per_sm = 0, sms = 0;
    AFB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kKernel, threads, shared));
    AFB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    AFB_CHECK(per_sm >= 1, "the kernel does not fit on this device");
    of[dev] = shared;
    ctas[dev] = (int64_t)per_sm * sms;
    return ctas[dev];
}

}  // namespace afb
