// Two threads ask for different amounts of a kernel's shared memory at the same time: the limit that is left allows the
// larger one.  The runtime's part of the first request takes longer than the whole of the second.
#include <cuda_runtime.h>

// the forms that take a kernel, which the runtime's header has for nvcc alone
static cudaError_t cudaFuncSetAttribute(void (*k)(int), cudaFuncAttribute a, int bytes) {
    return cudaFuncSetAttribute(reinterpret_cast<const void *>(k), a, bytes);
}
static cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessor(int *n, void (*k)(int), int threads, size_t shared) {
    return cudaOccupancyMaxActiveBlocksPerMultiprocessor(n, reinterpret_cast<const void *>(k), threads, shared);
}

#include "../alphafly_b200/csrc/launch.cuh"

#include "fake_runtime.h"

#include <atomic>
#include <chrono>
#include <thread>

static std::atomic<int> g_limit{0}, g_calls{0};

static void wait_ms(int ms) { std::this_thread::sleep_for(std::chrono::milliseconds(ms)); }

extern "C" cudaError_t cudaGetDevice(int *dev) { return *dev = 0, cudaSuccess; }
extern "C" cudaError_t cudaDeviceGetAttribute(int *value, cudaDeviceAttr, int) { return *value = 148, cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int bytes) {
    g_limit = bytes;
    if (g_calls++ == 0) wait_ms(300);
    return cudaSuccess;
}
extern "C" cudaError_t cudaOccupancyMaxActiveBlocksPerMultiprocessor(int *n, const void *, int, size_t shared) {
    const size_t fits = (228 << 10) / shared;
    wait_ms(1);
    return *n = (int)fits, cudaSuccess;
}

static void kernel(int) {}

int main() {
    std::thread large([] { afb::allow_shared<kernel>(200 << 10); });
    while (!g_calls) wait_ms(1);
    std::thread small([] { afb::allow_shared<kernel>(100 << 10); });
    large.join();
    small.join();
    afb::allow_shared<kernel>(200 << 10);        // allowed before
    EXPECT(g_limit >= 200 << 10);
    // and the CTAs of one size are never answered for the other
    std::atomic<int> wrong{0};
    auto ask = [&](size_t shared, int64_t ctas) {
        for (int i = 0; i < 200; ++i) wrong += afb::resident<kernel>(128, shared) != ctas;
    };
    std::thread a(ask, 100 << 10, 2 * 148), b(ask, 20 << 10, 11 * 148);
    a.join();
    b.join();
    EXPECT(wrong == 0);
    return 0;
}
