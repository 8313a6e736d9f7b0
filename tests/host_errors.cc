// A call of the runtime that fails is reported by the call that made it, and by no later one.
#include "../alphafly_b200/csrc/common.cuh"

#include "fake_runtime.h"

extern "C" cudaError_t cudaMalloc(void **, size_t) { return fails(cudaErrorMemoryAllocation); }
extern "C" cudaError_t cudaFree(void *) { return cudaSuccess; }

int main() {
    EXPECT(afb::guarded([] { afb::DevBuf<int> b(1000); }) == AFB_ECUDA);
    EXPECT(afb::guarded([] { AFB_LAUNCHED(); }) == AFB_OK);              // a launch that went well
    EXPECT(afb::guarded([] { fails(cudaErrorInvalidConfiguration); AFB_LAUNCHED(); }) == AFB_ECUDA);
    EXPECT(afb::guarded([] { AFB_LAUNCHED(); }) == AFB_OK);
    return 0;
}
