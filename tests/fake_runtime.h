// A stand-in for the CUDA runtime, for tests of the library's host code on machines without a GPU: each call does what
// the test has set.
#pragma once

#include <cuda_runtime.h>

#include <cstdio>
#include <cstdlib>

static cudaError_t g_last = cudaSuccess;         // what the runtime keeps of the last failure

static cudaError_t fails(cudaError_t e) { return g_last = e; }

extern "C" cudaError_t cudaGetLastError() {
    const cudaError_t e = g_last;
    g_last = cudaSuccess;
    return e;
}
extern "C" const char *cudaGetErrorString(cudaError_t) { return "planted"; }

namespace afb {
void set_last_error(const std::string &) {}
}  // namespace afb

#define EXPECT(cond)                                                   \
    do {                                                               \
        if (!(cond)) {                                                 \
            std::fprintf(stderr, "line %d: %s\n", __LINE__, #cond);    \
            std::exit(1);                                              \
        }                                                              \
    } while (0)
