// Element types of the entry points that take more than one (AFB_T_*): conversions and dispatch.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace afb {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// One rounding to the result's type, to nearest even.
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

inline bool known_type(int t) { return t == AFB_T_F32 || t == AFB_T_F16 || t == AFB_T_BF16; }
inline size_t type_size(int t) { return t == AFB_T_F32 ? 4 : 2; }

// f(element of the type): f receives a value whose type is the element type.
template <typename F>
void with_type(int t, F &&f) {
    if (t == AFB_T_F32) f(float{});
    else if (t == AFB_T_F16) f(__half{});
    else f(__nv_bfloat16{});
}

}  // namespace afb
