// Shared pieces of the 8-bit products and of distillation: element types (AFB_T_*), their conversions and dispatch, 16-byte
// pieces of rows.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "launch.cuh"

namespace afb {

constexpr float kInf = __builtin_huge_valf();

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

// 16 bytes of a row: kPer elements.
template <typename T>
struct Piece {
    static constexpr int kPer = 16 / (int)sizeof(T);
    union {
        uint4 raw;
        T e[kPer];
    };
    __device__ __forceinline__ Piece() : raw(make_uint4(0u, 0u, 0u, 0u)) {}
};

// Elements of a row's first 16-byte piece that lie before the row.
template <typename T>
__device__ __forceinline__ int lead_of(const T *row) {
    return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}

// The piece of a row of n elements that starts at element at (row + at on 16 bytes); what is not of the row is `fill`.
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T *row, int at, int n, T fill) {
    Piece<T> v;
    if (at >= 0 && at + Piece<T>::kPer <= n) {
        v.raw = __ldg(reinterpret_cast<const uint4 *>(row + at));
    } else {
#pragma unroll
        for (int e = 0; e < Piece<T>::kPer; ++e) v.e[e] = at + e >= 0 && at + e < n ? row[at + e] : fill;
    }
    return v;
}

// Stores a piece over the elements from `at` on, those of them that are of the row (row + at on 16 bytes).
template <typename T>
__device__ __forceinline__ void store_piece(T *row, int at, int n, const Piece<T> &v) {
    if (at >= 0 && at + Piece<T>::kPer <= n) {
        *reinterpret_cast<uint4 *>(row + at) = v.raw;
    } else {
#pragma unroll
        for (int e = 0; e < Piece<T>::kPer; ++e)
            if (at + e >= 0 && at + e < n) row[at + e] = v.e[e];
    }
}

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
