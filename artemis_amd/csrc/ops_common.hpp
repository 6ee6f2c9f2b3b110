// ops_common.hpp -- what the kernels of libartemis_ops.so share: element types, wave reductions, and
// the host side's error text.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <math.h>

#include "artemis_ops.h"

namespace aops {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using i32x4 = __attribute__((ext_vector_type(4))) int;
using u16x4 = __attribute__((ext_vector_type(4))) unsigned short;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using bf16x4 = __attribute__((ext_vector_type(4))) __bf16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x4 = __attribute__((ext_vector_type(4))) _Float16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;

// N consecutive elements of type T as one load or store of N * sizeof(T) bytes
template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

template <class T>
__device__ __forceinline__ float to_f32(T x) { return (float)x; }
template <class T>
__device__ __forceinline__ T from_f32(float x) { return (T)x; }

// sum / max over groups of `L` consecutive lanes (a power of two); every lane gets the result
template <int CTRL>
__device__ __forceinline__ float dpp(float x)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
template <int L>
__device__ __forceinline__ float group_sum(float x)
{
    if constexpr (L >= 2) x += dpp<0xB1>(x);    // lanes 1 0 3 2
    if constexpr (L >= 4) x += dpp<0x4E>(x);    // lanes 2 3 0 1
    if constexpr (L >= 8) x += dpp<0x141>(x);   // mirrored within 8
    if constexpr (L >= 16) x += dpp<0x140>(x);  // mirrored within 16
    if constexpr (L >= 32) x += __shfl_xor(x, 16);
    if constexpr (L >= 64) x += __shfl_xor(x, 32);
    return x;
}

int fail(int code, const char *fmt, ...);
int check_launch(const char *what);

}  // namespace aops
