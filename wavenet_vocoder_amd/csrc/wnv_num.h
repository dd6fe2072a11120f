// wnv_num.h -- element types and the gate function of the recurrence and 4-bit kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/wnv.h"

typedef __bf16 wnv_bf16;
typedef _Float16 wnv_f16;

static inline int wnv_dtype_size(int dtype) { return dtype == WNV_F32 ? 4 : dtype == WNV_BF16 || dtype == WNV_F16 ? 2 : 0; }

template <typename E> __device__ __forceinline__ float wnv_up(E x) { return (float)x; }
// one rounding to nearest even, of a value computed in 32 bits
template <typename E> __device__ __forceinline__ E wnv_down(float x) { return (E)x; }

// sigmoid(x) = 1 / (1 + exp(-x)), by the hardware's base-2 exponential and reciprocal (an ulp each): to a few ulps of itself at both
// ends, so that 1 - sigmoid(f), taken as sigmoid(-f), is as exact next to 0 as sigmoid(f) (1 - sigmoid(f) would leave it 2^-24
// absolute: at f = 9, 5e-4 of it).  exp overflows to infinity, whose reciprocal is the right 0; a NaN passes.
__device__ __forceinline__ float wnv_gate(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f));
}
// The same, and sigmoid(x) (1 - sigmoid(x)) = e / (1 + e)^2 with e = exp(-|x|) <= 1: exact at both ends too, no overflow.
__device__ __forceinline__ float wnv_gate(float x, float& slope) {
    const float e = __builtin_amdgcn_exp2f(fabsf(x) * -1.44269504088896340736f);
    const float r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
    slope = er * r;
    return x >= 0.f ? r : er;
}
