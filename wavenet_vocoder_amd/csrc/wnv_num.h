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

// keep = sigmoid(x) and its complement 1 - keep = e / (1 + e), e = exp(-x), both from one exponential and one reciprocal; the
// complement is exact to a few ulps where keep is next to 1 (1 - keep would leave it 2^-24 absolute: at x = 9, 5e-4 of it).
// The exponent stops at 126, so that 1 + e is finite and its reciprocal normal: keep <= 2^-126 and 1 - keep = 1 there, in
// place of inf * 0.  A NaN passes (the comparison is false).
__device__ __forceinline__ void wnv_gate(float x, float& keep, float& drop) {
    float p = x * -1.44269504088896340736f;
    p = p > 126.0f ? 126.0f : p;
    const float e = __builtin_amdgcn_exp2f(p);
    keep = __builtin_amdgcn_rcpf(1.0f + e);
    drop = e * keep;
}
