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

// sigmoid(x) = 1 / (1 + exp(-x)), by the hardware's base-2 exponential and reciprocal, an ulp each.  x log2(e) is rounded to 24 bits before
// that, so that next to 0 the result is within (1.5 |x| + 8) 2^-24 of itself: 11 ulps at x = -9, 64 at -80, and below 2^-126 it may
// read as 0.  1 - sigmoid(f), taken as sigmoid(-f), is that exact too (1 - sigmoid(f) would leave it 2^-24 absolute: at f = 9, 5e-4 of it).
// exp overflows to infinity, whose reciprocal is the right 0; a NaN passes.
__device__ __forceinline__ float wnv_gate(float x) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f));
}
// The same, and sigmoid(x) (1 - sigmoid(x)) = e / (1 + e)^2 with e = exp(-|x|) <= 1: as exact, at both ends, no overflow.
__device__ __forceinline__ float wnv_gate(float x, float& slope) {
    const float e = __builtin_amdgcn_exp2f(fabsf(x) * -1.44269504088896340736f);
    const float r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
    slope = er * r;
    return x >= 0.f ? r : er;
}
// sigmoid(f), and u = 1 - sigmoid(f) = sigmoid(-f), each as exact as above.
__device__ __forceinline__ float wnv_gates(float f, float& u) {
    const float e = __builtin_amdgcn_exp2f(fabsf(f) * -1.44269504088896340736f);
    const float more = __builtin_amdgcn_rcpf(1.0f + e), less = e * more;
    u = f > 0.f ? less : more;
    return f > 0.f ? more : less;
}
// sigmoid(f) h + (1 - sigmoid(f)) v.  Of the two weights the smaller, sigmoid(-|f|), is known to its own precision, and the other is 1 less
// that: a state that a gate remembers for n steps is not off by n roundings of a weight next to 1, and one that it forgets leaves what
// the formula leaves of it, not 2^-24 of what it was.  Nothing overflows that the result does not.  f = inf gives h, f = -inf gives v
// (both finite); a weight below 2^-126 may read as 0.
__device__ __forceinline__ float wnv_blend(float f, float h, float v) {
    const float e = __builtin_amdgcn_exp2f(fabsf(f) * -1.44269504088896340736f);
    const float less = e * __builtin_amdgcn_rcpf(1.0f + e);
    const bool keeps = f > 0.f;
    const float more = keeps ? h : v, rest = keeps ? v : h;
    return fmaf(less, rest, fmaf(-less, more, more));
}
