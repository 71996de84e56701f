// The activation of the gated transition: act(v) = v sigmoid(t(v)), for silu t = v, for gelu in its tanh form t = 2 sqrt(2 / pi) (v + 0.044715 v^3).
// Its derivative is s + v s (1 - s) t'(v) with s = sigmoid(t(v)).
#pragma once
#include <hip/hip_runtime.h>

#include "kutacc_hip.h"
#include "mfma_tiles.h"

namespace kutacc_dev {

constexpr float GELU_SLOPE = 1.5957691216057308f, GELU_CUBE = 0.044715f; // 2 sqrt(2 / pi)

// 2^(this) = exp(-t(v))
__device__ __forceinline__ float activation_exponent(float v, int activation)
{
    return activation == KUTACC_HIP_GELU ? v * fmaf(-LOG2E * GELU_SLOPE * GELU_CUBE, v * v, -LOG2E * GELU_SLOPE) : -LOG2E * v;
}

// act(v) of s = sigmoid(t(v)), and its derivative.  From |v| = 100 on s is 0 or 1, and so is the derivative: gelu's t'(v) stays what it is there, or a large v, times
// its square, would be an infinity times the zero of 1 - s.
__device__ __forceinline__ float activation_of_sigmoid(float v, float s, int activation, float &derivative)
{
    const float a = v * s, rest = 1.f - s;
    if (__builtin_constant_p(activation) && activation != KUTACC_HIP_GELU) {
        derivative = fmaf(a, rest, s);
    } else { // (with one expression for both, where the kernel is told which)
        derivative = fmaf(a * rest, activation == KUTACC_HIP_GELU ? fmaf(3.f * GELU_CUBE * GELU_SLOPE, fminf(v * v, 1e4f), GELU_SLOPE) : 1.f, s);
    }
    return a;
}

// act(v), and its derivative where it is asked for
template <bool DERIVATIVE>
__device__ __forceinline__ float activate(float v, int activation, float &derivative)
{
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(activation_exponent(v, activation)));
    if constexpr (DERIVATIVE) {
        return activation_of_sigmoid(v, s, activation, derivative);
    }
    return v * s;
}

// what the rounding of v to r left; of a result past bf16's range nothing, as infinity less infinity is no number
__device__ __forceinline__ bf16_t rounding_rest(float v, bf16_t r) { return (bf16_t)(fabsf((float)r) <= 3.4e38f ? v - (float)r : 0.f); }

} // namespace kutacc_dev
