// The activations of the row-scaled linears (the GEMM's epilogue and its backward), in fp32.
#pragma once
#include "gpic_device.h"

namespace gpic {

// sigmoid(x) = 1 / (1 + 2^(-x log2 e)) with the hardware's 2^t and reciprocal (1 ulp each). The product's rounding makes
// e^-x off by |x| 2^-24 relative, 6e-6 at most before it leaves fp32's range: far below the bf16 rounding (2^-9) of what is
// made of it, at a third of the instructions of the SwiGLU casts' sigmoid (gpic_device.h), whose bytes an oracle restates.
// -inf gives 0, +inf 1, NaN NaN.
__device__ __forceinline__ float fast_sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
}

constexpr float kGelu2C = 1.59576912f;            // 2 sqrt(2 / pi)
constexpr float kGelu2C3 = 0.0713548163f;         // 2 sqrt(2 / pi) 0.044715

// gelu_tanh(z) = z (1 + tanh u) / 2 = z sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3); e^-2u as 2^t, log2 e in the constants
__device__ __forceinline__ float gelu_sig(float z) {
  const float t = z * __builtin_fmaf(-1.44269504f * kGelu2C3, z * z, -1.44269504f * kGelu2C);
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t));
}

// act(z); act: GPIC_ACT_NONE / SILU / GELU_TANH (uniform over the wave)
__device__ __forceinline__ float act_fwd(float z, int act) {
  if (act == 1) return z * fast_sigmoid(z);
  if (act == 2) return z * gelu_sig(z);
  return z;
}

// act'(z): silu p (1 + z (1 - p)); gelu_tanh p + z p (1 - p) d(2 u)/dz
__device__ __forceinline__ float act_bwd(float z, int act) {
  if (act == 1) {
    const float p = fast_sigmoid(z);
    return p * __builtin_fmaf(z, 1.0f - p, 1.0f);
  }
  if (act == 2) {
    const float p = gelu_sig(z);
    // (z^2 bounded: p (1 - p) is 0 long before, and 0 times the overflowed square would be NaN)
    return __builtin_fmaf(z * p * (1.0f - p), __builtin_fmaf(3.0f * kGelu2C3, __builtin_fminf(z * z, 1e30f), kGelu2C), p);
  }
  return 1.0f;
}

}  // namespace gpic
