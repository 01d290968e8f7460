// Activations of the operators of models on frames and their slopes, on the device.
#pragma once
#include <hip/hip_runtime.h>

namespace tfa {

enum { kActNone = 0, kActSilu = 1, kActGelu = 2, kActRelu = 3 };

// e^-x by the hardware's exp2, a few 1e-7 of the result where it matters (x from -20 to 20)
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * -1.4426950408889634f); }
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + exp_neg(z)); }

// Phi(z), the normal distribution: 1 - erf by Abramowitz and Stegun 7.1.26 (1.5e-7 absolute), taken on the side where it is small;
// `bell` receives e^(-z^2 / 2), which the slope needs too.  GELU is off by 6e-7 at most (from -8 to 8); far out on the
// negative side that is a share of a value that is next to nothing (at -5, of 1.4e-6, 0.16 %; at -10, of 8e-23, 2 %).
__device__ __forceinline__ float normal_cdf(float z, float& bell) {
  const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.0f));
  bell = exp_neg(x * x);
  float q = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
  q = __builtin_fmaf(t, q, 1.421413741f);
  q = __builtin_fmaf(t, q, -0.284496736f);
  q = __builtin_fmaf(t, q, 0.254829592f);
  const float tail = 0.5f * q * t * bell;
  return z < 0.0f ? tail : 1.0f - tail;  // (NaN stays: it is in tail)
}

__device__ __forceinline__ float activate(float z, int act) {
  if (act == kActSilu) return z * sigmoid(z);
  if (act == kActGelu) {
    float bell;
    return z * normal_cdf(z, bell);
  }
  if (act == kActRelu) return z > 0.0f ? z : z != z ? z : 0.0f;  // NaN stays
  return z;
}

__device__ __forceinline__ float activation_slope(float z, int act) {
  if (act == kActSilu) {
    const float s = sigmoid(z);
    return s * __builtin_fmaf(z, 1.0f - s, 1.0f);
  }
  if (act == kActGelu) {
    float bell;
    const float cdf = normal_cdf(z, bell);
    return __builtin_fmaf(z * 0.39894228040143268f, bell, cdf);
  }
  if (act == kActRelu) return z > 0.0f ? 1.0f : 0.0f;
  return 1.0f;
}

}  // namespace tfa
