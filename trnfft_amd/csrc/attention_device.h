// Device helpers shared by the linear attention kernels.
#pragma once
#include "model_ops.h"

namespace tfa {

// A power of gamma as a sum of two fp32: products of it over a long memory keep fp32's precision (a rounded gamma of a
// memory of 256 tokens would be off by 256 half ulps, 8e-6).
struct Decay {
  float hi, lo;
  __device__ __forceinline__ explicit Decay(double x) : hi((float)x), lo((float)(x - (double)(float)x)) {}
  __device__ __forceinline__ float times(float m) const { return __builtin_fmaf(m, hi, m * lo); }
};

// log decays of -inf (no memory) are taken as -1e5: gamma^0 stays 1 and every other power is 0
__device__ __forceinline__ float log_decay_of(const float* g, int h) { return fmaxf(g[h], -1e5f); }

template <typename T>
__device__ __forceinline__ const T* head_base(const HeadsView& v, long long b, int h) {
  return static_cast<const T*>(v.p) + b * v.sb + (long long)(h / v.group) * v.sh;
}

__device__ __forceinline__ long long live_tokens(const AttnPass& p, long long b) {
  return p.lengths ? min(max(p.lengths[b], 0LL), p.tokens) : p.tokens;
}

}  // namespace tfa
