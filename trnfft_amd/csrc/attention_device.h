// Device helpers shared by the linear attention kernels.
#pragma once
#include "kernels.h"
#include "model_ops.h"

namespace tfa {

// A power of gamma as a sum of two fp32: products of it over a long memory keep fp32's precision (a rounded gamma of a
// memory of 256 tokens would be off by 256 half ulps, 8e-6).
struct Decay {
  float hi, lo;
  __device__ __forceinline__ explicit Decay(double x) : hi((float)x), lo((float)(x - (double)(float)x)) {}
  __device__ __forceinline__ float times(float m) const { return __builtin_fmaf(m, hi, m * lo); }
};

// The same as one fp32 factor a step: of the two fp32 around gamma, the one that brings the product so far nearer to the
// power, so that the product stays within a half ulp of it however many steps there are.
// (All of it the same in every lane, and kept in scalar registers: the errors, below 2^-23 of gamma, count in 2^-44ths.)
__device__ __forceinline__ float scalar(float x) {
  return __uint_as_float((unsigned)__builtin_amdgcn_readfirstlane((int)__float_as_uint(x)));
}
struct DecaySteps {
  float below, above;
  int err_below, err_above, err = 0;
  __device__ __forceinline__ explicit DecaySteps(double x) {
    const float near = (float)x;
    below = scalar((double)near <= x ? near : __uint_as_float(__float_as_uint(near) - 1));
    above = scalar((double)near >= x ? near : __uint_as_float(__float_as_uint(near) + 1));
    // (a gamma in the denormals or zero forgets all it carries: no error to keep account of; nor of NaN)
    const double unit = 0x1p44 / x;
    err_below = __builtin_amdgcn_readfirstlane(x > 1e-30 ? (int)(((double)below - x) * unit) : 0);
    err_above = __builtin_amdgcn_readfirstlane(x > 1e-30 ? (int)(((double)above - x) * unit) : 0);
  }
  __device__ __forceinline__ float next() {
    const bool down = err > 0;
    err += down ? err_below : err_above;
    return down ? below : above;
  }
};

// log decays of -inf (no memory) are taken as -1e5: gamma^0 stays 1 and every other power is 0.  (By a comparison that lets NaN through:
// a decay that has diverged is to be seen.)
__device__ __forceinline__ float log_decay_of(const float* g, int h) { return g[h] < -1e5f ? -1e5f : g[h]; }

template <typename T>
__device__ __forceinline__ const T* head_base(const HeadsView& v, long long b, int h) {
  return static_cast<const T*>(v.p) + b * v.sb + (long long)(h / v.group) * v.sh;
}

__device__ __forceinline__ long long live_tokens(const AttnPass& p, long long b) {
  return p.lengths ? min(max(p.lengths[b], 0LL), p.tokens) : p.tokens;
}

// Launches of `each` workgroups for every batch row, as many rows at a time as a launch holds.  (One row always fits: heads are
// below 2^16, slices of a head at most 8, and segments for few heads only.)
template <typename Args, typename Launch>
hipError_t for_batches(Args p, long long each, int threads, Launch launch) {
  const long long most = max_blocks(threads) / each;
  for (p.first = 0; p.first < p.batch; p.first += most) {
    launch(p, dim3((unsigned)(each * (p.batch - p.first < most ? p.batch - p.first : most))));
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace tfa
