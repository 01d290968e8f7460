// Arithmetic on lanes that the selective scan's kernels share (scan_blocks.h, kernels_scan.hip).
#pragma once
#include "model_ops.h"
#include "activations.h"

namespace tfa {

constexpr float kLog2E = 1.4426950408889634f;

// e^(s a) of a2 = a log2(e).  The hardware's exp2 is low by 7e-9 (results of 0.999 and above) to 1e-9 (0.95) on the average: nothing by itself, but
// over a memory of a thousand frames more than all roundings together.  Its mean is put back into the argument, which costs nothing.
__device__ __forceinline__ float decay_of(float s, float a2) { return __builtin_amdgcn_exp2f(__builtin_fmaf(s, a2, 6e-9f)); }

// log(1 + e^v) and its derivative, both a few 2^-24 of themselves for every v: with e = e^-|v|, log(1 + e) = 2 artanh(s) of
// s = e / (2 + e) <= 1/3, whose series to s^13 leaves 2e-8
__device__ __forceinline__ float softplus(float v, float& slope) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(v) * kLog2E);
  const float s = e * __builtin_amdgcn_rcpf(2.0f + e), w = s * s;
  float q = __builtin_fmaf(w, 1.0f / 13.0f, 1.0f / 11.0f);
  q = __builtin_fmaf(w, q, 1.0f / 9.0f);
  q = __builtin_fmaf(w, q, 1.0f / 7.0f);
  q = __builtin_fmaf(w, q, 1.0f / 5.0f);
  q = __builtin_fmaf(w, q, 1.0f / 3.0f);
  q = __builtin_fmaf(w, q, 1.0f);
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  slope = v < 0.0f ? e * r : r;
  return __builtin_fmaf(2.0f * s, q, fmaxf(v, 0.0f));  // (NaN stays: it is in s)
}

// x of the lane whose number differs by MASK (1, 2, 3, 7, 8: permutations within rows of 16 lanes; 4 is 7 after 3)
template <int MASK>
__device__ __forceinline__ float lane_xor(float x) {
  if constexpr (MASK == 4) return lane_xor<3>(lane_xor<7>(x));
  constexpr int ctrl = MASK == 1 ? 0xB1 : MASK == 2 ? 0x4E : MASK == 3 ? 0x1B : MASK == 7 ? 0x141 : 0x128;
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), ctrl, 15, 15, true));
}

// Sums over pairs of lanes whose numbers differ by MASK: lanes with MASK's highest bit clear receive a's sum, the others b's.
// Over all bits of a set of lanes, from the highest, whole sums of as many values come out, one a lane.
template <int MASK>
__device__ __forceinline__ float fold(float a, float b) {
  if constexpr (MASK >= 16) {
    const auto p = MASK == 32 ? __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false)
                              : __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
  } else {
    const bool up = threadIdx.x & (MASK == 7 ? 4 : MASK);
    const float keep = up ? b : a, give = up ? a : b;
    return keep + lane_xor<MASK>(give);
  }
}
// the sum over such pairs, in both lanes
template <int MASK>
__device__ __forceinline__ float fold(float a) {
  if constexpr (MASK >= 16)
    return fold<MASK>(a, a);
  else
    return a + lane_xor<MASK>(a);
}

}  // namespace tfa
