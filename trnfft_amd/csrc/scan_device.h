// Arithmetic on lanes that the selective scan's kernels share (scan_blocks.h, kernels_scan.hip).
#pragma once
#include "model_ops.h"
#include "activations.h"

#include <type_traits>
#include <utility>

namespace tfa {

constexpr float kLog2E = 1.4426950408889634f;

// e^(s a) of a2 = a log2(e).  The hardware's exp2 is low by 7e-9 (results of 0.999 and above) to 1e-9 (0.95) on the average: nothing by itself, but
// over a memory of a thousand frames more than all roundings together.  Its mean is put back into the argument, which costs nothing.
__device__ __forceinline__ float decay_of(float s, float a2) { return __builtin_amdgcn_exp2f(__builtin_fmaf(s, a2, 6e-9f)); }

// log(1 + e^v) and its derivative, off by a few 2^-24 of themselves and of v: with e = e^-|v| and u = 1 + e, log(1 + e) = log(u) + (e - (u - 1)),
// where the second term is what the sum u lost (the hardware's logarithm is good to its last bit next to 1 too).  Measured from -20 to 20:
// 3e-8 of it in the mean square for v > 0, 2e-7 at -8, 1e-6 at most; a series for the artanh took twice the instructions for the same.
__device__ __forceinline__ float softplus(float v, float& slope) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(v) * kLog2E), u = 1.0f + e;
  const float r = __builtin_fmaf(__builtin_amdgcn_logf(u), 0.69314718055994531f, e - (u - 1.0f));
  const float part = __builtin_amdgcn_rcpf(u);
  slope = v < 0.0f ? e * part : part;
  return __builtin_fmaf(v + fabsf(v), 0.5f, r);  // (NaN stays)
}

// x of the lane whose number differs by MASK (1, 2, 3, 7, 8: permutations within rows of 16 lanes; 4 is 7 after 3)
template <int MASK>
__device__ __forceinline__ float lane_xor(float x) {
  if constexpr (MASK == 4) return lane_xor<3>(lane_xor<7>(x));
  constexpr int ctrl = MASK == 1 ? 0xB1 : MASK == 2 ? 0x4E : MASK == 3 ? 0x1B : MASK == 7 ? 0x141 : 0x128;
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), ctrl, 15, 15, true));
}

// Products with x[r] of lane T of the lane's row of 16, which the instruction's operand takes from there.  (Waits as at
// fold_pairs.)
template <int T>
struct RowLane {
  template <int R>
  static __device__ __forceinline__ void products(const float (&x)[R], float u, float (&out)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) out[r] = lane(x[r]) * u;
  }
  template <int R>
  static __device__ __forceinline__ void add(const float (&x)[R], float u, float (&sum)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) sum[r] = __builtin_fmaf(lane(x[r]), u, sum[r]);
  }
  template <int R>
  static __device__ __forceinline__ float dot(const float (&x)[R], const float (&y)[R]) {
    float sum = lane(x[0]) * y[0];
#pragma unroll
    for (int r = 1; r < R; ++r) sum = __builtin_fmaf(lane(x[r]), y[r], sum);
    return sum;
  }
  static __device__ __forceinline__ float lane(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x150 + T, 15, 15, true));
  }
  // four at once without a move for each
#define TFA_ROW " row_newbcast:%c[t] row_mask:0xf bank_mask:0xf\n\t"
  static __device__ __forceinline__ void products(const float (&x)[4], float u, float (&out)[4]) {
    asm("s_nop 1\n\t"
        "v_mul_f32_dpp %0, %4, %8" TFA_ROW
        "v_mul_f32_dpp %1, %5, %8" TFA_ROW
        "v_mul_f32_dpp %2, %6, %8" TFA_ROW
        "v_mul_f32_dpp %3, %7, %8" TFA_ROW
        : "=&v"(out[0]), "=&v"(out[1]), "=&v"(out[2]), "=&v"(out[3])
        : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(u), [t] "n"(T));
  }
  static __device__ __forceinline__ void add(const float (&x)[4], float u, float (&sum)[4]) {
    asm("s_nop 1\n\t"
        "v_fmac_f32_dpp %0, %4, %8" TFA_ROW
        "v_fmac_f32_dpp %1, %5, %8" TFA_ROW
        "v_fmac_f32_dpp %2, %6, %8" TFA_ROW
        "v_fmac_f32_dpp %3, %7, %8" TFA_ROW
        : "+&v"(sum[0]), "+&v"(sum[1]), "+&v"(sum[2]), "+&v"(sum[3])
        : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(u), [t] "n"(T));
  }
  static __device__ __forceinline__ float dot(const float (&x)[4], const float (&y)[4]) {
    float sum;
    asm("s_nop 1\n\t"
        "v_mul_f32_dpp %0, %1, %5" TFA_ROW
        "v_fmac_f32_dpp %0, %2, %6" TFA_ROW
        "v_fmac_f32_dpp %0, %3, %7" TFA_ROW
        "v_fmac_f32_dpp %0, %4, %8" TFA_ROW
        "s_nop 1"
        : "=&v"(sum)
        : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(y[0]), "v"(y[1]), "v"(y[2]), "v"(y[3]), [t] "n"(T));
    return sum;
  }
#undef TFA_ROW
};
// f(0), f(1), ... f(N - 1) with numbers that are part of their type
template <typename F, int... I>
__device__ __forceinline__ void for_each_index(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void for_each(F f) {
  for_each_index(f, std::make_integer_sequence<int, N>());
}
#define TFA_INLINE __attribute__((always_inline))

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

// fold<MASK>(v[i], v[i + N]) of N pairs.  Within rows of 16 an addition that writes the lanes of some quads alone takes two
// instructions where selecting takes three.  (Permutations take values that are two instructions old: waits before, and behind for
// what the compiler does with the sums, since it does not see these instructions.)
template <int MASK, int N>
__device__ __forceinline__ void fold_pairs(const float (&v)[2 * N], float (&w)[N]) {
  if constexpr (MASK == 8 && N == 4) {
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %4, %4 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %0, %8, %8 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %1, %5, %5 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %1, %9, %9 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %2, %6, %6 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %2, %10, %10 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %3, %7, %7 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %3, %11, %11 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "s_nop 1"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3])
        : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[4]), "v"(v[5]), "v"(v[6]), "v"(v[7]));
  } else if constexpr (MASK == 7 && N == 4) {
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %4, %4 row_half_mirror row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %0, %8, %8 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
        "v_add_f32_dpp %1, %5, %5 row_half_mirror row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %1, %9, %9 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
        "v_add_f32_dpp %2, %6, %6 row_half_mirror row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %2, %10, %10 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
        "v_add_f32_dpp %3, %7, %7 row_half_mirror row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %3, %11, %11 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
        "s_nop 1"
        : "=&v"(w[0]), "=&v"(w[1]), "=&v"(w[2]), "=&v"(w[3])
        : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[4]), "v"(v[5]), "v"(v[6]), "v"(v[7]));
  } else if constexpr (MASK == 7 && N == 2) {
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %2, %2 row_half_mirror row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %0, %4, %4 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
        "v_add_f32_dpp %1, %3, %3 row_half_mirror row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %1, %5, %5 row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
        "s_nop 1"
        : "=&v"(w[0]), "=&v"(w[1])
        : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]));
  } else if constexpr (MASK == 8 && N == 2) {
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %2, %2 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %0, %4, %4 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %1, %3, %3 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %1, %5, %5 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "s_nop 1"
        : "=&v"(w[0]), "=&v"(w[1])
        : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = fold<MASK>(v[i], v[i + N]);
  }
}

}  // namespace tfa
