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

// a log2(e) as decay_of takes it.  A rate of -inf (no memory) becomes one that does the same for every step of 1e-35 and more, and with a step
// of zero, as padding has it, keeps the state instead of making NaN of it.  (NaN stays.)
__device__ __forceinline__ float rate_of(float a) { return (a < -1e38f ? -1e38f : a) * kLog2E; }

// log(1 + e^v) and its derivative, off by a few 2^-24 of themselves and of v: with e = e^-|v| and u = 1 + e, log(1 + e) = log(u) + (e - (u - 1)),
// where the second term is what the sum u lost (the hardware's logarithm is good to its last bit next to 1 too).  Measured from -20 to 20:
// 3e-8 of it in the mean square for v > 0, 2e-7 at -8, 1e-6 at most; a series for the artanh took twice the instructions for the same.
// -inf gives a step of 0 with slope 0: a frame that is masked so leaves the state.
__device__ __forceinline__ float softplus(float v, float& slope) {
  const float e = __builtin_amdgcn_exp2f(-fabsf(v) * kLog2E), u = 1.0f + e;
  const float r = __builtin_fmaf(__builtin_amdgcn_logf(u), 0.69314718055994531f, e - (u - 1.0f));
  const float part = __builtin_amdgcn_rcpf(u);
  slope = v < 0.0f ? e * part : part;
  return fmaxf(v, 0.0f) + r;  // (NaN stays: it is in r)
}

// x of the lane whose number differs by MASK (1, 2, 3, 7, 8: permutations within rows of 16 lanes; 4 is 7 after 3)
template <int MASK>
__device__ __forceinline__ float lane_xor(float x) {
  if constexpr (MASK == 4) return lane_xor<3>(lane_xor<7>(x));
  constexpr int ctrl = MASK == 1 ? 0xB1 : MASK == 2 ? 0x4E : MASK == 3 ? 0x1B : MASK == 7 ? 0x141 : 0x128;
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), ctrl, 15, 15, true));
}

// A permutation of lanes takes values that are two instructions old; the compiler keeps to that for its own instructions, and does not
// see those written here: they begin with a wait where what they permute may be new, and what they leave is made old by this before
// a permutation that the compiler writes.
template <int N>
__device__ __forceinline__ void settle(float (&v)[N]) {
  if constexpr (N == 4)
    asm volatile("s_nop 1" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
  else
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("s_nop 1" : "+v"(v[i]));
}

// Products with x[r] of lanes T and T + 1 of the lane's row of 16, which the instructions' operands take from there.
#define TFA_ROW_AT(lane) " row_newbcast:%c[" lane "] row_mask:0xf bank_mask:0xf\n\t"
template <int T>
struct RowLane {
  static __device__ __forceinline__ float lane(float x) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x150 + T, 15, 15, true));
  }
  // out = x (of T) u0 and x (of T + 1) u1
  template <int R>
  static __device__ __forceinline__ void products(const float (&x)[R], float u0, float u1, float (&out0)[R], float (&out1)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) out0[r] = lane(x[r]) * u0, out1[r] = RowLane<T + 1>::lane(x[r]) * u1;
  }
  static __device__ __forceinline__ void products(const float (&x)[4], float u0, float u1, float (&out0)[4], float (&out1)[4]) {
    asm("s_nop 1\n\t"
        "v_mul_f32_dpp %0, %8, %12" TFA_ROW_AT("t")
        "v_mul_f32_dpp %1, %9, %12" TFA_ROW_AT("t")
        "v_mul_f32_dpp %2, %10, %12" TFA_ROW_AT("t")
        "v_mul_f32_dpp %3, %11, %12" TFA_ROW_AT("t")
        "v_mul_f32_dpp %4, %8, %13" TFA_ROW_AT("n")
        "v_mul_f32_dpp %5, %9, %13" TFA_ROW_AT("n")
        "v_mul_f32_dpp %6, %10, %13" TFA_ROW_AT("n")
        "v_mul_f32_dpp %7, %11, %13" TFA_ROW_AT("n")
        : "=&v"(out0[0]), "=&v"(out0[1]), "=&v"(out0[2]), "=&v"(out0[3]), "=&v"(out1[0]), "=&v"(out1[1]), "=&v"(out1[2]), "=&v"(out1[3])
        : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(u0), "v"(u1), [t] "n"(T), [n] "n"(T + 1));
  }
  static __device__ __forceinline__ void products(const float (&x)[2], float u0, float u1, float (&out0)[2], float (&out1)[2]) {
    asm("s_nop 1\n\t"
        "v_mul_f32_dpp %0, %4, %6" TFA_ROW_AT("t")
        "v_mul_f32_dpp %1, %5, %6" TFA_ROW_AT("t")
        "v_mul_f32_dpp %2, %4, %7" TFA_ROW_AT("n")
        "v_mul_f32_dpp %3, %5, %7" TFA_ROW_AT("n")
        : "=&v"(out0[0]), "=&v"(out0[1]), "=&v"(out1[0]), "=&v"(out1[1])
        : "v"(x[0]), "v"(x[1]), "v"(u0), "v"(u1), [t] "n"(T), [n] "n"(T + 1));
  }
  // sum0 = x (of T) . y0, sum1 = x (of T + 1) . y1
  template <int R>
  static __device__ __forceinline__ void dots(const float (&x)[R], const float (&y0)[R], const float (&y1)[R], float& sum0, float& sum1) {
    sum0 = lane(x[0]) * y0[0], sum1 = RowLane<T + 1>::lane(x[0]) * y1[0];
#pragma unroll
    for (int r = 1; r < R; ++r)
      sum0 = __builtin_fmaf(lane(x[r]), y0[r], sum0), sum1 = __builtin_fmaf(RowLane<T + 1>::lane(x[r]), y1[r], sum1);
  }
  static __device__ __forceinline__ void dots(const float (&x)[4], const float (&y0)[4], const float (&y1)[4], float& sum0, float& sum1) {
    asm("s_nop 1\n\t"
        "v_mul_f32_dpp %0, %2, %6" TFA_ROW_AT("t")
        "v_mul_f32_dpp %1, %2, %10" TFA_ROW_AT("n")
        "v_fmac_f32_dpp %0, %3, %7" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %1, %3, %11" TFA_ROW_AT("n")
        "v_fmac_f32_dpp %0, %4, %8" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %1, %4, %12" TFA_ROW_AT("n")
        "v_fmac_f32_dpp %0, %5, %9" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %1, %5, %13" TFA_ROW_AT("n")
        : "=&v"(sum0), "=&v"(sum1)
        : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(y0[0]), "v"(y0[1]), "v"(y0[2]), "v"(y0[3]), "v"(y1[0]), "v"(y1[1]),
          "v"(y1[2]), "v"(y1[3]), [t] "n"(T), [n] "n"(T + 1));
  }
  static __device__ __forceinline__ void dots(const float (&x)[2], const float (&y0)[2], const float (&y1)[2], float& sum0, float& sum1) {
    asm("s_nop 1\n\t"
        "v_mul_f32_dpp %0, %2, %4" TFA_ROW_AT("t")
        "v_mul_f32_dpp %1, %2, %6" TFA_ROW_AT("n")
        "v_fmac_f32_dpp %0, %3, %5" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %1, %3, %7" TFA_ROW_AT("n")
        : "=&v"(sum0), "=&v"(sum1)
        : "v"(x[0]), "v"(x[1]), "v"(y0[0]), "v"(y0[1]), "v"(y1[0]), "v"(y1[1]), [t] "n"(T), [n] "n"(T + 1));
  }
  // sum += x (of T) u
  template <int R>
  static __device__ __forceinline__ void add(const float (&x)[R], float u, float (&sum)[R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) sum[r] = __builtin_fmaf(lane(x[r]), u, sum[r]);
  }
  static __device__ __forceinline__ void add(const float (&x)[4], float u, float (&sum)[4]) {
    asm("s_nop 1\n\t"
        "v_fmac_f32_dpp %0, %4, %8" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %1, %5, %8" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %2, %6, %8" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %3, %7, %8" TFA_ROW_AT("t")
        : "+&v"(sum[0]), "+&v"(sum[1]), "+&v"(sum[2]), "+&v"(sum[3])
        : "v"(x[0]), "v"(x[1]), "v"(x[2]), "v"(x[3]), "v"(u), [t] "n"(T));
  }
  // g += c (of T) u;  sum_b = b (of T) . g,  sum_c = c (of T) . h
  template <int R>
  static __device__ __forceinline__ void reverse(const float (&b)[R], const float (&c)[R], float u, const float (&h)[R], float (&g)[R], float& sum_b,
                                                 float& sum_c) {
    add(c, u, g);
    sum_b = lane(b[0]) * g[0], sum_c = lane(c[0]) * h[0];
#pragma unroll
    for (int r = 1; r < R; ++r) sum_b = __builtin_fmaf(lane(b[r]), g[r], sum_b), sum_c = __builtin_fmaf(lane(c[r]), h[r], sum_c);
  }
  static __device__ __forceinline__ void reverse(const float (&b)[4], const float (&c)[4], float u, const float (&h)[4], float (&g)[4], float& sum_b,
                                                 float& sum_c) {
    asm("s_nop 1\n\t"
        "v_fmac_f32_dpp %0, %10, %18" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %1, %11, %18" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %2, %12, %18" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %3, %13, %18" TFA_ROW_AT("t")
        "v_mul_f32_dpp %4, %6, %0" TFA_ROW_AT("t")
        "v_mul_f32_dpp %5, %10, %14" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %4, %7, %1" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %5, %11, %15" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %4, %8, %2" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %5, %12, %16" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %4, %9, %3" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %5, %13, %17" TFA_ROW_AT("t")
        : "+&v"(g[0]), "+&v"(g[1]), "+&v"(g[2]), "+&v"(g[3]), "=&v"(sum_b), "=&v"(sum_c)
        : "v"(b[0]), "v"(b[1]), "v"(b[2]), "v"(b[3]), "v"(c[0]), "v"(c[1]), "v"(c[2]), "v"(c[3]), "v"(h[0]), "v"(h[1]), "v"(h[2]), "v"(h[3]),
          "v"(u), [t] "n"(T));
  }
  static __device__ __forceinline__ void reverse(const float (&b)[2], const float (&c)[2], float u, const float (&h)[2], float (&g)[2], float& sum_b,
                                                 float& sum_c) {
    asm("s_nop 1\n\t"
        "v_fmac_f32_dpp %0, %6, %10" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %1, %7, %10" TFA_ROW_AT("t")
        "v_mul_f32_dpp %3, %6, %8" TFA_ROW_AT("t")
        "v_mul_f32_dpp %2, %4, %0" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %3, %7, %9" TFA_ROW_AT("t")
        "v_fmac_f32_dpp %2, %5, %1" TFA_ROW_AT("t")
        : "+&v"(g[0]), "+&v"(g[1]), "=&v"(sum_b), "=&v"(sum_c)
        : "v"(b[0]), "v"(b[1]), "v"(c[0]), "v"(c[1]), "v"(h[0]), "v"(h[1]), "v"(u), [t] "n"(T));
  }
};
#undef TFA_ROW_AT

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

// Sums over a row's 16 lanes of the 8 values of two tokens: lane l receives those of value 4 (l / 8) + 2 (l / 4 % 2) + l / 2 % 2.  An addition
// that writes the lanes of some quads alone takes two instructions where selecting takes three; below a quad lanes are selected by `odd`, those
// with bit 1 of their number set.
__device__ __forceinline__ void fold_row(const float (&v)[8], const float (&u)[8], unsigned long long odd, float& sum_v, float& sum_u) {
  float w0, w1, w2, w3, x0, x1, y0, y1, y2, y3, z0, z1;
#define TFA_HALVES(to, low, high) \
  "v_add_f32_dpp " to ", " low ", " low " row_ror:8 row_mask:0xf bank_mask:0x3\n\t" \
  "v_add_f32_dpp " to ", " high ", " high " row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
#define TFA_QUADS(to, low, high) \
  "v_add_f32_dpp " to ", " low ", " low " row_half_mirror row_mask:0xf bank_mask:0x5\n\t" \
  "v_add_f32_dpp " to ", " high ", " high " row_half_mirror row_mask:0xf bank_mask:0xa\n\t"
  asm("s_nop 1\n\t"
      TFA_HALVES("%0", "%4", "%8") TFA_HALVES("%2", "%6", "%10") TFA_HALVES("%1", "%5", "%9") TFA_HALVES("%3", "%7", "%11")
      : "=&v"(w0), "=&v"(w1), "=&v"(w2), "=&v"(w3)
      : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[4]), "v"(v[5]), "v"(v[6]), "v"(v[7]));
  asm("s_nop 1\n\t"
      TFA_HALVES("%0", "%4", "%8") TFA_HALVES("%2", "%6", "%10") TFA_HALVES("%1", "%5", "%9") TFA_HALVES("%3", "%7", "%11")
      : "=&v"(y0), "=&v"(y1), "=&v"(y2), "=&v"(y3)
      : "v"(u[0]), "v"(u[1]), "v"(u[2]), "v"(u[3]), "v"(u[4]), "v"(u[5]), "v"(u[6]), "v"(u[7]));
  float keep_v, give_v, keep_u, give_u;
  asm("s_nop 1\n\t"
      TFA_QUADS("%0", "%10", "%12") TFA_QUADS("%1", "%11", "%13") TFA_QUADS("%2", "%14", "%16") TFA_QUADS("%3", "%15", "%17")
      "v_cndmask_b32 %5, %1, %0, %18\n\t"  // (what the other lane keeps)
      "v_cndmask_b32 %7, %3, %2, %18\n\t"
      "v_cndmask_b32 %4, %0, %1, %18\n\t"
      "v_cndmask_b32 %6, %2, %3, %18\n\t"
      "v_add_f32_dpp %4, %5, %4 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
      "v_add_f32_dpp %6, %7, %6 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n\t"
      "s_nop 0\n\t"
      "v_add_f32_dpp %8, %4, %4 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n\t"
      "v_add_f32_dpp %9, %6, %6 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf"
      : "=&v"(x0), "=&v"(x1), "=&v"(z0), "=&v"(z1), "=&v"(keep_v), "=&v"(give_v), "=&v"(keep_u), "=&v"(give_u), "=&v"(sum_v), "=&v"(sum_u)
      : "v"(w0), "v"(w1), "v"(w2), "v"(w3), "v"(y0), "v"(y1), "v"(y2), "v"(y3), "s"(odd));
#undef TFA_HALVES
#undef TFA_QUADS
}

}  // namespace tfa
