// Linear attention with decays in blocks of C tokens on the bf16 matrix cores: one pass (model_ops.h, AttnPass)
//
//   out_i = scale ( sum_{j <= i} gamma^(i-j) (a_i . b_j) c_j  +  gamma^(i+e) a_i M ),
//   M    <- gamma^L M + sum_j gamma^(L-e-j) b_j c_j^T             i, j < L: places in the block, in the pass's order
//
// with e = 1 forward and 0 in a reversed pass (a state reaches its first token undecayed there).
//
// A workgroup carries one head's state, 32 columns a wave with all R rows of them in registers (accumulators of
// v_mfma_f32_32x32x16_bf16), through its tokens.  The accumulator layout (lane: column, register: row) is also the
// layout of a matrix operand (lane: column or row, register: contraction) up to an exchange of index bits 2 and 3, so with the
// rows that feed the product taken in that order (pi below) the state goes from accumulators to operands without leaving
// the registers.  Scores are 16 x 16 tiles (v_mfma_f32_16x16x32_bf16), shared out over the waves and joined in LDS.
// Outputs are computed transposed (lane: token), so that decays by token are one factor a lane and stores are 16 bytes.
//
// The log decay's gradient is the sum over all pairs of lag * flow, a flow being what a source (a token's b c^T, or
// the first state) contributes through a sink (a token's out . x, or the last state's gradient dS_T).  Pairs in one block: the
// query gradient's pass has their scores a . b, multiplies c . x out likewise, and sums lag gamma^lag of the two.  Pairs of
// different blocks: with the tokens in stretches of `stretch`, places in a stretch counted from 1, lag = (sink's stretch -
// source's) * stretch + sink's place - source's place, so their sum is
//   stretch * sum over the borders of S . dS  +  sum_t place_t q_t . dq_t  -  sum_s place_s k_s . dk_s
// of gradients through states alone.  The query gradient's pass adds the second sum and leaves the states S at the borders in
// memory; the key gradient's pass, which meets the same borders with dS, adds the first and the third.  (dS_T is a sink of place
// (T - 1) % stretch + 1 for all blocks but the last, whose tokens are told by their distance from the end.)  Places are at most
// 256 where lags are a head's memory: rounding counts some 256 / lag times in these, so states enter such passes in all
// their pieces (1e-7, not 1e-5), and a head without memory gets an exact 0.  (The state's derivative carried along in registers
// took the query gradient's pass from 150 to 500 us at 8 x 4096 tokens of 16 heads of 128.)
//
// Operands lie in LDS by token; products over features read them as they are, products over tokens through the transposing
// LDS read (ds_read_b64_tr_b16: 16 lanes take 4 tokens x 16 features, each receives one feature's 4 tokens).  The next block
// is on its way in registers while one is computed.
//
// What it measures: 32 x 1024 tokens of 16 bf16 heads of 128 forward 181 us (3.0 TB/s of operands and results; at the copy's rate
// 104), of 64 98 us (52); fp16 230 us, fp32 (3.1 TB/s) 345 us.  A training pass of 8 x 4096 tokens of 16 heads of 128: 1.09 ms, 1.4 in
// fp16, 2.1 in fp32.  What bounds it: a block's chain of dependent steps (stage, scores, decays and pieces, outputs, state) with two waves a
// SIMD at most, as the state leaves registers for no more (one where 512 workgroups of two waves are all there is: 64 columns and fewer): the
// matrix units are 30 to 44 % busy, vector units and memory less than that.
// Two blocks on their way instead of one, or heads in another order over the L2s, change nothing; 16 columns a wave (four
// waves a SIMD) read each operand from LDS twice as often: bf16 229 us for the 162 of 32, fp32 the other way (137 for 205 at
// 64 features).  One layout is kept for all types.
//
// Precision: operands are exact sums of bf16 pieces (bf16: 1, fp16: 2, fp32: 3).  Scores, states and decayed c's are fp32 where they
// are summed and kept, and are split into pieces to nearest as they enter a product: two for 16-bit outputs (2^-17, nothing beside their
// rounding), three for fp32 outputs and for what enters states.  Products of pieces i, j are taken where i + j is within the piece count,
// into fp32.
//
// What is not finite reaches what the recurrence lets it reach, and no token before it: scores of later tokens are replaced by zeros, and
// a c that is not finite (or rounds to infinity as bf16: fp32 above 3.39e38) is looked for as it is staged, taken out of its block and put
// in again as NaN from its token on, in its column (an infinity too: the state's splitting into pieces makes NaN of it anyway).  The decays'
// gradient of a head with such a value is NaN.  With the looking a training pass of 8 x 4096 tokens takes 1103 us for 1085, fp32 2095 for 2058.
#pragma once
#include <algorithm>
#include <type_traits>

#include "attention_device.h"

namespace tfa {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16;

__device__ __forceinline__ floatx16 mfma(uint4 a, uint4 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ floatx4 mfma(uint4 a, uint4 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// two fp32 as N packed pairs of bf16 pieces
template <int N>
__device__ __forceinline__ void split_pair(float x, float y, unsigned (&p)[N]) {
  floatx2 r = {x, y};
#pragma unroll
  for (int q = 0; q < N; ++q) {
    p[q] = __builtin_bit_cast(unsigned, __builtin_convertvector(r, bf16x2));
    if (q + 1 < N) {
      r[0] -= __uint_as_float(p[q] << 16);
      r[1] -= __uint_as_float(p[q] & 0xffff0000u);
    }
  }
}
// eight fp32 as an operand of N pieces
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], uint4 (&out)[N]) {
  unsigned p[4][N];
#pragma unroll
  for (int i = 0; i < 4; ++i) split_pair<N>(x[2 * i], x[2 * i + 1], p[i]);
#pragma unroll
  for (int q = 0; q < N; ++q) out[q] = make_uint4(p[0][q], p[1][q], p[2][q], p[3][q]);
}

// four tokens (rows `pitch` apart) of the lane's feature and the four after them
__device__ __forceinline__ uint4 read_transposed(const u16* src, int pitch) {
  typedef short shortx4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) shortx4* Lds;
  const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)src));
  const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(src + 4 * pitch)));
  return make_uint4(x.x, x.y, y.x, y.y);
}

// index bits 2 and 3 exchanged: the row that accumulator place m stands for
__device__ __forceinline__ int pi(int m) { return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1); }

// a value that the compiler takes as new: what follows from it is computed again, not kept in registers over a loop
__device__ __forceinline__ unsigned opaque(unsigned x) {
  asm volatile("" : "+v"(x));
  return x;
}

// the lane's number, computed where it is used
__device__ __forceinline__ int lane_again() {
  int x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
  return x;
}

template <typename T>
struct Kind;
template <>
struct Kind<__bf16> {
  static constexpr int pieces = 1, block = 64, out_pieces = 2;
};
template <>
struct Kind<_Float16> {
  static constexpr int pieces = 2, block = 32, out_pieces = 2;
};
template <>
struct Kind<float> {
  static constexpr int pieces = 3, block = 32, out_pieces = 3;
};

// Modes of the kernel: a pass with its outputs, the same with its part of the decays' gradient, or only the segments' own states
enum { kPass = 0, kLags = 1, kSums = 2 };

// pieces of two neighbouring features, from their raw bits: packed (f, f + 1)
template <typename T>
__device__ __forceinline__ void pair_pieces(const unsigned* w, unsigned (&p)[Kind<T>::pieces]) {
  if constexpr (sizeof(T) == 4)
    split_pair<3>(__uint_as_float(w[0]), __uint_as_float(w[1]), p);
  else if constexpr (Kind<T>::pieces == 2)
    split_pair<2>((float)__builtin_bit_cast(_Float16, (u16)w[0]), (float)__builtin_bit_cast(_Float16, (u16)(w[0] >> 16)), p);
  else
    p[0] = w[0];
}

template <typename T, int RP, int NW, int MODE>
struct Blocks {
  static constexpr bool out = MODE != kSums, lags = MODE == kLags;
  static constexpr int NP = Kind<T>::pieces, C = Kind<T>::block, JP = Kind<T>::out_pieces;
  static constexpr int J = lags ? 3 : JP;  // pieces of a state; of a score: JP
  static constexpr int CP = 32 * NW, threads = 64 * NW, TI = C / 32, RB = RP / 32;
  // score tiles (x, y, z): tokens i = 16 x + l against j = 32 y + 8 g + 4 z + r (lane l of group g, register r)
  static constexpr int all_tiles = TI == 2 ? 12 : 4, tiles = all_tiles / NW;
  static_assert(all_tiles % NW == 0, "the waves have equal shares");
  static constexpr int V = 16 / sizeof(T);
  // LDS in 16-bit units; rows start 4 banks apart, modulo 64
  static constexpr int pitch = RP + 8, pitch_c = CP + 8, pitch_s = C + 8;
  static constexpr int plane = C * pitch, plane_c = C * pitch_c, plane_s = C * pitch_s;
  static constexpr int a_end = out ? NP * plane : 0, s_size = out ? JP * plane_s : 0, bc_size = NP * (plane + plane_c);
  // x as it is in memory (16-bit units; rows 16 bytes longer than they need), before the scores take its place
  static constexpr int W = sizeof(T) / 2, pitch_x = (CP + V) * W, x_size = lags ? C * pitch_x : 0;
  // scores (and x) have a place of their own where two workgroups then still fit a compute unit; else a's, once a is done
  // with (and x is read from memory)
  static constexpr int sx_size = s_size > x_size ? s_size : x_size;
  static constexpr int marks = 4 * C * 4 + (out ? (CP + 4) * 4 : 0);  // bytes of the tables and of what `bad_c` leaves
  static constexpr bool own_scores = (a_end + sx_size + bc_size) * 2 + marks <= 80 * 1024;
  static constexpr bool x_in_lds = lags && own_scores;
  static constexpr int off_s = own_scores ? a_end : 0;
  static constexpr int off_b = own_scores ? a_end + sx_size : a_end > s_size ? a_end : s_size;
  static constexpr int off_c = off_b + NP * plane, off_end = off_c + NP * plane_c;
  // tables: scale gamma^(i - j) by i - j + C (zero before C), gamma^(C - e - j) by j (zero from C on)
  static constexpr int bytes = off_end * 2 + marks;
  // an operand's rows in 16-byte pieces: lanes over the features, then over the tokens
  template <int F>
  struct Rows {
    static constexpr int lanes = F / V, at_once = threads / lanes, passes = C / at_once;
    static_assert(C % at_once == 0, "whole passes");
    uint4 w[passes];
  };
};

template <typename T, int RP, int NW, int MODE>
__global__ __launch_bounds__(64 * NW, NW == 2 && RP == 128 ? 1 : 2) void attn_blocks_kernel(AttnPass p, int first_seg, int segs,
                                                                                              bool whole_o) {
  using B = Blocks<T, RP, NW, MODE>;
  constexpr int NP = B::NP, C = B::C, J = B::J, JP = B::JP, TI = B::TI, RB = B::RB, V = B::V;
  constexpr int STEPS = MODE == kPass ? 100 : 1;
  constexpr bool OUT = B::out, LAGS = B::lags;
  __shared__ __align__(16) unsigned char lds[B::bytes];
  u16* const L16 = reinterpret_cast<u16*>(lds);
  float* const pow_tab = reinterpret_cast<float*>(lds + B::off_end * 2);
  float* const upd_tab = pow_tab + 2 * C;
  int* const bad_from = reinterpret_cast<int*>(upd_tab + 2 * C);  // by column: the first token whose c is not finite
  int* const bad_block = bad_from + B::CP;                       // one past the last block with such a c

  const int t = threadIdx.x, lane = t & 63, half = lane >> 5, l32 = lane & 31, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  // Heads vary fastest and neighbours run on one XCD: tokens are rows of all heads, and one head alone keeps to few of an
  // L2's channels (16 heads of 256 bytes on 8 XCDs, head by XCD: two of its sixteen).
  unsigned block = xcd_tile_remap32(blockIdx.x, gridDim.x);
  const int h = (int)(block % p.heads);
  block /= p.heads;
  const int seg = first_seg + (int)(block % segs);
  const long long b = p.first + block / segs, bh = b * p.heads + h;
  const long long len = live_tokens(p, b);
  const long long seg_lo = seg * p.seg_tokens, seg_end = min(seg_lo + p.seg_tokens, p.tokens);
  const long long lo = min(seg_lo, len), hi = min(seg_end, len);
  const int rows = p.rows, cols = p.cols, e = p.reverse ? 0 : 1;
  const bool reverse = p.reverse;
  const double g = (double)log_decay_of(p.log_decay, h);

  for (int i = t; i < 2 * C; i += B::threads) {
    pow_tab[i] = i < C ? 0.0f : (float)(exp(g * (double)(i - C)) * (double)p.scale);
    upd_tab[i] = i < C ? (float)exp(g * (double)(C - e - i)) : 0.0f;
  }
  if (OUT && t == 0) *bad_block = 0;

  // the state: column 32 wave + l32, register r of block rb: row 32 rb + 16 (r / 8) + 8 half + r % 8
  floatx16 m[RB];
  const int ncol = 32 * wave + l32;
  const size_t m0 = (size_t)bh * rows * cols, seg_size = (size_t)p.batch * p.heads * rows * cols;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 32 * rb + 16 * (r >> 3) + 8 * half + (r & 7);
      float x = 0.0f;
      if (OUT && row < rows && ncol < cols) {
        const size_t at = m0 + (size_t)(row * p.m_r + ncol * p.m_n);
        if (p.segments > 1)
          x = p.seg_state[seg * seg_size + at];
        else if (p.m_in)
          x = p.m_in[at] * p.m_in_scale;
      }
      m[rb][r] = x;
    }
  double dg = 0.0;

  using RowsB = typename B::template Rows<RP>;
  using RowsC = typename B::template Rows<B::CP>;
  struct Set {
    RowsB a, b;
    RowsC c, x;
  };
  const int b_f = (t % RowsB::lanes) * V, b_u = t / RowsB::lanes, c_f = (t % RowsC::lanes) * V, c_u = t / RowsC::lanes;
  const bool b_on = b_f < rows, c_on = c_f < cols;

  // Row u of a block (in the pass's order) is u, or reversed C - 1 - u, token strides above the block's base; a partial
  // reversed block's base lies before its tokens, whose rows are not read.  Offsets in a block are 32-bit bytes.  Threads
  // past the features read feature 0 and keep zeros.
  const char* const base_a = OUT ? reinterpret_cast<const char*>(head_base<T>(p.a, b, h)) : nullptr;
  const char* const base_b = reinterpret_cast<const char*>(head_base<T>(p.b, b, h));
  const char* const base_c = reinterpret_cast<const char*>(head_base<T>(p.c, b, h));
  const char* const base_x = B::x_in_lds ? reinterpret_cast<const char*>(head_base<T>(p.x, b, h)) : nullptr;
  const long long st_x = B::x_in_lds ? p.x.st * (long long)sizeof(T) : 0;
  const long long st_a = OUT ? p.a.st * (long long)sizeof(T) : 0, st_b = p.b.st * (long long)sizeof(T), st_c = p.c.st * (long long)sizeof(T);
  auto offset = [&](long long st, int u, int f) {
    return (unsigned)(reverse ? C - 1 - u : u) * (unsigned)st + (unsigned)f * (unsigned)sizeof(T);
  };
  const unsigned off_a = offset(st_a, b_u, b_on ? b_f : 0), off_b = offset(st_b, b_u, b_on ? b_f : 0), off_c = offset(st_c, c_u, c_on ? c_f : 0),
                 off_x = offset(st_x, c_u, c_on ? c_f : 0);

  // blocks in the pass's order; their borders are the same tokens in both directions
  const int total = (int)((hi - lo + C - 1) / C);
  auto block_lo = [&](int i) { return lo + (long long)(reverse ? total - 1 - i : i) * C; };
  // (all: a whole block; else rows past the last one are zeros)
  auto fetch_rows = [&](auto& r, const char* base, unsigned off0, long long st, int u0, int count, auto all) {
    using R = std::remove_reference_t<decltype(r)>;
    const unsigned step = (unsigned)R::at_once * (reverse ? 0u - (unsigned)st : (unsigned)st);
    unsigned off = opaque(off0);
#pragma unroll
    for (int q = 0; q < R::passes; ++q, off += step) {
      if (!decltype(all)::value) r.w[q] = make_uint4(0, 0, 0, 0);
      if (decltype(all)::value || u0 + q * R::at_once < count) r.w[q] = *reinterpret_cast<const uint4*>(base + off);
    }
  };
  auto fetch = [&](int i, Set& set) {
    const long long c0 = block_lo(i);
    const int count = (int)min((long long)C, hi - c0);
    const long long at = reverse ? c0 - (C - count) : c0;
    auto each = [&](auto all) {
      if constexpr (OUT) fetch_rows(set.a, base_a + at * st_a, off_a, st_a, b_u, count, all);
      fetch_rows(set.b, base_b + at * st_b, off_b, st_b, b_u, count, all);
      fetch_rows(set.c, base_c + at * st_c, off_c, st_c, c_u, count, all);
      if constexpr (B::x_in_lds) fetch_rows(set.x, base_x + at * st_x, off_x, st_x, c_u, count, all);
    };
    if (count == C)
      each(std::true_type{});
    else
      each(std::false_type{});
  };
  // rows from registers to LDS, in pieces; `mark` becomes NaN where a leading piece is not finite
  auto stage_rows = [&](const auto& r, u16* dst, int step, int plane, bool on, auto check, float& mark) {
    using R = std::remove_cv_t<std::remove_reference_t<decltype(r)>>;
    auto look = [&](unsigned pair) {
      if constexpr (decltype(check)::value) mark = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), bf16x2{}, mark, false);
    };
#pragma unroll
    for (int q = 0; q < R::passes; ++q, dst += step) {
      const uint4 v = on ? r.w[q] : make_uint4(0, 0, 0, 0);
      if constexpr (NP == 1) {
        *reinterpret_cast<uint4*>(dst) = v;
        look(v.x), look(v.y), look(v.z), look(v.w);
      } else {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
        unsigned pc[V / 2][NP];
#pragma unroll
        for (int k = 0; k < V / 2; ++k) pair_pieces<T>(w + k * (int)sizeof(T) / 2, pc[k]), look(pc[k][0]);
#pragma unroll
        for (int z = 0; z < NP; ++z)
          if constexpr (V == 8)
            *reinterpret_cast<uint4*>(dst + z * plane) = make_uint4(pc[0][z], pc[1][z], pc[2][z], pc[3][z]);
          else
            *reinterpret_cast<uint2*>(dst + z * plane) = make_uint2(pc[0][z], pc[1][z]);
      }
    }
  };
  auto stage = [&](int i, const Set& set) {
    const int at = b_u * B::pitch + b_f, step = RowsB::at_once * B::pitch;
    float mark = 0.0f;
    if constexpr (OUT) stage_rows(set.a, L16 + at, step, B::plane, b_on, std::false_type{}, mark);
    stage_rows(set.b, L16 + B::off_b + at, step, B::plane, b_on, std::false_type{}, mark);
    if constexpr (B::x_in_lds) {
      u16* dst = L16 + B::off_s + c_u * B::pitch_x + c_f * B::W;
#pragma unroll
      for (int q = 0; q < RowsC::passes; ++q, dst += RowsC::at_once * B::pitch_x)
        *reinterpret_cast<uint4*>(dst) = c_on ? set.x.w[q] : make_uint4(0, 0, 0, 0);
    }
    stage_rows(set.c, L16 + B::off_c + c_u * B::pitch_c + c_f, RowsC::at_once * B::pitch_c, B::plane_c, c_on, std::bool_constant<OUT>{}, mark);
    if constexpr (OUT)
      if (__any(mark != mark) && lane == 0) *bad_block = i + 1;
  };
  // A c that is not finite may not meet the zeros that stand for the scores of tokens before it: it is taken out of the block, and its
  // column becomes NaN from its token on (poison).  Nothing of this runs where c is finite.
  auto take_out = [&]() {
    const int n = 64 * wave + lane_again();
    if (n < B::CP) {
      int from = C;
      for (int u = C - 1; u >= 0; --u) {
        u16* const at = L16 + B::off_c + u * B::pitch_c + n;
        if ((*at & 0x7f80) != 0x7f80) continue;
        from = u;
        for (int q = 0; q < NP; ++q) at[q * B::plane_c] = 0;
      }
      bad_from[n] = from;
    }
    __syncthreads();
  };
  // transposed operands: lane's row (feature) l32, in the order pi for b, tokens 8 half + 0 .. 7 of the sixteen from `src`
  const int tr_tok = 8 * half + ((lane & 15) >> 2), tr_f = lane & 16;
  const int tr_b = tr_tok * B::pitch + tr_f + 8 * (lane & 1) + 2 * (lane & 2), tr_c = tr_tok * B::pitch_c + tr_f + 4 * (lane & 3);

  // score tiles: token by l16, features 8 g + 0 .. 7; a score row stands for token 8 (l16 / 4) + l16 % 4
  const int l16 = lane & 15, grp = lane >> 4;
  const int at_a = l16 * B::pitch + 8 * grp, at_b = (8 * (l16 >> 2) + (l16 & 3)) * B::pitch + 8 * grp;
  int tile_x[B::tiles], tile_y[B::tiles], tile_z[B::tiles];
#pragma unroll
  for (int k = 0; k < B::tiles; ++k) {
    const int id = wave + NW * k, u = id >> 1;  // u: (0, 0), (1, 0), (2, 0), (3, 0), (2, 1), (3, 1)
    tile_z[k] = id & 1;
    tile_y[k] = u >> 2;
    tile_x[k] = u < 4 ? u : u - 2;
  }
  // states at the borders of stretches, as the lanes hold them
  float* const border = LAGS ? p.border_state + (size_t)bh * p.borders * (RB * 16 * B::threads) + t : nullptr;
  auto poison = [&](auto& o) {
    const float nan = __uint_as_float(0x7fc00000u);
    const int own = lane_again(), l32 = own & 31;
    const int* const from_of = bad_from + 32 * wave;
    if (from_of[l32] < C)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int r = 0; r < 16; ++r) m[rb][r] = nan;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int from = from_of[4 * (own >> 5) + 8 * (r >> 2) + (r & 3)];
#pragma unroll
      for (int x = 0; x < TI; ++x)
        if (32 * x + l32 >= from) o[x][r] = nan;
    }
    if (LAGS) dg = (double)nan;
  };
  DecaySteps gamma_full(exp(g * (double)C));
  const float gamma_part = scalar((float)exp(g * (double)((hi - lo) % C)));
  const float first = scalar((float)exp(g * (double)e));
  auto compute = [&](int i, Set& set) {
    const long long c0 = block_lo(i);
    const int count = (int)min((long long)C, hi - c0);
    __syncthreads();  // the block before is done with LDS
    stage(i, set);
    __syncthreads();
    const bool bad_c = OUT && __builtin_amdgcn_readfirstlane(*bad_block) == i + 1;
    if (i + 1 < total) fetch(i + 1, set);

    const bool at_border = LAGS && c0 > 0 && (c0 & (p.stretch - 1)) == 0;
    float* const held = LAGS && at_border ? border + (size_t)((c0 >> p.log_stretch) - 1) * (RB * 16 * B::threads) : nullptr;
    if constexpr (LAGS)
      if (at_border && !reverse)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int r = 0; r < 16; ++r) held[(rb * 16 + r) * B::threads] = m[rb][r];

    floatx16 o[OUT ? TI : 1];
    if constexpr (OUT) {
      // scores^T = b a^T, with their gamma^(i - j)
      floatx4 s[B::tiles];
#pragma unroll
      for (int k = 0; k < B::tiles; ++k) s[k] = floatx4{};
#pragma unroll
      for (int ks = 0; ks < RP / 32; ++ks) {
        uint4 fa[B::tiles][NP], fb[B::tiles][NP];
#pragma unroll
        for (int k = 0; k < B::tiles; ++k)
#pragma unroll
          for (int q = 0; q < NP; ++q) {
            fa[k][q] = *reinterpret_cast<const uint4*>(L16 + q * B::plane + 16 * tile_x[k] * B::pitch + 32 * ks + at_a);
            fb[k][q] = *reinterpret_cast<const uint4*>(L16 + B::off_b + q * B::plane + (32 * tile_y[k] + 4 * tile_z[k]) * B::pitch + 32 * ks + at_b);
          }
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
          for (int z = 0; z < NP; ++z)
            if (q + z < 3)
#pragma unroll
              for (int k = 0; k < B::tiles; ++k) s[k] = mfma(fb[k][q], fa[k][z], s[k]);  // (neighbours do not wait for each other)
      }
      if constexpr (LAGS)
        if (!reverse) {
          // pairs in the block: c . x beside a . b
          float sum = 0.0f;
#pragma unroll
          for (int k = 0; k < B::tiles; ++k) {
            floatx4 s2 = {};
            const int i = 16 * tile_x[k] + l16;
            const char* const xr = B::x_in_lds ? nullptr : reinterpret_cast<const char*>(head_base<T>(p.x, b, h) + (c0 + min(i, count - 1)) * p.x.st);
            (void)xr;
#pragma unroll
            for (int ks = 0; ks < B::CP / 32; ++ks) {
              const int f = 32 * ks + 8 * grp;
              unsigned raw[4 * sizeof(T) / 2];
#pragma unroll
              for (int y = 0; y < (int)sizeof(T) / 2; ++y) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if constexpr (B::x_in_lds)
                  v = *reinterpret_cast<const uint4*>(L16 + B::off_s + i * B::pitch_x + f * B::W + 8 * y);
                else if (i < count && f + y * V < cols)
                  v = *reinterpret_cast<const uint4*>(xr + f * (int)sizeof(T) + 16 * y);
                raw[4 * y] = v.x, raw[4 * y + 1] = v.y, raw[4 * y + 2] = v.z, raw[4 * y + 3] = v.w;
              }
              unsigned pc[4][NP];
#pragma unroll
              for (int y = 0; y < 4; ++y) pair_pieces<T>(raw + y * (int)sizeof(T) / 2, pc[y]);
#pragma unroll
              for (int q = 0; q < NP; ++q) {
                const uint4 fc = *reinterpret_cast<const uint4*>(L16 + B::off_c + q * B::plane_c + (32 * tile_y[k] + 4 * tile_z[k] + 8 * (l16 >> 2) + (l16 & 3)) * B::pitch_c + f);
#pragma unroll
                for (int z = 0; z < NP; ++z)
                  if (q + z < 3) s2 = mfma(fc, make_uint4(pc[0][z], pc[1][z], pc[2][z], pc[3][z]), s2);
              }
            }
            const int own = lane_again(), lag = 16 * (tile_x[k] - 2 * tile_y[k]) - 4 * tile_z[k] + (own & 15) - 8 * (own >> 4);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float with = __builtin_fmaf(s[k][r] * pow_tab[C + lag - r] * (float)(lag - r), s2[r], sum);
              sum = lag >= r ? with : sum;
            }
          }
          dg += (double)sum;
        }
      auto put_scores = [&]() {
#pragma unroll
        for (int k = 0; k < B::tiles; ++k) {
          const int own = lane_again(), i16 = own & 15, j8 = 8 * (own >> 4);
          const int j0 = 32 * tile_y[k] + 4 * tile_z[k], lag = 16 * tile_x[k] - j0 + i16 - j8;
          u16* const dst = L16 + B::off_s + (16 * tile_x[k] * B::pitch_s + j0) + (i16 * B::pitch_s + j8);
          float w[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float with = s[k][r] * pow_tab[C + lag - r];
            w[r] = lag >= r ? with : 0.0f;  // (not by a product: the score of a token that is not finite is NaN)
          }
          unsigned p0[JP], p1[JP];
          split_pair<JP>(w[0], w[1], p0);
          split_pair<JP>(w[2], w[3], p1);
#pragma unroll
          for (int q = 0; q < JP; ++q) *reinterpret_cast<uint2*>(dst + q * B::plane_s) = make_uint2(p0[q], p1[q]);
        }
      };
      if constexpr (B::own_scores && !LAGS) put_scores();
      // over the features: out^T = M^T a^T
#pragma unroll
      for (int x = 0; x < TI; ++x) o[x] = floatx16{};
#pragma unroll
      for (int ks = 0; ks < RP / 16; ++ks) {
        if (ks % STEPS == 0) __builtin_amdgcn_sched_barrier(0);  // (a few steps' operands at a time: registers)
        uint4 fa[NP][TI], fm[J];
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
          for (int x = 0; x < TI; ++x)
            fa[q][x] = *reinterpret_cast<const uint4*>(L16 + q * B::plane + (32 * x + l32) * B::pitch + 16 * ks + 8 * half);
        float mv[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mv[k] = m[ks / 2][8 * (ks & 1) + k];
        split8<J>(mv, fm);
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
          for (int z = 0; z < J; ++z)
            if (q + z < J)
#pragma unroll
              for (int x = 0; x < TI; ++x) o[x] = mfma(fm[z], fa[q][x], o[x]);
      }
      __builtin_amdgcn_sched_barrier(0);
      // a state reaches token i with gamma^(i + e)
#pragma unroll
      for (int x = 0; x < TI; ++x) {
        const float w = pow_tab[C + 32 * x + l32] * first;
#pragma unroll
        for (int r = 0; r < 16; ++r) o[x][r] *= w;
        if constexpr (LAGS) {
          const int own = lane_again(), u = 32 * x + (own & 31), n4 = 32 * wave + 4 * (own >> 5);
          if (u < count) {
            const long long tok = reverse ? c0 + count - 1 - u : c0 + u;
            const T* const xr = B::x_in_lds ? reinterpret_cast<const T*>(L16 + B::off_s + u * B::pitch_x) + n4 : head_base<T>(p.x, b, h) + tok * p.x.st + n4;
            float sum = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (B::x_in_lds || n4 + 8 * q < cols) {
                T xv[4];
                __builtin_memcpy(xv, __builtin_assume_aligned(xr + 8 * q, 4 * sizeof(T)), sizeof(xv));
#pragma unroll
                for (int k = 0; k < 4; ++k) sum = __builtin_fmaf(to_f32(xv[k]), o[x][4 * q + k], sum);
              }
            const int place = ((int)tok & (p.stretch - 1)) + 1;
            dg += (double)sum * (double)(!reverse ? place : c0 + count == len ? u : -place);
          }
        }
      }
      if constexpr (!B::own_scores || LAGS) {
        __syncthreads();  // a, or x, is done with
        put_scores();
      }
      __syncthreads();
    }
    {
      const float gamma = count == C ? gamma_full.next() : gamma_part;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int r = 0; r < 16; ++r) m[rb][r] *= gamma;
      if constexpr (LAGS)
        if (!reverse && p.m_sink && c0 + count == len) {  // dS_T as a sink of all blocks but this, the last
          const int row0 = (int)opaque(8u * half);
          float sum = 0.0f;
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int row = 32 * rb + 16 * (r >> 3) + row0 + (r & 7);
              if (row < rows && ncol < cols) sum = __builtin_fmaf(m[rb][r], p.m_sink[m0 + (size_t)(row * p.m_r + ncol * p.m_n)], sum);
            }
          dg += (double)sum * (double)(((int)(len - 1) & (p.stretch - 1)) + 1);
        }
    }
    if constexpr (OUT)
      if (bad_c) take_out();
    // over the tokens: out^T += c^T scores^T, M += b^T (decayed c)
#pragma unroll
    for (int kk = 0; kk < C / 16; ++kk) {
      if (kk % STEPS == 0) __builtin_amdgcn_sched_barrier(0);
      uint4 fc[NP];
#pragma unroll
      for (int q = 0; q < NP; ++q) fc[q] = read_transposed(L16 + B::off_c + q * B::plane_c + 16 * kk * B::pitch_c + 32 * wave + tr_c, B::pitch_c);
      if constexpr (OUT) {
        uint4 fp[JP][TI];
#pragma unroll
        for (int q = 0; q < JP; ++q)
#pragma unroll
          for (int x = kk / 2; x < TI; ++x)
            fp[q][x] = *reinterpret_cast<const uint4*>(L16 + B::off_s + q * B::plane_s + (32 * x + l32) * B::pitch_s + 16 * kk + 8 * half);
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
          for (int z = 0; z < JP; ++z)
            if (q + z < JP)
#pragma unroll
              for (int x = kk / 2; x < TI; ++x) o[x] = mfma(fc[q], fp[z][x], o[x]);
      }
      float cv[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) cv[k] = 0.0f;
#pragma unroll
      for (int q = NP - 1; q >= 0; --q) {
        const unsigned d[4] = {fc[q].x, fc[q].y, fc[q].z, fc[q].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          cv[2 * k] += __uint_as_float(d[k] << 16);
          cv[2 * k + 1] += __uint_as_float(d[k] & 0xffff0000u);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) cv[k] *= upd_tab[C - count + 16 * kk + 8 * half + k];
      uint4 fu[3];
      split8<3>(cv, fu);
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        uint4 fbt[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          fbt[rb] = read_transposed(L16 + B::off_b + q * B::plane + 16 * kk * B::pitch + 32 * rb + tr_b, B::pitch);
#pragma unroll
        for (int z = 0; z < 3; ++z)
          if (q + z < 3)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) m[rb] = mfma(fbt[rb], fu[z], m[rb]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (OUT)
      if (bad_c) poison(o);
    if constexpr (LAGS)
      if (at_border && reverse) {
        float sum = 0.0f;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int r = 0; r < 16; ++r) sum = __builtin_fmaf(held[(rb * 16 + r) * B::threads], m[rb][r], sum);
        dg += (double)sum * (double)p.scale * (double)p.stretch;
      }
    if constexpr (OUT) {
      // out: lane: token 32 x + l32, register r: column n4 + 8 (r / 4) + r % 4
      const int own = lane_again(), l32 = own & 31, half = own >> 5, n4 = 32 * wave + 4 * half;
#pragma unroll
      for (int x = 0; x < TI; ++x) {
        const int u = 32 * x + l32;
        const bool live = u < count;
        const long long tok = reverse ? c0 + count - 1 - u : c0 + u;
        const size_t row = (((size_t)b * p.tokens + tok) * p.heads + h) * cols;
        if (sizeof(T) == 4 || p.out_f32) {
          float* dst = static_cast<float*>(p.out) + row + n4;
          if (live)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if (whole_o) {
                if (n4 + 8 * q < cols) *reinterpret_cast<float4*>(dst + 8 * q) = make_float4(o[x][4 * q], o[x][4 * q + 1], o[x][4 * q + 2], o[x][4 * q + 3]);
              } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  if (n4 + 8 * q + k < cols) dst[8 * q + k] = o[x][4 * q + k];
              }
            }
        } else if constexpr (sizeof(T) == 2) {
          unsigned d[8];
#pragma unroll
          for (int k = 0; k < 8; ++k)
            d[k] = __builtin_bit_cast(u16, from_f32<T>(o[x][2 * k])) | (unsigned)__builtin_bit_cast(u16, from_f32<T>(o[x][2 * k + 1])) << 16;
          if (whole_o) {
            // the halves exchange so that each has 8 consecutive columns: 16 (q / 2) + 8 half
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
              const auto s0 = __builtin_amdgcn_permlane32_swap(d[2 * q], d[2 * q + 2], false, false);
              const auto s1 = __builtin_amdgcn_permlane32_swap(d[2 * q + 1], d[2 * q + 3], false, false);
              const int n = 32 * wave + 8 * q + 8 * half;
              if (live && n < cols) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row + n) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
            }
          } else if (live) {
            u16* dst = static_cast<u16*>(p.out) + row + n4;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int n = 8 * (k / 2) + 2 * (k % 2);
              if (n4 + n < cols) dst[n] = (u16)d[k];
              if (n4 + n + 1 < cols) dst[n + 1] = (u16)(d[k] >> 16);
            }
          }
        }
      }
    }
  };

  Set set;
  if (total > 0) fetch(0, set);
  for (int i = 0; i < total; ++i) compute(i, set);

  // padding: zeros
  if (OUT)
    for (long long tok = max(len, seg_lo) + t / 32; tok < seg_end; tok += B::threads / 32)
      for (int n = t % 32; n < cols; n += 32) {
        const size_t at = (((size_t)b * p.tokens + tok) * p.heads + h) * cols + n;
        if (p.out_f32)
          static_cast<float*>(p.out)[at] = 0.0f;
        else
          static_cast<T*>(p.out)[at] = from_f32<T>(0.0f);
      }
  const bool last = seg == (reverse ? 0 : p.segments - 1);
  const int row0 = (int)opaque(8u * half);
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 32 * rb + 16 * (r >> 3) + row0 + (r & 7);
      if (row >= rows || ncol >= cols) continue;
      const size_t at = m0 + (size_t)(row * p.m_r + ncol * p.m_n);
      if (!OUT)
        p.seg_state[seg * seg_size + at] = m[rb][r];
      else if (last && p.m_out)
        p.m_out[at] = m[rb][r] * p.m_out_scale;
    }
  if constexpr (LAGS) {
    double* sum = reinterpret_cast<double*>(lds);
    __syncthreads();
    sum[t] = dg;
    __syncthreads();
    if (t == 0) {
      double all = 0.0;
      for (int k = 0; k < B::threads; ++k) all += sum[k];
      p.dg_part[(bh * p.segments + seg) * 2 + (reverse ? 1 : 0)] = all;
    }
  }
}

template <typename T, int RP, int NW, int MODE>
static hipError_t blocks_launch(const AttnPass& p) {
  const int osize = p.out_f32 || sizeof(T) == 4 ? 4 : 2;
  const bool wo = p.cols % (16 / osize) == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  const int first = MODE == kSums && p.reverse ? 1 : 0, segs = MODE == kSums ? p.segments - 1 : p.segments;
  return for_batches(p, (long long)p.heads * segs, 64 * NW, [&](const AttnPass& q, dim3 grid) {
    hipLaunchKernelGGL((attn_blocks_kernel<T, RP, NW, MODE>), grid, dim3(64 * NW), 0, q.stream, q, first, segs, wo);
  });
}

template <typename T, int MODE>
static hipError_t blocks_dims(const AttnPass& p) {
  if (p.rows <= 64) return p.cols <= 64 ? blocks_launch<T, 64, 2, MODE>(p) : blocks_launch<T, 64, 4, MODE>(p);
  return p.cols <= 64 ? blocks_launch<T, 128, 2, MODE>(p) : blocks_launch<T, 128, 4, MODE>(p);
}

template <typename T>
static hipError_t blocks_modes(const AttnPass& p) {
  if (!p.out) return blocks_dims<T, kSums>(p);
  return p.dg_part ? blocks_dims<T, kLags>(p) : blocks_dims<T, kPass>(p);
}

}  // namespace tfa
