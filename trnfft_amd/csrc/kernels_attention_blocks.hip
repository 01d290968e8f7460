// Linear attention with decays in blocks of C tokens on the bf16 matrix cores: one pass (model_ops.h, AttnPass)
//
//   out_i = scale ( sum_{j <= i} gamma^(i-j) (a_i . b_j) c_j  +  gamma^(i+e) a_i M ),
//   M    <- gamma^L M + sum_j gamma^(L-e-j) b_j c_j^T             i, j < L: places in the block, in the pass's order
//
// with e = 1 forward and 0 in a reversed pass (a state reaches its first token undecayed there).  The tangent pass carries
// M' = dM/dg as well: M' <- gamma^L (M' + L M) + sum_j (L-1-j) gamma^(L-1-j) b_j c_j^T, and dg collects x_i against
// scale ( sum_j (i-j) gamma^(i-j) (a_i . b_j) c_j + gamma^(i+1) a_i (M' + (i+1) M) ).
//
// A workgroup carries one head's state for 32 columns a wave, all R rows of them in registers (32 x 32 accumulators of
// v_mfma_f32_32x32x16_bf16), through its tokens.  The accumulator layout (lane: column, register: row) is also the
// layout of a matrix operand (lane: column or row, register: contraction) up to an exchange of index bits 2 and 3, so with the
// rows that feed the product taken in that order (pi below) states and scores go from accumulators to operands
// without leaving the registers.  Each wave computes all scores of the block itself: 24 more MFMAs for 128 rows, and no
// barrier and no LDS between them and their use.  Outputs are computed transposed (lane: token), so that decays by token are
// one factor a lane and stores are 16 bytes.
//
// Operands in LDS: a and b by token (contraction over features), b and c by feature (contraction over tokens); the next
// block is on its way in registers while one is computed.
//
// Precision: operands are exact sums of bf16 pieces (bf16: 1, fp16: 2, fp32: 3).  Scores, states and decayed c's are split into
// pieces to nearest as they enter a product: two for 16-bit outputs (2^-17, nothing beside their rounding), three for fp32
// outputs and for what enters states.  Products of pieces i, j are taken where i + j is within the piece count, into fp32.
#include <algorithm>

#include "attention_device.h"

namespace tfa {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16;

__device__ __forceinline__ floatx16 mfma(uint4 a, uint4 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
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

// index bits 2 and 3 exchanged: the row that accumulator place m stands for
__device__ __forceinline__ int pi(int m) { return (m & ~12) | ((m & 4) << 1) | ((m & 8) >> 1); }

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

// Features f, f + 1 of one row, as raw bits: one dword (16 bits) or two (fp32)
template <typename T>
struct RawPair {
  unsigned w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ RawPair<T> raw_pair(const T* row, unsigned at, int f, int features, bool whole) {
  RawPair<T> r;
  if (whole) {
    if constexpr (sizeof(T) == 2) {
      r.w[0] = f < features ? *reinterpret_cast<const unsigned*>(row + at) : 0u;
    } else {
      const uint2 v = f < features ? *reinterpret_cast<const uint2*>(row + at) : make_uint2(0, 0);
      r.w[0] = v.x;
      r.w[1] = v.y;
    }
  } else {
    const T x = f < features ? row[at] : T(0.0f), y = f + 1 < features ? row[at + 1] : T(0.0f);
    if constexpr (sizeof(T) == 2) {
      r.w[0] = __builtin_bit_cast(u16, x) | (unsigned)__builtin_bit_cast(u16, y) << 16;
    } else {
      r.w[0] = __builtin_bit_cast(unsigned, x);
      r.w[1] = __builtin_bit_cast(unsigned, y);
    }
  }
  return r;
}

// pieces of a raw pair: packed (f, f + 1)
template <typename T>
__device__ __forceinline__ void pair_pieces(const RawPair<T>& r, unsigned (&p)[Kind<T>::pieces]) {
  if constexpr (sizeof(T) == 4) {
    split_pair<3>(__uint_as_float(r.w[0]), __uint_as_float(r.w[1]), p);
  } else if constexpr (Kind<T>::pieces == 2) {
    split_pair<2>((float)__builtin_bit_cast(_Float16, (u16)r.w[0]), (float)__builtin_bit_cast(_Float16, (u16)(r.w[0] >> 16)), p);
  } else {
    p[0] = r.w[0];
  }
}

template <typename T, int RP, int NW, bool TAN>
struct Blocks {
  static constexpr int NP = Kind<T>::pieces, C = Kind<T>::block, J = Kind<T>::out_pieces;
  static constexpr int CP = 32 * NW, threads = 64 * NW, TI = C / 32, RB = RP / 32;
  static constexpr int pitch_row = RP + 8, pitch_tok = C + 8;  // 16-bit units: rows start 4 banks apart, modulo 64
  static constexpr int row_plane = C * pitch_row, b_plane = RP * pitch_tok, c_plane = CP * pitch_tok;
  static constexpr int off_a = 0, off_b = off_a + NP * row_plane, off_bt = off_b + NP * row_plane;
  static constexpr int off_ct = off_bt + NP * b_plane, off_end = off_ct + NP * c_plane;
  // tables: gamma^(i - j) by i - j + C (zero before C), gamma^(L - e - j) by j
  static constexpr int bytes = off_end * 2 + (2 * C + C) * 4;

  // an operand's pair columns: lanes over pairs, token groups of 8
  template <int W>
  struct Pairs {
    static constexpr int lanes = W / 2, groups_at_once = threads / lanes;
    static constexpr int passes = (C / 8 + groups_at_once - 1) / groups_at_once;
    static constexpr bool partial = C / 8 < groups_at_once;  // some threads have no group
    RawPair<T> r[passes][8];
  };
};

// The places of a block's rows in memory: `base` the lowest token's row, place u at pos(u) rows above it
struct Rows {
  unsigned stride;  // in elements
  int count;        // live rows
  bool reverse;
  __device__ __forceinline__ unsigned at(int u) const {
    const int v = min(u, count - 1);
    return (unsigned)(reverse ? count - 1 - v : v) * stride;
  }
};

template <typename T, int RP, int NW, bool TAN>
__global__ __launch_bounds__(64 * NW, TAN ? 1 : 2) void attn_blocks_kernel(AttnPass p, int slices, int first_seg, int segs,
                                                                         bool whole_a, bool whole_b, bool whole_c,
                                                                         bool whole_o, bool whole_x) {
  using B = Blocks<T, RP, NW, TAN>;
  constexpr int NP = B::NP, C = B::C, J = B::J, TI = B::TI, RB = B::RB, V = 16 / sizeof(T);
  __shared__ __align__(16) unsigned char lds[B::bytes];
  u16* const L16 = reinterpret_cast<u16*>(lds);
  float* const pow_tab = reinterpret_cast<float*>(lds + B::off_end * 2);
  float* const upd_tab = pow_tab + 2 * C;

  const int t = threadIdx.x, lane = t & 63, half = lane >> 5, l32 = lane & 31, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  unsigned block = blockIdx.x;
  const int slice = (int)(block % slices);
  block /= slices;
  const int seg = first_seg + (int)(block % segs);
  const long long bh = block / segs, b = bh / p.heads;
  const int h = (int)(bh % p.heads);
  const int n0 = slice * B::CP;  // first column of the workgroup
  const long long len = live_tokens(p, b);
  const long long seg_lo = seg * p.seg_tokens, seg_end = min(seg_lo + p.seg_tokens, p.tokens);
  const long long lo = min(seg_lo, len), hi = min(seg_end, len);
  const T* A = p.out ? head_base<T>(p.a, b, h) : nullptr;
  const T* Bp = head_base<T>(p.b, b, h);
  const T* Cp = head_base<T>(p.c, b, h) + n0;
  const T* X = TAN ? head_base<T>(p.x, b, h) + n0 : nullptr;
  const int cols = min(p.cols - n0, B::CP);
  const double g = (double)log_decay_of(p.log_decay, h);
  const int e = p.reverse ? 0 : 1;
  const bool sums_only = p.out == nullptr;

  for (int i = t; i < 2 * C; i += B::threads) pow_tab[i] = i < C ? 0.0f : (float)exp(g * (double)(i - C));

  // the state: column n0 + 32 wave + l32, register r of block rb: row 32 rb + 16 (r / 8) + 8 half + r % 8
  floatx16 m[RB], rm[RB];
  const int ncol = 32 * wave + l32;
  const size_t m0 = (size_t)bh * p.rows * p.cols;
  const size_t seg_size = (size_t)p.batch * p.heads * p.rows * p.cols;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 32 * rb + 16 * (r >> 3) + 8 * half + (r & 7);
      float x = 0.0f;
      if (!sums_only && row < p.rows && ncol < cols) {
        const size_t at = m0 + (size_t)(row * p.m_r + (n0 + ncol) * p.m_n);
        if (p.segments > 1)
          x = p.seg_state[seg * seg_size + at];
        else if (p.m_in)
          x = p.m_in[at] * p.m_in_scale;
      }
      m[rb][r] = x;
      rm[rb][r] = 0.0f;
    }
  double dg = 0.0;

  using PB = typename B::template Pairs<RP>;
  using PC = typename B::template Pairs<B::CP>;
  constexpr int a_lanes = RP / V, a_rows = B::threads / a_lanes, a_passes = C / a_rows;
  static_assert(C % a_rows == 0, "whole passes");
  uint4 ra[a_passes];
  PB rb_raw;
  PC rc_raw;
  const int a_f = (t % a_lanes) * V, a_u = t / a_lanes;
  const int b_f = (t % PB::lanes) * 2, b_g = t / PB::lanes;
  const int c_f = (t % PC::lanes) * 2, c_g = t / PC::lanes;

  // blocks in the pass's order; their borders are the same tokens in both directions
  const int total = (int)((hi - lo + C - 1) / C);
  auto block_lo = [&](int i) { return lo + (long long)(p.reverse ? total - 1 - i : i) * C; };

  auto fetch = [&](int i) {
    const long long c0 = block_lo(i);
    const int count = (int)min((long long)C, hi - c0);
    const bool full = count == C;
    if (!sums_only) {
      const T* base = A + c0 * p.a.st;
      const Rows rows{(unsigned)p.a.st, count, p.reverse};
#pragma unroll
      for (int q = 0; q < a_passes; ++q) {
        const int u = a_u + q * a_rows;
        const unsigned at = rows.at(u) + a_f;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (whole_a) {
          if (a_f < p.rows) v = *reinterpret_cast<const uint4*>(base + at);
        } else {
          T x[V];
#pragma unroll
          for (int k = 0; k < V; ++k) x[k] = a_f + k < p.rows ? base[at + k] : T(0.0f);
          __builtin_memcpy(&v, x, 16);
        }
        if (!full && u >= count) v = make_uint4(0, 0, 0, 0);
        ra[q] = v;
      }
    }
    {
      const T* base = Bp + c0 * p.b.st;
      const Rows rows{(unsigned)p.b.st, count, p.reverse};
#pragma unroll
      for (int q = 0; q < PB::passes; ++q) {
        const int gidx = b_g + q * PB::groups_at_once;
        if (PB::partial && gidx >= C / 8) break;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int u = gidx * 8 + k;
          RawPair<T> v = raw_pair(base, rows.at(u) + b_f, b_f, p.rows, whole_b);
          if (!full && u >= count)
            for (unsigned& w : v.w) w = 0;
          rb_raw.r[q][k] = v;
        }
      }
    }
    {
      const T* base = Cp + c0 * p.c.st;
      const Rows rows{(unsigned)p.c.st, count, p.reverse};
#pragma unroll
      for (int q = 0; q < PC::passes; ++q) {
        const int gidx = c_g + q * PC::groups_at_once;
        if (PC::partial && gidx >= C / 8) break;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int u = gidx * 8 + k;
          RawPair<T> v = raw_pair(base, rows.at(u) + c_f, c_f, cols, whole_c);
          if (!full && u >= count)
            for (unsigned& w : v.w) w = 0;
          rc_raw.r[q][k] = v;
        }
      }
    }
  };

  // eight tokens of a pair, transposed: feature f's row gets 8 tokens, feature f + 1's too
  auto put_transposed = [&](const RawPair<T>(&r)[8], u16* plane0, int plane, int f, int tok, u16* rows0, int row_plane) {
    unsigned pc[8][NP];
#pragma unroll
    for (int k = 0; k < 8; ++k) pair_pieces<T>(r[k], pc[k]);
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      unsigned lo4[4], hi4[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        lo4[k] = (pc[2 * k][q] & 0xffffu) | (pc[2 * k + 1][q] << 16);
        hi4[k] = (pc[2 * k][q] >> 16) | (pc[2 * k + 1][q] & 0xffff0000u);
      }
      u16* dst = plane0 + q * plane + f * B::pitch_tok + tok;
      *reinterpret_cast<uint4*>(dst) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
      *reinterpret_cast<uint4*>(dst + B::pitch_tok) = make_uint4(hi4[0], hi4[1], hi4[2], hi4[3]);
      if (rows0)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          *reinterpret_cast<unsigned*>(rows0 + q * row_plane + (tok + k) * B::pitch_row + f) = pc[k][q];
    }
  };

  auto stage = [&]() {
    if (!sums_only) {
#pragma unroll
      for (int q = 0; q < a_passes; ++q) {
        u16* dst = L16 + B::off_a + (a_u + q * a_rows) * B::pitch_row + a_f;
        if constexpr (NP == 1) {
          *reinterpret_cast<uint4*>(dst) = ra[q];
        } else {
          const unsigned w[4] = {ra[q].x, ra[q].y, ra[q].z, ra[q].w};
#pragma unroll
          for (int k = 0; k < V / 2; ++k) {
            RawPair<T> r;
            if constexpr (sizeof(T) == 4) {
              r.w[0] = w[2 * k];
              r.w[1] = w[2 * k + 1];
            } else {
              r.w[0] = w[k];
            }
            unsigned pc[NP];
            pair_pieces<T>(r, pc);
#pragma unroll
            for (int z = 0; z < NP; ++z) *reinterpret_cast<unsigned*>(dst + z * B::row_plane + 2 * k) = pc[z];
          }
        }
      }
    }
#pragma unroll
    for (int q = 0; q < PB::passes; ++q) {
      const int gidx = b_g + q * PB::groups_at_once;
      if (PB::partial && gidx >= C / 8) break;
      put_transposed(rb_raw.r[q], L16 + B::off_bt, B::b_plane, b_f, gidx * 8, sums_only ? nullptr : L16 + B::off_b, B::row_plane);
    }
#pragma unroll
    for (int q = 0; q < PC::passes; ++q) {
      const int gidx = c_g + q * PC::groups_at_once;
      if (PC::partial && gidx >= C / 8) break;
      put_transposed(rc_raw.r[q], L16 + B::off_ct, B::c_plane, c_f, gidx * 8, nullptr, 0);
    }
  };

  const Decay gamma_full(exp(g * (double)C));
  int table_for = 0;
  if (total > 0) fetch(0);
  for (int i = 0; i < total; ++i) {
    const long long c0 = block_lo(i);
    const int count = (int)min((long long)C, hi - c0);
    __syncthreads();  // the block before is done with LDS
    if (table_for != count) {
      table_for = count;
      for (int j = t; j < C; j += B::threads) upd_tab[j] = j < count ? (float)exp(g * (double)(count - e - j)) : 0.0f;
    }
    stage();
    __syncthreads();
    if (i + 1 < total) fetch(i + 1);

    floatx16 o[TI], s[TI][TI], ol[TAN ? TI : 1];
    if (!sums_only) {
#pragma unroll
      for (int x = 0; x < TI; ++x) {
        o[x] = floatx16{};
        if (TAN) ol[x] = floatx16{};
#pragma unroll
        for (int y = 0; y < TI; ++y) s[x][y] = floatx16{};
      }
      // over the features: scores^T = b a^T (rows in the order pi) and out^T = M^T a^T
#pragma unroll
      for (int ks = 0; ks < RP / 16; ++ks) {
        uint4 fa[NP][TI], fb[NP][TI], fm[J];
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
          for (int x = 0; x < TI; ++x) {
            fa[q][x] = *reinterpret_cast<const uint4*>(L16 + B::off_a + q * B::row_plane + (32 * x + l32) * B::pitch_row + 16 * ks + 8 * half);
            fb[q][x] = *reinterpret_cast<const uint4*>(L16 + B::off_b + q * B::row_plane + (32 * x + pi(l32)) * B::pitch_row + 16 * ks + 8 * half);
          }
        float mv[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) mv[k] = m[ks / 2][8 * (ks & 1) + k];
        split8<J>(mv, fm);
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
          for (int z = 0; z < J; ++z)
            if (q + z < (J > 2 ? 3 : 2))
#pragma unroll
              for (int x = 0; x < TI; ++x) o[x] = mfma(fm[z], fa[q][x], o[x]);
        if constexpr (TAN) {
          uint4 fr[3];
#pragma unroll
          for (int k = 0; k < 8; ++k) mv[k] = rm[ks / 2][8 * (ks & 1) + k];
          split8<3>(mv, fr);
#pragma unroll
          for (int q = 0; q < NP; ++q)
#pragma unroll
            for (int z = 0; z < 3; ++z)
              if (q + z < 3)
#pragma unroll
                for (int x = 0; x < TI; ++x) ol[x] = mfma(fr[z], fa[q][x], ol[x]);
        }
#pragma unroll
        for (int q = 0; q < NP; ++q)
#pragma unroll
          for (int z = 0; z < NP; ++z)
            if (q + z < 3)
#pragma unroll
              for (int x = 0; x < TI; ++x)
#pragma unroll
                for (int y = 0; y <= x; ++y) s[x][y] = mfma(fb[q][y], fa[z][x], s[x][y]);
      }
      // a state reaches token i with gamma^(i + e)
#pragma unroll
      for (int x = 0; x < TI; ++x) {
        const float w = e ? pow_tab[C + 32 * x + l32] * pow_tab[C + 1] : pow_tab[C + 32 * x + l32];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          o[x][r] *= w;
          if (TAN) ol[x][r] = __builtin_fmaf(ol[x][r], w, (float)(32 * x + l32 + 1) * o[x][r]);
        }
      }
    }
    // the state takes gamma^L M, its tangent gamma^L (M' + L M)
    {
      const Decay gamma = count == C ? gamma_full : Decay(exp(g * (double)count));
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          if (TAN) rm[rb][r] = gamma.times(__builtin_fmaf((float)count, m[rb][r], rm[rb][r]));
          m[rb][r] = gamma.times(m[rb][r]);
        }
    }
    // over the tokens: out^T += c^T scores^T, M += b^T (decayed c)
#pragma unroll
    for (int kk = 0; kk < C / 16; ++kk) {
      uint4 fc[NP];
#pragma unroll
      for (int q = 0; q < NP; ++q)
        fc[q] = *reinterpret_cast<const uint4*>(L16 + B::off_ct + q * B::c_plane + ncol * B::pitch_tok + 16 * kk + 8 * half);
      if (!sums_only) {
        const int y = kk / 2, r0 = 8 * (kk & 1);
#pragma unroll
        for (int x = y; x < TI; ++x) {
          float w[8], wl[8];
          // token i = 32 x + l32, j = 16 kk + 8 half + k
          const int lag = 32 * x + l32 - 16 * kk - 8 * half;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            w[k] = s[x][y][r0 + k] * pow_tab[C + lag - k];
            wl[k] = w[k] * (float)(lag - k);
          }
          uint4 fp[J];
          split8<J>(w, fp);
#pragma unroll
          for (int q = 0; q < NP; ++q)
#pragma unroll
            for (int z = 0; z < J; ++z)
              if (q + z < (J > 2 ? 3 : 2)) o[x] = mfma(fc[q], fp[z], o[x]);
          if constexpr (TAN) {
            uint4 fl[3];
            split8<3>(wl, fl);
#pragma unroll
            for (int q = 0; q < NP; ++q)
#pragma unroll
              for (int z = 0; z < 3; ++z)
                if (q + z < 3) ol[x] = mfma(fc[q], fl[z], ol[x]);
          }
        }
      }
      float cv[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) cv[k] = 0.0f;
#pragma unroll
      for (int q = NP - 1; q >= 0; --q) {
        const unsigned w[4] = {fc[q].x, fc[q].y, fc[q].z, fc[q].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          cv[2 * k] += __uint_as_float(w[k] << 16);
          cv[2 * k + 1] += __uint_as_float(w[k] & 0xffff0000u);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) cv[k] *= upd_tab[16 * kk + 8 * half + k];
      uint4 fu[3], ft[TAN ? 3 : 1];
      split8<3>(cv, fu);
      if constexpr (TAN) {
        float tv[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) tv[k] = cv[k] * (float)(count - 1 - 16 * kk - 8 * half - k);
        split8<3>(tv, ft);
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          const uint4 fbt = *reinterpret_cast<const uint4*>(L16 + B::off_bt + q * B::b_plane + (32 * rb + pi(l32)) * B::pitch_tok + 16 * kk + 8 * half);
#pragma unroll
          for (int z = 0; z < 3; ++z)
            if (q + z < 3) {
              m[rb] = mfma(fbt, fu[z], m[rb]);
              if constexpr (TAN) rm[rb] = mfma(fbt, ft[z], rm[rb]);
            }
        }
    }
    if (sums_only) continue;
    // out: lane: token 32 x + l32, register r: column 32 wave + 8 (r / 4) + 4 half + r % 4
#pragma unroll
    for (int x = 0; x < TI; ++x) {
      const int u = 32 * x + l32;
      const bool live = u < count;
      const long long tok = p.reverse ? c0 + count - 1 - u : c0 + u;
      const int nw = 32 * wave;
      if constexpr (TAN) {
        float sum = 0.0f;
        if (live) {
          const T* xr = X + tok * p.x.st + nw + 4 * half;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            T xv[4];
            if (whole_x) {
              if (nw + 8 * q + 4 * half < cols)
                __builtin_memcpy(xv, __builtin_assume_aligned(xr + 8 * q, 4 * sizeof(T)), sizeof(xv));
              else
                for (T& z : xv) z = T(0.0f);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k) xv[k] = nw + 8 * q + 4 * half + k < cols ? xr[8 * q + k] : T(0.0f);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) sum = __builtin_fmaf(to_f32(xv[k]), ol[x][4 * q + k], sum);
          }
        }
        dg += (double)sum * (double)p.scale;
      }
      float ov[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) ov[r] = o[x][r] * p.scale;
      const size_t row = ((size_t)b * p.tokens + tok) * p.heads + h;
      if (p.out_f32 || sizeof(T) == 4) {
        float* dst = static_cast<float*>(p.out) + row * p.cols + n0 + nw + 4 * half;
        if (live)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int n = nw + 8 * q + 4 * half;
            if (whole_o) {
              if (n < cols) *reinterpret_cast<float4*>(dst + 8 * q) = make_float4(ov[4 * q], ov[4 * q + 1], ov[4 * q + 2], ov[4 * q + 3]);
            } else {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (n + k < cols) dst[8 * q + k] = ov[4 * q + k];
            }
          }
      } else if constexpr (sizeof(T) == 2) {
        unsigned d[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          d[k] = __builtin_bit_cast(u16, from_f32<T>(ov[2 * k])) | (unsigned)__builtin_bit_cast(u16, from_f32<T>(ov[2 * k + 1])) << 16;
        if (whole_o) {
          // the halves exchange so that each has 8 consecutive columns: 16 (q / 2) + 8 half
#pragma unroll
          for (int q = 0; q < 4; q += 2) {
            const auto s0 = __builtin_amdgcn_permlane32_swap(d[2 * q], d[2 * q + 2], false, false);
            const auto s1 = __builtin_amdgcn_permlane32_swap(d[2 * q + 1], d[2 * q + 3], false, false);
            const int n = nw + 8 * q + 8 * half;
            if (live && n < cols)
              *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row * p.cols + n0 + n) = make_uint4(s0[0], s1[0], s0[1], s1[1]);
          }
        } else if (live) {
          u16* dst = static_cast<u16*>(p.out) + row * p.cols + n0 + nw + 4 * half;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int n = 8 * (k / 2) + 2 * (k % 2);
            if (nw + 4 * half + n < cols) dst[n] = (u16)d[k];
            if (nw + 4 * half + n + 1 < cols) dst[n + 1] = (u16)(d[k] >> 16);
          }
        }
      }
    }
  }

  // padding: zeros
  if (!sums_only)
    for (long long tok = max(len, seg_lo) + t / 32; tok < seg_end; tok += B::threads / 32)
      for (int n = t % 32; n < cols; n += 32) {
        const size_t at = (((size_t)b * p.tokens + tok) * p.heads + h) * p.cols + n0 + n;
        if (p.out_f32)
          static_cast<float*>(p.out)[at] = 0.0f;
        else
          static_cast<T*>(p.out)[at] = from_f32<T>(0.0f);
      }
  const bool last = seg == (p.reverse ? 0 : p.segments - 1);
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 32 * rb + 16 * (r >> 3) + 8 * half + (r & 7);
      if (row >= p.rows || ncol >= cols) continue;
      const size_t at = m0 + (size_t)(row * p.m_r + (n0 + ncol) * p.m_n);
      if (sums_only)
        p.seg_state[seg * seg_size + at] = m[rb][r];
      else if (last && p.m_out)
        p.m_out[at] = m[rb][r] * p.m_out_scale;
      if (TAN) {
        const float sink = p.segments > 1 ? p.seg_sink[seg * seg_size + at] * p.scale : p.m_sink ? p.m_sink[at] : 0.0f;
        dg += (double)rm[rb][r] * (double)sink;
      }
    }
  if constexpr (TAN) {
    double* sum = reinterpret_cast<double*>(lds);
    __syncthreads();
    sum[t] = dg;
    __syncthreads();
    if (t == 0) {
      double all = 0.0;
      for (int k = 0; k < B::threads; ++k) all += sum[k];
      p.dg_part[(bh * p.segments + seg) * slices + slice] = all;
    }
  }
}

static int block_slices(const AttnPass& p) { return p.cols <= 64 ? 1 : (p.cols + 127) / 128; }

int attn_blocks_dg_parts(const AttnPass& p) { return block_slices(p) * std::max(1, p.segments); }

static bool aligned(const HeadsView& v, int dtype, int bytes) {
  const int size = dtype == 0 ? 4 : 2, n = bytes / size;
  return reinterpret_cast<uintptr_t>(v.p) % bytes == 0 && v.sb % n == 0 && v.st % n == 0 && v.sh % n == 0;
}

template <typename T, int RP, int NW, bool TAN>
static hipError_t blocks_launch(const AttnPass& p) {
  const int size = (int)sizeof(T), slices = block_slices(p);
  const bool wa = p.out && p.rows % (16 / size) == 0 && aligned(p.a, p.dtype, 16);
  const bool wb = p.rows % 2 == 0 && aligned(p.b, p.dtype, 2 * size), wc = p.cols % 2 == 0 && aligned(p.c, p.dtype, 2 * size);
  const int osize = p.out_f32 ? 4 : size;
  const bool wo = p.cols % (osize == 4 ? 4 : 8) == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
  const bool wx = TAN && p.cols % 4 == 0 && aligned(p.x, p.dtype, 4 * size);
  const int first = !p.out && p.reverse ? 1 : 0, segs = p.out ? p.segments : p.segments - 1;
  const long long grid = p.batch * p.heads * slices * segs;
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL((attn_blocks_kernel<T, RP, NW, TAN>), dim3((unsigned)grid), dim3(64 * NW), 0, p.stream, p, slices, first, segs,
                     wa, wb, wc, wo, wx);
  return hipGetLastError();
}

template <typename T, bool TAN>
static hipError_t blocks_dims(const AttnPass& p) {
  if (p.rows <= 64) return p.cols <= 64 ? blocks_launch<T, 64, 2, TAN>(p) : blocks_launch<T, 64, 4, TAN>(p);
  return p.cols <= 64 ? blocks_launch<T, 128, 2, TAN>(p) : blocks_launch<T, 128, 4, TAN>(p);
}

hipError_t launch_attn_blocks(const AttnPass& p) {
  if (p.dtype == 0) return p.dg_part ? blocks_dims<float, true>(p) : blocks_dims<float, false>(p);
  if (p.dtype == 1) return p.dg_part ? blocks_dims<__bf16, true>(p) : blocks_dims<__bf16, false>(p);
  return p.dg_part ? blocks_dims<_Float16, true>(p) : blocks_dims<_Float16, false>(p);
}

// seg_state[s] of each segment's own sum becomes the state it starts from; one thread an element
__global__ __launch_bounds__(256) void attn_join_kernel(AttnPass p) {
  const size_t size = (size_t)p.rows * p.cols, all = (size_t)p.batch * p.heads * size;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  const long long bh = (long long)(i / size), len = live_tokens(p, bh / p.heads);
  const double g = (double)log_decay_of(p.log_decay, (int)(bh % p.heads));
  const Decay whole(exp(g * (double)p.seg_tokens));
  float m = p.m_in ? p.m_in[i] * p.m_in_scale : 0.0f;
  for (int k = 0; k < p.segments; ++k) {
    const int s = p.reverse ? p.segments - 1 - k : k;
    float* at = p.seg_state + s * all + i;
    const bool end = k == p.segments - 1;
    const float own = end ? 0.0f : *at;
    *at = m;
    const long long tokens = min(max(len - s * p.seg_tokens, 0LL), p.seg_tokens);
    m = (tokens == p.seg_tokens ? whole : Decay(exp(g * (double)tokens))).times(m) + own;
  }
}

hipError_t launch_attn_join(const AttnPass& p) {
  const size_t all = (size_t)p.batch * p.heads * p.rows * p.cols, blocks = (all + 255) / 256;
  if (blocks > 0x7fffffff) return hipErrorInvalidValue;
  hipLaunchKernelGGL(attn_join_kernel, dim3((unsigned)blocks), dim3(256), 0, p.stream, p);
  return hipGetLastError();
}

}  // namespace tfa
