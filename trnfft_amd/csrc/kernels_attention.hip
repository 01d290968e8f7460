// Linear attention with a decay for each head.
//
//   S_t = gamma S_{t-1} + k_t v_t^T,   o_t = scale S_t^T q_t,   gamma = exp(log_decay[h])
//
// Forward and gradients are one form, out_t = scale sum_s gamma^|t-s| (a_t . b_s) c_s, over s <= t or, with time
// reversed, s >= t:
//          a   b   c   order     state M = sum gamma^(..) b c^T
//   o      q   k   v   forward   S            from S_0, ends as S_T
//   dq     do  v   k   forward   S^T          from S_0^T
//   dk     v   do  q   reversed  (dS)^T       from dS_T^T
//   dv     k   q   do  reversed  dS           from dS_T, ends as dS_0
// (forward, a state reaches token t with gamma^(t+1); reversed, dS_T reaches token s with gamma^(T-1-s): the decay
// comes after the token instead of before it).  Scores, states and sums are held in fp32 whatever the inputs' type; in blocks they enter
// the products of 16-bit outputs as 16 to 17 bits of theirs (attention_blocks.h).
//
// The log decay's gradient is the sum over all pairs of lag * flow.  Token by token it is carried by the state's derivative
// dM/dg: M' <- gamma (M' + M), with each token's contribution a M' . x (the dq pass, x = q), and M' . dS_T^T at the end; in
// blocks it comes from the query and key gradients themselves (attention_blocks.h).
#include "attention_device.h"

#include <algorithm>

namespace tfa {

// ------------------------------------------------------------------------------------------------
// Token by token, for heads of 129 to 256 features (and where there is no token: states and zeros only).  A workgroup carries 32
// columns of one head's state: thread (column, row group) holds RPT rows of its column in registers, 16 tokens are
// staged in LDS at a time, and the row groups' parts of the outputs are joined once per 16 tokens.  Bound by the fp32
// FMAs (3 a state element and token, 6 with the tangent) and, more, by their LDS operands: 8 x 1024 tokens of 8 bf16 heads of 256,
// 3.2 ms, 8 TFLOP/s.
// ------------------------------------------------------------------------------------------------

constexpr int kScanCols = 32, kScanGroups = 8, kScanTokens = 16;

template <typename T, int RPT, bool TANGENT>
__global__ __launch_bounds__(256) void attn_scan_kernel(AttnPass p, int slices) {
  constexpr int R = RPT * kScanGroups;
  __shared__ float sa[kScanTokens][R], sb[kScanTokens][R], sc[kScanTokens][kScanCols], sx[kScanTokens][kScanCols];
  __shared__ float part[kScanTokens][kScanGroups][kScanCols];
  const int t = threadIdx.x, col = t % kScanCols, rg = t / kScanCols;
  const int slice = blockIdx.x % slices;
  const long long bh = p.first * p.heads + blockIdx.x / slices, b = bh / p.heads;
  const int h = (int)(bh % p.heads), n = slice * kScanCols + col;
  const long long len = live_tokens(p, b);
  const T* A = head_base<T>(p.a, b, h);
  const T* B = head_base<T>(p.b, b, h);
  const T* C = head_base<T>(p.c, b, h);
  const T* X = TANGENT ? head_base<T>(p.x, b, h) : nullptr;
  const Decay gamma(exp((double)log_decay_of(p.log_decay, h)));
  const long long m0 = bh * p.rows * p.cols;

  float m[RPT], tm[RPT];
#pragma unroll
  for (int j = 0; j < RPT; ++j) {
    const int r = rg + kScanGroups * j;
    m[j] = p.m_in && r < p.rows && n < p.cols ? p.m_in[m0 + r * p.m_r + n * p.m_n] * p.m_in_scale : 0.0f;
    tm[j] = 0.0f;
  }
  double dg = 0.0;
  const long long o_t = (long long)p.heads * p.cols, o0 = b * p.tokens * o_t + (long long)h * p.cols;
  for (long long t0 = 0; t0 < len; t0 += kScanTokens) {
    const int count = (int)min((long long)kScanTokens, len - t0);
    for (int i = t; i < kScanTokens * R; i += 256) {
      const int k = i / R, r = i % R;
      const bool in = k < count && r < p.rows;
      const long long at = p.reverse ? len - 1 - t0 - k : t0 + k;
      sa[k][r] = in ? to_f32(A[at * p.a.st + r]) : 0.0f;
      sb[k][r] = in ? to_f32(B[at * p.b.st + r]) : 0.0f;
    }
    for (int i = t; i < kScanTokens * kScanCols; i += 256) {
      const int k = i / kScanCols, cn = slice * kScanCols + i % kScanCols;
      const bool in = k < count && cn < p.cols;
      const long long at = p.reverse ? len - 1 - t0 - k : t0 + k;
      sc[k][i % kScanCols] = in ? to_f32(C[at * p.c.st + cn]) : 0.0f;
      if (TANGENT) sx[k][i % kScanCols] = in ? to_f32(X[at * p.x.st + cn]) : 0.0f;
    }
    __syncthreads();
    float dgt = 0.0f;
    for (int k = 0; k < count; ++k) {
      const float c = sc[k][col];
      float acc = 0.0f, tacc = 0.0f;
#pragma unroll
      for (int j = 0; j < RPT; ++j) {
        const float a = sa[k][rg + kScanGroups * j], bb = sb[k][rg + kScanGroups * j];
        if (TANGENT) {
          tm[j] = gamma.times(tm[j] + m[j]);
          tacc = __builtin_fmaf(a, tm[j], tacc);
        }
        if (p.reverse) {
          m[j] = __builtin_fmaf(bb, c, m[j]);
          acc = __builtin_fmaf(a, m[j], acc);
          m[j] = gamma.times(m[j]);
        } else {
          m[j] = __builtin_fmaf(bb, c, gamma.times(m[j]));
          acc = __builtin_fmaf(a, m[j], acc);
        }
      }
      part[k][rg][col] = acc;
      if (TANGENT) dgt = __builtin_fmaf(tacc, sx[k][col], dgt);
    }
    if (TANGENT) dg += (double)dgt * (double)p.scale;
    __syncthreads();
    for (int k = rg; k < count; k += kScanGroups) {
      float s = 0.0f;
#pragma unroll
      for (int g = 0; g < kScanGroups; ++g) s += part[k][g][col];
      const long long at = p.reverse ? len - 1 - t0 - k : t0 + k;
      if (n < p.cols) {
        if (p.out_f32)
          static_cast<float*>(p.out)[o0 + at * o_t + n] = s * p.scale;
        else
          static_cast<T*>(p.out)[o0 + at * o_t + n] = from_f32<T>(s * p.scale);
      }
    }
  }
  // padding: nothing was read there, and its outputs are zeros
  for (long long at = len + rg; at < p.tokens; at += kScanGroups)
    if (n < p.cols) {
      if (p.out_f32)
        static_cast<float*>(p.out)[o0 + at * o_t + n] = 0.0f;
      else
        static_cast<T*>(p.out)[o0 + at * o_t + n] = from_f32<T>(0.0f);
    }
#pragma unroll
  for (int j = 0; j < RPT; ++j) {
    const int r = rg + kScanGroups * j;
    if (r < p.rows && n < p.cols) {
      if (p.m_out) p.m_out[m0 + r * p.m_r + n * p.m_n] = m[j] * p.m_out_scale;
      if (TANGENT && p.m_sink) dg += (double)tm[j] * (double)p.m_sink[m0 + r * p.m_r + n * p.m_n];
    }
  }
  if (TANGENT) {
    __shared__ double sum[256];
    sum[t] = dg;
    __syncthreads();
    for (int s = 128; s > 0; s /= 2) {
      if (t < s) sum[t] += sum[t + s];
      __syncthreads();
    }
    if (t == 0) p.dg_part[bh * slices + slice] = sum[0];
  }
}

int attn_scan_dg_parts(const AttnPass& p) { return (p.cols + kScanCols - 1) / kScanCols; }

template <typename T, int RPT>
static hipError_t scan_launch(const AttnPass& p) {
  const int slices = (p.cols + kScanCols - 1) / kScanCols;
  return for_batches(p, (long long)p.heads * slices, 256, [&](const AttnPass& q, dim3 grid) {
    if (q.dg_part)
      hipLaunchKernelGGL((attn_scan_kernel<T, RPT, true>), grid, dim3(256), 0, q.stream, q, slices);
    else
      hipLaunchKernelGGL((attn_scan_kernel<T, RPT, false>), grid, dim3(256), 0, q.stream, q, slices);
  });
}

template <typename T>
static hipError_t scan_rows(const AttnPass& p) {
  if (p.rows <= 8 * kScanGroups) return scan_launch<T, 8>(p);
  return p.rows <= 16 * kScanGroups ? scan_launch<T, 16>(p) : scan_launch<T, 32>(p);
}

hipError_t launch_attn_scan(const AttnPass& p) {
  if (p.dtype == 0) return scan_rows<float>(p);
  return p.dtype == 1 ? scan_rows<__bf16>(p) : scan_rows<_Float16>(p);
}

// ------------------------------------------------------------------------------------------------
// In blocks of tokens (attention_blocks.h): dispatch, and what surrounds the segments of a long sequence.
// ------------------------------------------------------------------------------------------------

hipError_t launch_attn_blocks_f32(const AttnPass& p);
hipError_t launch_attn_blocks_bf16(const AttnPass& p);
hipError_t launch_attn_blocks_f16(const AttnPass& p);

hipError_t launch_attn_blocks(const AttnPass& p) {
  if (p.dtype == 0) return launch_attn_blocks_f32(p);
  return p.dtype == 1 ? launch_attn_blocks_bf16(p) : launch_attn_blocks_f16(p);
}

int attn_blocks_dg_parts(const AttnPass& p) { return 2 * p.segments; }
size_t attn_border_bytes(int rows, int cols) { return sizeof(float) * (rows <= 64 ? 64 : 128) * (cols <= 64 ? 64 : 128); }

// seg_state[s] of each segment's own sum becomes the state it starts from; one thread an element, 8 segments' sums on their way at a
// time.  Bound by memory: 4 segments of 128 heads of 128 x 128, 17 us, 3.9 TB/s.
__global__ __launch_bounds__(256) void attn_join_kernel(AttnPass p) {
  const size_t size = (size_t)p.rows * p.cols, all = (size_t)p.batch * p.heads * size;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  const long long bh = (long long)(i / size), len = live_tokens(p, bh / p.heads);
  const double g = (double)log_decay_of(p.log_decay, (int)(bh % p.heads));
  const Decay whole(exp(g * (double)p.seg_tokens));
  float m = p.m_in ? p.m_in[i] * p.m_in_scale : 0.0f;
  constexpr int U = 8;  // sums on their way at a time
  for (int k0 = 0; k0 < p.segments; k0 += U) {
    float own[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u, s = p.reverse ? p.segments - 1 - k : k;
      own[u] = k < p.segments - 1 ? p.seg_state[s * all + i] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u, s = p.reverse ? p.segments - 1 - k : k;
      if (k >= p.segments) break;
      p.seg_state[s * all + i] = m;
      const long long tokens = min(max(len - s * p.seg_tokens, 0LL), p.seg_tokens);
      if (tokens > 0) m = (tokens == p.seg_tokens ? whole : Decay(exp(g * (double)tokens))).times(m) + own[u];
    }
  }
}

hipError_t launch_attn_join(const AttnPass& p) {
  const size_t all = (size_t)p.batch * p.heads * p.rows * p.cols, blocks = (all + 255) / 256;
  if ((long long)blocks > max_blocks(256)) return hipErrorInvalidValue;  // (segments are for few heads)
  hipLaunchKernelGGL(attn_join_kernel, dim3((unsigned)blocks), dim3(256), 0, p.stream, p);
  return hipGetLastError();
}

// Workgroups of 256 for `total` threads' work, in a loop past 2^20 of them
static unsigned looping_blocks(long long total) { return (unsigned)std::min((total + 255) / 256, 1LL << 20); }

// (batch, token, head, features) of any strides as a dense tensor of `padded` features, zeros past the last: operands that are
// not in whole 16-byte pieces, which the blocks' loads need.  32 x 1024 tokens of 16 bf16 heads of 127: 3 copies and a
// pass 415 us (a value a thread: 860), where heads of 128 take 181.
// A thread writes one piece of 16 bytes, and reads it in one load (at whatever address: the hardware takes any) where it is whole.
template <typename U>
__global__ __launch_bounds__(256) void attn_pack_kernel(const U* __restrict__ in, U* __restrict__ out, long long total,
                                                        unsigned tokens, unsigned heads, int features, unsigned pieces, long long sb,
                                                        long long st, long long sh) {
  constexpr int N = 16 / sizeof(U);
  struct __attribute__((aligned(sizeof(U)))) Any {
    U v[N];
  };
  for (long long i0 = (long long)blockIdx.x * 256; i0 + threadIdx.x < total; i0 += (long long)gridDim.x * 256) {
    const long long row = (long long)heads * pieces, bt0 = i0 / row, b0 = bt0 / tokens;
    const unsigned p = (unsigned)(i0 - bt0 * row) + threadIdx.x, r = p % (unsigned)row;
    const unsigned t = (unsigned)(bt0 - b0 * tokens) + p / (unsigned)row, h = r / pieces;
    const int f = (int)(r % pieces) * N;
    const U* src = in + (b0 + t / tokens) * sb + (long long)(t % tokens) * st + h * sh + f;
    Any x;
    if (f + N <= features) {
      x = *reinterpret_cast<const Any*>(src);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x.v[j] = f + j < features ? src[j] : U(0);
    }
    *reinterpret_cast<uint4*>(out + (i0 + threadIdx.x) * N) = __builtin_bit_cast(uint4, x);
  }
}

hipError_t launch_attn_pack(const HeadsView& v, void* out, int dtype, long long batch, long long tokens, int heads, int features,
                            int padded, hipStream_t stream) {
  const int pieces = padded / (dtype == 0 ? 4 : 8);
  const long long total = batch * tokens * heads * pieces;
  const dim3 grid(looping_blocks(total)), block(256);
  if (dtype == 0)
    hipLaunchKernelGGL((attn_pack_kernel<unsigned>), grid, block, 0, stream, static_cast<const unsigned*>(v.p),
                       static_cast<unsigned*>(out), total, (unsigned)tokens, (unsigned)heads, features, (unsigned)pieces, v.sb, v.st, v.sh);
  else
    hipLaunchKernelGGL((attn_pack_kernel<unsigned short>), grid, block, 0, stream, static_cast<const unsigned short*>(v.p),
                       static_cast<unsigned short*>(out), total, (unsigned)tokens, (unsigned)heads, features, (unsigned)pieces, v.sb, v.st, v.sh);
  return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------
// Sums of the gradients' parts, in a fixed order.
// ------------------------------------------------------------------------------------------------

__global__ __launch_bounds__(256) void attn_dg_sum_kernel(const double* __restrict__ parts, float* __restrict__ out,
                                                          long long batch, int heads, int each) {
  __shared__ double sum[256];
  const int h = blockIdx.x, t = threadIdx.x;
  double s = 0.0;
  for (long long i = t; i < batch * each; i += 256) s += parts[((i / each) * heads + h) * each + i % each];
  sum[t] = s;
  __syncthreads();
  for (int k = 128; k > 0; k /= 2) {
    if (t < k) sum[t] += sum[t + k];
    __syncthreads();
  }
  if (t == 0) out[h] = (float)sum[0];
}

hipError_t launch_attn_dg_sum(const double* parts, float* out, long long batch, int heads, int each,
                              hipStream_t stream) {
  hipLaunchKernelGGL(attn_dg_sum_kernel, dim3(heads), dim3(256), 0, stream, parts, out, batch, heads, each);
  return hipGetLastError();
}

template <typename T>
__global__ __launch_bounds__(256) void attn_head_sum_kernel(const float* __restrict__ in, T* __restrict__ out,
                                                            long long total, int group, int d) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const float* src = in + (i / d) * group * d + i % d;
    float s = 0.0f;
    for (int g = 0; g < group; ++g) s += src[(long long)g * d];
    out[i] = from_f32<T>(s);
  }
}

hipError_t launch_attn_head_sum(const float* in, void* out, int dtype, long long rows, int heads_out, int group, int d,
                                hipStream_t stream) {
  const long long total = rows * heads_out * d;
  const dim3 grid(looping_blocks(total)), block(256);
  if (dtype == 0)
    hipLaunchKernelGGL((attn_head_sum_kernel<float>), grid, block, 0, stream, in, static_cast<float*>(out), total, group, d);
  else if (dtype == 1)
    hipLaunchKernelGGL((attn_head_sum_kernel<__bf16>), grid, block, 0, stream, in, static_cast<__bf16*>(out), total, group, d);
  else
    hipLaunchKernelGGL((attn_head_sum_kernel<_Float16>), grid, block, 0, stream, in, static_cast<_Float16*>(out), total, group, d);
  return hipGetLastError();
}

// ------------------------------------------------------------------------------------------------
// One token of every stream: S <- gamma S + k v^T in place, o = scale S^T q.  Bound by reading and writing the states
// (8 bytes an element), each of them once: 256 streams of 16 heads of 128 x 128, 108 us, 4.9 TB/s.  A workgroup takes 32 columns,
// so that one stream of 8 heads of 64 is 16 workgroups: 8 lanes of four columns (a 128-byte line together), 32 row groups of 4
// rows a pass, all of a pass's 16-byte loads ahead of its arithmetic.  (At addresses that are no multiples of 16 bytes the same
// accesses take 163 us.  Where columns are no multiple of 4 a row's last ones go by the value: 126 columns, 180 us; all of them so, 199.)
// ------------------------------------------------------------------------------------------------

// four neighbours at any address of a float (one access: the hardware asks for no more)
struct __attribute__((aligned(4))) AnyFour {
  float v[4];
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void attn_step_kernel(AttnStep p, int slices) {
  __shared__ float part[4][32];
  const int t = threadIdx.x, c4 = t % 8, rg = t / 8, wave = t / 64;
  const int slice = blockIdx.x % slices;
  const long long bh = p.first * p.heads + blockIdx.x / slices, b = bh / p.heads;
  const int h = (int)(bh % p.heads), n = slice * 32 + c4 * 4;
  const T* q = static_cast<const T*>(p.q) + b * p.q_sb + (long long)(h / p.q_group) * p.q_sh;
  const T* k = static_cast<const T*>(p.k) + b * p.k_sb + (long long)(h / p.k_group) * p.k_sh;
  const T* v = static_cast<const T*>(p.v) + b * p.v_sb + (long long)(h / p.v_group) * p.v_sh;
  float* S = p.state + bh * p.rows * p.cols;
  const Decay gamma(exp((double)log_decay_of(p.log_decay, h)));  // (rounded once more at every frame, it would add up)
  float vv[4], acc[4] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) vv[j] = n + j < p.cols ? to_f32(v[n + j]) : 0.0f;
  for (int r0 = 0; r0 < p.rows; r0 += 128) {
    float s[4][4], qr[4], kr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + rg + 32 * i;
      const bool in = r < p.rows;
      qr[i] = in ? to_f32(q[r]) : 0.0f;
      kr[i] = in ? to_f32(k[r]) : 0.0f;
      const float* src = S + (long long)r * p.cols + n;
      if (in && (VEC ? n < p.cols : n + 3 < p.cols)) {
        const AnyFour x = *reinterpret_cast<const AnyFour*>(src);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = x.v[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = !VEC && in && n + j < p.cols ? src[j] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = r0 + rg + 32 * i;
      float* dst = S + (long long)r * p.cols + n;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = __builtin_fmaf(kr[i], vv[j], gamma.times(s[i][j]));
        acc[j] = __builtin_fmaf(qr[i], s[i][j], acc[j]);
      }
      if (r < p.rows) {
        if (VEC ? n < p.cols : n + 3 < p.cols) {
          *reinterpret_cast<AnyFour*>(dst) = AnyFour{{s[i][0], s[i][1], s[i][2], s[i][3]}};
        } else if (!VEC) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < p.cols) dst[j] = s[i][j];
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int o = 8; o < 64; o *= 2) acc[j] += __shfl_xor(acc[j], o);
    if (t % 64 < 8) part[wave][c4 * 4 + j] = acc[j];
  }
  __syncthreads();
  if (t < 32 && slice * 32 + t < p.cols)
    static_cast<T*>(p.out)[bh * p.cols + slice * 32 + t] =
        from_f32<T>((part[0][t] + part[1][t] + part[2][t] + part[3][t]) * p.scale);
}

template <typename T>
static hipError_t step_launch(const AttnStep& p) {
  const int slices = (p.cols + 31) / 32;
  return for_batches(p, (long long)p.heads * slices, 256, [&](const AttnStep& q, dim3 grid) {
    if (q.cols % 4 == 0)
      hipLaunchKernelGGL((attn_step_kernel<T, true>), grid, dim3(256), 0, q.stream, q, slices);
    else
      hipLaunchKernelGGL((attn_step_kernel<T, false>), grid, dim3(256), 0, q.stream, q, slices);
  });
}

hipError_t launch_attn_step(const AttnStep& p) {
  if (p.dtype == 0) return step_launch<float>(p);
  return p.dtype == 1 ? step_launch<__bf16>(p) : step_launch<_Float16>(p);
}

}  // namespace tfa
