// Operators of models on frames: decayed linear attention, group norm with an activation, AdamW steps, causal convolution,
// selective scan, gradient norms.  Argument blocks and launch functions shared by the kernels (kernels_attention.hip,
// kernels_norm.hip, kernels_adamw.hip, kernels_conv.hip, kernels_scan.hip, kernels_clip.hip) and their C entry points
// (model_ops.hip, state_space_ops.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace tfa {

// Workgroups of a launch: a dispatch counts its threads along x in 32 bits, and what is past them is dropped without an error.
constexpr long long max_blocks(int threads) { return 0xffffffffLL / threads; }

// Sets the calling thread's error text (tfa_last_error) and returns `code`; never throws.
int set_error(int code, const char* text) noexcept;

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  return static_cast<float>(x);
}
template <>
__device__ __forceinline__ float to_f32<__bf16>(__bf16 x) {
  return __uint_as_float((unsigned)__builtin_bit_cast(unsigned short, x) << 16);
}
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  return static_cast<T>(x);  // to nearest, ties to even
}

// V neighbouring values, one access
template <typename T, int V>
struct __attribute__((aligned(V * sizeof(T)))) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_pack(const T* p, float (&x)[V]) {
  const Pack<T, V> u = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = to_f32(u.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const float (&x)[V]) {
  Pack<T, V> u;
#pragma unroll
  for (int i = 0; i < V; ++i) u.v[i] = from_f32<T>(x[i]);
  *reinterpret_cast<Pack<T, V>*>(p) = u;
}

// ------------------------------------------------------------------------------------------------
// decayed linear attention
// ------------------------------------------------------------------------------------------------

// (batch, token, head, feature) operand: strides in elements, features contiguous; head h of the call reads h / group
struct HeadsView {
  const void* p;
  long long sb, st, sh;
  int group;
};

// One pass  out_t = scale (sum_s gamma^|t-s| (a_t . b_s) c_s + gamma^(..) a_t M_in)  over s <= t, or s >= t when
// `reverse`; M is the (R, N) state sum_s gamma^(..) b_s c_s^T that the pass carries.  The forward of the attention and
// each of its gradients is one such pass (the table is in kernels_attention.hip).
struct AttnPass {
  HeadsView a, b, c;
  int rows, cols;  // R: features of a and b, N: features of c
  bool reverse;
  int dtype;
  long long batch, tokens;
  long long first;             // batch row of the launch's first workgroup (launches set it)
  int heads;
  const float* log_decay;      // (heads)
  const long long* lengths;    // (batch) or nullptr: tokens at and past it are padding
  const float* m_in;           // (batch, heads, ...) or nullptr; element (r, n) at r * m_r + n * m_n
  float* m_out;                // or nullptr; laid out as m_in, must not alias it
  long long m_r, m_n;
  float m_in_scale, m_out_scale;
  void* out;                   // (batch, tokens, heads, N), fp32 where out_f32, else `dtype`
  bool out_f32;
  float scale;
  // the decays' gradient, sum over pairs of lag * flow: x (batch, token, head, N) the operand that `out` is the gradient of,
  // m_sink the gradient of the end state (laid out as m_in) or nullptr, dg_part attn_*_dg_parts(pass) values for each (batch, head)
  HeadsView x;
  const float* m_sink;
  double* dg_part;
  // A long sequence in segments of seg_tokens (a multiple of 64), each a workgroup of its own: seg_state (segments,
  // batch, heads, ...) are the states they start from, laid out as m_in.  out = nullptr: writes the segments' own sums there.
  int segments;
  long long seg_tokens;
  float* seg_state;
  // In blocks, with dg_part: the forward pass of the query gradient leaves the states at every `stretch` tokens (a divisor of
  // seg_tokens) but the first, `borders` of them for each (batch, head), for the reversed pass of the key gradient
  float* border_state;
  long long borders;
  int stretch, log_stretch;  // a power of two
  hipStream_t stream;
};

// token by token (any dimensions up to 256)
hipError_t launch_attn_scan(const AttnPass& p);
int attn_scan_dg_parts(const AttnPass& p);
// in blocks of tokens on the matrix cores: dimensions up to 128; a, b and c "whole" (addresses, strides and features are
// multiples of 16 bytes, or stride 0) with token strides below 2^24 elements
int attn_blocks_dg_parts(const AttnPass& p);
size_t attn_border_bytes(int rows, int cols);  // of one border's state
hipError_t launch_attn_blocks(const AttnPass& p);
// a dense copy (batch, tokens, heads, padded) of an operand, zeros past its features
hipError_t launch_attn_pack(const HeadsView& v, void* out, int dtype, long long batch, long long tokens, int heads, int features,
                            int padded, hipStream_t stream);
// the states that segments of a long sequence start from, p.seg_state, from the segments' own sums: in place
hipError_t launch_attn_join(const AttnPass& p);
// dlog_decay[h] = sum over batch and parts
hipError_t launch_attn_dg_sum(const double* parts, float* out, long long batch, int heads, int each, hipStream_t stream);
// out (rows, heads_out, d) of `dtype` = sums of `group` neighbouring heads of (rows, heads_out * group, d) fp32
hipError_t launch_attn_head_sum(const float* in, void* out, int dtype, long long rows, int heads_out, int group, int d,
                                hipStream_t stream);

struct AttnStep {
  const void *q, *k, *v;  // (batch, q_heads, rows), (batch, k_heads, rows), (batch, v_heads, cols)
  long long q_sb, q_sh, k_sb, k_sh, v_sb, v_sh;
  int q_group, k_group, v_group;
  int rows, cols, heads, dtype;
  long long batch;
  long long first;  // as AttnPass's
  const float* log_decay;
  float* state;  // (batch, heads, rows, cols)
  void* out;     // (batch, heads, cols)
  float scale;
  hipStream_t stream;
};
hipError_t launch_attn_step(const AttnStep& p);

// ------------------------------------------------------------------------------------------------
// group norm with an activation, channels last
// ------------------------------------------------------------------------------------------------

struct NormArgs {
  const void* x;  // (batch, positions, channels)
  const void* dy;
  void* y;        // forward: y; backward: dx
  const float* weight;  // or nullptr: 1
  const float* bias;    // or nullptr: 0
  float* mean;    // (batch, groups)
  float* rstd;
  float* dweight;  // backward, or nullptr
  float* dbias;
  const long long* lengths;  // (batch) or nullptr: positions at and past lengths[n] * inner are padding
  long long batch, positions, inner;
  int channels, groups, act, dtype;
  float eps;
  float* ws;  // norm_workspace_bytes
  hipStream_t stream;
};
size_t norm_workspace_bytes(const NormArgs& a, bool backward);
bool norm_aligned(const NormArgs& a);
hipError_t launch_norm_forward(const NormArgs& a);
hipError_t launch_norm_backward(const NormArgs& a);

// ------------------------------------------------------------------------------------------------
// AdamW over many tensors
// ------------------------------------------------------------------------------------------------

struct AdamTensor {
  void* p;
  const void* g;
  void* m;         // fp32, or int8 codes
  void* v;         // fp32, or uint8 codes
  float* m_scale;  // 8 bits: one per block of 256
  float* v_scale;
  float* master;   // or nullptr
  long long n;
};
struct AdamArgs {
  int p_dtype, g_dtype, bits;
  float decay;             // 1 - lr * weight_decay
  float beta1, one_beta1, beta2, one_beta2;
  float step_size;         // lr / (1 - beta1^step)
  float inv_root_bc2, eps;  // 1 / sqrt(1 - beta2^step)
};
hipError_t launch_adamw(const AdamTensor* tensors, long long count, const AdamArgs& a, hipStream_t stream);
// out[i] = the values that 8-bit codes stand for (second moments where `squares`)
struct CodeTensor {
  const void* codes;
  const float* scales;
  float* out;
  long long n;
};
hipError_t launch_adam_values(const CodeTensor* tensors, long long count, bool squares, hipStream_t stream);

// ------------------------------------------------------------------------------------------------
// causal convolution along frames, a filter for each channel
// ------------------------------------------------------------------------------------------------

struct ConvArgs {
  const void* x;  // (batch, tokens, channels) at x_sb, x_st
  long long x_sb, x_st;
  const float* weight;  // (channels, width)
  const float* bias;    // or nullptr
  const long long* lengths;
  const void* state_in;  // (batch, width - 1, channels) or nullptr: zeros
  void* y;               // contiguous
  void* state_out;       // or nullptr
  int channels, width, act, dtype;
  long long batch, tokens;
  // backward: dy contiguous, dstate_out or nullptr; dx, dstate_in, dweight and dbias or nullptr
  const void* dy;
  const void* dstate_out;
  void* dx;
  void* dstate_in;
  float* dweight;
  float* dbias;
  float* ws;  // conv_workspace_bytes
  hipStream_t stream;
};
size_t conv_workspace_bytes(const ConvArgs& a);
hipError_t launch_conv_forward(const ConvArgs& a);
hipError_t launch_conv_backward(const ConvArgs& a);
// one token: state_out (= state_in) is shifted in place
hipError_t launch_conv_step(const ConvArgs& a);

// ------------------------------------------------------------------------------------------------
// selective scan
// ------------------------------------------------------------------------------------------------

struct ScanArgs {
  // (batch, tokens, channels) at strides of batch and token, channels contiguous; z may be nullptr (no gate)
  const void *x, *dt, *z;
  long long x_sb, x_st, dt_sb, dt_st, z_sb, z_st;
  // (batch, tokens, groups, n) at strides of batch, token and group, n contiguous
  const void *b, *c;
  long long b_sb, b_st, b_sg, c_sb, c_st, c_sg;
  const float *a;             // (channels, n)
  const float *d, *dt_bias;   // (channels) or nullptr
  const long long* lengths;   // (batch) or nullptr
  const float* state_in;      // (batch, channels, n) or nullptr: zeros
  float* state_out;           // or nullptr
  void* y;                    // contiguous
  bool softplus;
  int channels, groups, n, dtype;
  long long batch, tokens;
  // states at every kScanStretch tokens but the first, as the kernels lay them out: written by the forward, read by the backward
  float* kept;
  // a long sequence in segments: their own sums and decays, then the states they start from
  float* seg_state;
  float* seg_steps;
  // backward: dy contiguous; dx, ddt, dz, db and dc contiguous (db, dc: (batch, tokens, groups, n)), or nullptr
  const void* dy;
  const float* dstate_out;
  void *dx, *ddt, *dz, *db, *dc;
  float *da, *dd, *ddt_bias, *dstate_in;
  float* shared_parts;   // sums over workgroups' channels of db and dc
  float* channel_parts;  // sums over rows and segments of da, dd and ddt_bias
  int segments;
  long long seg_tokens;  // a multiple of kScanStretch, and of as many times `fine`
  int fine;              // parts of a segment whose sums are made by themselves
  hipStream_t stream;
};
constexpr int kScanTile = 16;     // tokens that are worked on together
constexpr int kScanStretch = 16;  // tokens between kept states
constexpr int kScanMostStates = 64;
// Sizes in bytes of what a call needs (segments and seg_tokens set)
struct ScanSizes {
  size_t kept, seg_state, seg_steps, shared_parts, channel_parts;
};
long long scan_waves(const ScanArgs& p);  // of a segment
bool scan_has_pairs(const ScanArgs& p);   // whether two waves can take the same channels, forward
ScanSizes scan_sizes(const ScanArgs& p);
hipError_t launch_scan_forward(const ScanArgs& p);
hipError_t launch_scan_backward(const ScanArgs& p);
struct ScanStep {
  const void *x, *dt, *z, *b, *c;
  long long x_sb, dt_sb, z_sb, b_sb, b_sg, c_sb, c_sg;
  const float *a, *d, *dt_bias;
  float* state;
  void* y;
  bool softplus;
  int channels, groups, n, dtype;
  long long batch;
  hipStream_t stream;
};
hipError_t launch_scan_step(const ScanStep& p);

// ------------------------------------------------------------------------------------------------
// the gradients' global norm and their clipping
// ------------------------------------------------------------------------------------------------

struct GradTensor {
  void* p;
  long long n;
};
// tensors of a dtype (the index), any number of each
struct GradLists {
  const GradTensor* tensors[3];
  long long count[3];
};
long long grad_parts(const GradLists& g);  // doubles of the workspace
// norm[0] = sqrt(sum of squares); then, where `scale`, every value times min(1, max_norm / (norm + 1e-6))
hipError_t launch_grad_norm(const GradLists& g, double* parts, float* norm, bool scale, double max_norm, hipStream_t stream);

}  // namespace tfa
