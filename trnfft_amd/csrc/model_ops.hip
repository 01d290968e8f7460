// C entry points of the operators of models on frames (include/trnfft_amd.h): argument checks, workspaces, launches.
#include "model_ops.h"

#include <algorithm>
#include <cmath>

#include "../../include/trnfft_amd.h"

using tfa::set_error;

namespace {

int launched(hipError_t e) { return e == hipSuccess ? TFA_OK : set_error(TFA_ERR_HIP, hipGetErrorString(e)); }

bool dtype_ok(int32_t d) { return d == TFA_DTYPE_F32 || d == TFA_DTYPE_BF16 || d == TFA_DTYPE_F16; }
size_t dtype_size(int32_t d) { return d == TFA_DTYPE_F32 ? 4 : 2; }

constexpr int64_t kMaxBlocks = 0x7fffffff;
constexpr int32_t kMaxHeadDim = 256;

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

int check_heads(const tfa_attn_desc* d) {
  if (!d) return set_error(TFA_ERR_INVALID, "null descriptor");
  if (!dtype_ok(d->dtype)) return set_error(TFA_ERR_INVALID, "dtype must be TFA_DTYPE_F32, _BF16 or _F16");
  if (d->batch < 0 || d->tokens < 0) return set_error(TFA_ERR_INVALID, "negative dimension");
  if (d->heads < 1 || d->key_dim < 1 || d->value_dim < 1) return set_error(TFA_ERR_INVALID, "need at least one head and feature");
  for (const int32_t n : {d->q_heads, d->k_heads, d->v_heads})
    if (n < 1 || d->heads % n) return set_error(TFA_ERR_INVALID, "heads must be a multiple of each operand's heads");
  if (!(std::isfinite(d->scale) && d->scale != 0.0f)) return set_error(TFA_ERR_INVALID, "scale must be finite and not zero");
  if (d->key_dim > kMaxHeadDim || d->value_dim > kMaxHeadDim)
    return set_error(TFA_ERR_UNSUPPORTED, "head dimensions above 256 are not implemented");
  if (d->heads > 65535 || d->batch > kMaxBlocks / 16 / d->heads)
    return set_error(TFA_ERR_UNSUPPORTED, "batch * heads beyond the launch grid");
  if (d->tokens > INT32_MAX) return set_error(TFA_ERR_UNSUPPORTED, "more than 2^31 tokens");
  return TFA_OK;
}

tfa::HeadsView view(const void* p, const tfa_attn_desc* d, const int64_t* stride, int32_t own) {
  // (a stride along one row says nothing)
  return {p, d->batch > 1 ? stride[0] : 0, d->tokens > 1 ? stride[1] : 0, own > 1 ? stride[2] : 0, d->heads / own};
}

tfa::HeadsView dense(const void* p, const tfa_attn_desc* d, int32_t features) {
  return {p, (long long)d->tokens * d->heads * features, (long long)d->heads * features, features, 1};
}

// the forward pass of every gradient and of the output, without its operands
tfa::AttnPass pass_of(const tfa_attn_desc* d, const float* log_decay, const int64_t* lengths, tfa_stream stream) {
  tfa::AttnPass p{};
  p.dtype = d->dtype;
  p.batch = d->batch;
  p.tokens = d->tokens;
  p.heads = d->heads;
  p.log_decay = log_decay;
  p.lengths = reinterpret_cast<const long long*>(lengths);
  p.m_in_scale = p.m_out_scale = 1.0f;
  p.scale = d->scale;
  p.stream = static_cast<hipStream_t>(stream);
  return p;
}

// Heads of up to kBlockDim features go in blocks of tokens on the matrix cores, wider ones (whose state does not fit a wave's
// registers) token by token.  Blocks are the better choice from the first token on: 256 x 4 tokens of 16 bf16 heads of 128, 136 against 168 us,
// training 538 against 1037; 16 tokens 137 against 422 us; 64 x 4 of 8 heads of 64, 16 against 15 us.
constexpr int32_t kBlockDim = 128;
// A long sequence is cut into segments where batch * heads alone leave compute units idle: about kWantBlocks
// workgroups in all, segments of at least kSegTokens.  Twice as many workgroups: 64 x 626 tokens of 8 heads of 64 99 against
// 71 us, 1 x 65536 of 16 heads of 128 487 against 454, training on 8 x 4096 1205 against 1040 (sums and joins repeat the
// keys' and values' reading).  Segments of at least 256: training on 4 x 1001 of 6 fp32 heads 350 against 223 us.
constexpr int64_t kWantBlocks = 512, kSegTokens = 128;
// Tokens between the states that the decays' gradient keeps: a quarter of the traffic of keeping each 64-token block's
// (training on 8 x 4096 tokens of 16 heads of 128: 1017 us, with 64 tokens 1383; 64 x 626 of 8 heads of 64: 341 and 398).
constexpr int64_t kStretch = 256;

struct Plan {
  bool blocks;
  int segments;
  int64_t seg_tokens;
  size_t state_bytes;  // of the segments' states
  // operands q, k, v, grad_out that are not laid out in whole 16-byte pieces are copied so first
  int padded[4];        // features of the copy, 0: taken as it is
  size_t pack_bytes[4];
};

Plan plan_of(const tfa_attn_desc* d, bool backward) {
  Plan plan{};
  plan.segments = 1;
  plan.seg_tokens = std::max<int64_t>(1, (d->tokens + 63) / 64 * 64);
  plan.blocks = d->tokens > 0 && d->key_dim <= kBlockDim && d->value_dim <= kBlockDim;
  if (!plan.blocks || d->batch == 0) return plan;
  const int piece = 16 / (int)dtype_size(d->dtype);
  const int64_t* strides[3] = {d->q_stride, d->k_stride, d->v_stride};
  const int32_t own[4] = {d->q_heads, d->k_heads, d->v_heads, d->heads};
  for (int i = 0; i < (backward ? 4 : 3); ++i) {
    const int32_t features = i < 2 ? d->key_dim : d->value_dim;
    bool whole = features % piece == 0;
    if (i < 3) {
      const tfa::HeadsView v = view(nullptr, d, strides[i], own[i]);
      whole = whole && v.sb % piece == 0 && v.st % piece == 0 && v.sh % piece == 0 && v.st >= 0 && v.st < (1 << 24);
    }
    if (whole) continue;
    plan.padded[i] = (features + piece - 1) / piece * piece;
    plan.pack_bytes[i] = align256((size_t)d->batch * d->tokens * own[i] * plan.padded[i] * dtype_size(d->dtype));
  }
  const int64_t rows = d->batch * d->heads;
  const int64_t want = std::min((kWantBlocks + rows - 1) / rows, d->tokens / kSegTokens);
  if (want > 1) {
    plan.seg_tokens = ((d->tokens + want - 1) / want + 63) / 64 * 64;
    plan.segments = (int)((d->tokens + plan.seg_tokens - 1) / plan.seg_tokens);
    if (plan.segments > 1) plan.state_bytes = align256((size_t)plan.segments * rows * d->key_dim * d->value_dim * sizeof(float));
  }
  return plan;
}

size_t packed_bytes(const Plan& plan) { return plan.pack_bytes[0] + plan.pack_bytes[1] + plan.pack_bytes[2] + plan.pack_bytes[3]; }

// Operand i as the kernels take it, copied to `*space` where the plan says so; `*space` moves past the copy.
int operand(const tfa_attn_desc* d, const Plan& plan, int i, int32_t own, int32_t features, tfa::HeadsView* v, char** space,
            hipStream_t stream) {
  if (!plan.blocks) return TFA_OK;
  if (!plan.padded[i]) {
    if (reinterpret_cast<uintptr_t>(v->p) % 16) return set_error(TFA_ERR_INVALID, "operands must be 16-byte aligned");
    return TFA_OK;
  }
  const hipError_t e = tfa::launch_attn_pack(*v, *space, d->dtype, d->batch, d->tokens, own, features, plan.padded[i], stream);
  if (e != hipSuccess) return launched(e);
  const long long row = (long long)own * plan.padded[i];
  *v = {*space, d->tokens * row, row, plan.padded[i], v->group};
  *space += plan.pack_bytes[i];
  return TFA_OK;
}

hipError_t run_pass(tfa::AttnPass p, const Plan& plan, float* states) {
  p.segments = plan.segments;
  p.seg_tokens = plan.seg_tokens;
  p.seg_state = states;
  return plan.blocks ? tfa::launch_attn_blocks(p) : tfa::launch_attn_scan(p);
}

// the states that a pass's segments start from
hipError_t segment_states(tfa::AttnPass p, const Plan& plan, float* states) {
  if (plan.segments == 1) return hipSuccess;
  p.out = nullptr;
  p.dg_part = nullptr;
  const hipError_t e = run_pass(p, plan, states);
  if (e != hipSuccess) return e;
  p.segments = plan.segments;
  p.seg_tokens = plan.seg_tokens;
  p.seg_state = states;
  return tfa::launch_attn_join(p);
}

struct BackwardSpace {
  size_t dq = 0, dk = 0, dv = 0, dg = 0, total = 0;  // offsets; gradients of shared heads before their sum
  size_t packed = 0, states = 0, grad_states = 0, border = 0;
  int64_t stretch = 0, borders = 0;
  int dg_each = 0;
  Plan plan;
};

BackwardSpace backward_space(const tfa_attn_desc* d, bool decays) {
  BackwardSpace s;
  s.plan = plan_of(d, true);
  const size_t rows = (size_t)d->batch * d->tokens * d->heads * sizeof(float);
  if (d->q_heads != d->heads) s.dq = s.total, s.total += align256(rows * d->key_dim);
  if (d->k_heads != d->heads) s.dk = s.total, s.total += align256(rows * d->key_dim);
  if (d->v_heads != d->heads) s.dv = s.total, s.total += align256(rows * d->value_dim);
  s.packed = s.total, s.total += packed_bytes(s.plan);
  s.states = s.total, s.total += s.plan.state_bytes;
  s.grad_states = s.total, s.total += s.plan.state_bytes;
  tfa::AttnPass p{};
  p.rows = d->value_dim;
  p.cols = d->key_dim;
  p.segments = s.plan.segments;
  s.dg_each = s.plan.blocks ? tfa::attn_blocks_dg_parts(p) : tfa::attn_scan_dg_parts(p);
  s.dg = s.total;
  s.total += align256((size_t)d->batch * d->heads * s.dg_each * sizeof(double));
  if (decays && s.plan.blocks) {
    s.stretch = kStretch;
    while (s.plan.seg_tokens % s.stretch) s.stretch /= 2;
    s.borders = (d->tokens - 1) / s.stretch;
    s.border = s.total;
    s.total += align256((size_t)d->batch * d->heads * s.borders * tfa::attn_border_bytes(p.rows, p.cols));
  }
  return s;
}

}  // namespace

extern "C" {

int tfa_linear_attention_workspace_size(const tfa_attn_desc* desc, int32_t backward, size_t* bytes) {
  if (!bytes) return set_error(TFA_ERR_INVALID, "null bytes pointer");
  *bytes = 0;
  if (const int rc = check_heads(desc)) return rc;
  if (backward) {
    *bytes = backward_space(desc, backward == 2).total;
  } else {
    const Plan plan = plan_of(desc, false);
    *bytes = packed_bytes(plan) + plan.state_bytes;
  }
  return TFA_OK;
}

int tfa_linear_attention(const tfa_attn_desc* desc, const void* q, const void* k, const void* v, const float* log_decay,
                         const int64_t* lengths, const float* state_in, void* out, float* state_out, void* workspace,
                         tfa_stream stream) {
  if (const int rc = check_heads(desc)) return rc;
  if (desc->batch == 0) return TFA_OK;
  if (!log_decay || (desc->tokens > 0 && (!q || !k || !v || !out))) return set_error(TFA_ERR_INVALID, "null data pointer");
  if (state_out && state_out == state_in) return set_error(TFA_ERR_INVALID, "state_out must not be state_in");
  tfa::AttnPass p = pass_of(desc, log_decay, lengths, stream);
  p.a = view(q, desc, desc->q_stride, desc->q_heads);
  p.b = view(k, desc, desc->k_stride, desc->k_heads);
  p.c = view(v, desc, desc->v_stride, desc->v_heads);
  p.rows = desc->key_dim;
  p.cols = desc->value_dim;
  p.m_in = state_in;
  p.m_out = state_out;
  p.m_r = desc->value_dim;
  p.m_n = 1;
  p.out = out;
  const Plan plan = plan_of(desc, false);
  if (packed_bytes(plan) + plan.state_bytes && !workspace) return set_error(TFA_ERR_INVALID, "null workspace");
  char* space = static_cast<char*>(workspace);
  if (const int rc = operand(desc, plan, 0, desc->q_heads, desc->key_dim, &p.a, &space, p.stream)) return rc;
  if (const int rc = operand(desc, plan, 1, desc->k_heads, desc->key_dim, &p.b, &space, p.stream)) return rc;
  if (const int rc = operand(desc, plan, 2, desc->v_heads, desc->value_dim, &p.c, &space, p.stream)) return rc;
  float* states = reinterpret_cast<float*>(space);
  if (const hipError_t e = segment_states(p, plan, states)) return launched(e);
  return launched(run_pass(p, plan, states));
}

int tfa_linear_attention_backward(const tfa_attn_desc* desc, const void* q, const void* k, const void* v,
                                  const float* log_decay, const int64_t* lengths, const float* state_in,
                                  const void* grad_out, const float* grad_state_out, void* grad_q, void* grad_k,
                                  void* grad_v, float* grad_log_decay, float* grad_state_in, void* workspace,
                                  tfa_stream stream) {
  if (const int rc = check_heads(desc)) return rc;
  const tfa_attn_desc& d = *desc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const BackwardSpace space = backward_space(desc, grad_log_decay != nullptr);
  if (!log_decay || (!workspace && space.total)) return set_error(TFA_ERR_INVALID, "null data pointer");
  if (d.batch > 0 && d.tokens > 0 && (!q || !k || !v || !grad_out)) return set_error(TFA_ERR_INVALID, "null data pointer");
  if (grad_log_decay && d.batch > 0 && d.tokens > 0 && (!grad_q || !grad_k)) return set_error(TFA_ERR_INVALID, "grad_log_decay needs grad_q and grad_k");
  if (grad_state_in && grad_state_in == grad_state_out) return set_error(TFA_ERR_INVALID, "grad_state_in must not be grad_state_out");
  char* ws = static_cast<char*>(workspace);
  double* parts = reinterpret_cast<double*>(ws + space.dg);
  const long long rows = (long long)d.batch * d.tokens;
  tfa::HeadsView qv = view(q, desc, d.q_stride, d.q_heads), kv = view(k, desc, d.k_stride, d.k_heads),
                       vv = view(v, desc, d.v_stride, d.v_heads), gv = dense(grad_out, desc, d.value_dim);
  const Plan& plan = space.plan;
  if (d.batch > 0) {
    char* packed = ws + space.packed;
    if (const int rc = operand(desc, plan, 0, d.q_heads, d.key_dim, &qv, &packed, s)) return rc;
    if (const int rc = operand(desc, plan, 1, d.k_heads, d.key_dim, &kv, &packed, s)) return rc;
    if (const int rc = operand(desc, plan, 2, d.v_heads, d.value_dim, &vv, &packed, s)) return rc;
    if (const int rc = operand(desc, plan, 3, d.heads, d.value_dim, &gv, &packed, s)) return rc;
  }
  float* states = reinterpret_cast<float*>(ws + space.states);
  float* grad_states = reinterpret_cast<float*>(ws + space.grad_states);
  // the value gradient's pass; its states are those of the key gradient too, and where the decays' tangent ends
  tfa::AttnPass pv = pass_of(desc, log_decay, lengths, stream);
  pv.a = kv;
  pv.b = qv;
  pv.c = gv;
  pv.rows = d.key_dim;
  pv.cols = d.value_dim;
  pv.reverse = true;
  pv.m_in = grad_state_out;
  pv.m_out = grad_state_in;
  pv.m_in_scale = 1.0f / d.scale;
  pv.m_out_scale = d.scale;
  pv.m_r = d.value_dim;
  pv.m_n = 1;
  if (d.batch > 0 && plan.segments > 1) {
    if (const hipError_t e = segment_states(pv, plan, grad_states)) return launched(e);
    if (grad_q || grad_log_decay) {
      tfa::AttnPass p = pass_of(desc, log_decay, lengths, stream);
      p.b = kv;
      p.c = vv;
      p.rows = d.key_dim;
      p.cols = d.value_dim;
      p.m_in = state_in;
      p.m_r = d.value_dim;
      p.m_n = 1;
      if (const hipError_t e = segment_states(p, plan, states)) return launched(e);
    }
  }
  if (d.batch > 0 && (grad_q || grad_log_decay)) {
    tfa::AttnPass p = pass_of(desc, log_decay, lengths, stream);
    p.a = gv;
    p.b = vv;
    p.c = kv;
    p.rows = d.value_dim;
    p.cols = d.key_dim;
    p.m_in = state_in;
    p.m_r = 1;
    p.m_n = d.value_dim;
    p.out_f32 = d.q_heads != d.heads;
    p.out = p.out_f32 ? ws + space.dq : grad_q;
    if (grad_log_decay) {
      p.x = qv;
      p.m_sink = grad_state_out;
      p.dg_part = parts;
      p.border_state = reinterpret_cast<float*>(ws + space.border);
      p.borders = space.borders;
      p.stretch = (int)space.stretch;
      p.log_stretch = __builtin_ctz((unsigned)space.stretch);
    }
    if (const hipError_t e = run_pass(p, plan, states)) return launched(e);
    if (p.out_f32 && grad_q && rows)
      if (const hipError_t e = tfa::launch_attn_head_sum(reinterpret_cast<const float*>(ws + space.dq), grad_q, d.dtype, rows,
                                                         d.q_heads, d.heads / d.q_heads, d.key_dim, s))
        return launched(e);
  }
  if (d.batch > 0 && (grad_k || grad_log_decay)) {
    tfa::AttnPass p = pass_of(desc, log_decay, lengths, stream);
    p.a = vv;
    p.b = gv;
    p.c = qv;
    p.rows = d.value_dim;
    p.cols = d.key_dim;
    p.reverse = true;
    p.m_in = grad_state_out;
    p.m_in_scale = 1.0f / d.scale;
    p.m_r = 1;
    p.m_n = d.value_dim;
    p.out_f32 = d.k_heads != d.heads;
    p.out = p.out_f32 ? ws + space.dk : grad_k;
    if (grad_log_decay && plan.blocks) {
      p.x = kv;
      p.dg_part = parts;
      p.border_state = reinterpret_cast<float*>(ws + space.border);
      p.borders = space.borders;
      p.stretch = (int)space.stretch;
      p.log_stretch = __builtin_ctz((unsigned)space.stretch);
    }
    if (const hipError_t e = run_pass(p, plan, grad_states)) return launched(e);
    if (p.out_f32 && rows)
      if (const hipError_t e = tfa::launch_attn_head_sum(reinterpret_cast<const float*>(ws + space.dk), grad_k, d.dtype, rows,
                                                         d.k_heads, d.heads / d.k_heads, d.key_dim, s))
        return launched(e);
  }
  if (grad_log_decay)
    if (const hipError_t e = tfa::launch_attn_dg_sum(parts, grad_log_decay, d.batch, d.heads, space.dg_each, s))
      return launched(e);
  if (d.batch > 0 && (grad_v || grad_state_in)) {
    tfa::AttnPass p = pv;
    p.out_f32 = d.v_heads != d.heads;
    p.out = p.out_f32 ? ws + space.dv : grad_v;
    if (!p.out && rows) return set_error(TFA_ERR_INVALID, "grad_state_in needs grad_v");
    if (const hipError_t e = run_pass(p, plan, grad_states)) return launched(e);
    if (p.out_f32 && grad_v && rows)
      if (const hipError_t e = tfa::launch_attn_head_sum(reinterpret_cast<const float*>(ws + space.dv), grad_v, d.dtype, rows,
                                                         d.v_heads, d.heads / d.v_heads, d.value_dim, s))
        return launched(e);
  }
  return TFA_OK;
}

int tfa_linear_attention_step(const tfa_attn_desc* desc, const void* q, const void* k, const void* v,
                              const float* log_decay, float* state, void* out, tfa_stream stream) {
  if (const int rc = check_heads(desc)) return rc;
  const tfa_attn_desc& d = *desc;
  if (d.tokens != 1) return set_error(TFA_ERR_INVALID, "a step is one token");
  if (d.batch == 0) return TFA_OK;
  if (!q || !k || !v || !log_decay || !state || !out) return set_error(TFA_ERR_INVALID, "null data pointer");
  tfa::AttnStep p{};
  p.q = q, p.k = k, p.v = v;
  p.q_sb = d.q_stride[0], p.q_sh = d.q_stride[2], p.q_group = d.heads / d.q_heads;
  p.k_sb = d.k_stride[0], p.k_sh = d.k_stride[2], p.k_group = d.heads / d.k_heads;
  p.v_sb = d.v_stride[0], p.v_sh = d.v_stride[2], p.v_group = d.heads / d.v_heads;
  p.rows = d.key_dim, p.cols = d.value_dim, p.heads = d.heads, p.dtype = d.dtype, p.batch = d.batch;
  p.log_decay = log_decay, p.state = state, p.out = out, p.scale = d.scale;
  p.stream = static_cast<hipStream_t>(stream);
  return launched(tfa::launch_attn_step(p));
}

// ------------------------------------------------------------------------------------------------

static int check_norm(const tfa_norm_desc* d) {
  if (!d) return set_error(TFA_ERR_INVALID, "null descriptor");
  if (!dtype_ok(d->dtype)) return set_error(TFA_ERR_INVALID, "dtype must be TFA_DTYPE_F32, _BF16 or _F16");
  if (d->batch < 0 || d->positions < 0) return set_error(TFA_ERR_INVALID, "negative dimension");
  if (d->inner < 1 || d->positions % d->inner) return set_error(TFA_ERR_INVALID, "positions must be a multiple of inner");
  if (d->channels < 1 || d->groups < 1 || d->channels % d->groups)
    return set_error(TFA_ERR_INVALID, "channels must be a multiple of groups");
  if (d->activation < TFA_ACT_NONE || d->activation > TFA_ACT_RELU) return set_error(TFA_ERR_INVALID, "unknown activation");
  if (!(std::isfinite(d->eps) && d->eps >= 0.0f)) return set_error(TFA_ERR_INVALID, "eps must be finite and not negative");
  if (d->channels > (1 << 20) || d->batch > kMaxBlocks / d->groups)
    return set_error(TFA_ERR_UNSUPPORTED, "batch or channels beyond the launch grid");
  return TFA_OK;
}

static tfa::NormArgs norm_args(const tfa_norm_desc* d) {
  tfa::NormArgs a{};
  a.batch = d->batch, a.positions = d->positions, a.inner = d->inner;
  a.channels = d->channels, a.groups = d->groups, a.act = d->activation, a.dtype = d->dtype, a.eps = d->eps;
  return a;
}

int tfa_group_norm_workspace_size(const tfa_norm_desc* desc, int32_t backward, size_t* bytes) {
  if (!bytes) return set_error(TFA_ERR_INVALID, "null bytes pointer");
  *bytes = 0;
  if (const int rc = check_norm(desc)) return rc;
  *bytes = tfa::norm_workspace_bytes(norm_args(desc), backward != 0);
  return TFA_OK;
}

int tfa_group_norm(const tfa_norm_desc* desc, const void* x, const float* weight, const float* bias,
                   const int64_t* lengths, void* y, float* mean, float* rstd, void* workspace, tfa_stream stream) {
  if (const int rc = check_norm(desc)) return rc;
  if (desc->batch == 0 || desc->positions == 0) return TFA_OK;
  tfa::NormArgs a = norm_args(desc);
  if (!x || !y || !mean || !rstd || (!workspace && tfa::norm_workspace_bytes(a, false)))
    return set_error(TFA_ERR_INVALID, "null data pointer");
  a.x = x, a.y = y, a.weight = weight, a.bias = bias, a.mean = mean, a.rstd = rstd;
  a.lengths = reinterpret_cast<const long long*>(lengths);
  a.ws = static_cast<float*>(workspace), a.stream = static_cast<hipStream_t>(stream);
  if (!tfa::norm_aligned(a)) return set_error(TFA_ERR_INVALID, "x and y must be 16-byte aligned");
  return launched(tfa::launch_norm_forward(a));
}

int tfa_group_norm_backward(const tfa_norm_desc* desc, const void* x, const void* grad_y, const float* weight,
                            const float* bias, const int64_t* lengths, const float* mean, const float* rstd,
                            void* grad_x, float* grad_weight, float* grad_bias, void* workspace, tfa_stream stream) {
  if (const int rc = check_norm(desc)) return rc;
  if (desc->batch == 0 || desc->positions == 0) return TFA_OK;
  if (!x || !grad_y || !grad_x || !mean || !rstd || !workspace) return set_error(TFA_ERR_INVALID, "null data pointer");
  tfa::NormArgs a = norm_args(desc);
  a.x = x, a.dy = grad_y, a.y = grad_x, a.weight = weight, a.bias = bias;
  a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd), a.dweight = grad_weight, a.dbias = grad_bias;
  a.lengths = reinterpret_cast<const long long*>(lengths);
  a.ws = static_cast<float*>(workspace), a.stream = static_cast<hipStream_t>(stream);
  if (!tfa::norm_aligned(a)) return set_error(TFA_ERR_INVALID, "x, grad_y and grad_x must be 16-byte aligned");
  return launched(tfa::launch_norm_backward(a));
}

// ------------------------------------------------------------------------------------------------

int tfa_adamw_step(int64_t count, const tfa_adam_tensor* tensors, const tfa_adam_desc* desc, tfa_stream stream) {
  if (count < 0 || !desc || (count > 0 && !tensors)) return set_error(TFA_ERR_INVALID, "bad argument");
  const tfa_adam_desc& d = *desc;
  if (!dtype_ok(d.param_dtype) || !dtype_ok(d.grad_dtype)) return set_error(TFA_ERR_INVALID, "dtype must be TFA_DTYPE_F32, _BF16 or _F16");
  if (d.grad_dtype != d.param_dtype && d.grad_dtype != TFA_DTYPE_F32)
    return set_error(TFA_ERR_UNSUPPORTED, "gradients must have the parameters' type or be fp32");
  if (d.state_bits != 32 && d.state_bits != 8) return set_error(TFA_ERR_INVALID, "states have 32 or 8 bits");
  if (d.step < 1) return set_error(TFA_ERR_INVALID, "steps count from 1");
  if (!(d.beta1 >= 0.0 && d.beta1 < 1.0 && d.beta2 >= 0.0 && d.beta2 < 1.0)) return set_error(TFA_ERR_INVALID, "betas must be in [0, 1)");
  if (!(d.eps >= 0.0) || !std::isfinite(d.lr) || !std::isfinite(d.weight_decay)) return set_error(TFA_ERR_INVALID, "bad learning rate, eps or weight decay");
  for (int64_t i = 0; i < count; ++i) {
    const tfa_adam_tensor& t = tensors[i];
    if (t.n < 0) return set_error(TFA_ERR_INVALID, "negative size");
    if (t.n == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return set_error(TFA_ERR_INVALID, "null data pointer");
    if (d.state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) return set_error(TFA_ERR_INVALID, "8-bit states need their scales");
  }
  tfa::AdamArgs a{};
  a.p_dtype = d.param_dtype, a.g_dtype = d.grad_dtype, a.bits = d.state_bits;
  a.decay = (float)(1.0 - d.lr * d.weight_decay);
  a.beta1 = (float)d.beta1, a.one_beta1 = (float)(1.0 - d.beta1), a.beta2 = (float)d.beta2, a.one_beta2 = (float)(1.0 - d.beta2);
  a.step_size = (float)(d.lr / (1.0 - std::pow(d.beta1, (double)d.step)));
  a.inv_root_bc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(d.beta2, (double)d.step)));
  a.eps = (float)d.eps;
  static_assert(sizeof(tfa_adam_tensor) == sizeof(tfa::AdamTensor), "one layout");
  const hipError_t e = tfa::launch_adamw(reinterpret_cast<const tfa::AdamTensor*>(tensors), count, a, static_cast<hipStream_t>(stream));
  if (e == hipErrorInvalidValue) return set_error(TFA_ERR_UNSUPPORTED, "tensor beyond the launch grid");
  return launched(e);
}

int tfa_adamw_state_values(int64_t count, const tfa_code_tensor* tensors, int32_t squares, tfa_stream stream) {
  if (count < 0 || (count > 0 && !tensors)) return set_error(TFA_ERR_INVALID, "bad argument");
  for (int64_t i = 0; i < count; ++i) {
    if (tensors[i].n < 0) return set_error(TFA_ERR_INVALID, "negative size");
    if (tensors[i].n > 0 && (!tensors[i].codes || !tensors[i].scales || !tensors[i].out)) return set_error(TFA_ERR_INVALID, "null data pointer");
  }
  static_assert(sizeof(tfa_code_tensor) == sizeof(tfa::CodeTensor), "one layout");
  const hipError_t e = tfa::launch_adam_values(reinterpret_cast<const tfa::CodeTensor*>(tensors), count, squares != 0,
                                               static_cast<hipStream_t>(stream));
  if (e == hipErrorInvalidValue) return set_error(TFA_ERR_UNSUPPORTED, "tensor beyond the launch grid");
  return launched(e);
}

}  // extern "C"
