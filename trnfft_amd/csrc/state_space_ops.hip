// C entry points of the state space layer's operators and of gradient clipping (include/trnfft_amd.h): argument checks,
// workspaces, launches.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "../../include/trnfft_amd.h"
#include "model_ops.h"

using tfa::set_error;

namespace {

int launched(hipError_t e) { return e == hipSuccess ? TFA_OK : set_error(TFA_ERR_HIP, hipGetErrorString(e)); }

bool dtype_ok(int32_t d) { return d == TFA_DTYPE_F32 || d == TFA_DTYPE_BF16 || d == TFA_DTYPE_F16; }

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

// Sizes up to which no count of threads, values or bytes of a workspace passes 63 bits
constexpr int32_t kMostChannels = 1 << 20;
constexpr int64_t kMostBatch = 1 << 28, kMostTokens = INT32_MAX;
constexpr double kMostValues = 1LL << 44;

int check_sequence(int32_t dtype, int64_t batch, int64_t tokens, int32_t channels) {
  if (!dtype_ok(dtype)) return set_error(TFA_ERR_INVALID, "dtype must be TFA_DTYPE_F32, _BF16 or _F16");
  if (batch < 0 || tokens < 0) return set_error(TFA_ERR_INVALID, "negative dimension");
  if (channels < 1) return set_error(TFA_ERR_INVALID, "need at least one channel");
  if (channels > kMostChannels) return set_error(TFA_ERR_UNSUPPORTED, "more than 2^20 channels");
  if (batch > kMostBatch) return set_error(TFA_ERR_UNSUPPORTED, "more than 2^28 batch rows");
  if (tokens > kMostTokens) return set_error(TFA_ERR_UNSUPPORTED, "more than 2^31 tokens");
  if ((double)batch * (double)tokens * channels > kMostValues) return set_error(TFA_ERR_UNSUPPORTED, "more than 2^44 values");
  return TFA_OK;
}

int check_conv(const tfa_conv_desc* d) {
  if (!d) return set_error(TFA_ERR_INVALID, "null descriptor");
  if (const int rc = check_sequence(d->dtype, d->batch, d->tokens, d->channels)) return rc;
  if (d->width < 1) return set_error(TFA_ERR_INVALID, "need at least one tap");
  if (d->width > 8) return set_error(TFA_ERR_UNSUPPORTED, "filters of more than 8 taps are not implemented");
  if (d->activation < TFA_ACT_NONE || d->activation > TFA_ACT_RELU) return set_error(TFA_ERR_INVALID, "unknown activation");
  return TFA_OK;
}

tfa::ConvArgs conv_args(const tfa_conv_desc* d, const void* x, const float* weight, const float* bias, const int64_t* lengths,
                        const void* state_in, tfa_stream stream) {
  tfa::ConvArgs a{};
  a.dtype = d->dtype, a.channels = d->channels, a.width = d->width, a.act = d->activation;
  a.batch = d->batch, a.tokens = d->tokens;
  // (a stride along one row or token says nothing)
  a.x_sb = d->batch > 1 ? d->x_stride[0] : 0, a.x_st = d->tokens > 1 ? d->x_stride[1] : 0;
  a.x = x, a.weight = weight, a.bias = bias, a.state_in = d->width > 1 ? state_in : nullptr;
  a.lengths = reinterpret_cast<const long long*>(lengths);
  a.stream = static_cast<hipStream_t>(stream);
  return a;
}

int check_scan(const tfa_scan_desc* d) {
  if (!d) return set_error(TFA_ERR_INVALID, "null descriptor");
  if (const int rc = check_sequence(d->dtype, d->batch, d->tokens, d->channels)) return rc;
  if (d->groups < 1 || d->channels % d->groups) return set_error(TFA_ERR_INVALID, "channels must be a multiple of groups");
  if (d->states < 1) return set_error(TFA_ERR_INVALID, "need at least one state");
  if (d->states > tfa::kScanMostStates) return set_error(TFA_ERR_UNSUPPORTED, "more than 64 states are not implemented");
  return TFA_OK;
}

// A sequence is cut into segments where its rows and channels alone leave the vector units idle, at a cost: the segments' sums are 0.6 (forward)
// and 0.25 (backward) of the pass itself.  Forward below 1024 waves into segments that make about 4096, backward below 2048 into
// such that make 2048 (a wave takes half of a SIMD's registers there), at most 64 of at least 32 tokens, of sequences of at least 256.
// 16 states, bf16: 8 x 4096 tokens of 2048 channels (1024 waves) forward 400 us whole, 505 in 4 segments; backward 1340 whole, 1100 in 2,
// 1140 in 4.  1 x 65536 of 1024 (64 waves) 753 in 16, 544 in 32, 491 in 64.  1 x 16384 of 256 (16 waves) 83 in 64, 131 in 256.  1 x 1000 of 512
// 73 in 3, 40 in 7, 27 in 15, 24 in 31; 4 x 1001 of 384 in 15 and 31: forward 36 and 30, backward with its sums 54 and 40.  1 x 128 of 1024 21
// whole, 27 in 2.
// Where two waves take the same channels (scan_pairs.h) a token takes 0.1 us whole up to 1024 waves; segments take as much at 924, less in
// proportion to the waves below, and some 15 us for their launches: whole and in segments 7 x 4096 of 2048 (896 waves) 392 and 445, 6 rows (768)
// 381 and 354, 12 x 1024 of 1024 (768) 97 and 100, 16 x 300 of 512 (512) 27 and 34.
// Other numbers of states, bf16, forward and whole training passes (the backward's segments beside the rule's own forward), the rule's, then the
// best of 1, 2, 4 ... 64 segments: 4 states, 8 x 4096 of 1024 (512 waves) 144 and 503, 128 (in 32) and 466 (in 16); 2 x 4096 of 1024 (128) 47 and
// 150, 48 and 141; 1 x 65536 of 256 (16) 183 and 450, 184 and 449.  8 states, 1 x 16384 of 1024 (64) 97 and 320, 97 and 317.  32 states,
// 8 x 4096 of 512 (512) 229 and 784, 199 and 784; 1 x 1000 of 512 (64) 26 and 111, 26 and 110.  64 states, 8 x 4096 of 256 (512) 221 and
// 1043, 209 and 1041; 4 x 1001 of 384 (384) 55 and 261, 55 and 231 (in 8).  It does not fit where other numbers than 9 to 16 states make 1024 waves
// exactly: 8 x 4096 of 2048 whole 597 (4 states) and 551 (8), 283 and 327 in 16 segments; 8 x 4096 of 512 of 64 states 512, 383.
constexpr int64_t kForwardWaves = 1024, kForwardWant = 4096, kBackwardWaves = 2048, kBackwardWant = 2048;
constexpr int64_t kMostSegments = 64, kSegTokens = 32, kSplitTokens = 256;
// Sums of so few long segments are made in halves: 8 x 4096 of 2048, whose sums backwards are 1024 waves', 173 and 132 us.
constexpr int64_t kFineTokens = 512;  // of such a segment
constexpr int64_t kPairWaves = 924, kPairWork = 150000;  // tokens times the waves that are missing

tfa::ScanArgs scan_args(const tfa_scan_desc* d, bool backward) {
  tfa::ScanArgs p{};
  p.dtype = d->dtype, p.channels = d->channels, p.groups = d->groups, p.n = d->states;
  p.batch = d->batch, p.tokens = d->tokens, p.softplus = d->softplus != 0;
  p.segments = 1, p.fine = 1;
  p.seg_tokens = std::max<int64_t>(1, (d->tokens + tfa::kScanStretch - 1) / tfa::kScanStretch) * tfa::kScanStretch;
  if (d->batch == 0) return p;
  const int64_t waves = tfa::scan_waves(p);
  if (waves >= (backward ? kBackwardWaves : kForwardWaves) || d->tokens < kSplitTokens) return p;
  if (!backward && tfa::scan_has_pairs(p) && (waves >= kPairWaves || d->tokens <= kPairWork / (kPairWaves - waves))) return p;
  const int64_t want = std::min({((backward ? kBackwardWant : kForwardWant) + waves - 1) / waves, d->tokens / kSegTokens, kMostSegments});
  if (want > 1) {
    if (backward && waves * (want - 1) < kBackwardWant && d->tokens / want >= kFineTokens) p.fine = 2;
    const int64_t step = tfa::kScanStretch * p.fine;
    p.seg_tokens = ((d->tokens + want - 1) / want + step - 1) / step * step;
    p.segments = (int)((d->tokens + p.seg_tokens - 1) / p.seg_tokens);
  }
  return p;
}

struct ScanInputs {
  const void *x, *dt, *b, *c, *z;
  const float *a, *d, *dt_bias;
};
template <typename P>
void scan_inputs(P& p, const tfa_scan_desc* d, const ScanInputs& in) {
  const bool rows = d->batch > 1, groups = d->groups > 1;
  p.x = in.x, p.dt = in.dt, p.z = in.z, p.b = in.b, p.c = in.c, p.a = in.a, p.d = in.d, p.dt_bias = in.dt_bias;
  p.x_sb = rows ? d->x_stride[0] : 0, p.dt_sb = rows ? d->dt_stride[0] : 0, p.z_sb = rows ? d->z_stride[0] : 0;
  p.b_sb = rows ? d->b_stride[0] : 0, p.c_sb = rows ? d->c_stride[0] : 0;
  p.b_sg = groups ? d->b_stride[2] : 0, p.c_sg = groups ? d->c_stride[2] : 0;
}
// what the kernels read and write by 16 bytes
int check_aligned(const void* kept, const void* workspace) {
  if ((reinterpret_cast<uintptr_t>(kept) | reinterpret_cast<uintptr_t>(workspace)) % 16)
    return set_error(TFA_ERR_INVALID, "kept states and workspace must be 16-byte aligned");
  return TFA_OK;
}
// (a lane's own part of an address has 32 bits: tokens of a tile are less than 2^32 bytes apart)
int check_token_strides(const tfa_scan_desc* d) {
  if (d->tokens < 2) return TFA_OK;
  for (const int64_t st : {d->x_stride[1], d->dt_stride[1], d->z_stride[1], d->b_stride[1], d->c_stride[1], (int64_t)d->channels})
    if (st < 0 || st >= 1 << 24) return set_error(TFA_ERR_UNSUPPORTED, "token strides must be from 0 to 2^24 - 1 elements");
  return TFA_OK;
}
void scan_tokens(tfa::ScanArgs& p, const tfa_scan_desc* d) {
  const bool many = d->tokens > 1;
  p.x_st = many ? d->x_stride[1] : 0, p.dt_st = many ? d->dt_stride[1] : 0, p.z_st = many ? d->z_stride[1] : 0;
  p.b_st = many ? d->b_stride[1] : 0, p.c_st = many ? d->c_stride[1] : 0;
}

int check_grads(const tfa_grad_lists* g) {
  if (!g) return set_error(TFA_ERR_INVALID, "null lists");
  for (int d = 0; d < 3; ++d) {
    if (g->count[d] < 0 || (g->count[d] > 0 && !g->tensors[d])) return set_error(TFA_ERR_INVALID, "bad list");
    for (int64_t i = 0; i < g->count[d]; ++i) {
      if (g->tensors[d][i].n < 0) return set_error(TFA_ERR_INVALID, "negative size");
      if (g->tensors[d][i].n > 0 && !g->tensors[d][i].data) return set_error(TFA_ERR_INVALID, "null data pointer");
    }
  }
  return TFA_OK;
}

tfa::GradLists grad_lists(const tfa_grad_lists* g) {
  static_assert(sizeof(tfa_grad_tensor) == sizeof(tfa::GradTensor), "one layout");
  tfa::GradLists l;
  for (int d = 0; d < 3; ++d) {
    l.tensors[d] = reinterpret_cast<const tfa::GradTensor*>(g->tensors[d]);
    l.count[d] = g->count[d];
  }
  return l;
}

// whether two of the tensors share memory, which two workgroups would then scale
bool overlapping(const tfa_grad_lists* g) {
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  spans.reserve(g->count[0] + g->count[1] + g->count[2]);
  for (int d = 0; d < 3; ++d)
    for (int64_t i = 0; i < g->count[d]; ++i)
      if (g->tensors[d][i].n > 0) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(g->tensors[d][i].data);
        spans.emplace_back(at, at + (uintptr_t)g->tensors[d][i].n * (d == TFA_DTYPE_F32 ? 4 : 2));
      }
  if (!std::is_sorted(spans.begin(), spans.end())) std::sort(spans.begin(), spans.end());  // (as a model's gradients mostly lie, at a third of the time)
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return true;
  return false;
}

int grad_norm(const tfa_grad_lists* grads, float* norm, void* workspace, bool scale, double max_norm, tfa_stream stream) {
  if (!norm || !workspace) return set_error(TFA_ERR_INVALID, "null data pointer");
  if (reinterpret_cast<uintptr_t>(workspace) % 8) return set_error(TFA_ERR_INVALID, "the workspace must be 8-byte aligned");
  const hipError_t e = tfa::launch_grad_norm(grad_lists(grads), static_cast<double*>(workspace), norm, scale, max_norm,
                                             static_cast<hipStream_t>(stream));
  if (e == hipErrorInvalidValue) return set_error(TFA_ERR_UNSUPPORTED, "tensor beyond the launch grid");
  return launched(e);
}

}  // namespace

extern "C" {

int tfa_causal_conv(const tfa_conv_desc* desc, const void* x, const float* weight, const float* bias, const int64_t* lengths,
                    const void* state_in, void* y, void* state_out, tfa_stream stream) {
  if (const int rc = check_conv(desc)) return rc;
  if (desc->batch == 0) return TFA_OK;
  if (!weight || (desc->tokens > 0 && (!x || !y))) return set_error(TFA_ERR_INVALID, "null data pointer");
  tfa::ConvArgs a = conv_args(desc, x, weight, bias, lengths, state_in, stream);
  if (state_out && state_out == state_in) return set_error(TFA_ERR_INVALID, "state_out must not be state_in");
  a.y = y, a.state_out = desc->width > 1 ? state_out : nullptr;
  if (desc->tokens == 0 && !a.state_out) return TFA_OK;
  return launched(tfa::launch_conv_forward(a));
}

int tfa_causal_conv_workspace_size(const tfa_conv_desc* desc, size_t* bytes) {
  if (!bytes) return set_error(TFA_ERR_INVALID, "null bytes pointer");
  *bytes = 0;
  if (const int rc = check_conv(desc)) return rc;
  *bytes = tfa::conv_workspace_bytes(conv_args(desc, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr));
  return TFA_OK;
}

int tfa_causal_conv_backward(const tfa_conv_desc* desc, const void* x, const float* weight, const float* bias,
                             const int64_t* lengths, const void* state_in, const void* grad_y, const void* grad_state_out,
                             void* grad_x, float* grad_weight, float* grad_bias, void* grad_state_in, void* workspace,
                             tfa_stream stream) {
  if (const int rc = check_conv(desc)) return rc;
  if (desc->batch > 0 && (!weight || (desc->tokens > 0 && (!x || !grad_y)))) return set_error(TFA_ERR_INVALID, "null data pointer");
  tfa::ConvArgs a = conv_args(desc, x, weight, bias, lengths, state_in, stream);
  if ((grad_weight || grad_bias) && !workspace && tfa::conv_workspace_bytes(a)) return set_error(TFA_ERR_INVALID, "null workspace");
  if (grad_state_in && grad_state_in == grad_state_out) return set_error(TFA_ERR_INVALID, "grad_state_in must not be grad_state_out");
  a.dy = grad_y, a.dx = grad_x, a.dweight = grad_weight, a.dbias = grad_bias;
  if (desc->width > 1) a.dstate_out = grad_state_out, a.dstate_in = grad_state_in;
  a.ws = static_cast<float*>(workspace);
  return launched(tfa::launch_conv_backward(a));
}

int tfa_causal_conv_step(const tfa_conv_desc* desc, const void* x, const float* weight, const float* bias, void* state, void* y,
                         tfa_stream stream) {
  if (const int rc = check_conv(desc)) return rc;
  if (desc->tokens != 1) return set_error(TFA_ERR_INVALID, "a step is one token");
  if (desc->batch == 0) return TFA_OK;
  if (!x || !weight || !y || (!state && desc->width > 1)) return set_error(TFA_ERR_INVALID, "null data pointer");
  tfa::ConvArgs a = conv_args(desc, x, weight, bias, nullptr, nullptr, stream);
  a.y = y, a.state_out = state;
  return launched(tfa::launch_conv_step(a));
}

// ------------------------------------------------------------------------------------------------

int tfa_selective_scan_sizes(const tfa_scan_desc* desc, size_t* kept, size_t* workspace, size_t* backward_workspace) {
  if (!kept || !workspace || !backward_workspace) return set_error(TFA_ERR_INVALID, "null bytes pointer");
  *kept = *workspace = *backward_workspace = 0;
  if (const int rc = check_scan(desc)) return rc;
  const tfa::ScanSizes f = tfa::scan_sizes(scan_args(desc, false)), b = tfa::scan_sizes(scan_args(desc, true));
  *kept = f.kept;
  *workspace = align256(f.seg_state) + align256(f.seg_steps);
  *backward_workspace = align256(b.seg_state) + align256(b.seg_steps) + align256(b.channel_parts) + (desc->bc_fixed ? 0 : align256(b.shared_parts));
  return TFA_OK;
}

int tfa_selective_scan(const tfa_scan_desc* desc, const void* x, const void* dt, const float* a, const void* b, const void* c,
                       const float* d, const void* z, const float* dt_bias, const int64_t* lengths, const float* state_in,
                       void* y, float* state_out, void* kept, void* workspace, tfa_stream stream) {
  if (const int rc = check_scan(desc)) return rc;
  if (const int rc = check_token_strides(desc)) return rc;
  if (desc->batch == 0) return TFA_OK;
  if (!a || (desc->tokens > 0 && (!x || !dt || !b || !c || !y))) return set_error(TFA_ERR_INVALID, "null data pointer");
  if (state_out && state_out == state_in) return set_error(TFA_ERR_INVALID, "state_out must not be state_in");
  tfa::ScanArgs p = scan_args(desc, false);
  scan_inputs(p, desc, {x, dt, b, c, z, a, d, dt_bias});
  scan_tokens(p, desc);
  const tfa::ScanSizes size = tfa::scan_sizes(p);
  if (size.seg_state && !workspace) return set_error(TFA_ERR_INVALID, "null workspace");
  if (const int rc = check_aligned(kept, workspace)) return rc;
  p.lengths = reinterpret_cast<const long long*>(lengths);
  p.state_in = state_in, p.state_out = state_out, p.y = y;
  p.kept = size.kept ? static_cast<float*>(kept) : nullptr;
  p.seg_state = static_cast<float*>(workspace);
  p.seg_steps = reinterpret_cast<float*>(static_cast<char*>(workspace) + align256(size.seg_state));
  p.stream = static_cast<hipStream_t>(stream);
  return launched(tfa::launch_scan_forward(p));
}

int tfa_selective_scan_backward(const tfa_scan_desc* desc, const void* x, const void* dt, const float* a, const void* b,
                                const void* c, const float* d, const void* z, const float* dt_bias, const int64_t* lengths,
                                const float* state_in, const void* kept, const tfa_scan_grads* grads, void* workspace,
                                tfa_stream stream) {
  if (const int rc = check_scan(desc)) return rc;
  if (const int rc = check_token_strides(desc)) return rc;
  if (!grads) return set_error(TFA_ERR_INVALID, "null gradients");
  const tfa_scan_grads& g = *grads;
  const bool some = desc->batch > 0 && desc->tokens > 0;
  if (desc->batch > 0 && !a) return set_error(TFA_ERR_INVALID, "null data pointer");
  if (some && (!x || !dt || !b || !c || !g.grad_y)) return set_error(TFA_ERR_INVALID, "null data pointer");
  if (g.z && !z) return set_error(TFA_ERR_INVALID, "no gate, no gradient of one");
  if (desc->bc_fixed && (g.b || g.c)) return set_error(TFA_ERR_INVALID, "bc_fixed leaves no room for gradients of b and c");
  if (g.state_in && g.state_in == g.grad_state_out) return set_error(TFA_ERR_INVALID, "the states' gradients must not be one");
  tfa::ScanArgs p = scan_args(desc, true);
  scan_inputs(p, desc, {x, dt, b, c, z, a, d, dt_bias});
  scan_tokens(p, desc);
  const tfa::ScanSizes size = tfa::scan_sizes(p);
  if (size.kept && !kept) return set_error(TFA_ERR_INVALID, "the forward's states are needed");
  if (!workspace && size.seg_state + size.channel_parts + (desc->bc_fixed ? 0 : size.shared_parts)) return set_error(TFA_ERR_INVALID, "null workspace");
  if (const int rc = check_aligned(kept, workspace)) return rc;
  p.lengths = reinterpret_cast<const long long*>(lengths);
  p.state_in = state_in, p.kept = static_cast<float*>(const_cast<void*>(kept));
  p.dy = g.grad_y, p.dstate_out = g.grad_state_out;
  p.dx = g.x, p.ddt = g.dt, p.dz = g.z, p.db = g.b, p.dc = g.c;
  p.da = g.a, p.dd = g.d, p.ddt_bias = g.dt_bias, p.dstate_in = g.state_in;
  char* space = static_cast<char*>(workspace);
  p.seg_state = reinterpret_cast<float*>(space), space += align256(size.seg_state);
  p.seg_steps = reinterpret_cast<float*>(space), space += align256(size.seg_steps);
  if (g.a || g.d || g.dt_bias) p.channel_parts = reinterpret_cast<float*>(space);
  space += align256(size.channel_parts);
  if (g.b || g.c) p.shared_parts = reinterpret_cast<float*>(space);
  p.stream = static_cast<hipStream_t>(stream);
  return launched(tfa::launch_scan_backward(p));
}

int tfa_selective_scan_step(const tfa_scan_desc* desc, const void* x, const void* dt, const float* a, const void* b,
                            const void* c, const float* d, const void* z, const float* dt_bias, float* state, void* y,
                            tfa_stream stream) {
  if (const int rc = check_scan(desc)) return rc;
  if (desc->tokens != 1) return set_error(TFA_ERR_INVALID, "a step is one token");
  if (desc->batch == 0) return TFA_OK;
  if (!x || !dt || !a || !b || !c || !state || !y) return set_error(TFA_ERR_INVALID, "null data pointer");
  tfa::ScanStep p{};
  scan_inputs(p, desc, {x, dt, b, c, z, a, d, dt_bias});
  p.dtype = desc->dtype, p.channels = desc->channels, p.groups = desc->groups, p.n = desc->states;
  p.batch = desc->batch, p.softplus = desc->softplus != 0, p.state = state, p.y = y;
  p.stream = static_cast<hipStream_t>(stream);
  return launched(tfa::launch_scan_step(p));
}

// ------------------------------------------------------------------------------------------------

int tfa_grad_norm_workspace_size(const tfa_grad_lists* grads, size_t* bytes) {
  if (!bytes) return set_error(TFA_ERR_INVALID, "null bytes pointer");
  *bytes = 0;
  if (const int rc = check_grads(grads)) return rc;
  *bytes = (size_t)tfa::grad_parts(grad_lists(grads)) * sizeof(double);
  return TFA_OK;
}

int tfa_grad_norm(const tfa_grad_lists* grads, float* norm, void* workspace, tfa_stream stream) {
  if (const int rc = check_grads(grads)) return rc;
  return grad_norm(grads, norm, workspace, false, 0.0, stream);
}

int tfa_clip_grads(const tfa_grad_lists* grads, double max_norm, float* norm, void* workspace, tfa_stream stream) {
  if (const int rc = check_grads(grads)) return rc;
  if (!(max_norm >= 0.0)) return set_error(TFA_ERR_INVALID, "max_norm must not be negative");
  try {
    if (overlapping(grads)) return set_error(TFA_ERR_INVALID, "tensors must not overlap");
  } catch (const std::bad_alloc&) {
    return set_error(TFA_ERR_HIP, "out of host memory");
  }
  return grad_norm(grads, norm, workspace, true, max_norm, stream);
}

}  // extern "C"
