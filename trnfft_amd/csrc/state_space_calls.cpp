// The host's side of the state space operators (trnfft_amd/state_space.py) where their questions to tensors, or a passage through Python
// on autograd's thread, would take longer than their work on the GPU.
//
// Steps of streams: where every operand is as the C ABI takes it, the call is made from here; asked from Python nine tensors cost 8 of the
// 13.8 us of a small scan's step.  Anything else is left to Python, which converts or refuses it: filters, biases, d and dt_bias of 16 bits are
// converted to fp32 by a launch each (1 x 1024: convolution's step 20.5 us for 5.2, scan's 24.5 for 5.3).
//
// Whole sequences likewise (a scan takes 15 us of the host from Python, 7.6 from here), and their nodes of autograd's graph: a backward
// pass in Python took 70 us on autograd's thread, which had to wake up for it and to take Python's lock; a small training pass of the scan takes
// 123 us of the host instead of 218 (a layer norm's: 66).
#include <Python.h>

#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include "../../include/trnfft_amd.h"

#include <cstdint>
#include <exception>
#include <iterator>
#include <optional>
#include <tuple>
#include <unordered_set>
#include <vector>

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The C ABI's entries, which Python has loaded.
struct Entries {
  decltype(&tfa_causal_conv) conv;
  decltype(&tfa_causal_conv_workspace_size) conv_size;
  decltype(&tfa_causal_conv_backward) conv_backward;
  decltype(&tfa_causal_conv_step) conv_step;
  decltype(&tfa_selective_scan_sizes) scan_sizes;
  decltype(&tfa_selective_scan) scan;
  decltype(&tfa_selective_scan_backward) scan_backward;
  decltype(&tfa_selective_scan_step) scan_step;
  decltype(&tfa_last_error) last_error;
} entries;

// A status of the C ABI: of a forward call it is returned to Python, which raises the exception that belongs to it.
struct Refused {
  int rc;
};
void run(int rc) {
  if (rc) throw Refused{rc};
}
void run_backward(int rc, const char* what) { TORCH_CHECK(rc == TFA_OK, what, " backward: ", entries.last_error()); }

tfa_stream stream_of(int64_t device) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }

int dtype_of(at::ScalarType t) {
  return t == at::kFloat ? TFA_DTYPE_F32 : t == at::kBFloat16 ? TFA_DTYPE_BF16 : t == at::kHalf ? TFA_DTYPE_F16 : -1;
}
void* data(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* floats(const at::Tensor& t) { return static_cast<float*>(data(t)); }
int64_t* whole_numbers(const at::Tensor& t) { return static_cast<int64_t*>(data(t)); }
at::Tensor bytes_like(const at::Tensor& x, size_t n) { return n ? at::empty({(int64_t)n}, x.options().dtype(at::kByte)) : at::Tensor(); }
typedef std::optional<at::Tensor> Optional;
Optional optional_of(const at::Tensor& t) { return t.defined() ? Optional(t) : std::nullopt; }
at::Tensor tensor_of(const Optional& t) { return t ? *t : at::Tensor(); }
at::Tensor dense(const at::Tensor& g) { return g.defined() ? g.resolve_neg().contiguous() : g; }

// ------------------------------------------------------------------------------------------------
// nodes of the graph
// ------------------------------------------------------------------------------------------------

// A gradient that must not be differentiated again: a graph through it ends here.
struct Once : torch::autograd::Function<Once> {
  static at::Tensor forward(AutogradContext*, const at::Tensor& g) { return g.alias(); }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "trying to differentiate twice through causal_conv or selective_scan, whose gradients are once_differentiable");
  }
};
variable_list once(variable_list grads) {
  if (c10::GradMode::is_enabled()) {
    for (at::Tensor& g : grads)
      if (g.defined()) g = Once::apply(g.requires_grad_());
  }
  return grads;
}

// A leaf's gradients go to a node that belongs to the stream on which the leaf was first used, for as long as any graph with it lives.
// A backward pass that is captured cannot reach one of the default stream: the attempt ends the process.  So a captured call refuses to
// become part of such a graph.
void refuse_eager_graphs(const at::Tensor* tensors, size_t count) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  std::vector<std::shared_ptr<torch::autograd::Node>> todo;
  std::unordered_set<torch::autograd::Node*> seen;
  const auto add = [&](const std::shared_ptr<torch::autograd::Node>& node) {
    if (node && seen.insert(node.get()).second) todo.push_back(node);
  };
  for (size_t i = 0; i < count; ++i)
    if (tensors[i].defined() && tensors[i].requires_grad())
      add(tensors[i].grad_fn() ? tensors[i].grad_fn() : torch::autograd::impl::try_get_grad_accumulator(tensors[i]));
  while (!todo.empty()) {
    const auto node = todo.back();
    todo.pop_back();
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(node.get())) {
      const auto stream = node->stream();
      TORCH_CHECK(!stream || stream->id() != c10::hip::getDefaultHIPStream(stream->device_index()).id(),
                  "a graph of an eager pass through these tensors lives: delete its results before a pass through them is captured");
    }
    for (const auto& edge : node->next_edges()) add(edge.function);
  }
}

// Room for the gradients of the first N of a node's operands, where they are wanted (operands that were left out have no edge in the graph).
void make_grads(AutogradContext* ctx, const variable_list& saved, size_t n, variable_list& grads) {
  size_t edge = 0;
  for (size_t i = 0; i < n; ++i)
    if (saved[i].defined() && ctx->needs_input_grad(edge++)) grads[i] = at::empty(saved[i].sizes(), saved[i].options());
}

tfa_conv_desc conv_desc(const at::Tensor& x, const at::Tensor& weight, int64_t activation) {
  tfa_conv_desc d{};
  d.dtype = dtype_of(x.scalar_type()), d.channels = (int32_t)x.size(2), d.width = (int32_t)weight.size(1), d.activation = (int32_t)activation;
  d.batch = x.size(0), d.tokens = x.size(1), d.x_stride[0] = x.stride(0), d.x_stride[1] = x.stride(1);
  return d;
}

// y, and the state after each row's last frame where it is wanted
variable_list conv_forward(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, const at::Tensor& state, const at::Tensor& lengths,
                           int64_t activation, bool want_state) {
  const c10::DeviceGuard guard(x.device());
  const tfa_conv_desc desc = conv_desc(x, weight, activation);
  variable_list out{at::empty(x.sizes(), x.options())};
  if (want_state) out.push_back(at::empty({x.size(0), weight.size(1) - 1, x.size(2)}, x.options()));
  run(entries.conv(&desc, data(x), floats(weight), floats(bias), whole_numbers(lengths), data(state), data(out[0]),
                   want_state ? data(out[1]) : nullptr, stream_of(x.get_device())));
  return out;
}

struct ConvFn : torch::autograd::Function<ConvFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const Optional& given_bias,
                               const Optional& given_state, const Optional& given_lengths, int64_t activation, bool want_state) {
    const at::Tensor bias = tensor_of(given_bias), state = tensor_of(given_state), lengths = tensor_of(given_lengths);
    ctx->set_materialize_grads(false);
    ctx->saved_data["activation"] = activation;
    ctx->save_for_backward({x, weight, bias, state, lengths});
    return conv_forward(x, weight, bias, state, lengths, activation, want_state);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list grads(7);
    {
      const at::NoGradGuard no_grad;
      const variable_list saved = ctx->get_saved_variables();
      const at::Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &state = saved[3], &lengths = saved[4];
      const c10::DeviceGuard guard(x.device());
      const tfa_conv_desc desc = conv_desc(x, weight, ctx->saved_data["activation"].toInt());
      make_grads(ctx, saved, 4, grads);
      const at::Tensor dy = g[0].defined() ? dense(g[0]) : at::zeros(x.sizes(), x.options()), dlast = g.size() > 1 ? dense(g[1]) : at::Tensor();
      at::Tensor workspace;
      if (grads[1].defined() || grads[2].defined()) {
        size_t n = 0;
        run_backward(entries.conv_size(&desc, &n), "causal_conv");
        workspace = bytes_like(x, n);
      }
      run_backward(entries.conv_backward(&desc, data(x), floats(weight), floats(bias), whole_numbers(lengths), data(state), data(dy), data(dlast),
                                         data(grads[0]), floats(grads[1]), floats(grads[2]), data(grads[3]), data(workspace),
                                         stream_of(x.get_device())),
                   "causal_conv");
    }
    return once(std::move(grads));
  }
};

tfa_scan_desc scan_desc(const at::Tensor& x, const at::Tensor& dt, const at::Tensor& a, const at::Tensor& b, const at::Tensor& c, const at::Tensor& z,
                        bool softplus) {
  tfa_scan_desc d{};
  d.dtype = dtype_of(x.scalar_type()), d.channels = (int32_t)x.size(2), d.groups = (int32_t)b.size(2), d.states = (int32_t)a.size(1);
  d.softplus = softplus, d.batch = x.size(0), d.tokens = x.size(1);
  for (int i = 0; i < 2; ++i) d.x_stride[i] = x.stride(i), d.dt_stride[i] = dt.stride(i), d.z_stride[i] = z.defined() ? z.stride(i) : 0;
  for (int i = 0; i < 3; ++i) d.b_stride[i] = b.stride(i), d.c_stride[i] = c.stride(i);
  return d;
}

// y, the state after each row's last frame where it is wanted, and what a backward pass needs of this one
std::tuple<variable_list, at::Tensor> scan_forward(const at::Tensor& x, const at::Tensor& dt, const at::Tensor& a, const at::Tensor& b,
                                                   const at::Tensor& c, const at::Tensor& d, const at::Tensor& z, const at::Tensor& bias,
                                                   const at::Tensor& state, const at::Tensor& lengths, bool softplus, bool want_state, bool want_kept) {
  const c10::DeviceGuard guard(x.device());
  const tfa_scan_desc desc = scan_desc(x, dt, a, b, c, z, softplus);
  size_t kept_size = 0, size = 0, backward_size = 0;
  run(entries.scan_sizes(&desc, &kept_size, &size, &backward_size));
  const at::Tensor kept = bytes_like(x, want_kept ? kept_size : 0), workspace = bytes_like(x, size);
  variable_list out{at::empty(x.sizes(), x.options())};
  if (want_state) out.push_back(at::empty({x.size(0), a.size(0), a.size(1)}, a.options()));
  run(entries.scan(&desc, data(x), data(dt), floats(a), data(b), data(c), floats(d), data(z), floats(bias), whole_numbers(lengths), floats(state),
                   data(out[0]), want_state ? floats(out[1]) : nullptr, data(kept), data(workspace), stream_of(x.get_device())));
  return {std::move(out), kept};
}

struct ScanFn : torch::autograd::Function<ScanFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& dt, const at::Tensor& a, const at::Tensor& b,
                               const at::Tensor& c, const Optional& given_d, const Optional& given_z, const Optional& given_bias,
                               const Optional& given_state, const Optional& given_lengths, bool softplus, bool want_state) {
    const at::Tensor d = tensor_of(given_d), z = tensor_of(given_z), bias = tensor_of(given_bias), state = tensor_of(given_state),
                     lengths = tensor_of(given_lengths);
    ctx->set_materialize_grads(false);
    ctx->saved_data["softplus"] = softplus;
    auto [out, kept] = scan_forward(x, dt, a, b, c, d, z, bias, state, lengths, softplus, want_state, true);
    ctx->save_for_backward({x, dt, a, b, c, d, z, bias, state, lengths, kept});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list grads(12);
    {
      const at::NoGradGuard no_grad;
      const variable_list saved = ctx->get_saved_variables();
      const at::Tensor &x = saved[0], &dt = saved[1], &a = saved[2], &b = saved[3], &c = saved[4], &d = saved[5], &z = saved[6], &bias = saved[7],
                       &state = saved[8], &lengths = saved[9], &kept = saved[10];
      const c10::DeviceGuard guard(x.device());
      tfa_scan_desc desc = scan_desc(x, dt, a, b, c, z, ctx->saved_data["softplus"].toBool());
      make_grads(ctx, saved, 9, grads);
      desc.bc_fixed = !grads[3].defined() && !grads[4].defined();
      size_t kept_size = 0, forward_size = 0, size = 0;
      run_backward(entries.scan_sizes(&desc, &kept_size, &forward_size, &size), "selective_scan");
      const at::Tensor workspace = bytes_like(x, size);
      const at::Tensor dy = g[0].defined() ? dense(g[0]) : at::zeros(x.sizes(), x.options()), dlast = g.size() > 1 ? dense(g[1]) : at::Tensor();
      tfa_scan_grads out{};
      out.grad_y = data(dy), out.grad_state_out = floats(dlast);
      out.x = data(grads[0]), out.dt = data(grads[1]), out.a = floats(grads[2]), out.b = data(grads[3]), out.c = data(grads[4]);
      out.d = floats(grads[5]), out.z = data(grads[6]), out.dt_bias = floats(grads[7]), out.state_in = floats(grads[8]);
      run_backward(entries.scan_backward(&desc, data(x), data(dt), floats(a), data(b), data(c), floats(d), data(z), floats(bias),
                                         whole_numbers(lengths), floats(state), data(kept), &out, data(workspace), stream_of(x.get_device())),
                   "selective_scan");
    }
    return once(std::move(grads));
  }
};

// ------------------------------------------------------------------------------------------------
// calls from Python
// ------------------------------------------------------------------------------------------------

const char kBindDoc[] = "bind(addresses): the C ABI's entries in the order of ENTRIES.";
const char kConvDoc[] =
    "causal_conv(x, weight, bias, state, lengths, activation, want_state, checked) -> y or (y, last), an error's status, or None where operands\n"
    "that are not checked are not as the C ABI takes them.";
const char kScanDoc[] =
    "selective_scan(x, dt, a, b, c, d, z, dt_bias, state, lengths, softplus, want_state, checked) -> y or (y, last), an error's status, or\n"
    "None, as causal_conv.";
const char kConvStepDoc[] =
    "conv_step(device, x, state, weight, bias, activation) -> y, an error's status, or None where an operand is not as the C ABI takes it\n"
    "(or needs a gradient).";
const char kScanStepDoc[] = "scan_step(device, x, dt, a, b, c, state, d, z, dt_bias, softplus) -> y, an error's status, or None, as conv_step.";

constexpr const char* kEntries[] = {"tfa_causal_conv",          "tfa_causal_conv_workspace_size", "tfa_causal_conv_backward",
                                    "tfa_causal_conv_step",     "tfa_selective_scan_sizes",       "tfa_selective_scan",
                                    "tfa_selective_scan_backward", "tfa_selective_scan_step",     "tfa_last_error"};

PyObject* bind_of(PyObject* args) {
  unsigned long long p[9];
  if (!PyArg_ParseTuple(args, "KKKKKKKKK", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, p + 7, p + 8)) return nullptr;
  static_assert(sizeof(Entries) == 9 * sizeof(void*) && sizeof(kEntries) == sizeof(Entries));
  entries = Entries{reinterpret_cast<decltype(entries.conv)>(p[0]),          reinterpret_cast<decltype(entries.conv_size)>(p[1]),
                    reinterpret_cast<decltype(entries.conv_backward)>(p[2]), reinterpret_cast<decltype(entries.conv_step)>(p[3]),
                    reinterpret_cast<decltype(entries.scan_sizes)>(p[4]),    reinterpret_cast<decltype(entries.scan)>(p[5]),
                    reinterpret_cast<decltype(entries.scan_backward)>(p[6]), reinterpret_cast<decltype(entries.scan_step)>(p[7]),
                    reinterpret_cast<decltype(entries.last_error)>(p[8])};
  Py_RETURN_NONE;
}

struct WithoutGil {
  PyThreadState* const state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

// The tensor of an argument; None gives an undefined one.
at::Tensor argument(PyObject* o) {
  if (o == Py_None) return at::Tensor();
  TORCH_CHECK(THPVariable_Check(o), "a tensor or None expected");
  return THPVariable_Unpack(o);
}

// A tensor of the device with contiguous last axis, which (grads) needs no gradient; None gives an undefined one where it may be left out.
struct Operand {
  const at::Tensor* t = nullptr;
  bool good = false;
  Operand(PyObject* o, int64_t device, bool grads, bool optional = false) {
    if (o == Py_None) {
      good = optional;
      return;
    }
    if (!THPVariable_CheckExact(o) && !THPVariable_Check(o)) return;
    const at::Tensor& v = THPVariable_Unpack(o);
    if (!v.defined() || v.layout() != at::kStrided || !v.is_cuda() || v.get_device() != device || v.is_neg() || (grads && v.requires_grad())) return;
    if (v.dim() < 1 || v.dim() > 4 || (v.size(v.dim() - 1) != 1 && v.stride(v.dim() - 1) != 1)) return;
    t = &v;
    good = true;
  }
  bool is(at::ScalarType type, std::initializer_list<int64_t> sizes) const { return !t || (t->scalar_type() == type && t->sizes() == at::IntArrayRef(sizes)); }
  bool whole(at::ScalarType type, std::initializer_list<int64_t> sizes) const { return !t || (is(type, sizes) && t->is_contiguous()); }
  at::Tensor tensor() const { return t ? *t : at::Tensor(); }
};

PyObject* none() { Py_RETURN_NONE; }

// y, or y and the last state
PyObject* result_of(const variable_list& v) {
  PyObject* const y = THPVariable_Wrap(v[0]);
  if (!y || v.size() == 1) return y;
  PyObject* const last = THPVariable_Wrap(v[1]);
  PyObject* const both = last ? PyTuple_Pack(2, y, last) : nullptr;
  Py_DECREF(y);
  Py_XDECREF(last);
  return both;
}

bool want_gradients(const at::Tensor* t, size_t count) {
  if (c10::GradMode::is_enabled())
    for (size_t i = 0; i < count; ++i)
      if (t[i].defined() && t[i].requires_grad()) return true;
  return false;
}
// a sequence's operand whose frames are as close as the kernels' addresses take them
bool close_frames(const Operand& o) { return !o.t || o.t->size(1) < 2 || (o.t->stride(1) >= 0 && o.t->stride(1) < 1 << 24); }

// Whole sequences: operands x, weight, bias, state and lengths.  `checked`: by Python, which has made them what the C ABI takes; else they are left
// to it unless they are so already.
PyObject* conv_of(PyObject* args) {
  PyObject* o[5];
  int activation, want_state, checked;
  if (!PyArg_ParseTuple(args, "OOOOOipp", o, o + 1, o + 2, o + 3, o + 4, &activation, &want_state, &checked)) return nullptr;
  if (!checked) {
    if (!THPVariable_Check(o[0])) return none();
    const int64_t device = THPVariable_Unpack(o[0]).get_device();
    const Operand x(o[0], device, false), weight(o[1], device, false), bias(o[2], device, false, true), state(o[3], device, false, true),
        lengths(o[4], device, false, true);
    for (const Operand* v : {&x, &weight, &bias, &state, &lengths})
      if (!v->good) return none();
    if (x.t->dim() != 3 || weight.t->dim() != 2 || !close_frames(x)) return none();
    const at::ScalarType type = x.t->scalar_type();
    const int64_t b = x.t->size(0), c = x.t->size(2), width = weight.t->size(1);
    if (dtype_of(type) < 0 || c < 1 || width < 1 || c > INT32_MAX || width > INT32_MAX) return none();
    if (!weight.whole(at::kFloat, {c, width}) || !bias.whole(at::kFloat, {c}) || !state.whole(type, {b, width - 1, c}) ||
        !lengths.whole(at::kLong, {b}))
      return none();
  }
  at::Tensor t[5];
  for (int i = 0; i < 5; ++i) t[i] = argument(o[i]);
  const bool grads = want_gradients(t, 4);
  if (grads) refuse_eager_graphs(t, 4);
  variable_list out;
  {
    const WithoutGil released;
    out = grads ? ConvFn::apply(t[0], t[1], optional_of(t[2]), optional_of(t[3]), optional_of(t[4]), (int64_t)activation, (bool)want_state)
                : conv_forward(t[0], t[1], t[2], t[3], t[4], activation, want_state);
  }
  return result_of(out);
}

// as conv_of: x, dt, a, b, c, d, z, dt_bias, state and lengths
PyObject* scan_of(PyObject* args) {
  PyObject* o[10];
  int softplus, want_state, checked;
  if (!PyArg_ParseTuple(args, "OOOOOOOOOOppp", o, o + 1, o + 2, o + 3, o + 4, o + 5, o + 6, o + 7, o + 8, o + 9, &softplus, &want_state, &checked))
    return nullptr;
  if (!checked) {
    if (!THPVariable_Check(o[0])) return none();
    const int64_t device = THPVariable_Unpack(o[0]).get_device();
    const Operand x(o[0], device, false), dt(o[1], device, false), a(o[2], device, false), b(o[3], device, false), c(o[4], device, false),
        d(o[5], device, false, true), z(o[6], device, false, true), bias(o[7], device, false, true), state(o[8], device, false, true),
        lengths(o[9], device, false, true);
    for (const Operand* v : {&x, &dt, &a, &b, &c, &d, &z, &bias, &state, &lengths})
      if (!v->good) return none();
    if (x.t->dim() != 3 || a.t->dim() != 2 || b.t->dim() != 4) return none();
    const at::ScalarType type = x.t->scalar_type();
    const int64_t rows = x.t->size(0), tokens = x.t->size(1), channels = x.t->size(2), n = a.t->size(1), groups = b.t->size(2);
    if (dtype_of(type) < 0 || channels < 1 || n < 1 || groups < 1 || channels % groups || channels > INT32_MAX || n > INT32_MAX) return none();
    if (!dt.is(type, {rows, tokens, channels}) || !z.is(type, {rows, tokens, channels}) || !b.is(type, {rows, tokens, groups, n}) ||
        !c.is(type, {rows, tokens, groups, n}))
      return none();
    for (const Operand* v : {&x, &dt, &b, &c, &z})
      if (!close_frames(*v)) return none();
    if (!a.whole(at::kFloat, {channels, n}) || !d.whole(at::kFloat, {channels}) || !bias.whole(at::kFloat, {channels}) ||
        !state.whole(at::kFloat, {rows, channels, n}) || !lengths.whole(at::kLong, {rows}))
      return none();
  }
  at::Tensor t[10];
  for (int i = 0; i < 10; ++i) t[i] = argument(o[i]);
  const bool grads = want_gradients(t, 9);
  if (grads) refuse_eager_graphs(t, 9);
  variable_list out;
  {
    const WithoutGil released;
    if (grads)
      out = ScanFn::apply(t[0], t[1], t[2], t[3], t[4], optional_of(t[5]), optional_of(t[6]), optional_of(t[7]), optional_of(t[8]),
                          optional_of(t[9]), (bool)softplus, (bool)want_state);
    else
      out = std::get<0>(scan_forward(t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], t[9], softplus, want_state, false));
  }
  return result_of(out);
}

// y where the call went well, its status otherwise; the state has changed
PyObject* stepped(int rc, const at::Tensor& y, const at::Tensor& state) {
  if (rc) return PyLong_FromLong(rc);
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return THPVariable_Wrap(y);
}

PyObject* conv_step_of(PyObject* args) {
  PyObject *ox, *ostate, *oweight, *obias;
  long long device;
  int activation;
  if (!PyArg_ParseTuple(args, "LOOOOi", &device, &ox, &ostate, &oweight, &obias, &activation)) return nullptr;
  const bool grads = c10::GradMode::is_enabled();
  const Operand x(ox, device, grads), state(ostate, device, grads), weight(oweight, device, grads), bias(obias, device, grads, true);
  if (!x.good || !state.good || !weight.good || !bias.good || x.t->dim() != 2 || weight.t->dim() != 2) return none();
  const at::ScalarType type = x.t->scalar_type();
  const int64_t b = x.t->size(0), c = x.t->size(1), width = weight.t->size(1);
  if (dtype_of(type) < 0 || c < 1 || width < 1 || c > INT32_MAX || width > INT32_MAX) return none();
  if (!weight.whole(at::kFloat, {c, width}) || !bias.whole(at::kFloat, {c}) || !state.whole(type, {b, width - 1, c})) return none();
  tfa_conv_desc desc{};
  desc.dtype = dtype_of(type), desc.channels = (int32_t)c, desc.width = (int32_t)width, desc.activation = activation;
  desc.batch = b, desc.tokens = 1, desc.x_stride[0] = x.t->stride(0);
  const at::Tensor y = at::empty({b, c}, x.t->options());
  return stepped(entries.conv_step(&desc, data(*x.t), floats(*weight.t), floats(bias.tensor()), data(*state.t), data(y), stream_of(device)), y, *state.t);
}

PyObject* scan_step_of(PyObject* args) {
  PyObject *ox, *odt, *oa, *ob, *oc, *ostate, *od, *oz, *obias;
  long long device;
  int soft;
  if (!PyArg_ParseTuple(args, "LOOOOOOOOOp", &device, &ox, &odt, &oa, &ob, &oc, &ostate, &od, &oz, &obias, &soft)) return nullptr;
  const bool grads = c10::GradMode::is_enabled();
  const Operand x(ox, device, grads), dt(odt, device, grads), a(oa, device, grads), b(ob, device, grads), c(oc, device, grads);
  const Operand state(ostate, device, grads), d(od, device, grads, true), z(oz, device, grads, true), bias(obias, device, grads, true);
  for (const Operand* o : {&x, &dt, &a, &b, &c, &state, &d, &z, &bias})
    if (!o->good) return none();
  if (x.t->dim() != 2 || a.t->dim() != 2 || b.t->dim() != 3) return none();
  const at::ScalarType type = x.t->scalar_type();
  const int64_t rows = x.t->size(0), channels = x.t->size(1), n = a.t->size(1), groups = b.t->size(1);
  if (dtype_of(type) < 0 || channels < 1 || n < 1 || groups < 1 || channels % groups || channels > INT32_MAX || n > INT32_MAX) return none();
  if (!dt.is(type, {rows, channels}) || !z.is(type, {rows, channels}) || !b.is(type, {rows, groups, n}) || !c.is(type, {rows, groups, n})) return none();
  if (!a.whole(at::kFloat, {channels, n}) || !d.whole(at::kFloat, {channels}) || !bias.whole(at::kFloat, {channels})) return none();
  if (!state.whole(at::kFloat, {rows, channels, n})) return none();
  tfa_scan_desc desc{};
  desc.dtype = dtype_of(type), desc.channels = (int32_t)channels, desc.groups = (int32_t)groups, desc.states = (int32_t)n, desc.softplus = soft;
  desc.batch = rows, desc.tokens = 1;
  desc.x_stride[0] = x.t->stride(0), desc.dt_stride[0] = dt.t->stride(0), desc.z_stride[0] = z.t ? z.t->stride(0) : 0;
  desc.b_stride[0] = b.t->stride(0), desc.b_stride[2] = b.t->stride(1), desc.c_stride[0] = c.t->stride(0), desc.c_stride[2] = c.t->stride(1);
  const at::Tensor y = at::empty({rows, channels}, x.t->options());
  return stepped(entries.scan_step(&desc, data(*x.t), data(*dt.t), floats(*a.t), data(*b.t), data(*c.t), floats(d.tensor()), data(z.tensor()),
                                   floats(bias.tensor()), floats(*state.t), data(y), stream_of(device)),
                 y, *state.t);
}

// C++ exceptions end here: a status of the C ABI is returned, torch's become Python's.
template <PyObject* (*F)(PyObject*)>
PyObject* guarded(PyObject*, PyObject* args) {
  HANDLE_TH_ERRORS
  try {
    return F(args);
  } catch (const Refused& r) {
    return PyLong_FromLong(r.rc);
  }
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {{"bind", guarded<bind_of>, METH_VARARGS, kBindDoc},
                          {"causal_conv", guarded<conv_of>, METH_VARARGS, kConvDoc},
                          {"selective_scan", guarded<scan_of>, METH_VARARGS, kScanDoc},
                          {"conv_step", guarded<conv_step_of>, METH_VARARGS, kConvStepDoc},
                          {"scan_step", guarded<scan_step_of>, METH_VARARGS, kScanStepDoc},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_state_space", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__state_space() {
  PyObject* const m = PyModule_Create(&kModule);
  PyObject* const names = m ? PyTuple_New(std::size(kEntries)) : nullptr;
  if (!names) return nullptr;
  for (size_t i = 0; i < std::size(kEntries); ++i) PyTuple_SET_ITEM(names, (Py_ssize_t)i, PyUnicode_FromString(kEntries[i]));
  if (PyModule_AddObject(m, "ENTRIES", names)) return nullptr;
  return m;
}
