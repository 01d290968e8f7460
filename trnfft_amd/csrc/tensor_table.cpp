// Host side of calls whose questions to their tensors take longer than their work on the GPU.
//
// Operators on lists of tensors (trnfft_amd/optim.py): checks the lists and lays their addresses out in the C ABI's table.  A step has
// hundreds of tensors in up to seven lists; asked from Python, five questions each, they cost 0.25 us a tensor and list, which
// bounded the step of a model of 320 tensors and 8-bit states (0.99 ms).
//
// Steps of streams (trnfft_amd/state_space.py): where every operand is as the C ABI takes it, the call is made from here; asked from Python
// nine tensors cost 8 of the 13.8 us of a small scan's step.  Anything else is left to Python, which converts or refuses it.
#include <Python.h>

#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>

#include "../../include/trnfft_amd.h"

#include <cstdint>
#include <cstring>
#include <exception>

namespace {

constexpr int64_t kBlock = 256;  // values that share a scale

const char kDoc[] =
    "table(what, names, lists, dtypes, device) -> bytes: rows of 64-bit words, one for each tensor of lists[0]: the address\n"
    "of its entry in each list (0 where a list is None), then its size.  Tensors must be contiguous, no negating views, on the GPU of that\n"
    "index and of the list's dtype, with as many values as lists[0]'s (a name that ends in 'scales': one for every 256).";

// An error of list `name` (a new Python exception of the given type).
PyObject* refuse(PyObject* type, PyObject* what, PyObject* name, const char* text) {
  PyErr_Format(type, "%U: %U %s", what, name, text);
  return nullptr;
}

bool ends_in_scales(PyObject* name) {
  Py_ssize_t n = 0;
  const char* s = PyUnicode_AsUTF8AndSize(name, &n);
  return s && n >= 6 && !strcmp(s + n - 6, "scales");
}

PyObject* table_of(PyObject* args) {
  PyObject *what, *names, *lists, *dtypes;
  long long device;
  if (!PyArg_ParseTuple(args, "UO!O!O!L", &what, &PyTuple_Type, &names, &PyTuple_Type, &lists, &PyTuple_Type, &dtypes, &device))
    return nullptr;
  const Py_ssize_t columns = PyTuple_GET_SIZE(lists);
  if (columns < 1 || PyTuple_GET_SIZE(names) != columns || PyTuple_GET_SIZE(dtypes) != columns || !PyList_Check(PyTuple_GET_ITEM(lists, 0))) {
    PyErr_SetString(PyExc_ValueError, "table: names, lists and dtypes must agree");
    return nullptr;
  }
  const Py_ssize_t count = PyList_GET_SIZE(PyTuple_GET_ITEM(lists, 0)), width = columns + 1;
  PyObject* const bytes = PyBytes_FromStringAndSize(nullptr, count * width * (Py_ssize_t)sizeof(int64_t));
  if (!bytes) return nullptr;
  struct Owned {  // given up where the table is complete
    PyObject* p;
    ~Owned() { Py_XDECREF(p); }
  } owned{bytes};
  int64_t* const words = reinterpret_cast<int64_t*>(PyBytes_AS_STRING(bytes));
  for (Py_ssize_t c = 0; c < columns; ++c) {
    PyObject* const list = PyTuple_GET_ITEM(lists, c);
    PyObject* const name = PyTuple_GET_ITEM(names, c);
    PyObject* const dtype = PyTuple_GET_ITEM(dtypes, c);
    if (!PyUnicode_Check(name)) {
      PyErr_SetString(PyExc_TypeError, "table: names are strings");
      return nullptr;
    }
    if (list == Py_None) {
      for (Py_ssize_t i = 0; i < count; ++i) words[i * width + c] = 0;
      continue;
    }
    if (!PyList_Check(list) || !THPDtype_Check(dtype)) {
      PyErr_SetString(PyExc_TypeError, "table: lists of tensors and their dtypes expected");
      return nullptr;
    }
    if (PyList_GET_SIZE(list) != count) {
      PyErr_Format(PyExc_ValueError, "%U: %zd %U, but %zd %U", what, count, PyTuple_GET_ITEM(names, 0), PyList_GET_SIZE(list), name);
      return nullptr;
    }
    const at::ScalarType type = reinterpret_cast<THPDtype*>(dtype)->scalar_type;
    const bool scales = ends_in_scales(name);
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject* const item = PyList_GET_ITEM(list, i);
      if (!THPVariable_Check(item)) return refuse(PyExc_TypeError, what, name, "must be tensors");
      const at::Tensor& t = THPVariable_Unpack(item);
      if (t.scalar_type() != type) {
        PyErr_Format(PyExc_TypeError, "%U: %U must be %S, got %S", what, name, dtype, reinterpret_cast<PyObject*>(torch::getTHPDtype(t.scalar_type())));
        return nullptr;
      }
      if (t.is_neg()) return refuse(PyExc_ValueError, what, name, "must not be negating views (resolve_neg)");
      if (!t.is_cuda() || t.get_device() != device) return refuse(PyExc_ValueError, what, name, "must be on the GPU of the first");
      if (t.layout() != at::kStrided || !t.is_contiguous()) return refuse(PyExc_ValueError, what, name, "must be contiguous");
      const int64_t n = t.numel();
      if (c == 0) words[i * width + columns] = n;
      const int64_t own = words[i * width + columns];
      if (n != (scales ? (own + kBlock - 1) / kBlock : own)) return refuse(PyExc_ValueError, what, name, "must have the size that the first list asks for");
      words[i * width + c] = reinterpret_cast<int64_t>(t.data_ptr());
    }
  }
  owned.p = nullptr;
  return bytes;
}

PyObject* table(PyObject*, PyObject* args) {
  try {
    return table_of(args);
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "table: unknown error");
  }
  return nullptr;
}

// ------------------------------------------------------------------------------------------------

const char kConvStepDoc[] =
    "conv_step(entry, stream, device, x, state, weight, bias, activation) -> y, an error's status, or None where an operand is not as the\n"
    "C ABI takes it (or needs a gradient).  entry: the address of tfa_causal_conv_step.";
const char kScanStepDoc[] =
    "scan_step(entry, stream, device, x, dt, a, b, c, state, d, z, dt_bias, softplus) -> y, an error's status, or None, as conv_step.\n"
    "entry: the address of tfa_selective_scan_step.";

int dtype_of(at::ScalarType t) {
  return t == at::kFloat ? TFA_DTYPE_F32 : t == at::kBFloat16 ? TFA_DTYPE_BF16 : t == at::kHalf ? TFA_DTYPE_F16 : -1;
}

// A tensor of the device with contiguous last axis that needs no gradient; None gives an undefined one where it may be left out.
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
    if (v.dim() < 1 || v.dim() > 3 || (v.size(v.dim() - 1) != 1 && v.stride(v.dim() - 1) != 1)) return;
    t = &v;
    good = true;
  }
  bool is(at::ScalarType type, std::initializer_list<int64_t> sizes) const { return !t || (t->scalar_type() == type && t->sizes() == at::IntArrayRef(sizes)); }
  bool whole(at::ScalarType type, std::initializer_list<int64_t> sizes) const { return !t || (is(type, sizes) && t->is_contiguous()); }
  const void* data() const { return t ? t->data_ptr() : nullptr; }
  const float* floats() const { return static_cast<const float*>(data()); }
};

PyObject* none() { Py_RETURN_NONE; }

// y where the call went well, its status otherwise; the state has changed
PyObject* stepped(int rc, const at::Tensor& y, const at::Tensor& state) {
  if (rc) return PyLong_FromLong(rc);
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return THPVariable_Wrap(y);
}

PyObject* conv_step_of(PyObject* args) {
  PyObject *ox, *ostate, *oweight, *obias;
  unsigned long long entry, stream;
  long long device;
  int activation;
  if (!PyArg_ParseTuple(args, "KKLOOOOi", &entry, &stream, &device, &ox, &ostate, &oweight, &obias, &activation)) return nullptr;
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
  const auto call = reinterpret_cast<decltype(&tfa_causal_conv_step)>(entry);
  return stepped(call(&desc, x.data(), weight.floats(), bias.floats(), state.t->data_ptr(), y.data_ptr(), reinterpret_cast<tfa_stream>(stream)), y,
                 *state.t);
}

PyObject* scan_step_of(PyObject* args) {
  PyObject *ox, *odt, *oa, *ob, *oc, *ostate, *od, *oz, *obias;
  unsigned long long entry, stream;
  long long device;
  int soft;
  if (!PyArg_ParseTuple(args, "KKLOOOOOOOOOp", &entry, &stream, &device, &ox, &odt, &oa, &ob, &oc, &ostate, &od, &oz, &obias, &soft)) return nullptr;
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
  const auto call = reinterpret_cast<decltype(&tfa_selective_scan_step)>(entry);
  return stepped(call(&desc, x.data(), dt.data(), a.floats(), b.data(), c.data(), d.floats(), z.data(), bias.floats(),
                      static_cast<float*>(state.t->data_ptr()), y.data_ptr(), reinterpret_cast<tfa_stream>(stream)),
                 y, *state.t);
}

// C++ exceptions end here
template <PyObject* (*F)(PyObject*)>
PyObject* guarded(PyObject*, PyObject* args) {
  try {
    return F(args);
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown error");
  }
  return nullptr;
}

PyMethodDef kMethods[] = {{"table", table, METH_VARARGS, kDoc},
                          {"conv_step", guarded<conv_step_of>, METH_VARARGS, kConvStepDoc},
                          {"scan_step", guarded<scan_step_of>, METH_VARARGS, kScanStepDoc},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tensor_table", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_table() { return PyModule_Create(&kModule); }
