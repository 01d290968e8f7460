// Host side of the operators on lists of tensors (trnfft_amd/optim.py): checks the lists and lays their addresses out in
// the C ABI's table.  A step has hundreds of tensors in up to seven lists; asked from Python, five questions each,
// they cost 0.25 us a tensor and list, which bounded the step of a model of 320 tensors and 8-bit states (0.99 ms).
#include <Python.h>

#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>

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

PyMethodDef kMethods[] = {{"table", table, METH_VARARGS, kDoc}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_tensor_table", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_table() { return PyModule_Create(&kModule); }
