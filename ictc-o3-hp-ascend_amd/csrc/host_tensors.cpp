// Host side of the calls over many tensors: checks lists of tensors and reads their addresses and
// sizes, as the arrays that the C entry points take.
//
// A step over a model's parameters looks at dtype, device, layout, size and address of every
// parameter and gradient.  From Python that is about 1.3 us a tensor, many times the update itself for
// hundreds of small ones; here it is about 0.025 us (pairs 0.019, written 0.006; 300 tensors).
#include <ATen/ATen.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <vector>

namespace {

// The tensor behind item `i` of a list, or null (with an exception unless the item is an allowed None).
const at::Tensor* item(PyObject* list, Py_ssize_t i, bool none, const char* what) {
  PyObject* o = PyList_GET_ITEM(list, i);
  if (o == Py_None && none) return nullptr;
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_ValueError, "%s must be tensors", what);
    return nullptr;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.scalar_type() != at::kFloat || t.layout() != at::kStrided || t.is_neg()) {
    PyErr_Format(PyExc_ValueError, "%s must be dense FP32 tensors on a ROCm GPU", what);
    return nullptr;
  }
  return &t;
}

bool same_device(int& device, const at::Tensor& t, const char* what) {
  if (device < 0) device = t.get_device();
  if (device == t.get_device()) return true;
  PyErr_Format(PyExc_ValueError, "%s must be on the same GPU", what);
  return false;
}

PyObject* bytes_of(const std::vector<int64_t>& v) {
  return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(v.data()),
                                   static_cast<Py_ssize_t>(v.size() * sizeof(int64_t)));
}

// addresses(tensors, what) -> (device index, addresses, sizes, contiguous): 64-bit arrays as bytes.
// `contiguous` is false where a tensor is not (its address is then of no use).
PyObject* addresses(PyObject*, PyObject* args) {
  PyObject* list;
  const char* what;
  if (!PyArg_ParseTuple(args, "O!s", &PyList_Type, &list, &what)) return nullptr;
  const Py_ssize_t n = PyList_GET_SIZE(list);
  std::vector<int64_t> at(n), size(n);
  int device = -1;
  bool contiguous = true;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t = item(list, i, false, what);
    if (!t || !same_device(device, *t, what)) return nullptr;
    contiguous = contiguous && t->is_contiguous();
    at[i] = reinterpret_cast<int64_t>(t->const_data_ptr());
    size[i] = t->numel();
  }
  return Py_BuildValue("iNNO", device, bytes_of(at), bytes_of(size), contiguous ? Py_True : Py_False);
}

// pairs(params, grads, block) -> (device index, parameter addresses, gradient addresses, sizes, values,
// contiguous): a gradient may be None (address 0; one without elements has another address); values is
// the sum of the sizes, each rounded up to whole blocks; `contiguous` speaks of the gradients.
PyObject* pairs(PyObject*, PyObject* args) {
  PyObject *params, *grads;
  long long block;
  if (!PyArg_ParseTuple(args, "O!O!L", &PyList_Type, &params, &PyList_Type, &grads, &block)) return nullptr;
  const Py_ssize_t n = PyList_GET_SIZE(params);
  if (n == 0 || PyList_GET_SIZE(grads) != n || block < 1) {
    PyErr_SetString(PyExc_ValueError, "expected one gradient (or None) for each parameter");
    return nullptr;
  }
  std::vector<int64_t> p_at(n), g_at(n), size(n);
  int device = -1;
  bool contiguous = true;
  long long values = 0;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* p = item(params, i, false, "parameters");
    if (!p || !same_device(device, *p, "parameters")) return nullptr;
    if (!p->is_contiguous()) {
      PyErr_SetString(PyExc_ValueError, "parameters must be contiguous");
      return nullptr;
    }
    const at::Tensor* g = item(grads, i, true, "gradients");
    if (!g && PyErr_Occurred()) return nullptr;
    p_at[i] = reinterpret_cast<int64_t>(p->const_data_ptr());
    size[i] = p->numel();
    values += (size[i] + block - 1) / block * block;
    g_at[i] = 0;
    if (!g) continue;
    if (!same_device(device, *g, "parameters and gradients")) return nullptr;
    if (g->sizes() != p->sizes()) {
      PyErr_SetString(PyExc_ValueError, "a gradient must have its parameter's shape");
      return nullptr;
    }
    contiguous = contiguous && g->is_contiguous();
    g_at[i] = size[i] ? reinterpret_cast<int64_t>(g->const_data_ptr()) : 16;
  }
  return Py_BuildValue("iNNNLO", device, bytes_of(p_at), bytes_of(g_at), bytes_of(size), values,
                       contiguous ? Py_True : Py_False);
}

// matrices(tensors, what) -> (device index, addresses, rows, columns, batches, contiguous) of tensors [..., rows,
// columns], leading axes counting matrices: 64-bit arrays as bytes.
PyObject* matrices(PyObject*, PyObject* args) {
  PyObject* list;
  const char* what;
  if (!PyArg_ParseTuple(args, "O!s", &PyList_Type, &list, &what)) return nullptr;
  const Py_ssize_t n = PyList_GET_SIZE(list);
  std::vector<int64_t> at(n), rows(n), columns(n), batches(n);
  int device = -1;
  bool contiguous = true;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t = item(list, i, false, what);
    if (!t || !same_device(device, *t, what)) return nullptr;
    const int64_t axes = t->dim();
    if (axes < 2) {
      PyErr_Format(PyExc_ValueError, "%s must be matrices (or have leading axes that count them)", what);
      return nullptr;
    }
    contiguous = contiguous && t->is_contiguous();
    at[i] = reinterpret_cast<int64_t>(t->const_data_ptr());
    rows[i] = t->size(axes - 2), columns[i] = t->size(axes - 1);
    batches[i] = 1;
    for (int64_t k = 0; k < axes - 2; ++k) batches[i] *= t->size(k);
  }
  return Py_BuildValue("iNNNNO", device, bytes_of(at), bytes_of(rows), bytes_of(columns), bytes_of(batches),
                       contiguous ? Py_True : Py_False);
}

// apart(params, momentum, grads): refuses written memory (params, momentum) that another one of the lists' tensors
// overlaps, of those whose gradient is not None.  Gradients may share memory with each other.
PyObject* apart(PyObject*, PyObject* args) {
  PyObject* lists[3];
  if (!PyArg_ParseTuple(args, "O!O!O!", &PyList_Type, &lists[0], &PyList_Type, &lists[1], &PyList_Type, &lists[2]))
    return nullptr;
  struct Piece {
    uintptr_t from, to;
    bool written;
  };
  std::vector<Piece> pieces;
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(lists[2]); ++i) {
    if (PyList_GET_ITEM(lists[2], i) == Py_None) continue;
    for (int k = 0; k < 3; ++k) {
      if (i >= PyList_GET_SIZE(lists[k])) continue;
      const at::Tensor* t = item(lists[k], i, false, "parameters, momentum and gradients");
      if (!t) return nullptr;
      if (t->numel() == 0) continue;
      const uintptr_t from = reinterpret_cast<uintptr_t>(t->const_data_ptr());
      pieces.push_back({from, from + t->numel() * sizeof(float), k < 2});
    }
  }
  std::sort(pieces.begin(), pieces.end(), [](const Piece& a, const Piece& b) { return a.from < b.from; });
  uintptr_t written = 0, any = 0;      // where what begins earlier ends
  for (const Piece& p : pieces) {
    if (p.from < (p.written ? any : written)) {
      PyErr_SetString(PyExc_ValueError, "parameters and momentum must not overlap each other or the gradients");
      return nullptr;
    }
    any = std::max(any, p.to);
    if (p.written) written = std::max(written, p.to);
  }
  Py_RETURN_NONE;
}

// alike(tensors) -> new contiguous tensors of their shapes
PyObject* alike(PyObject*, PyObject* args) {
  PyObject* list;
  if (!PyArg_ParseTuple(args, "O!", &PyList_Type, &list)) return nullptr;
  const Py_ssize_t n = PyList_GET_SIZE(list);
  PyObject* made = PyList_New(n);
  if (!made) return nullptr;
  try {
    for (Py_ssize_t i = 0; i < n; ++i) {
      const at::Tensor* t = item(list, i, false, "tensors");
      if (!t) {
        Py_DECREF(made);
        return nullptr;
      }
      PyList_SET_ITEM(made, i, THPVariable_Wrap(at::empty(t->sizes(), t->options())));
    }
  } catch (...) {
    Py_DECREF(made);
    throw;
  }
  return made;
}

// written(params, grads): raises the version counter of every parameter whose gradient is not None.
PyObject* written(PyObject*, PyObject* args) {
  PyObject *params, *grads;
  if (!PyArg_ParseTuple(args, "O!O!", &PyList_Type, &params, &PyList_Type, &grads)) return nullptr;
  const Py_ssize_t n = PyList_GET_SIZE(params);
  for (Py_ssize_t i = 0; i < n && i < PyList_GET_SIZE(grads); ++i) {
    PyObject* o = PyList_GET_ITEM(params, i);
    if (PyList_GET_ITEM(grads, i) == Py_None || !THPVariable_Check(o)) continue;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  Py_RETURN_NONE;
}

// No C++ exception leaves through Python's C interface.
template <PyObject* (*F)(PyObject*, PyObject*)>
PyObject* guarded(PyObject* self, PyObject* args) {
  try {
    return F(self, args);
  } catch (const std::exception&) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"addresses", guarded<addresses>, METH_VARARGS,
     "(device, addresses, sizes, contiguous) of a list of FP32 GPU tensors"},
    {"pairs", guarded<pairs>, METH_VARARGS, "(device, parameters, gradients, sizes, values, contiguous) of two lists"},
    {"matrices", guarded<matrices>, METH_VARARGS,
     "(device, addresses, rows, columns, batches, contiguous) of a list of matrices"},
    {"apart", guarded<apart>, METH_VARARGS, "refuse parameters and momentum that overlap"},
    {"alike", guarded<alike>, METH_VARARGS, "new contiguous tensors of a list's shapes"},
    {"written", guarded<written>, METH_VARARGS,
     "raise the version counters of parameters written through their addresses"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "ictc_host_tensors", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_ictc_host_tensors() { return PyModule_Create(&module); }
