// Host side of the layers that a model calls by the hundred: the autograd nodes of the layer norm and of the
// embedding, on the library's C entry points.
//
// A node of Python's costs its forward pass 15 us and its backward pass 40 to 60: the engine's own thread has to
// take the interpreter's lock from the thread that waits for it.  These take 5 to 8 each, more than the kernels of a
// model's usual sizes.  What is beyond the kernels' orders is composed of torch operations in Python
// (`formula`, given to `bind` with the entry points' addresses).
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <exception>
#include <optional>
#include <stdexcept>
#include <string>

#include "ictc_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entries {
  decltype(&ictc_hip_status_string) status = nullptr;
  decltype(&ictc_hip_layer_norm_workspace) norm_workspace = nullptr;
  decltype(&ictc_hip_layer_norm_forward) norm_forward = nullptr;
  decltype(&ictc_hip_layer_norm_backward) norm_backward = nullptr;
  decltype(&ictc_hip_layer_norm_second) norm_second = nullptr;
  decltype(&ictc_hip_embedding_forward) embedding_forward = nullptr;
  decltype(&ictc_hip_embedding_workspace) embedding_workspace = nullptr;
  decltype(&ictc_hip_embedding_table_grad) embedding_table_grad = nullptr;
  PyObject* formula = nullptr;
};

Entries lib;

void check(int64_t status, const char* what) {
  if (status != 0)
    throw std::runtime_error(std::string(what) + " failed: " + lib.status(static_cast<int>(status)) + " (status " +
                             std::to_string(status) + ")");
}

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

const float* in(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }
float* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr<float>() : nullptr; }

// As the kernels read it: rows one after another, and no sign that is only noted (torch.imag of a conjugate).
Tensor dense(const Tensor& t) { return t.resolve_neg().contiguous(); }

Tensor given(const std::optional<Tensor>& t) { return t ? *t : Tensor(); }

// The workspace of a call, or nothing for a size of 0.
Tensor workspace(int64_t units, const Tensor& beside, const char* what) {
  if (units < 0) check(-units, what);
  return at::empty({units}, beside.options().dtype(at::kFloat));
}

// Rows [N, W] of a norm and what belongs to them; bias may be undefined.
struct Spec {
  int activation;
  float eps;
};

Tensor norm_forward(const Spec& s, const Tensor& x, const Tensor& weight, const Tensor& bias) {
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty_like(x);
  if (x.numel())
    check(lib.norm_forward(in(x), in(weight), in(bias), out(y), static_cast<int>(x.size(1)), s.activation, s.eps,
                           x.size(0), stream_of(x)),
          "ictc_hip_layer_norm_forward");
  return y;
}

// A weight's gradient to be written, or zeros where there are no rows.
Tensor weight_grad(const Tensor& x, const Tensor& weight, bool need) {
  return !need ? Tensor() : x.numel() ? at::empty_like(weight) : at::zeros_like(weight);
}

// Gradients to (x, weight, bias), undefined where not needed.
variable_list norm_backward(const Spec& s, const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& dy,
                            const bool (&need)[3]) {
  const c10::DeviceGuard guard(x.device());
  Tensor dx = need[0] ? at::empty_like(x) : Tensor();
  Tensor dw = weight_grad(x, weight, need[1]), db = weight_grad(x, bias, need[2]);
  if (x.numel()) {
    const int width = static_cast<int>(x.size(1));
    Tensor ws;
    if (need[1] || need[2]) ws = workspace(lib.norm_workspace(width, x.size(0)), x, "ictc_hip_layer_norm_workspace");
    check(lib.norm_backward(in(x), in(weight), in(bias), in(dy), out(dx), out(dw), out(db), out(ws),
                            ws.defined() ? ws.numel() : 0, width, s.activation, s.eps, x.size(0), stream_of(x)),
          "ictc_hip_layer_norm_backward");
  }
  return {dx, dw, db};
}

// Gradients of <u, dx> to (x, weight, bias, dy), undefined where not needed.
variable_list norm_second(const Spec& s, const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& dy,
                          const Tensor& u, const bool (&need)[4]) {
  const c10::DeviceGuard guard(x.device());
  Tensor gx = need[0] ? at::empty_like(x) : Tensor(), gdy = need[3] ? at::empty_like(dy) : Tensor();
  Tensor gw = weight_grad(x, weight, need[1]), gb = weight_grad(x, bias, need[2]);
  if (x.numel()) {
    const int width = static_cast<int>(x.size(1));
    Tensor ws;
    if (need[1] || need[2]) ws = workspace(lib.norm_workspace(width, x.size(0)), x, "ictc_hip_layer_norm_workspace");
    check(lib.norm_second(in(x), in(weight), in(bias), in(dy), in(u), out(gx), out(gdy), out(gw), out(gb), out(ws),
                          ws.defined() ? ws.numel() : 0, width, s.activation, s.eps, x.size(0), stream_of(x)),
          "ictc_hip_layer_norm_second");
  }
  return {gx, gw, gb, gdy};
}

// Python's formula: gradients of <cots, gradients(x, weight, bias, dy)> where needed, recorded where grad mode is on.
variable_list composed(const Spec& s, const variable_list& inputs, const bool (&need)[4], const variable_list& cots) {
  if (!lib.formula) throw std::runtime_error("the host module has no formula");
  const PyGILState_STATE state = PyGILState_Ensure();
  PyObject* result = nullptr;
  variable_list grads(4);
  std::optional<python_error> error;      // (an exception of the formula's goes on as what it is)
  bool failed = false;
  {
    PyObject* ins = PyTuple_New(4);
    for (int k = 0; k < 4; ++k) PyTuple_SET_ITEM(ins, k, THPVariable_Wrap(inputs[k]));
    PyObject* tops = PyTuple_New(3);
    for (int k = 0; k < 3; ++k) PyTuple_SET_ITEM(tops, k, THPVariable_Wrap(cots[k]));
    PyObject* needs = Py_BuildValue("(iiii)", need[0], need[1], need[2], need[3]);
    result = PyObject_CallFunction(lib.formula, "(id)OOO", s.activation, static_cast<double>(s.eps), ins, needs, tops);
    Py_XDECREF(ins);
    Py_XDECREF(tops);
    Py_XDECREF(needs);
  }
  if (!result) {
    error.emplace();
    error->persist();
  } else if (!PyTuple_Check(result) || PyTuple_GET_SIZE(result) != 4) {
    failed = true;
  } else {
    for (int k = 0; k < 4; ++k) {
      PyObject* g = PyTuple_GET_ITEM(result, k);
      if (THPVariable_Check(g)) grads[k] = THPVariable_Unpack(g);
    }
  }
  Py_XDECREF(result);
  PyGILState_Release(state);
  if (error) throw *error;
  if (failed) throw std::runtime_error("the composed gradients are not four");
  return grads;
}

// Of a node's inputs (x, weight, bias if there is one, ...) which gradients the engine will use.
template <int N>
void needed(const AutogradContext* ctx, bool bias, bool (&need)[N]) {
  size_t edge = 0;
  for (int k = 0; k < N; ++k) need[k] = (k != 2 || bias) && ctx->needs_input_grad(edge++);
}

void keep(AutogradContext* ctx, const Spec& s, variable_list tensors) {
  ctx->saved_data["activation"] = static_cast<int64_t>(s.activation);
  ctx->saved_data["eps"] = static_cast<double>(s.eps);
  ctx->save_for_backward(std::move(tensors));
}

Spec kept(AutogradContext* ctx) {
  return {static_cast<int>(ctx->saved_data["activation"].toInt()), static_cast<float>(ctx->saved_data["eps"].toDouble())};
}

// The gradients that are needed (a mask of three bits), as a function of (x, weight, bias, dy).
struct LayerNormGradient : torch::autograd::Function<LayerNormGradient> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                               const std::optional<Tensor>& bias, const Tensor& dy, int64_t activation, double eps,
                               int64_t mask) {
    const Spec s{static_cast<int>(activation), static_cast<float>(eps)};
    const Tensor b = given(bias);
    ctx->set_materialize_grads(false);
    ctx->saved_data["mask"] = mask;
    keep(ctx, s, {x, weight, b, dy});
    const bool need[3] = {(mask & 1) != 0, (mask & 2) != 0, (mask & 4) != 0};
    variable_list all = norm_backward(s, x, weight, b, dy, need), made;
    for (int k = 0; k < 3; ++k)
      if (need[k]) made.push_back(all[k]);
    return made;
  }

  static variable_list backward(AutogradContext* ctx, variable_list tops) {
    const variable_list inputs = ctx->get_saved_variables();
    const Spec s = kept(ctx);
    const int64_t mask = ctx->saved_data["mask"].toInt();
    variable_list cots(3), grads(4);
    for (int k = 0, at = 0; k < 3; ++k)
      if (mask >> k & 1) cots[k] = tops[at++];
    bool need[4];
    needed(ctx, inputs[2].defined(), need);
    if (cots[1].defined() || cots[2].defined() || (cots[0].defined() && at::GradMode::is_enabled())) {
      grads = composed(s, inputs, need, cots);
    } else if (cots[0].defined()) {
      if (!s.activation) need[2] = false;          // without an activation the bias is in none of the gradients
      if (need[0] || need[1] || need[2] || need[3])
        grads = norm_second(s, inputs[0], inputs[1], inputs[2], inputs[3], dense(cots[0]), need);
    }
    return {grads[0], grads[1], grads[2], grads[3], Tensor(), Tensor(), Tensor()};
  }
};

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
                        int64_t activation, double eps) {
    const Spec s{static_cast<int>(activation), static_cast<float>(eps)};
    const Tensor b = given(bias);
    ctx->set_materialize_grads(false);
    keep(ctx, s, {x, weight, b});
    return norm_forward(s, x, weight, b);
  }

  static variable_list backward(AutogradContext* ctx, variable_list tops) {
    variable_list grads(5);
    const variable_list inputs = ctx->get_saved_variables();
    const Spec s = kept(ctx);
    bool need[3];
    needed(ctx, inputs[2].defined(), need);
    if (!tops[0].defined() || !(need[0] || need[1] || need[2])) return grads;
    const Tensor dy = dense(tops[0]);
    if (at::GradMode::is_enabled()) {
      const std::optional<Tensor> bias = inputs[2].defined() ? std::optional<Tensor>(inputs[2]) : std::nullopt;
      const int64_t mask = need[0] | need[1] << 1 | need[2] << 2;
      const variable_list made =
          LayerNormGradient::apply(inputs[0], inputs[1], bias, dy, s.activation, static_cast<double>(s.eps), mask);
      for (int k = 0, at = 0; k < 3; ++k)
        if (need[k]) grads[k] = made[at++];
    } else {
      const variable_list made = norm_backward(s, inputs[0], inputs[1], inputs[2], dy, need);
      for (int k = 0; k < 3; ++k) grads[k] = made[k];
    }
    return grads;
  }
};

Tensor lookup(const Tensor& table, const Tensor& tokens, double scale) {
  const c10::DeviceGuard guard(table.device());
  Tensor y = at::empty({tokens.size(0), table.size(1)}, table.options());
  if (tokens.size(0))
    check(lib.embedding_forward(tokens.const_data_ptr(), static_cast<int>(tokens.element_size()), in(table), out(y),
                                table.size(0), static_cast<int>(table.size(1)), static_cast<float>(scale),
                                tokens.size(0), stream_of(table)),
          "ictc_hip_embedding_forward");
  return y;
}

Tensor table_grad(const Tensor& grad, const Tensor& tokens, int64_t rows, double scale) {
  const c10::DeviceGuard guard(grad.device());
  const int64_t count = grad.size(0);
  const int width = static_cast<int>(grad.size(1));
  if (count == 0) return at::zeros({rows, width}, grad.options());
  Tensor y = at::empty({rows, width}, grad.options());
  const Tensor ws =
      workspace(lib.embedding_workspace(rows, width, count), grad, "ictc_hip_embedding_workspace");
  check(lib.embedding_table_grad(tokens.const_data_ptr(), static_cast<int>(tokens.element_size()), in(grad), out(y), rows,
                                 width, static_cast<float>(scale), count, out(ws), ws.numel(), stream_of(grad)),
        "ictc_hip_embedding_table_grad");
  return y;
}

// The lookup and the table's gradient are linear and each other's adjoint, so they cover every order.
struct TableGrad;

struct Lookup : torch::autograd::Function<Lookup> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& tokens, double scale);
  static variable_list backward(AutogradContext* ctx, variable_list tops);
};

struct TableGrad : torch::autograd::Function<TableGrad> {
  static Tensor forward(AutogradContext* ctx, const Tensor& grad, const Tensor& tokens, int64_t rows, double scale);
  static variable_list backward(AutogradContext* ctx, variable_list tops);
};

Tensor Lookup::forward(AutogradContext* ctx, const Tensor& table, const Tensor& tokens, double scale) {
  ctx->set_materialize_grads(false);
  ctx->saved_data["rows"] = table.size(0);
  ctx->saved_data["scale"] = scale;
  ctx->save_for_backward({tokens});
  return lookup(table, tokens, scale);
}

variable_list Lookup::backward(AutogradContext* ctx, variable_list tops) {
  if (!tops[0].defined()) return {Tensor(), Tensor(), Tensor()};
  const Tensor tokens = ctx->get_saved_variables()[0], grad = dense(tops[0]);
  const int64_t rows = ctx->saved_data["rows"].toInt();
  const double scale = ctx->saved_data["scale"].toDouble();
  return {at::GradMode::is_enabled() ? TableGrad::apply(grad, tokens, rows, scale) : table_grad(grad, tokens, rows, scale),
          Tensor(), Tensor()};
}

Tensor TableGrad::forward(AutogradContext* ctx, const Tensor& grad, const Tensor& tokens, int64_t rows, double scale) {
  ctx->set_materialize_grads(false);
  ctx->saved_data["scale"] = scale;
  ctx->save_for_backward({tokens});
  return table_grad(grad, tokens, rows, scale);
}

variable_list TableGrad::backward(AutogradContext* ctx, variable_list tops) {
  if (!tops[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
  const Tensor tokens = ctx->get_saved_variables()[0], cot = dense(tops[0]);
  const double scale = ctx->saved_data["scale"].toDouble();
  return {at::GradMode::is_enabled() ? Lookup::apply(cot, tokens, scale) : lookup(cot, tokens, scale), Tensor(), Tensor(),
          Tensor()};
}

// ---------------------------------------------------------------------------------------------------------
// Python's interface
// ---------------------------------------------------------------------------------------------------------

// What a caller gave wrong: a ValueError.
struct Refused : std::invalid_argument {
  using std::invalid_argument::invalid_argument;
};

const Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) throw Refused("expected a tensor");
  return THPVariable_Unpack(o);
}

void require_gpu_fp32(const Tensor& t, const Tensor& beside) {
  if (!t.is_cuda() || t.scalar_type() != at::kFloat || t.layout() != at::kStrided)
    throw Refused("ictc_o3 HIP operators require FP32 tensors on a ROCm GPU; precision is never changed automatically");
  if (t.device() != beside.device()) throw Refused("All operands must be on the same GPU");
}

// A Python number as a double that is finite as a float, too (bool is none).
double number(PyObject* o, const char* what) {
  const double v = PyBool_Check(o) || !(PyFloat_Check(o) || PyLong_Check(o)) ? NAN : PyFloat_AsDouble(o);
  if (!std::isfinite(static_cast<float>(v)) || PyErr_Occurred()) {       // (an integer beyond a double's range is -1 with an exception)
    PyErr_Clear();
    throw Refused(what);
  }
  return v;
}

// bind(status_string, norm workspace, forward, backward, second, embedding forward, workspace, table_grad, formula)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long at[8];
  PyObject* formula;
  if (!PyArg_ParseTuple(args, "KKKKKKKKO", at, at + 1, at + 2, at + 3, at + 4, at + 5, at + 6, at + 7, &formula))
    return nullptr;
  lib.status = reinterpret_cast<decltype(lib.status)>(at[0]);
  lib.norm_workspace = reinterpret_cast<decltype(lib.norm_workspace)>(at[1]);
  lib.norm_forward = reinterpret_cast<decltype(lib.norm_forward)>(at[2]);
  lib.norm_backward = reinterpret_cast<decltype(lib.norm_backward)>(at[3]);
  lib.norm_second = reinterpret_cast<decltype(lib.norm_second)>(at[4]);
  lib.embedding_forward = reinterpret_cast<decltype(lib.embedding_forward)>(at[5]);
  lib.embedding_workspace = reinterpret_cast<decltype(lib.embedding_workspace)>(at[6]);
  lib.embedding_table_grad = reinterpret_cast<decltype(lib.embedding_table_grad)>(at[7]);
  Py_INCREF(formula);
  Py_XDECREF(lib.formula);
  lib.formula = formula;
  Py_RETURN_NONE;
}

// layer_norm(features [..., W], weight, bias or None, activation, eps)
PyObject* layer_norm(PyObject*, PyObject* args) {
  PyObject *x, *weight, *bias, *given_eps;
  int activation;
  if (!PyArg_ParseTuple(args, "OOOiO", &x, &weight, &bias, &activation, &given_eps)) return nullptr;
  if (!lib.norm_forward) throw std::runtime_error("the host module is not bound to the library");
  const double eps = number(given_eps, "eps must be a positive number");
  if (!(static_cast<float>(eps) > 0.f)) throw Refused("eps must be a positive number");
  const Tensor& features = tensor(x);
  if (features.dim() < 1 || features.size(-1) < 1 || features.size(-1) > ICTC_LAYER_NORM_MAX_WIDTH)
    throw Refused("features must have between 1 and " + std::to_string(ICTC_LAYER_NORM_MAX_WIDTH) + " columns");
  const int64_t width = features.size(-1);
  const auto check_weight = [&](const Tensor& w) {
    if (w.dim() != 1 || w.size(0) != width)
      throw Refused("weight and bias must have shape [" + std::to_string(width) + "]");
    require_gpu_fp32(w, features);
  };
  require_gpu_fp32(features, features);
  check_weight(tensor(weight));
  std::optional<Tensor> b;
  if (bias != Py_None) {
    check_weight(tensor(bias));
    b = dense(tensor(bias));
  }
  const bool rows = features.dim() == 2;
  const Tensor y = LayerNorm::apply(dense(rows ? features : features.reshape({-1, width})),
                                    dense(tensor(weight)), b, activation, eps);
  return THPVariable_Wrap(rows ? y : y.view(features.sizes()));
}

// embedding(tokens of any shape, table, scale)
PyObject* embedding(PyObject*, PyObject* args) {
  PyObject *given_tokens, *given_table, *given_scale;
  if (!PyArg_ParseTuple(args, "OOO", &given_tokens, &given_table, &given_scale)) return nullptr;
  if (!lib.embedding_forward) throw std::runtime_error("the host module is not bound to the library");
  const Tensor &t = tensor(given_tokens), &table = tensor(given_table);
  if (table.dim() != 2 || table.size(0) < 1 || table.size(1) < 1) throw Refused("the table must have shape [rows, width]");
  if (t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) throw Refused("tokens must be int32 or int64");
  const double scale = number(given_scale, "scale must be a finite number");
  require_gpu_fp32(table, table);
  if (t.device() != table.device()) throw Refused("All operands must be on the same GPU");
  const bool flat = t.dim() == 1;
  const Tensor y = Lookup::apply(dense(table), flat ? t.contiguous() : t.reshape({-1}).contiguous(), scale);
  if (flat) return THPVariable_Wrap(y);
  auto shape = t.sizes().vec();
  shape.push_back(y.size(1));
  return THPVariable_Wrap(y.view(shape));
}

// No C++ exception leaves through Python's C interface.
template <PyObject* (*F)(PyObject*, PyObject*)>
PyObject* guarded(PyObject* self, PyObject* args) {
  try {
    return F(self, args);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception&) {      // (memory that ran out, a hook's own exception: each as torch's calls raise it)
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

PyMethodDef methods[] = {
    {"bind", guarded<bind>, METH_VARARGS, "addresses of the library's entry points, and the composed gradients"},
    {"layer_norm", guarded<layer_norm>, METH_VARARGS, "layer norm of rows, differentiable"},
    {"embedding", guarded<embedding>, METH_VARARGS, "rows of a table by token, differentiable"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "ictc_host_layers", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_ictc_host_layers() { return PyModule_Create(&module); }
