// The Python module beside the ops, a library of its own: gnb200_torch.so is loaded by libtorch programs without Python too.
//
// plain_call(x, weight, bias, num_groups, eps, act, num_channels) -> tensor, or None where the module's Python code has
// to look at the call: anything but exact tensors and parameters, a torch-function mode, other argument types, a shape that it
// refuses.  Called without torch.ops' argument matching, which took 3 us.
//
// rms_norm(x, weight, residual, eps, offset) -> y or (y, sum), rms_quant(x, weight, residual, eps, offset, block, format) ->
// (codes, scales[, sum]), rotary(q, k, positions, inv_freq, sections, q_weight, k_weight, eps, offset, interleaved) -> (q, k): the same for the
// operators on token rows; None, for an absent tensor, is an argument like any other there.  So are quantize_4bit(x, block, scale),
// dequantize_4bit(codes, scales, channels, scale, dtype), rms_quant_4bit(x, weight, residual, eps, offset, block, scale),
// linear_4bit(codes, scales, weight_codes, weight_scales, scale, weight_scale, bias, dtype) and dropout_add(x, residual, p, seed, layer), whose seed
// is a tensor or a number.
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <utility>
#include <vector>

#include "gn_torch.h"

namespace {

const at::Tensor* exact_tensor(PyObject* o) {
  if (Py_TYPE(o) != (PyTypeObject*)THPVariableClass && Py_TYPE(o) != (PyTypeObject*)ParameterClass) return nullptr;
  return &THPVariable_Unpack(o);
}

PyObject* plain_call(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 7 || !PyLong_CheckExact(args[3]) || !PyFloat_CheckExact(args[4]) || !PyLong_CheckExact(args[5]) ||
      !PyLong_CheckExact(args[6]) || at::impl::torch_function_mode_enabled())
    Py_RETURN_NONE;
  const at::Tensor *x = exact_tensor(args[0]), *w = exact_tensor(args[1]), *b = exact_tensor(args[2]);
  if (!x || !w || !b) Py_RETURN_NONE;
  const long long G = PyLong_AsLongLong(args[3]), act = PyLong_AsLongLong(args[5]), C = PyLong_AsLongLong(args[6]);
  if (PyErr_Occurred()) return nullptr;
  if (!x->is_cuda() || x->dim() < 3 || x->size(1) != C) Py_RETURN_NONE;
  const double eps = PyFloat_AS_DOUBLE(args[4]);
  at::Tensor y;
  {
    pybind11::gil_scoped_release no_gil;
    y = gnb200_ops::group_norm_act_direct(*x, *w, *b, G, eps, act);
  }
  if (!y.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// an exact tensor, or an undefined one for None; false for everything else
bool tensor_or_none(PyObject* o, at::Tensor* out) {
  if (o == Py_None) return true;
  const at::Tensor* t = exact_tensor(o);
  if (t) *out = *t;
  return t != nullptr;
}

PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor x, weight, residual, y, sum;
  if (nargs != 5 || !exact_tensor(args[0]) || !tensor_or_none(args[0], &x) || !tensor_or_none(args[1], &weight) ||
      !tensor_or_none(args[2], &residual) || !PyFloat_CheckExact(args[3]) || !PyFloat_CheckExact(args[4]) ||
      at::impl::torch_function_mode_enabled())
    Py_RETURN_NONE;
  const double eps = PyFloat_AS_DOUBLE(args[3]), offset = PyFloat_AS_DOUBLE(args[4]);
  bool ok = false;
  {
    pybind11::gil_scoped_release no_gil;
    std::tie(y, sum) = gnb200_ops::rms_norm_direct(x, weight, residual, eps, offset, &ok);
  }
  if (!ok) Py_RETURN_NONE;
  if (!sum.defined()) return THPVariable_Wrap(std::move(y));
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(y)), THPVariable_Wrap(std::move(sum)));
  END_HANDLE_TH_ERRORS
}

PyObject* rms_quant(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor x, weight, residual, q, scale, sum;
  if (nargs != 7 || !exact_tensor(args[0]) || !tensor_or_none(args[0], &x) || !tensor_or_none(args[1], &weight) ||
      !tensor_or_none(args[2], &residual) || !PyFloat_CheckExact(args[3]) || !PyFloat_CheckExact(args[4]) || !PyLong_CheckExact(args[5]) ||
      !PyLong_CheckExact(args[6]) || at::impl::torch_function_mode_enabled())
    Py_RETURN_NONE;
  const double eps = PyFloat_AS_DOUBLE(args[3]), offset = PyFloat_AS_DOUBLE(args[4]);
  const long long block = PyLong_AsLongLong(args[5]), format = PyLong_AsLongLong(args[6]);
  if (PyErr_Occurred()) return nullptr;
  bool ok = false;
  {
    pybind11::gil_scoped_release no_gil;
    std::tie(q, scale, sum) = gnb200_ops::rms_quant_direct(x, weight, residual, eps, offset, block, format, &ok);
  }
  if (!ok) Py_RETURN_NONE;
  if (!sum.defined()) return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(q)), THPVariable_Wrap(std::move(scale)));
  return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(q)), THPVariable_Wrap(std::move(scale)), THPVariable_Wrap(std::move(sum)));
  END_HANDLE_TH_ERRORS
}

PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor q, k, positions, inv_freq, qw, kw, qo, ko;
  if (nargs != 10 || !exact_tensor(args[0]) || !tensor_or_none(args[0], &q) || !tensor_or_none(args[1], &k) || !exact_tensor(args[2]) ||
      !tensor_or_none(args[2], &positions) || !exact_tensor(args[3]) || !tensor_or_none(args[3], &inv_freq) || !PyTuple_CheckExact(args[4]) ||
      !tensor_or_none(args[5], &qw) || !tensor_or_none(args[6], &kw) || !PyFloat_CheckExact(args[7]) || !PyFloat_CheckExact(args[8]) ||
      !PyBool_Check(args[9]) || at::impl::torch_function_mode_enabled())
    Py_RETURN_NONE;
  const double eps = PyFloat_AS_DOUBLE(args[7]), offset = PyFloat_AS_DOUBLE(args[8]);
  const bool interleaved = args[9] == Py_True;
  std::vector<int64_t> sections;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(args[4]); ++i) {
    PyObject* o = PyTuple_GET_ITEM(args[4], i);
    if (!PyLong_CheckExact(o)) Py_RETURN_NONE;
    sections.push_back(PyLong_AsLongLong(o));
  }
  if (PyErr_Occurred()) return nullptr;
  bool ok = false;
  {
    pybind11::gil_scoped_release no_gil;
    std::tie(qo, ko) = gnb200_ops::rotary_direct(q, k, positions, inv_freq, sections, qw, kw, eps, offset, interleaved, &ok);
  }
  if (!ok) Py_RETURN_NONE;
  PyObject* second = ko.defined() ? THPVariable_Wrap(std::move(ko)) : Py_NewRef(Py_None);
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(qo)), second);
  END_HANDLE_TH_ERRORS
}

bool dtype_of(PyObject* o, at::ScalarType* out) {
  if (!THPDtype_Check(o)) return false;
  *out = reinterpret_cast<THPDtype*>(o)->scalar_type;
  return true;
}

PyObject* quantize_4bit(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor x, scale, codes, scales;
  if (nargs != 3 || !exact_tensor(args[0]) || !tensor_or_none(args[0], &x) || !PyLong_CheckExact(args[1]) || !tensor_or_none(args[2], &scale) ||
      at::impl::torch_function_mode_enabled())
    Py_RETURN_NONE;
  const long long block = PyLong_AsLongLong(args[1]);
  if (PyErr_Occurred()) return nullptr;
  bool ok = false;
  {
    pybind11::gil_scoped_release no_gil;
    std::tie(codes, scales) = gnb200_ops::quantize_4bit_direct(x, block, scale, &ok);
  }
  if (!ok) Py_RETURN_NONE;
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(codes)), THPVariable_Wrap(std::move(scales)));
  END_HANDLE_TH_ERRORS
}

PyObject* dequantize_4bit(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor codes, scales, scale, out;
  at::ScalarType dtype;
  if (nargs != 5 || !exact_tensor(args[0]) || !tensor_or_none(args[0], &codes) || !exact_tensor(args[1]) || !tensor_or_none(args[1], &scales) ||
      !PyLong_CheckExact(args[2]) || !tensor_or_none(args[3], &scale) || !dtype_of(args[4], &dtype) || at::impl::torch_function_mode_enabled())
    Py_RETURN_NONE;
  const long long channels = PyLong_AsLongLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  bool ok = false;
  {
    pybind11::gil_scoped_release no_gil;
    out = gnb200_ops::dequantize_4bit_direct(codes, scales, channels, scale, dtype, &ok);
  }
  if (!ok) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* rms_quant_4bit(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor x, weight, residual, scale, codes, scales, sum;
  if (nargs != 7 || !exact_tensor(args[0]) || !tensor_or_none(args[0], &x) || !tensor_or_none(args[1], &weight) ||
      !tensor_or_none(args[2], &residual) || !PyFloat_CheckExact(args[3]) || !PyFloat_CheckExact(args[4]) || !PyLong_CheckExact(args[5]) ||
      !tensor_or_none(args[6], &scale) || at::impl::torch_function_mode_enabled())
    Py_RETURN_NONE;
  const double eps = PyFloat_AS_DOUBLE(args[3]), offset = PyFloat_AS_DOUBLE(args[4]);
  const long long block = PyLong_AsLongLong(args[5]);
  if (PyErr_Occurred()) return nullptr;
  bool ok = false;
  {
    pybind11::gil_scoped_release no_gil;
    std::tie(codes, scales, sum) = gnb200_ops::rms_quant_4bit_direct(x, weight, residual, eps, offset, block, scale, &ok);
  }
  if (!ok) Py_RETURN_NONE;
  if (!sum.defined()) return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(codes)), THPVariable_Wrap(std::move(scales)));
  return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(codes)), THPVariable_Wrap(std::move(scales)), THPVariable_Wrap(std::move(sum)));
  END_HANDLE_TH_ERRORS
}

PyObject* linear_4bit(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[7], out;
  at::ScalarType dtype;
  if (nargs != 8 || !dtype_of(args[7], &dtype) || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  for (int i = 0; i < 7; ++i)
    if ((i < 4 && !exact_tensor(args[i])) || !tensor_or_none(args[i], &t[i])) Py_RETURN_NONE;
  bool ok = false;
  {
    pybind11::gil_scoped_release no_gil;
    out = gnb200_ops::linear_4bit_direct(t[0], t[1], t[2], t[3], t[4], t[5], t[6], dtype, &ok);
  }
  if (!ok) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* dropout_add(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor x, residual, seed_at, out;
  if (nargs != 5 || !exact_tensor(args[0]) || !tensor_or_none(args[0], &x) || !tensor_or_none(args[1], &residual) || !PyFloat_CheckExact(args[2]) ||
      !PyLong_CheckExact(args[4]) || at::impl::torch_function_mode_enabled())
    Py_RETURN_NONE;
  long long seed = 0;
  if (PyLong_CheckExact(args[3]))
    seed = PyLong_AsLongLong(args[3]);
  else if (args[3] == Py_None || !tensor_or_none(args[3], &seed_at))
    Py_RETURN_NONE;
  const long long layer = PyLong_AsLongLong(args[4]);
  if (PyErr_Occurred()) {  // beyond 64 bits: Python looks at it
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const double p = PyFloat_AS_DOUBLE(args[2]);
  bool ok = false;
  {
    pybind11::gil_scoped_release no_gil;
    out = gnb200_ops::dropout_add_direct(x, residual, p, seed_at, seed, layer, &ok);
  }
  if (!ok) Py_RETURN_NONE;
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {{"plain_call", (PyCFunction)(void (*)())plain_call, METH_FASTCALL, nullptr},
                          {"rms_norm", (PyCFunction)(void (*)())rms_norm, METH_FASTCALL, nullptr},
                          {"rms_quant", (PyCFunction)(void (*)())rms_quant, METH_FASTCALL, nullptr},
                          {"rotary", (PyCFunction)(void (*)())rotary, METH_FASTCALL, nullptr},
                          {"quantize_4bit", (PyCFunction)(void (*)())quantize_4bit, METH_FASTCALL, nullptr},
                          {"dequantize_4bit", (PyCFunction)(void (*)())dequantize_4bit, METH_FASTCALL, nullptr},
                          {"rms_quant_4bit", (PyCFunction)(void (*)())rms_quant_4bit, METH_FASTCALL, nullptr},
                          {"linear_4bit", (PyCFunction)(void (*)())linear_4bit, METH_FASTCALL, nullptr},
                          {"dropout_add", (PyCFunction)(void (*)())dropout_add, METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "gnb200_python", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_gnb200_python(void) { return PyModule_Create(&kModule); }
