// qrb200 -- the short way from Python to the layer operators.
//
// A call on small tensors is bound by the host: of the 8 us that rms_norm of one token took through
// torch.ops, 1.5 us went into finding the operator by its schema.  These two functions take their
// arguments straight from Python instead.  They answer only for plain CUDA tensors with nothing else
// listening (no tensor subclass, no dispatch or function mode, no functorch transform); for anything
// else (under torch.inference_mode(), which excludes autograd's keys, too) they return NotImplemented, and
// the caller takes torch.ops, which every such feature knows.
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "qrb_torch_layers.h"

namespace {

using qrb200::OptTensor;

bool nothing_listens() {
  const auto keys = c10::impl::tls_local_dispatch_key_set();
  return !c10::impl::TorchDispatchModeTLS::any_modes_set() && at::impl::PythonTorchFunctionTLS::stack_len() == 0 &&
         (keys.included_ - c10::default_included_set).empty() && !keys.excluded_.has_any(c10::autograd_dispatch_keyset);
}
// obj as a plain CUDA tensor; None as nothing where that is allowed.
bool take(PyObject* obj, bool optional, OptTensor& out) {
  if (obj == Py_None) return optional;
  if (!THPVariable_CheckExact(obj)) return false;
  const at::Tensor& t = THPVariable_Unpack(obj);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.key_set().has(c10::DispatchKey::Python) || t.is_conj() || t.is_neg())
    return false;
  out = t;
  return true;
}
bool take_dtype(PyObject* obj, std::optional<at::ScalarType>& out) {
  if (obj == Py_None) return true;
  if (!THPDtype_Check(obj)) return false;
  out = reinterpret_cast<THPDtype*>(obj)->scalar_type;
  return true;
}
PyObject* not_taken() { Py_RETURN_NOTIMPLEMENTED; }

// rms_norm(x, weight, residual, eps, out_dtype) -> y, (y, h), (y, scale) or (y, scale, h)
PyObject* py_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  OptTensor x, weight, residual;
  std::optional<at::ScalarType> out;
  if (n != 5 || !nothing_listens() || !take(args[0], false, x) || !take(args[1], true, weight) ||
      !take(args[2], true, residual) || !PyFloat_CheckExact(args[3]) || !take_dtype(args[4], out))
    return not_taken();
  const double eps = PyFloat_AS_DOUBLE(args[3]);
  std::tuple<at::Tensor, at::Tensor, at::Tensor> r;
  {
    pybind11::gil_scoped_release no_gil;
    r = qrb200::rms_norm(*x, weight, residual, eps, out);
  }
  auto& [y, scale, h] = r;
  const int count = 1 + scale.defined() + h.defined();
  if (count == 1) return THPVariable_Wrap(std::move(y));
  PyObject* t = PyTuple_New(count);
  if (!t) return nullptr;
  int at = 0;
  for (at::Tensor* o : {&y, &scale, &h})
    if (o->defined()) PyTuple_SET_ITEM(t, at++, THPVariable_Wrap(std::move(*o)));
  return t;
  END_HANDLE_TH_ERRORS
}

// linear(x, weight, bias, residual, activation, x_scale, weight_scale, out_dtype) -> y
PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  OptTensor x, weight, bias, residual, xs, ws;
  std::optional<at::ScalarType> out;
  if (n != 8 || !nothing_listens() || !take(args[0], false, x) || !take(args[1], false, weight) || !take(args[2], true, bias) ||
      !take(args[3], true, residual) || !PyLong_CheckExact(args[4]) || !take(args[5], true, xs) || !take(args[6], true, ws) ||
      !take_dtype(args[7], out))
    return not_taken();
  const long act = PyLong_AsLong(args[4]);
  std::tuple<at::Tensor, at::Tensor> r;
  {
    pybind11::gil_scoped_release no_gil;
    r = qrb200::linear(*x, *weight, bias, residual, act, xs, ws, out, false);
  }
  return THPVariable_Wrap(std::move(std::get<0>(r)));
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_rms_norm)), METH_FASTCALL, nullptr},
                         {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_linear)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_layers", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layers() { return PyModule_Create(&module); }
