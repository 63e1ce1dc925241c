// What the host helper modules of the operators share (not part of the C ABI): the tensors that a call takes,
// its results straight from the allocator, and Python's side of a call.  Each module includes it once and
// defines kModuleName before.
#pragma once

#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <cstring>
#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/fastmoe_amd.h"

namespace {

using at::Tensor;

// fmoe_last_error, once the module is bound.
const char* (*last_error)() = nullptr;

// A negative status of a C entry point.
struct StatusError : std::runtime_error {
  int code;
  StatusError(int c, const std::string& what) : std::runtime_error(what), code(c) {}
};

inline void check(int rc, const char* what) {
  if (rc == FMOE_OK) return;
  std::string msg = std::string(what) + ": ";
  if (rc != FMOE_EINVAL && rc != FMOE_ERANGE) msg += "status " + std::to_string(rc) + ": ";
  throw StatusError(rc, msg + last_error());
}

inline int code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return FMOE_F32;
    case at::kBFloat16: return FMOE_BF16;
    case at::kHalf: return FMOE_F16;
    case at::kLong: return FMOE_I64;
    case at::kInt: return FMOE_I32;
    default: throw std::runtime_error("fastmoe_amd: unsupported dtype");
  }
}
inline at::ScalarType type_of(int c) {
  return c == FMOE_F32 ? at::kFloat : c == FMOE_BF16 ? at::kBFloat16 : at::kHalf;
}

// The device of a call's tensors, and its current stream.
struct Place {
  c10::DeviceGuard guard;
  void* stream;
  explicit Place(const Tensor& t)
      : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// Straight from the allocator: through the dispatcher the norm's four results took 1.2 us more.
inline Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType t) {
  return Tensor(at::detail::empty_cuda(sizes, t, like.device(), std::nullopt));
}
inline Tensor empty(at::IntArrayRef sizes, const Tensor& like) { return empty(sizes, like, like.scalar_type()); }

// Elements from row to row; a single row's stride may be anything.
inline int64_t pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
inline void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

inline bool capturing() {
  return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}

inline bool is_float(const Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 ||
         t.scalar_type() == at::kHalf;
}
// A tensor whose memory holds its values: neither a view that stands for their negatives, nor a subclass that
// answers in Python, nor one that stands for zeros, which have no memory of their own (their null
// address would pass for an absent residual, bias or index).
inline bool plain(const Tensor& t) {
  return t.is_cuda() && t.layout() == c10::kStrided && t.has_storage() && !t.is_neg() &&
         !t.key_set().has(c10::DispatchKey::Python) && !t._is_zerotensor();
}
// A gradient, of either mode, would be recorded.
inline bool recorded(const Tensor& t) {
  return t.defined() &&
         ((t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined());
}
inline bool good_matrix(const Tensor& t) {
  return t.defined() && plain(t) && t.dim() == 2 && is_float(t) && t.size(1) >= 1 &&
         (t.size(1) == 1 || t.stride(1) == 1 || t.size(0) == 0);
}
// A gradient's rows with unit column stride, as their memory stands.
inline Tensor by_rows(Tensor t) {
  if (t._is_zerotensor()) t = at::zeros_like(t);
  t = (t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous()).resolve_neg();
  if (!plain(t))
    throw std::runtime_error("fastmoe_amd: this backward does not take a gradient without memory of its own");
  return t;
}

// ---- Python's side ------------------------------------------------------------------------------
inline Tensor tensor(PyObject* o) {
  if (o == Py_None) return Tensor();
  if (!THPVariable_Check(o)) throw std::invalid_argument("fastmoe_amd: expected a tensor");
  return THPVariable_Unpack(o);
}
inline int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw std::invalid_argument("fastmoe_amd: expected a number");
  return v;
}
inline double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1 && PyErr_Occurred()) throw std::invalid_argument("fastmoe_amd: expected a number");
  return v;
}
// The argument is no tensor, or not as the function takes it.
inline PyObject* not_taken() { Py_RETURN_NOTIMPLEMENTED; }
inline bool tensors(std::initializer_list<PyObject*> os) {
  for (PyObject* o : os)
    if (o != Py_None && !THPVariable_Check(o)) return false;
  return true;
}
inline PyObject* wrap(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
template <typename... Ts> PyObject* tuple(const Ts&... ts) {
  PyObject* items[] = {wrap(ts)...};
  constexpr Py_ssize_t n = sizeof...(Ts);
  PyObject* res = PyTuple_New(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!items[i] && res) Py_CLEAR(res);
    if (res) PyTuple_SET_ITEM(res, i, items[i]);
  }
  return res;
}

// A new reference to module.name, an exception type; RuntimeError if there is none.
inline PyObject* attribute(const char* module, const char* name) {
  PyObject* m = PyImport_ImportModule(module);
  PyObject* v = m ? PyObject_GetAttrString(m, name) : nullptr;
  Py_XDECREF(m);
  if (v) return v;
  PyErr_Clear();
  Py_INCREF(PyExc_RuntimeError);
  return PyExc_RuntimeError;
}

// torch.jit.trace or make_fx records the program: results that come straight from the allocator would
// enter the record as constants, whatever the inputs.
inline bool traced() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  return torch::jit::tracer::isTracing() ||
         Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
}

// Runs f with its `want` arguments; no C++ exception leaves it.
template <Py_ssize_t want, typename F> PyObject* guarded(Py_ssize_t given, F&& f) {
  if (given != want) {
    PyErr_Format(PyExc_TypeError, "%s: expected %zd arguments, got %zd", kModuleName, want, given);
    return nullptr;
  }
  if (!last_error) {
    PyErr_Format(PyExc_RuntimeError, "%s: bind() has not been called", kModuleName);
    return nullptr;
  }
  if (traced()) return not_taken();
  try {
    return f();
  } catch (python_error& e) {  // Python's own, from a hook on saved tensors: activation checkpointing's way out
    e.restore();
  } catch (const StatusError& e) {
    PyObject* type = e.code == FMOE_EINVAL    ? PyExc_ValueError
                     : e.code == FMOE_ERANGE ? PyExc_OverflowError
                                             : nullptr;
    if (type) Py_INCREF(type);
    else type = attribute("fastmoe_amd._abi", "FastMoEError");
    PyErr_SetString(type, e.what());
    Py_DECREF(type);
  } catch (const std::invalid_argument& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* type = attribute("torch", "OutOfMemoryError");
    PyErr_SetString(type, e.what_without_backtrace());
    Py_DECREF(type);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

#define FMOE_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL

}  // namespace
