// What the sources of the torch operator layer share: statuses as exceptions, tensor checks, the arguments of CPython
// functions.  Every definition sits in an unnamed namespace of the including translation unit.
#pragma once
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/hip/HIPStream.h>
#include <c10/util/Exception.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>

#include "pplx_a2a.h"

namespace {

inline const char *status_name(int status) {
  switch (status) {
    case PPLX_A2A_INVALID_ARGUMENT: return "invalid argument";
    case PPLX_A2A_INVALID_STATE: return "invalid state";
    case PPLX_A2A_HIP_ERROR: return "HIP error";
    case PPLX_A2A_UNSUPPORTED: return "unsupported";
    default: return "error";
  }
}

#define A2A_CHECK(status)                                                                     \
  do {                                                                                        \
    const int st_ = (status);                                                                 \
    TORCH_CHECK(st_ == PPLX_A2A_OK, "pplx_kernels: ", status_name(st_), ": ", pplx_a2a_last_error()); \
  } while (0)

// Tensor checks (csrc/bindings/all_to_all_ops.cpp:19-24,135-161,249-259)
inline void check_tensor(const at::Tensor &x, int64_t ndim, const char *name) {
  TORCH_CHECK(x.is_cuda(), "Tensor ", name, " must be on GPU");
  TORCH_CHECK(x.is_contiguous(), "Tensor ", name, " must be contiguous");
  TORCH_CHECK(x.dim() == ndim, "Tensor ", name, " must be ", ndim, " dimensional");
}

inline void check_bound_m(const at::Tensor *bound_m) {
  if (!bound_m) return;
  check_tensor(*bound_m, 1, "boundM.value()");
  TORCH_CHECK(bound_m->scalar_type() == at::kUInt32, "boundM must be of type UInt32");
  TORCH_CHECK(bound_m->numel() == 1, "boundM must be a scalar tensor");
}

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return PPLX_A2A_F32;
    case at::kBFloat16: return PPLX_A2A_BF16;
    case at::kHalf: return PPLX_A2A_F16;
    default: return -1;
  }
}

inline void *current_stream_of(const at::Tensor &t) {
  return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

inline const at::Tensor *opt(const std::optional<at::Tensor> &t) { return t.has_value() ? &*t : nullptr; }

inline const at::Tensor &tensor_arg(PyObject *obj, const char *name) {
  TORCH_CHECK_TYPE(THPVariable_Check(obj), name, " must be a Tensor, not ", Py_TYPE(obj)->tp_name);
  return THPVariable_Unpack(obj);
}

inline const at::Tensor *optional_tensor_arg(PyObject *obj, const char *name) {
  return obj == Py_None ? nullptr : &tensor_arg(obj, name);
}

inline int64_t int_arg(PyObject *obj, const char *name) {
  const long long v = PyLong_AsLongLong(obj);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, name, " must be an int, not ", Py_TYPE(obj)->tp_name);
  }
  return v;
}

inline bool bool_arg(PyObject *obj) {
  const int v = PyObject_IsTrue(obj);
  if (v < 0) throw python_error();  // (what its __bool__ raised)
  return v;
}

inline void arity(const char *fn, Py_ssize_t got, Py_ssize_t want) {
  TORCH_CHECK_TYPE(got == want, fn, "() takes ", want, " positional arguments but ", got, " were given");
}

// The library call itself runs without the interpreter lock.
struct WithoutGil {
  PyThreadState *state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

template <class Fn>
int without_gil(Fn &&fn) {
  WithoutGil released;
  return fn();
}

}  // namespace
