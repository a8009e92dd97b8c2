// What the sources of the operators on plain tensors share (torch_experts.cpp, torch_router.cpp): checks, fresh tensors,
// calls through the dispatcher.  Every definition sits in an unnamed namespace of the including translation unit.
#pragma once
#include <Python.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <string>

#include "pplx_a2a.h"
#include "torch_common.h"

namespace {

using opt_tensor = const std::optional<at::Tensor> &;

// ---------------------------------------------------------------------------
// Checks
// ---------------------------------------------------------------------------
inline void check_on(const at::Tensor &x, const at::Tensor &with, const char *name) {
  TORCH_CHECK(x.is_cuda(), "Tensor ", name, " must be on GPU");
  TORCH_CHECK(x.device() == with.device(), "Tensor ", name, " must be on ", with.device(), ", not on ", x.device());
}

// Rows of the last dimension that lie in one piece, at 16-byte boundaries.
inline void check_rows_of(const at::Tensor &x, const char *name) {
  const int64_t dims = x.dim(), bytes = (int64_t)x.element_size();
  TORCH_CHECK(x.sizes()[dims - 1] <= 1 || x.strides()[dims - 1] == 1, "the rows of ", name, " must be contiguous");
  for (int64_t d = 0; d + 1 < dims; ++d) {
    TORCH_CHECK(x.sizes()[d] <= 1 || x.strides()[d] * bytes % 16 == 0, "the rows of ", name, " must be 16-byte aligned");
  }
  TORCH_CHECK(reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0, "Tensor ", name, " must be 16-byte aligned");
}

// Stride of dimension d (elements); where there is one entry it is not used, and 0.
inline int64_t step_of(const at::Tensor &x, int64_t d) { return x.sizes()[d] <= 1 ? 0 : x.strides()[d]; }
inline int64_t byte_step_of(const at::Tensor &x, int64_t d) { return step_of(x, d) * (int64_t)x.element_size(); }

inline void check_dense(const at::Tensor &x, at::ScalarType type, int64_t dims, const at::Tensor &with, const char *name) {
  check_on(x, with, name);
  TORCH_CHECK(x.dim() == dims, "Tensor ", name, " must be ", dims, " dimensional");
  TORCH_CHECK(x.scalar_type() == type, name, " must be of type ", type);
  TORCH_CHECK(x.is_contiguous(), "Tensor ", name, " must be contiguous");
}

inline void check_float(const at::Tensor &x, const char *name) {
  TORCH_CHECK(dtype_code(x.scalar_type()) >= 0, "Unsupported dtype for ", name);
}

// What is written holds no element twice and none of what is read.
inline void check_written(const at::Tensor &out, const char *name, std::initializer_list<const at::Tensor *> read) {
  TORCH_CHECK(at::has_internal_overlap(out) != at::MemOverlap::Yes, "Tensor ", name, " holds elements more than once");
  for (const at::Tensor *x : read) {
    if (!x || !out.is_alias_of(*x)) continue;
    const at::MemOverlapStatus status = at::get_overlap_status(out, *x);
    TORCH_CHECK(status != at::MemOverlapStatus::Full && status != at::MemOverlapStatus::Partial, "Tensor ", name,
                " overlaps a tensor that is read or written too");
  }
}

// The writes are seen by autograd's check of saved tensors.
inline void written(const at::Tensor &x) {
  if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

template <class T> T *data_of(const at::Tensor *x) { return x ? static_cast<T *>(x->data_ptr()) : nullptr; }

// ---------------------------------------------------------------------------
// Results
// ---------------------------------------------------------------------------
inline at::Tensor fresh(at::IntArrayRef sizes, const at::Tensor &with, at::ScalarType type) {
  return at::empty(sizes, at::TensorOptions(with.device()).dtype(type));
}

// The same of sizes that a trace may not know.
inline at::Tensor fresh_traced(c10::SymIntArrayRef sizes, const at::Tensor &with, at::ScalarType type) {
  return at::empty_symint(sizes, at::TensorOptions(with.device()).dtype(type));
}

inline const at::Tensor *defined(const at::Tensor &t) { return t.defined() ? &t : nullptr; }

// ---------------------------------------------------------------------------
// Ops and their gradients
// ---------------------------------------------------------------------------
// A registered op, through the dispatcher, so that a step can be traced.
template <class Fn> auto op_handle(const char *name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Fn>();
}

// Gradients come in any layout (that of a sum is one element, expanded).  Those of a traced step have no address, and sizes
// that may not be known.
inline at::Tensor as_rows(const at::Tensor &g) {
  if (g.is_meta() || g.key_set().has(c10::DispatchKey::Python) || g.key_set().has(c10::DispatchKey::Functionalize)) return g.contiguous();
  const int64_t bytes = (int64_t)g.element_size();
  const bool fits =
      g.strides()[1] == 1 && g.strides()[0] * bytes % 16 == 0 && reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 == 0;
  return fits ? g : g.clone(at::MemoryFormat::Contiguous);
}

// Gradients that are asked for their own (create_graph) say that they have none when they are.
inline torch::autograd::variable_list differentiable_once(torch::autograd::variable_list grads, const char *of) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::variable_list made;
  for (const at::Tensor &g : grads) {
    if (g.defined()) made.push_back(g);
  }
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string("pplx_kernels: the gradients of ") + of + " are differentiable once", (int64_t)made.size());
  for (at::Tensor &g : made) {
    g = g.detach();
    g.requires_grad_(true);
  }
  made = (*error)(std::move(made));
  size_t next = 0;
  for (at::Tensor &g : grads) {
    if (g.defined()) g = made[next++];
  }
  return grads;
}

// Tangents of forward-mode differentiation are refused, not dropped.
inline void check_no_tangent(std::initializer_list<const at::Tensor *> read, const char *of) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const at::Tensor *x : read) {
    TORCH_CHECK(!x || !x->defined() || !x->_fw_grad(0).defined(),
                "pplx_kernels: ", of, " and their gradients have no forward-mode derivatives");
  }
}

// Meta kernels: a traced call does nothing.
template <class Fn> struct Nothing;
template <class... A> struct Nothing<void (*)(A...)> {
  static void run(A...) {}
};

template <class Fn> void define(torch::Library &m, const char *name, const char *schema, Fn fn) {
  m.def((std::string(name) + schema).c_str());
  m.impl(name, c10::kCUDA, fn);
  m.impl(name, c10::kMeta, &Nothing<Fn>::run);
}

// ---------------------------------------------------------------------------
// Functions of pplx_kernels._C
// ---------------------------------------------------------------------------
// Whether the dispatcher would go straight to the kernel (or to autograd, which the functions see to).  A tracer, a mode, a
// transform or a tensor that is more than its data has to see the registered op: behind its back the results would be taken for
// what `empty` made.
inline bool straight(std::initializer_list<const at::Tensor *> tensors) {
  static const uint64_t usual =
      c10::full_backend_mask | c10::autocast_dispatch_keyset.raw_repr() |
      c10::DispatchKeySet({c10::DispatchKey::Dense, c10::DispatchKey::BackendSelect, c10::DispatchKey::ADInplaceOrView,
                           c10::DispatchKey::AutogradFunctionality}).raw_repr();
  const auto local = c10::impl::tls_local_dispatch_key_set();
  c10::DispatchKeySet keys = local.included_;
  for (const at::Tensor *x : tensors) {
    if (x) keys = keys | x->key_set();
  }
  return ((keys - local.excluded_).raw_repr() & ~usual) == 0;
}

inline std::optional<at::Tensor> maybe(const at::Tensor *x) { return x ? std::optional<at::Tensor>(*x) : std::nullopt; }

inline PyObject *wrap_or_none(const at::Tensor &t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}

}  // namespace
