// The torch layer of the operators between dispatch and combine: ops of pplx_kernels that write tensors of the caller,
// and the same as functions of pplx_kernels._C, which also make the tensors where they are asked to (pplx_kernels/experts.py).
#include <ATen/ops/empty_like.h>
#include <torch/csrc/Dtype.h>

#include <tuple>

#include "torch_tensors.h"

namespace {

uint64_t sort_workspace(int64_t m, int64_t k, int64_t experts) {
  TORCH_CHECK(m <= UINT32_MAX && k <= UINT32_MAX && experts >= 0 && experts <= UINT32_MAX,
              "pplx_kernels: invalid argument: size out of range");
  uint64_t bytes = 0;
  A2A_CHECK(pplx_a2a_sort_workspace((uint32_t)m, (uint32_t)k, (uint32_t)experts, &bytes));
  return bytes;
}

// ---------------------------------------------------------------------------
// The operators on tensors of the caller
// ---------------------------------------------------------------------------
void sort_tokens(const at::Tensor &rows, const at::Tensor *scale, const at::Tensor &slots, const at::Tensor &offsets,
                 const at::Tensor *workspace, const at::Tensor &x, const at::Tensor &indices, const at::Tensor *bound_m) {
  TORCH_CHECK(x.is_cuda(), "Tensor x must be on GPU");
  TORCH_CHECK(x.dim() == 2, "Tensor x must be 2 dimensional");
  check_float(x, "x");
  check_rows_of(x, "x");
  check_dense(indices, at::kUInt32, 2, x, "indices");
  const int64_t m = x.sizes()[0], k = indices.sizes()[1], experts = offsets.numel() - 1;
  TORCH_CHECK(indices.sizes()[0] == m, "indices.size(0) must be equal to x.size(0)");
  check_bound_m(bound_m);
  if (bound_m) check_on(*bound_m, x, "bound_m");
  check_dense(offsets, at::kInt, 1, x, "offsets");
  check_dense(slots, at::kInt, 2, x, "slots");
  TORCH_CHECK(slots.sizes() == indices.sizes(), "slots must have the shape of indices");
  check_on(rows, x, "rows");
  TORCH_CHECK(rows.dim() == 2 && rows.sizes()[0] == m * k && rows.sizes()[1] == x.sizes()[1], "rows must be [", m * k, ", ",
              x.sizes()[1], "]");
  check_rows_of(rows, "rows");
  if (scale) {
    check_dense(*scale, at::kFloat, 1, x, "scale");
    TORCH_CHECK(scale->sizes()[0] == m * k, "scale must be [", m * k, "]");
    TORCH_CHECK(rows.scalar_type() == at::kChar, "quantised rows must be of type Char");
  } else {
    TORCH_CHECK(rows.scalar_type() == x.scalar_type(), "rows must have the dtype of x");
  }
  const uint64_t bytes = sort_workspace(m, k, experts);
  if (bytes) {
    TORCH_CHECK(workspace, "a step of this size needs a workspace of ", bytes, " bytes");
    check_dense(*workspace, at::kInt, 1, x, "workspace");
    TORCH_CHECK(4 * (uint64_t)workspace->numel() >= bytes, "the workspace has fewer than ", bytes, " bytes");
  }
  check_written(rows, "rows", {&x, &indices, bound_m, scale, &slots, &offsets, workspace});
  check_written(slots, "slots", {&indices, bound_m, &x, scale, &offsets, workspace});
  check_written(offsets, "offsets", {&indices, bound_m, &x, scale, workspace});
  if (scale) check_written(*scale, "scale", {&indices, bound_m, &x, workspace});
  if (bytes) check_written(*workspace, "workspace", {&indices, bound_m, &x});

  pplx_a2a_sort_args_t a{};
  a.x = x.data_ptr();
  a.x_stride_row = byte_step_of(x, 0);
  a.dtype = dtype_code(x.scalar_type());
  a.m = (uint32_t)m;
  a.experts_per_token = (uint32_t)k;
  a.num_experts = (uint32_t)experts;
  a.hidden_dim = (uint64_t)x.sizes()[1];
  a.indices = data_of<const uint32_t>(&indices);
  a.bound_m = data_of<const uint32_t>(bound_m);
  a.out_rows = rows.data_ptr();
  a.out_stride_row = byte_step_of(rows, 0);
  a.out_scale = data_of<float>(scale);
  a.slots = data_of<int32_t>(&slots);
  a.offsets = data_of<int32_t>(&offsets);
  a.workspace = bytes ? workspace->data_ptr() : nullptr;
  A2A_CHECK(pplx_a2a_sort_tokens(x.device().index(), &a, current_stream_of(x)));
  written(rows);
  written(slots);
  written(offsets);
  if (scale) written(*scale);
}

void check_slots(const at::Tensor &slots, const at::Tensor *weights, const at::Tensor &with, int64_t m) {
  check_dense(slots, at::kInt, 2, with, "slots");
  TORCH_CHECK(slots.sizes()[0] == m, "slots must have a row for each of the ", m, " tokens");
  if (!weights) return;
  check_dense(*weights, at::kFloat, 2, with, "weights");
  TORCH_CHECK(weights->sizes() == slots.sizes(), "weights must have the shape of slots");
}

void check_offsets(const at::Tensor &offsets, const at::Tensor &with) {
  check_dense(offsets, at::kInt, 1, with, "offsets");
  TORCH_CHECK(offsets.numel() >= 1, "offsets must not be empty");
}

void unsort_tokens(const at::Tensor &out, const at::Tensor &y, const at::Tensor &slots, const at::Tensor *weights) {
  TORCH_CHECK(y.is_cuda(), "Tensor y must be on GPU");
  TORCH_CHECK(y.dim() == 2, "Tensor y must be 2 dimensional");
  check_float(y, "y");
  check_rows_of(y, "y");
  check_on(out, y, "out");
  TORCH_CHECK(out.dim() == 2 && out.sizes()[1] == y.sizes()[1], "out must be [tokens, ", y.sizes()[1], "]");
  check_float(out, "out");
  check_rows_of(out, "out");
  const int64_t m = out.sizes()[0];
  check_slots(slots, weights, y, m);
  TORCH_CHECK(m <= UINT32_MAX, "pplx_kernels: unsupported: 2^32 tokens or more");
  check_written(out, "out", {&y, &slots, weights});

  pplx_a2a_unsort_args_t a{};
  a.out = out.data_ptr();
  a.out_stride_row = byte_step_of(out, 0);
  a.out_dtype = dtype_code(out.scalar_type());
  a.y_dtype = dtype_code(y.scalar_type());
  a.y = y.data_ptr();
  a.y_stride_row = byte_step_of(y, 0);
  a.y_rows = y.sizes()[0];
  a.slots = data_of<const int32_t>(&slots);
  a.weights = data_of<const float>(weights);
  a.m = (uint32_t)m;
  a.experts_per_token = (uint32_t)slots.sizes()[1];
  a.hidden_dim = (uint64_t)y.sizes()[1];
  A2A_CHECK(pplx_a2a_unsort_tokens(y.device().index(), &a, current_stream_of(y)));
  written(out);
}

void unsort_tokens_backward(const at::Tensor *grad_y, const at::Tensor *grad_weights, const at::Tensor &grad_out,
                            const at::Tensor &y, const at::Tensor &slots, const at::Tensor &offsets,
                            const at::Tensor *weights) {
  TORCH_CHECK(y.is_cuda(), "Tensor y must be on GPU");
  TORCH_CHECK(y.dim() == 2, "Tensor y must be 2 dimensional");
  check_float(y, "y");
  check_rows_of(y, "y");
  check_on(grad_out, y, "grad_out");
  check_float(grad_out, "grad_out");
  TORCH_CHECK(grad_out.dim() == 2 && grad_out.sizes()[1] == y.sizes()[1], "grad_out must be [tokens, ", y.sizes()[1], "]");
  check_rows_of(grad_out, "grad_out");
  const int64_t m = grad_out.sizes()[0];
  check_slots(slots, weights, y, m);
  check_offsets(offsets, y);
  TORCH_CHECK(m <= UINT32_MAX, "pplx_kernels: unsupported: 2^32 tokens or more");
  if (grad_y) {
    check_on(*grad_y, y, "grad_y");
    TORCH_CHECK(grad_y->sizes() == y.sizes() && grad_y->scalar_type() == y.scalar_type(),
                "grad_y must have the shape and dtype of y");
    check_rows_of(*grad_y, "grad_y");
    check_written(*grad_y, "grad_y", {&grad_out, &y, &slots, &offsets, weights, grad_weights});
  }
  if (grad_weights) {
    check_dense(*grad_weights, at::kFloat, 2, y, "grad_weights");
    TORCH_CHECK(grad_weights->sizes() == slots.sizes(), "grad_weights must have the shape of slots");
    check_written(*grad_weights, "grad_weights", {&grad_out, &y, &slots, &offsets, weights});
  }

  pplx_a2a_unsort_backward_args_t a{};
  if (grad_y) {
    a.grad_y = grad_y->data_ptr();
    a.grad_y_stride_row = byte_step_of(*grad_y, 0);
  }
  a.grad_weights = data_of<float>(grad_weights);
  a.grad_out = grad_out.data_ptr();
  a.grad_out_stride_row = byte_step_of(grad_out, 0);
  a.grad_dtype = dtype_code(grad_out.scalar_type());
  a.dtype = dtype_code(y.scalar_type());
  a.y = y.data_ptr();
  a.y_stride_row = byte_step_of(y, 0);
  a.y_rows = y.sizes()[0];
  a.slots = data_of<const int32_t>(&slots);
  a.num_rows = data_of<const int32_t>(&offsets) + (offsets.numel() - 1);
  a.weights = data_of<const float>(weights);
  a.m = (uint32_t)m;
  a.experts_per_token = (uint32_t)slots.sizes()[1];
  a.hidden_dim = (uint64_t)y.sizes()[1];
  A2A_CHECK(pplx_a2a_unsort_tokens_backward(y.device().index(), &a, current_stream_of(y)));
  if (grad_y) written(*grad_y);
  if (grad_weights) written(*grad_weights);
}

// Where the rows of x [rows, ..] or [experts, rows, ..] lie.
pplx_a2a_rows_t rows_of(const at::Tensor &x, const at::Tensor *num_tokens, const at::Tensor *offsets) {
  TORCH_CHECK(!num_tokens || !offsets, "num_tokens and offsets exclude each other");
  pplx_a2a_rows_t r{};
  if (num_tokens) {
    TORCH_CHECK(x.dim() == 3, "num_tokens goes with rows [experts, rows, ..]");
    check_dense(*num_tokens, at::kInt, 1, x, "num_tokens");
    TORCH_CHECK(num_tokens->sizes()[0] == x.sizes()[0], "num_tokens must have an entry for each expert");
    TORCH_CHECK(x.sizes()[0] >= 1 && x.sizes()[0] <= UINT32_MAX, "pplx_kernels: invalid argument: number of experts");
    r.layout = PPLX_A2A_ROWS_PADDED;
    r.num_experts = (uint32_t)x.sizes()[0];
    r.rows = (uint64_t)x.sizes()[1];
    r.starts_or_counts = data_of<const int32_t>(num_tokens);
  } else {
    TORCH_CHECK(x.dim() == 2, "rows [experts, rows, ..] need num_tokens");
    r.rows = (uint64_t)x.sizes()[0];
    r.num_experts = 1;
    if (offsets) {
      check_dense(*offsets, at::kInt, 1, x, "offsets");
      TORCH_CHECK(offsets->numel() >= 2 && offsets->numel() <= UINT32_MAX, "offsets must be [experts + 1]");
      r.layout = PPLX_A2A_ROWS_SORTED;
      r.num_experts = (uint32_t)(offsets->numel() - 1);
      r.starts_or_counts = data_of<const int32_t>(offsets);
    }
  }
  return r;
}

// Shape and strides of what goes along with x: [.., width], or one number for each row (width < 0).
void check_beside(const at::Tensor &t, const at::Tensor &x, int64_t width, const char *name) {
  check_on(t, x, name);
  const int64_t dims = x.dim() - (width < 0 ? 1 : 0);
  bool same = t.dim() == dims;
  for (int64_t d = 0; same && d < x.dim() - 1; ++d) same = t.sizes()[d] == x.sizes()[d];
  if (same && width >= 0) same = t.sizes()[dims - 1] == width;
  TORCH_CHECK(same, name, " must have the rows of x", width < 0 ? "" : " and ", width < 0 ? "" : std::to_string(width),
              width < 0 ? "" : " columns");
}

void quantize_rows(const at::Tensor &out, const at::Tensor &scale, const at::Tensor &x, const at::Tensor *num_tokens,
                   const at::Tensor *offsets, bool swiglu) {
  TORCH_CHECK(x.is_cuda(), "Tensor x must be on GPU");
  check_float(x, "x");
  TORCH_CHECK(x.dim() == 2 || x.dim() == 3, "Tensor x must be 2 or 3 dimensional");
  check_rows_of(x, "x");
  pplx_a2a_quantize_args_t a{};
  a.rows = rows_of(x, num_tokens, offsets);
  const int64_t row = x.dim() - 2, columns = x.sizes()[row + 1];
  TORCH_CHECK(!swiglu || columns % 2 == 0, "swiglu takes rows of two halves");
  const int64_t width = swiglu ? columns / 2 : columns;
  TORCH_CHECK(out.scalar_type() == at::kChar, "out must be of type Char");
  check_beside(out, x, width, "out");
  check_rows_of(out, "out");
  TORCH_CHECK(scale.scalar_type() == at::kFloat, "scale must be of type Float");
  check_beside(scale, x, -1, "scale");
  check_written(out, "out", {&x, num_tokens, offsets, &scale});
  check_written(scale, "scale", {&x, num_tokens, offsets});
  const bool padded = row == 1;
  a.out = out.data_ptr();
  a.out_stride_row = byte_step_of(out, row);
  a.out_stride_expert = padded ? byte_step_of(out, 0) : 0;
  a.out_scale = data_of<float>(&scale);
  a.out_scale_stride_row = step_of(scale, row);
  a.out_scale_stride_expert = padded ? step_of(scale, 0) : 0;
  a.x = x.data_ptr();
  a.x_stride_row = byte_step_of(x, row);
  a.x_stride_expert = padded ? byte_step_of(x, 0) : 0;
  a.dtype = dtype_code(x.scalar_type());
  a.swiglu = swiglu;
  a.width = (uint64_t)width;
  A2A_CHECK(pplx_a2a_quantize_rows(x.device().index(), &a, current_stream_of(x)));
  written(out);
  written(scale);
}

void int8_matmul(const at::Tensor &out, const at::Tensor &x, const at::Tensor &x_scale, const at::Tensor &weight,
                 const at::Tensor &weight_scale, const at::Tensor *num_tokens, const at::Tensor *offsets) {
  TORCH_CHECK(x.is_cuda(), "Tensor x must be on GPU");
  TORCH_CHECK(x.scalar_type() == at::kChar, "x must be of type Char");
  TORCH_CHECK(x.dim() == 2 || x.dim() == 3, "Tensor x must be 2 or 3 dimensional");
  check_rows_of(x, "x");
  pplx_a2a_int8_matmul_args_t a{};
  a.rows = rows_of(x, num_tokens, offsets);
  const int64_t row = x.dim() - 2, depth = x.sizes()[row + 1];
  const bool experts = num_tokens || offsets;
  check_dense(weight, at::kChar, experts ? 3 : 2, x, "weight");
  const int64_t n = weight.sizes()[experts ? 1 : 0];
  TORCH_CHECK(weight.sizes()[experts ? 2 : 1] == depth, "weight and x must have rows of one length");
  TORCH_CHECK(!experts || weight.sizes()[0] == (int64_t)a.rows.num_experts, "weight must have an entry for each of the ",
              a.rows.num_experts, " experts");
  check_dense(weight_scale, at::kFloat, experts ? 2 : 1, x, "weight_scale");
  TORCH_CHECK(weight_scale.sizes() == weight.sizes().slice(0, experts ? 2 : 1), "weight_scale must have an entry for each row of weight");
  TORCH_CHECK(x_scale.scalar_type() == at::kFloat, "x_scale must be of type Float");
  check_beside(x_scale, x, -1, "x_scale");
  check_float(out, "out");
  check_beside(out, x, n, "out");
  TORCH_CHECK(n <= 1 || out.strides()[row + 1] == 1, "the rows of out must be contiguous");
  check_written(out, "out", {&x, &x_scale, &weight, &weight_scale, num_tokens, offsets});
  const bool padded = row == 1;
  a.out = out.data_ptr();
  a.out_stride_row = step_of(out, row);
  a.out_stride_expert = padded ? step_of(out, 0) : 0;
  a.out_dtype = dtype_code(out.scalar_type());
  a.x = data_of<const int8_t>(&x);
  a.x_stride_row = byte_step_of(x, row);
  a.x_stride_expert = padded ? byte_step_of(x, 0) : 0;
  a.x_scale = data_of<const float>(&x_scale);
  a.x_scale_stride_row = step_of(x_scale, row);
  a.x_scale_stride_expert = padded ? step_of(x_scale, 0) : 0;
  a.weight = data_of<const int8_t>(&weight);
  a.weight_scale = data_of<const float>(&weight_scale);
  a.n = (uint64_t)n;
  a.k = (uint64_t)depth;
  A2A_CHECK(pplx_a2a_int8_matmul(x.device().index(), &a, current_stream_of(x)));
  written(out);
}

// ---------------------------------------------------------------------------
// The registered ops
// ---------------------------------------------------------------------------
void sort_tokens_op(at::Tensor &rows, opt_tensor scale, at::Tensor &slots, at::Tensor &offsets, opt_tensor workspace,
                    const at::Tensor &x, const at::Tensor &indices, opt_tensor bound_m) {
  sort_tokens(rows, opt(scale), slots, offsets, opt(workspace), x, indices, opt(bound_m));
}
void unsort_tokens_op(at::Tensor &out, const at::Tensor &y, const at::Tensor &slots, opt_tensor weights) {
  unsort_tokens(out, y, slots, opt(weights));
}
void unsort_tokens_backward_op(opt_tensor grad_y, opt_tensor grad_weights, const at::Tensor &grad_out, const at::Tensor &y,
                               const at::Tensor &slots, const at::Tensor &offsets, opt_tensor weights) {
  unsort_tokens_backward(opt(grad_y), opt(grad_weights), grad_out, y, slots, offsets, opt(weights));
}
void quantize_rows_op(at::Tensor &out, at::Tensor &scale, const at::Tensor &x, opt_tensor num_tokens, opt_tensor offsets,
                      bool swiglu) {
  quantize_rows(out, scale, x, opt(num_tokens), opt(offsets), swiglu);
}
void int8_matmul_op(at::Tensor &out, const at::Tensor &x, const at::Tensor &x_scale, const at::Tensor &weight,
                    const at::Tensor &weight_scale, opt_tensor num_tokens, opt_tensor offsets) {
  int8_matmul(out, x, x_scale, weight, weight_scale, opt(num_tokens), opt(offsets));
}
int64_t sort_workspace_op(int64_t m, int64_t k, int64_t experts) {
  TORCH_CHECK(m >= 0 && k >= 0, "pplx_kernels: invalid argument: negative size");
  return (int64_t)((sort_workspace(m, k, experts) + 3) / 4);
}

// ---------------------------------------------------------------------------
// The differentiable ones, which make their results
// ---------------------------------------------------------------------------
struct Sorted {
  at::Tensor rows, scale, slots, offsets, workspace;
};

Sorted new_sorted(const at::Tensor &x, const at::Tensor &indices, int64_t experts, bool int8) {
  TORCH_CHECK(x.dim() == 2, "Tensor x must be 2 dimensional");
  TORCH_CHECK(indices.dim() == 2, "Tensor indices must be 2 dimensional");
  TORCH_CHECK(experts >= 1, "pplx_kernels: invalid argument: num_experts must be positive");
  const int64_t m = indices.sizes()[0], k = indices.sizes()[1], words = (int64_t)(sort_workspace(m, k, experts) / 4);
  Sorted s;
  s.rows = fresh({m * k, x.sizes()[1]}, x, int8 ? at::kChar : x.scalar_type());
  if (int8) s.scale = fresh({m * k}, x, at::kFloat);
  s.slots = fresh({m, k}, x, at::kInt);
  s.offsets = fresh({experts + 1}, x, at::kInt);
  if (words) s.workspace = fresh({words}, x, at::kInt);
  return s;
}

Sorted sort_new(const at::Tensor &x, const at::Tensor &indices, int64_t experts, const at::Tensor *bound_m, bool int8) {
  TORCH_CHECK(x.is_cuda(), "Tensor x must be on GPU");
  Sorted s = new_sorted(x, indices, experts, int8);
  sort_tokens(s.rows, defined(s.scale), s.slots, s.offsets, defined(s.workspace), x, indices, bound_m);
  return s;
}

// (rows, scale, slots, offsets); without int8 the scale is empty
using SortedTuple = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
SortedTuple as_tuple(const Sorted &s) {
  return {s.rows, s.scale.defined() ? s.scale : fresh({0}, s.rows, at::kFloat), s.slots, s.offsets};
}
SortedTuple sorted_tokens_op(const at::Tensor &x, const at::Tensor &indices, int64_t experts, opt_tensor bound_m, bool int8) {
  return as_tuple(sort_new(x, indices, experts, opt(bound_m), int8));
}
SortedTuple sorted_tokens_meta(const at::Tensor &x, const at::Tensor &indices, int64_t experts, opt_tensor, bool int8) {
  TORCH_CHECK(x.dim() == 2, "Tensor x must be 2 dimensional");
  TORCH_CHECK(indices.dim() == 2, "Tensor indices must be 2 dimensional");
  const c10::SymInt m = indices.sym_size(0), k = indices.sym_size(1);
  return {fresh_traced({m * k, x.sym_size(1)}, x, int8 ? at::kChar : x.scalar_type()),
          fresh_traced({int8 ? m * k : c10::SymInt(0)}, x, at::kFloat), fresh_traced({m, k}, x, at::kInt),
          fresh({experts + 1}, x, at::kInt)};
}

at::Tensor unsorted_tokens_meta(const at::Tensor &y, const at::Tensor &slots, const at::Tensor &, opt_tensor,
                                std::optional<at::ScalarType> out_dtype) {
  TORCH_CHECK(y.dim() == 2, "Tensor y must be 2 dimensional");
  TORCH_CHECK(slots.dim() == 2, "Tensor slots must be 2 dimensional");
  return fresh_traced({slots.sym_size(0), y.sym_size(1)}, y, out_dtype.value_or(y.scalar_type()));
}
at::Tensor unsorted_tokens_op(const at::Tensor &y, const at::Tensor &slots, const at::Tensor &offsets, opt_tensor weights,
                              std::optional<at::ScalarType> out_dtype) {
  TORCH_CHECK(y.is_cuda(), "Tensor y must be on GPU");
  TORCH_CHECK(y.dim() == 2, "Tensor y must be 2 dimensional");
  TORCH_CHECK(slots.dim() == 2, "Tensor slots must be 2 dimensional");
  check_offsets(offsets, y);  // (the gradient reads them)
  at::Tensor out = fresh({slots.sizes()[0], y.sizes()[1]}, y, out_dtype.value_or(y.scalar_type()));
  unsort_tokens(out, y, slots, opt(weights));
  return out;
}

constexpr char kDifferentiable[] = "sort_tokens and unsort_tokens";  // (in messages)

SortedTuple call_sorted_tokens(const at::Tensor &x, const at::Tensor &indices, int64_t experts, opt_tensor bound_m, bool int8) {
  at::AutoDispatchBelowADInplaceOrView below;
  static auto op = op_handle<SortedTuple(const at::Tensor &, const at::Tensor &, int64_t, opt_tensor, bool)>(
      "pplx_kernels::sorted_tokens");
  return op.call(x, indices, experts, bound_m, int8);
}

struct SortFunction : torch::autograd::Function<SortFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x,
                                                const at::Tensor &indices, int64_t experts,
                                                const std::optional<at::Tensor> &bound_m) {
    auto [rows, scale, slots, offsets] = call_sorted_tokens(x, indices, experts, bound_m, false);
    ctx->save_for_backward({slots});
    ctx->mark_non_differentiable({scale, slots, offsets});
    ctx->set_materialize_grads(false);
    return {rows, scale, slots, offsets};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    at::Tensor grad_x;
    check_no_tangent({&grads[0]}, kDifferentiable);
    if (grads[0].defined()) {
      const at::Tensor slots = ctx->get_saved_variables()[0];
      at::NoGradGuard plain;
      static auto op = op_handle<void(at::Tensor &, const at::Tensor &, const at::Tensor &, opt_tensor)>(
          "pplx_kernels::unsort_tokens");
      const at::Tensor g = as_rows(grads[0]);
      grad_x = fresh_traced({slots.sym_size(0), g.sym_size(1)}, g, g.scalar_type());
      op.call(grad_x, g, slots, std::nullopt);
    }
    return differentiable_once({grad_x, at::Tensor(), at::Tensor(), at::Tensor()}, kDifferentiable);
  }
};

struct UnsortFunction : torch::autograd::Function<UnsortFunction> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &y, const at::Tensor &slots,
                            const at::Tensor &offsets, const std::optional<at::Tensor> &weights,
                            std::optional<at::ScalarType> out_dtype) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = op_handle<at::Tensor(const at::Tensor &, const at::Tensor &, const at::Tensor &, opt_tensor,
                                          std::optional<at::ScalarType>)>("pplx_kernels::unsorted_tokens");
    at::Tensor out = op.call(y, slots, offsets, weights, out_dtype);
    ctx->save_for_backward({y, slots, offsets, weights.value_or(at::Tensor())});
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &y = saved[0], &weights = saved[3];
    at::Tensor grad_y, grad_weights;
    check_no_tangent({&grads[0], &y, &weights}, kDifferentiable);
    {
      at::NoGradGuard plain;
      static auto op = op_handle<void(opt_tensor, opt_tensor, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                                      const at::Tensor &, opt_tensor)>("pplx_kernels::unsort_tokens_backward");
      if (ctx->needs_input_grad(0)) grad_y = fresh_traced(y.sym_sizes(), y, y.scalar_type());
      if (weights.defined() && ctx->needs_input_grad(3)) grad_weights = fresh_traced(weights.sym_sizes(), weights, at::kFloat);
      auto if_defined = [](const at::Tensor &t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; };
      if (saved[1].sym_size(0) == 0) {  // (without tokens)
        if (grad_y.defined()) grad_y.zero_();
      } else {
        op.call(if_defined(grad_y), if_defined(grad_weights), as_rows(grads[0]), y, saved[1], saved[2], if_defined(weights));
      }
    }
    return differentiable_once({grad_y, at::Tensor(), at::Tensor(), grad_weights, at::Tensor()}, kDifferentiable);
  }
};

SortedTuple sorted_tokens_autograd(const at::Tensor &x, const at::Tensor &indices, int64_t experts, opt_tensor bound_m,
                                   bool int8) {
  if (int8) return call_sorted_tokens(x, indices, experts, bound_m, true);
  check_no_tangent({&x}, kDifferentiable);
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    TORCH_CHECK(x.dim() == 2 && x.sym_size(1) % 8 == 0, "x must have rows of a multiple of 8 elements for its gradient");
  }
  auto made = SortFunction::apply(x, indices, experts, bound_m);
  return {made[0], made[1], made[2], made[3]};
}
at::Tensor unsorted_tokens_autograd(const at::Tensor &y, const at::Tensor &slots, const at::Tensor &offsets,
                                    opt_tensor weights, std::optional<at::ScalarType> out_dtype) {
  check_no_tangent({&y, opt(weights)}, kDifferentiable);
  return UnsortFunction::apply(y, slots, offsets, weights, out_dtype);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pplx_kernels, m) {
  define(m, "sort_tokens",
         "(Tensor! rows, Tensor!? scale, Tensor! slots, Tensor! offsets, Tensor!? workspace, Tensor x, Tensor indices, "
         "Tensor? bound_m) -> ()",
         &sort_tokens_op);
  define(m, "unsort_tokens", "(Tensor! out, Tensor y, Tensor slots, Tensor? weights) -> ()", &unsort_tokens_op);
  define(m, "unsort_tokens_backward",
         "(Tensor!? grad_y, Tensor!? grad_weights, Tensor grad_out, Tensor y, Tensor slots, Tensor offsets, "
         "Tensor? weights) -> ()",
         &unsort_tokens_backward_op);
  define(m, "quantize_rows",
         "(Tensor! out, Tensor! scale, Tensor x, Tensor? num_tokens, Tensor? offsets, bool swiglu) -> ()", &quantize_rows_op);
  define(m, "int8_matmul",
         "(Tensor! out, Tensor x, Tensor x_scale, Tensor weight, Tensor weight_scale, Tensor? num_tokens, Tensor? offsets) "
         "-> ()",
         &int8_matmul_op);
  m.def("sorted_tokens(Tensor x, Tensor indices, int num_experts, Tensor? bound_m, bool int8) -> (Tensor, Tensor, Tensor, Tensor)");
  m.impl("sorted_tokens", c10::kCUDA, &sorted_tokens_op);
  m.impl("sorted_tokens", c10::kMeta, &sorted_tokens_meta);
  m.impl("sorted_tokens", c10::DispatchKey::Autograd, &sorted_tokens_autograd);
  m.def("unsorted_tokens(Tensor y, Tensor slots, Tensor offsets, Tensor? weights, ScalarType? out_dtype) -> Tensor");
  m.impl("unsorted_tokens", c10::kCUDA, &unsorted_tokens_op);
  m.impl("unsorted_tokens", c10::kMeta, &unsorted_tokens_meta);
  m.impl("unsorted_tokens", c10::DispatchKey::Autograd, &unsorted_tokens_autograd);
  m.def("sort_workspace", &sort_workspace_op);
}

// ---------------------------------------------------------------------------
// Functions of pplx_kernels._C
// ---------------------------------------------------------------------------
namespace {

// sort_tokens(x, indices, num_experts, bound_m, int8) -> (rows, scale, slots, offsets, workspace): on new tensors
PyObject *py_sort_tokens(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("sort_tokens", nargs, 5);
  const at::Tensor &x = tensor_arg(args[0], "x"), &indices = tensor_arg(args[1], "indices");
  const int64_t experts = int_arg(args[2], "num_experts");
  const at::Tensor *bound_m = optional_tensor_arg(args[3], "bound_m");
  const bool int8 = bool_arg(args[4]);
  Sorted s;
  if (straight({&x, &indices, bound_m})) {
    s = sort_new(x, indices, experts, bound_m, int8);
  } else {
    static auto op = op_handle<decltype(sorted_tokens_op)>("pplx_kernels::sorted_tokens");
    std::tie(s.rows, s.scale, s.slots, s.offsets) = op.call(x, indices, experts, maybe(bound_m), int8);
    if (!int8) s.scale = at::Tensor();
  }
  PyObject *out = PyTuple_New(5);
  if (!out) throw python_error();
  const at::Tensor *made[] = {&s.rows, &s.scale, &s.slots, &s.offsets, &s.workspace};
  for (int i = 0; i < 5; ++i) PyTuple_SET_ITEM(out, i, wrap_or_none(*made[i]));
  return out;
  END_HANDLE_TH_ERRORS
}

// sort_tokens_out(rows, scale, slots, offsets, workspace, x, indices, bound_m)
PyObject *py_sort_tokens_out(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("sort_tokens_out", nargs, 8);
  const at::Tensor &rows = tensor_arg(args[0], "rows"), &slots = tensor_arg(args[2], "slots"),
                   &offsets = tensor_arg(args[3], "offsets"), &x = tensor_arg(args[5], "x"),
                   &indices = tensor_arg(args[6], "indices");
  const at::Tensor *scale = optional_tensor_arg(args[1], "scale"), *workspace = optional_tensor_arg(args[4], "workspace"),
                   *bound_m = optional_tensor_arg(args[7], "bound_m");
  if (straight({&rows, scale, &slots, &offsets, workspace, &x, &indices, bound_m})) {
    sort_tokens(rows, scale, slots, offsets, workspace, x, indices, bound_m);
  } else {
    static auto op = op_handle<decltype(sort_tokens_op)>("pplx_kernels::sort_tokens");
    at::Tensor to_rows = rows, to_slots = slots, to_offsets = offsets;
    op.call(to_rows, maybe(scale), to_slots, to_offsets, maybe(workspace), x, indices, maybe(bound_m));
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// differentiable: sorted_tokens(x, indices, num_experts, bound_m) -> (rows, slots, offsets)
PyObject *py_sorted_tokens(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("sorted_tokens", nargs, 4);
  const at::Tensor *bound_m = optional_tensor_arg(args[3], "bound_m");
  auto [rows, scale, slots, offsets] =
      sorted_tokens_autograd(tensor_arg(args[0], "x"), tensor_arg(args[1], "indices"), int_arg(args[2], "num_experts"),
                             bound_m ? std::optional<at::Tensor>(*bound_m) : std::nullopt, false);
  PyObject *out = PyTuple_New(3);
  if (!out) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(rows));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(slots));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(offsets));
  return out;
  END_HANDLE_TH_ERRORS
}

// differentiable: unsorted_tokens(y, slots, offsets, weights, out_dtype) -> out
PyObject *py_unsorted_tokens(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("unsorted_tokens", nargs, 5);
  const at::Tensor *weights = optional_tensor_arg(args[3], "weights");
  std::optional<at::ScalarType> dtype;
  if (args[4] != Py_None) {
    TORCH_CHECK_TYPE(THPDtype_Check(args[4]), "out_dtype must be a torch.dtype");
    dtype = reinterpret_cast<THPDtype *>(args[4])->scalar_type;
  }
  return THPVariable_Wrap(unsorted_tokens_autograd(tensor_arg(args[0], "y"), tensor_arg(args[1], "slots"),
                                                   tensor_arg(args[2], "offsets"),
                                                   weights ? std::optional<at::Tensor>(*weights) : std::nullopt, dtype));
  END_HANDLE_TH_ERRORS
}

// unsort_tokens(out, y, slots, weights)
PyObject *py_unsort_tokens(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("unsort_tokens", nargs, 4);
  const at::Tensor &out = tensor_arg(args[0], "out"), &y = tensor_arg(args[1], "y"), &slots = tensor_arg(args[2], "slots");
  const at::Tensor *weights = optional_tensor_arg(args[3], "weights");
  if (straight({&out, &y, &slots, weights})) {
    unsort_tokens(out, y, slots, weights);
  } else {
    static auto op = op_handle<decltype(unsort_tokens_op)>("pplx_kernels::unsort_tokens");
    at::Tensor to = out;
    op.call(to, y, slots, maybe(weights));
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// unsort_tokens_backward(grad_y, grad_weights, grad_out, y, slots, offsets, weights)
PyObject *py_unsort_tokens_backward(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("unsort_tokens_backward", nargs, 7);
  const at::Tensor *grad_y = optional_tensor_arg(args[0], "grad_y"), *grad_weights = optional_tensor_arg(args[1], "grad_weights"),
                   *weights = optional_tensor_arg(args[6], "weights");
  const at::Tensor &grad_out = tensor_arg(args[2], "grad_out"), &y = tensor_arg(args[3], "y"), &slots = tensor_arg(args[4], "slots"),
                   &offsets = tensor_arg(args[5], "offsets");
  if (straight({grad_y, grad_weights, &grad_out, &y, &slots, &offsets, weights})) {
    unsort_tokens_backward(grad_y, grad_weights, grad_out, y, slots, offsets, weights);
  } else {
    static auto op = op_handle<decltype(unsort_tokens_backward_op)>("pplx_kernels::unsort_tokens_backward");
    op.call(maybe(grad_y), maybe(grad_weights), grad_out, y, slots, offsets, maybe(weights));
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// quantize_rows(out, scale, x, num_tokens, offsets, swiglu)
PyObject *py_quantize_rows(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("quantize_rows", nargs, 6);
  const at::Tensor &out = tensor_arg(args[0], "out"), &scale = tensor_arg(args[1], "scale"), &x = tensor_arg(args[2], "x");
  const at::Tensor *num_tokens = optional_tensor_arg(args[3], "num_tokens"), *offsets = optional_tensor_arg(args[4], "offsets");
  const bool swiglu = bool_arg(args[5]);
  if (straight({&out, &scale, &x, num_tokens, offsets})) {
    quantize_rows(out, scale, x, num_tokens, offsets, swiglu);
  } else {
    static auto op = op_handle<decltype(quantize_rows_op)>("pplx_kernels::quantize_rows");
    at::Tensor to = out, to_scale = scale;
    op.call(to, to_scale, x, maybe(num_tokens), maybe(offsets), swiglu);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// int8_matmul(out, x, x_scale, weight, weight_scale, num_tokens, offsets)
PyObject *py_int8_matmul(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("int8_matmul", nargs, 7);
  const at::Tensor &out = tensor_arg(args[0], "out"), &x = tensor_arg(args[1], "x"), &x_scale = tensor_arg(args[2], "x_scale"),
                   &weight = tensor_arg(args[3], "weight"), &weight_scale = tensor_arg(args[4], "weight_scale");
  const at::Tensor *num_tokens = optional_tensor_arg(args[5], "num_tokens"), *offsets = optional_tensor_arg(args[6], "offsets");
  if (straight({&out, &x, &x_scale, &weight, &weight_scale, num_tokens, offsets})) {
    int8_matmul(out, x, x_scale, weight, weight_scale, num_tokens, offsets);
  } else {
    static auto op = op_handle<decltype(int8_matmul_op)>("pplx_kernels::int8_matmul");
    at::Tensor to = out;
    op.call(to, x, x_scale, weight, weight_scale, maybe(num_tokens), maybe(offsets));
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#ifndef PPLX_EXPERTS_SOURCE_ID
#define PPLX_EXPERTS_SOURCE_ID "unknown"
#endif
PyObject *py_experts_build_id(PyObject *, PyObject *) { return PyUnicode_FromString(PPLX_EXPERTS_SOURCE_ID); }
#ifndef PPLX_EXPERTS_HEADERS_ID
#define PPLX_EXPERTS_HEADERS_ID "unknown"
#endif
PyObject *py_experts_headers_id(PyObject *, PyObject *) { return PyUnicode_FromString(PPLX_EXPERTS_HEADERS_ID); }

#define PPLX_FASTCALL(fn) (PyCFunction)(void (*)(void))fn, METH_FASTCALL
PyMethodDef kExpertsMethods[] = {
    {"sort_tokens", PPLX_FASTCALL(py_sort_tokens),
     "sort_tokens(x, indices, num_experts, bound_m, int8) -> (rows, scale, slots, offsets, workspace)"},
    {"sort_tokens_out", PPLX_FASTCALL(py_sort_tokens_out),
     "sort_tokens_out(rows, scale, slots, offsets, workspace, x, indices, bound_m)"},
    {"sorted_tokens", PPLX_FASTCALL(py_sorted_tokens),
     "sorted_tokens(x, indices, num_experts, bound_m) -> (rows, slots, offsets), differentiable"},
    {"unsorted_tokens", PPLX_FASTCALL(py_unsorted_tokens),
     "unsorted_tokens(y, slots, offsets, weights, out_dtype) -> out, differentiable"},
    {"unsort_tokens", PPLX_FASTCALL(py_unsort_tokens), "unsort_tokens(out, y, slots, weights)"},
    {"unsort_tokens_backward", PPLX_FASTCALL(py_unsort_tokens_backward),
     "unsort_tokens_backward(grad_y, grad_weights, grad_out, y, slots, offsets, weights)"},
    {"quantize_rows", PPLX_FASTCALL(py_quantize_rows), "quantize_rows(out, scale, x, num_tokens, offsets, swiglu)"},
    {"int8_matmul", PPLX_FASTCALL(py_int8_matmul),
     "int8_matmul(out, x, x_scale, weight, weight_scale, num_tokens, offsets)"},
    {"experts_build_id", py_experts_build_id, METH_NOARGS, "hash of the sources that these functions were built from"},
    {"experts_headers_id", py_experts_headers_id, METH_NOARGS, "hash of the binding's headers that they were built with"},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

PyMethodDef *experts_methods() { return kExpertsMethods; }
