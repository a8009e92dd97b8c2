// The torch layer of the operators before dispatch: ops of pplx_kernels that write tensors of the caller, those that make their
// results and have gradients, and the same as functions of pplx_kernels._C (pplx_kernels/router.py).
#include <tuple>

#include "torch_tensors.h"

namespace {

// ---------------------------------------------------------------------------
// Checks
// ---------------------------------------------------------------------------
uint32_t tokens_of(const at::Tensor &x) {
  TORCH_CHECK(x.sizes()[0] < (1ll << 31), "pplx_kernels: unsupported: 2^31 tokens or more");
  return (uint32_t)x.sizes()[0];
}

// Rows [tokens, columns] of one type, 16-byte aligned.
void check_matrix(const at::Tensor &x, const char *name) {
  TORCH_CHECK(x.is_cuda(), "Tensor ", name, " must be on GPU");
  TORCH_CHECK(x.dim() == 2, "Tensor ", name, " must be 2 dimensional");
  check_float(x, name);
  check_rows_of(x, name);
}
void check_like(const at::Tensor &t, const at::Tensor &x, const char *name, const char *of) {
  check_on(t, x, name);
  TORCH_CHECK(t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type(), name, " must have the shape and dtype of ", of);
  check_rows_of(t, name);
}
// Rows whose elements lie in one piece, at any element.
void check_lines(const at::Tensor &x, const char *name) {
  TORCH_CHECK(x.dim() == 2, "Tensor ", name, " must be 2 dimensional");
  check_float(x, name);
  TORCH_CHECK(x.sizes()[1] <= 1 || x.strides()[1] == 1, "the rows of ", name, " must be contiguous");
}
void check_weight_type(const at::Tensor &weight, const at::Tensor &x) {
  TORCH_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat,
              "weight must have the dtype of x or be of type Float");
}

// `out` may be `x` itself: the same elements at the same places.
bool is_same(const at::Tensor *out, const at::Tensor *x) {
  return out && x && out->data_ptr() == x->data_ptr() && out->sizes() == x->sizes() && step_of(*out, 0) == step_of(*x, 0) &&
         out->scalar_type() == x->scalar_type();
}
const at::Tensor *unless_same(const at::Tensor *x, const at::Tensor *out) { return is_same(out, x) ? nullptr : x; }

float as_float(double v) { return (float)v; }

// Bytes for a call's own use: the caller's, `given`, checked against what else the call reads and writes, or memory of torch's
// allocator, which goes back to it with the call: a later one on the same stream may have it, and a capture by torch keeps it in its
// graph's pool.
at::Tensor space(uint64_t bytes, const at::Tensor &with, const at::Tensor *given, std::initializer_list<const at::Tensor *> others) {
  if (!given) return fresh({(int64_t)bytes}, with, at::kByte);
  check_dense(*given, at::kByte, 1, with, "workspace");
  TORCH_CHECK((uint64_t)given->numel() >= bytes, "the workspace has fewer than ", bytes, " bytes");
  TORCH_CHECK(bytes == 0 || reinterpret_cast<uintptr_t>(given->data_ptr()) % 16 == 0, "workspace must be 16-byte aligned");
  if (bytes) check_written(*given, "workspace", others);
  return *given;
}

// ---------------------------------------------------------------------------
// The operators on tensors of the caller
// ---------------------------------------------------------------------------
constexpr int64_t kBlock = 128;  // columns that share a scale of e4m3 rows

void rms_norm(const at::Tensor *y, const at::Tensor *sum, const at::Tensor *q, const at::Tensor *scale, const at::Tensor &x,
              const at::Tensor &weight, const at::Tensor *residual, double eps) {
  check_matrix(x, "x");
  const int64_t m = x.sizes()[0], h = x.sizes()[1];
  check_weight_type(weight, x);
  check_dense(weight, weight.scalar_type(), 1, x, "weight");
  TORCH_CHECK(weight.sizes()[0] == h, "weight must be [", h, "]");
  TORCH_CHECK((residual != nullptr) == (sum != nullptr), "sum goes with residual");
  TORCH_CHECK((q != nullptr) == (scale != nullptr), "scale goes with q");
  if (residual) {
    check_like(*residual, x, "residual", "x");
    check_like(*sum, x, "sum", "x");
    check_written(*sum, "sum", {unless_same(&x, sum), unless_same(residual, sum), &weight, y, q, scale});
  }
  if (y) {
    check_like(*y, x, "y", "x");
    check_written(*y, "y", {unless_same(&x, y), unless_same(residual, y), &weight, q, scale});
  }
  pplx_a2a_rms_norm_args_t a{};
  if (q) {
    check_on(*q, x, "q");
    TORCH_CHECK(q->sizes() == x.sizes(), "q must have the shape of x");
    check_rows_of(*q, "q");
    TORCH_CHECK(q->scalar_type() == at::kChar || q->scalar_type() == at::kFloat8_e4m3fn, "q must be of type Char or Float8_e4m3fn");
    a.format = q->scalar_type() == at::kChar ? PPLX_A2A_ROWS_INT8 : PPLX_A2A_ROWS_E4M3;
    check_on(*scale, x, "scale");
    TORCH_CHECK(scale->scalar_type() == at::kFloat, "scale must be of type Float");
    const int64_t blocks = (h + kBlock - 1) / kBlock;
    if (a.format == PPLX_A2A_ROWS_INT8) {
      TORCH_CHECK(scale->dim() == 1 && scale->sizes()[0] == m, "scale must be [", m, "]");
    } else {
      TORCH_CHECK(scale->dim() == 2 && scale->sizes()[0] == m && scale->sizes()[1] == blocks, "scale must be [", m, ", ", blocks, "]");
    }
    check_written(*q, "q", {&x, residual, &weight, scale});
    check_written(*scale, "scale", {&x, residual, &weight});
    a.q = q->data_ptr();
    a.q_stride_row = byte_step_of(*q, 0);
    a.scale = data_of<float>(scale);
    a.scale_stride_row = step_of(*scale, 0);
    a.scale_stride_block = a.format == PPLX_A2A_ROWS_E4M3 ? step_of(*scale, 1) : 0;
  }
  a.x = x.data_ptr();
  a.x_stride_row = byte_step_of(x, 0);
  if (residual) {
    a.residual = residual->data_ptr();
    a.residual_stride_row = byte_step_of(*residual, 0);
    a.sum = sum->data_ptr();
    a.sum_stride_row = byte_step_of(*sum, 0);
  }
  a.weight = weight.data_ptr();
  a.dtype = dtype_code(x.scalar_type());
  a.weight_dtype = dtype_code(weight.scalar_type());
  a.eps = as_float(eps);
  a.m = tokens_of(x);
  a.hidden_dim = (uint64_t)h;
  if (y) {
    a.y = y->data_ptr();
    a.y_stride_row = byte_step_of(*y, 0);
  }
  A2A_CHECK(pplx_a2a_rms_norm(x.device().index(), &a, current_stream_of(x)));
  for (const at::Tensor *t : {y, sum, q, scale}) {
    if (t) written(*t);
  }
}

void rms_norm_backward(const at::Tensor *grad_h, const at::Tensor *grad_weight, const at::Tensor &grad_y, const at::Tensor *grad_sum,
                       const at::Tensor &h, const at::Tensor &weight, double eps, const at::Tensor *workspace) {
  check_matrix(h, "h");
  check_weight_type(weight, h);
  check_dense(weight, weight.scalar_type(), 1, h, "weight");
  TORCH_CHECK(weight.sizes()[0] == h.sizes()[1], "weight must be [", h.sizes()[1], "]");
  check_like(grad_y, h, "grad_y", "h");
  if (grad_sum) check_like(*grad_sum, h, "grad_sum", "h");
  if (grad_h) {
    check_like(*grad_h, h, "grad_h", "h");
    check_written(*grad_h, "grad_h", {unless_same(&grad_y, grad_h), unless_same(grad_sum, grad_h), &h, &weight, grad_weight});
  }
  if (grad_weight) {
    check_dense(*grad_weight, weight.scalar_type(), 1, h, "grad_weight");
    TORCH_CHECK(grad_weight->sizes() == weight.sizes(), "grad_weight must have the shape of weight");
    check_written(*grad_weight, "grad_weight", {&grad_y, grad_sum, &h, &weight});
  }
  const uint32_t m = tokens_of(h);
  if (m == 0) {
    if (grad_weight) grad_weight->zero_();
    return;
  }
  pplx_a2a_rms_norm_backward_args_t a{};
  a.grad_y = grad_y.data_ptr();
  a.grad_y_stride_row = byte_step_of(grad_y, 0);
  if (grad_sum) {
    a.grad_sum = grad_sum->data_ptr();
    a.grad_sum_stride_row = byte_step_of(*grad_sum, 0);
  }
  a.h = h.data_ptr();
  a.h_stride_row = byte_step_of(h, 0);
  a.weight = weight.data_ptr();
  a.dtype = dtype_code(h.scalar_type());
  a.weight_dtype = dtype_code(weight.scalar_type());
  a.eps = as_float(eps);
  a.m = m;
  a.hidden_dim = (uint64_t)h.sizes()[1];
  if (grad_h) {
    a.grad_h = grad_h->data_ptr();
    a.grad_h_stride_row = byte_step_of(*grad_h, 0);
  }
  at::Tensor work;
  if (grad_weight) {
    uint64_t bytes = 0;
    A2A_CHECK(pplx_a2a_rms_norm_workspace(m, a.hidden_dim, &bytes));
    work = space(bytes, h, workspace, {&grad_y, grad_sum, &h, &weight, grad_h, grad_weight});
    a.grad_weight = grad_weight->data_ptr();
    a.workspace = work.data_ptr();
  }
  A2A_CHECK(pplx_a2a_rms_norm_backward(h.device().index(), &a, current_stream_of(h)));
  if (grad_h) written(*grad_h);
  if (grad_weight) written(*grad_weight);
}

void check_router(const at::Tensor &x, const at::Tensor &weight) {
  check_matrix(x, "x");
  check_weight_type(weight, x);
  check_on(weight, x, "weight");
  check_matrix(weight, "weight");
  TORCH_CHECK(weight.sizes()[1] == x.sizes()[1], "weight and x must have rows of one length");
  TORCH_CHECK(weight.sizes()[0] <= UINT32_MAX, "pplx_kernels: invalid argument: number of experts");
}

void router_logits(const at::Tensor &logits, const at::Tensor &x, const at::Tensor &weight, const at::Tensor *workspace) {
  check_router(x, weight);
  check_on(logits, x, "logits");
  check_lines(logits, "logits");
  TORCH_CHECK(logits.scalar_type() == at::kFloat, "logits must be of type Float");
  TORCH_CHECK(logits.sizes()[0] == x.sizes()[0] && logits.sizes()[1] == weight.sizes()[0], "logits must be [", x.sizes()[0], ", ",
              weight.sizes()[0], "]");
  check_written(logits, "logits", {&x, &weight});
  pplx_a2a_router_logits_args_t a{};
  a.x = x.data_ptr();
  a.x_stride_row = byte_step_of(x, 0);
  a.weight = weight.data_ptr();
  a.weight_stride_row = byte_step_of(weight, 0);
  a.dtype = dtype_code(x.scalar_type());
  a.weight_dtype = dtype_code(weight.scalar_type());
  a.m = tokens_of(x);
  a.num_experts = (uint32_t)weight.sizes()[0];
  a.hidden_dim = (uint64_t)x.sizes()[1];
  a.logits = data_of<float>(&logits);
  a.logits_stride_row = step_of(logits, 0);
  uint64_t bytes = 0;
  A2A_CHECK(pplx_a2a_router_workspace(a.m, a.num_experts, a.hidden_dim, a.dtype, a.weight_dtype, 0, &bytes));
  at::Tensor work;
  if (bytes) {
    work = space(bytes, x, workspace, {&x, &weight, &logits});
    a.workspace = work.data_ptr();
  }
  A2A_CHECK(pplx_a2a_router_logits(x.device().index(), &a, current_stream_of(x)));
  written(logits);
}

void router_logits_backward(const at::Tensor *grad_x, const at::Tensor *grad_weight, const at::Tensor &grad_logits,
                            const at::Tensor &x, const at::Tensor &weight, const at::Tensor *workspace) {
  check_router(x, weight);
  check_on(grad_logits, x, "grad_logits");
  check_lines(grad_logits, "grad_logits");
  TORCH_CHECK(grad_logits.scalar_type() == at::kFloat, "grad_logits must be of type Float");
  TORCH_CHECK(grad_logits.sizes()[0] == x.sizes()[0] && grad_logits.sizes()[1] == weight.sizes()[0], "grad_logits must be [",
              x.sizes()[0], ", ", weight.sizes()[0], "]");
  if (grad_x) {
    check_like(*grad_x, x, "grad_x", "x");
    check_written(*grad_x, "grad_x", {&grad_logits, &x, &weight, grad_weight});
  }
  if (grad_weight) {
    check_like(*grad_weight, weight, "grad_weight", "weight");
    check_written(*grad_weight, "grad_weight", {&grad_logits, &x, &weight});
  }
  const uint32_t m = tokens_of(x);
  if (m == 0) {
    if (grad_weight) grad_weight->zero_();
    return;
  }
  pplx_a2a_router_logits_backward_args_t a{};
  a.grad_logits = data_of<const float>(&grad_logits);
  a.grad_logits_stride_row = step_of(grad_logits, 0);
  a.x = x.data_ptr();
  a.x_stride_row = byte_step_of(x, 0);
  a.weight = weight.data_ptr();
  a.weight_stride_row = byte_step_of(weight, 0);
  a.dtype = dtype_code(x.scalar_type());
  a.weight_dtype = dtype_code(weight.scalar_type());
  a.m = m;
  a.num_experts = (uint32_t)weight.sizes()[0];
  a.hidden_dim = (uint64_t)x.sizes()[1];
  if (grad_x) {
    a.grad_x = grad_x->data_ptr();
    a.grad_x_stride_row = byte_step_of(*grad_x, 0);
  }
  if (grad_weight) {
    a.grad_weight = grad_weight->data_ptr();
    a.grad_weight_stride_row = byte_step_of(*grad_weight, 0);
  }
  uint64_t bytes = 0;
  A2A_CHECK(pplx_a2a_router_workspace(m, a.num_experts, a.hidden_dim, a.dtype, a.weight_dtype, 1, &bytes));
  const at::Tensor work = space(bytes, x, workspace, {&grad_logits, &x, &weight, grad_x, grad_weight});
  a.workspace = work.data_ptr();
  A2A_CHECK(pplx_a2a_router_logits_backward(x.device().index(), &a, current_stream_of(x)));
  if (grad_x) written(*grad_x);
  if (grad_weight) written(*grad_weight);
}

struct Choice {
  int64_t num_groups, top_groups, group_top;
  bool sigmoid, renormalize;
  double scale;
};

void route_tokens(const at::Tensor &indices, const at::Tensor &weights, const at::Tensor &logits, const at::Tensor *bias,
                  const at::Tensor *bound_m, const Choice &c) {
  TORCH_CHECK(logits.is_cuda(), "Tensor logits must be on GPU");
  check_lines(logits, "logits");
  const int64_t experts = logits.sizes()[1];
  check_dense(indices, at::kUInt32, 2, logits, "indices");
  TORCH_CHECK(indices.sizes()[0] == logits.sizes()[0], "indices.size(0) must be equal to logits.size(0)");
  check_dense(weights, at::kFloat, 2, logits, "weights");
  TORCH_CHECK(weights.sizes() == indices.sizes(), "weights must have the shape of indices");
  if (bias) {
    check_dense(*bias, at::kFloat, 1, logits, "bias");
    TORCH_CHECK(bias->sizes()[0] == experts, "bias must be [", experts, "]");
  }
  check_bound_m(bound_m);
  if (bound_m) check_on(*bound_m, logits, "bound_m");
  check_written(indices, "indices", {&logits, bias, bound_m, &weights});
  check_written(weights, "weights", {&logits, bias, bound_m});
  for (int64_t v : {experts, indices.sizes()[1], c.num_groups, c.top_groups, c.group_top}) {
    TORCH_CHECK(v >= 0 && v <= UINT32_MAX, "pplx_kernels: invalid argument: size out of range");
  }
  pplx_a2a_route_args_t a{};
  a.logits = logits.data_ptr();
  a.logits_stride_row = step_of(logits, 0);
  a.dtype = dtype_code(logits.scalar_type());
  a.m = tokens_of(logits);
  a.num_experts = (uint32_t)experts;
  a.experts_per_token = (uint32_t)indices.sizes()[1];
  a.bias = data_of<const float>(bias);
  a.bound_m = data_of<const uint32_t>(bound_m);
  a.num_groups = (uint32_t)c.num_groups;
  a.top_groups = (uint32_t)c.top_groups;
  a.group_top = (uint32_t)c.group_top;
  a.scores = c.sigmoid ? PPLX_A2A_SIGMOID : PPLX_A2A_SOFTMAX;
  a.renormalize = c.renormalize;
  a.weight_scale = as_float(c.scale);
  a.indices = data_of<uint32_t>(&indices);
  a.weights = data_of<float>(&weights);
  A2A_CHECK(pplx_a2a_route_tokens(logits.device().index(), &a, current_stream_of(logits)));
  written(indices);
  written(weights);
}

void route_tokens_backward(const at::Tensor &grad_logits, const at::Tensor &grad_weights, const at::Tensor &logits,
                           const at::Tensor &indices, bool sigmoid, bool renormalize, double scale) {
  TORCH_CHECK(logits.is_cuda(), "Tensor logits must be on GPU");
  check_lines(logits, "logits");
  check_dense(indices, at::kUInt32, 2, logits, "indices");
  TORCH_CHECK(indices.sizes()[0] == logits.sizes()[0], "indices.size(0) must be equal to logits.size(0)");
  check_dense(grad_weights, at::kFloat, 2, logits, "grad_weights");
  TORCH_CHECK(grad_weights.sizes() == indices.sizes(), "grad_weights must have the shape of indices");
  check_on(grad_logits, logits, "grad_logits");
  check_lines(grad_logits, "grad_logits");
  TORCH_CHECK(grad_logits.sizes() == logits.sizes() && grad_logits.scalar_type() == logits.scalar_type(),
              "grad_logits must have the shape and dtype of logits");
  check_written(grad_logits, "grad_logits", {&grad_weights, &logits, &indices});
  TORCH_CHECK(logits.sizes()[1] <= UINT32_MAX && indices.sizes()[1] <= UINT32_MAX, "pplx_kernels: invalid argument: size out of range");
  pplx_a2a_route_backward_args_t a{};
  a.grad_weights = data_of<const float>(&grad_weights);
  a.logits = logits.data_ptr();
  a.logits_stride_row = step_of(logits, 0);
  a.indices = data_of<const uint32_t>(&indices);
  a.dtype = dtype_code(logits.scalar_type());
  a.m = tokens_of(logits);
  a.num_experts = (uint32_t)logits.sizes()[1];
  a.experts_per_token = (uint32_t)indices.sizes()[1];
  a.scores = sigmoid ? PPLX_A2A_SIGMOID : PPLX_A2A_SOFTMAX;
  a.renormalize = renormalize;
  a.weight_scale = as_float(scale);
  a.grad_logits = grad_logits.data_ptr();
  a.grad_logits_stride_row = step_of(grad_logits, 0);
  A2A_CHECK(pplx_a2a_route_tokens_backward(logits.device().index(), &a, current_stream_of(logits)));
  written(grad_logits);
}

// ---------------------------------------------------------------------------
// The registered ops
// ---------------------------------------------------------------------------
void rms_norm_op(opt_tensor y, opt_tensor sum, opt_tensor q, opt_tensor scale, const at::Tensor &x, const at::Tensor &weight,
                 opt_tensor residual, double eps) {
  rms_norm(opt(y), opt(sum), opt(q), opt(scale), x, weight, opt(residual), eps);
}
void rms_norm_backward_op(opt_tensor grad_h, opt_tensor grad_weight, const at::Tensor &grad_y, opt_tensor grad_sum,
                          const at::Tensor &h, const at::Tensor &weight, double eps, opt_tensor workspace) {
  rms_norm_backward(opt(grad_h), opt(grad_weight), grad_y, opt(grad_sum), h, weight, eps, opt(workspace));
}
void router_logits_op(at::Tensor &logits, const at::Tensor &x, const at::Tensor &weight, opt_tensor workspace) {
  router_logits(logits, x, weight, opt(workspace));
}
void router_logits_backward_op(opt_tensor grad_x, opt_tensor grad_weight, const at::Tensor &grad_logits, const at::Tensor &x,
                               const at::Tensor &weight, opt_tensor workspace) {
  router_logits_backward(opt(grad_x), opt(grad_weight), grad_logits, x, weight, opt(workspace));
}
void route_tokens_op(at::Tensor &indices, at::Tensor &weights, const at::Tensor &logits, opt_tensor bias, opt_tensor bound_m,
                     int64_t num_groups, int64_t top_groups, int64_t group_top, bool sigmoid, bool renormalize, double scale) {
  route_tokens(indices, weights, logits, opt(bias), opt(bound_m), {num_groups, top_groups, group_top, sigmoid, renormalize, scale});
}
void route_tokens_backward_op(at::Tensor &grad_logits, const at::Tensor &grad_weights, const at::Tensor &logits,
                              const at::Tensor &indices, bool sigmoid, bool renormalize, double scale) {
  route_tokens_backward(grad_logits, grad_weights, logits, indices, sigmoid, renormalize, scale);
}

// ---------------------------------------------------------------------------
// The differentiable ones, which make their results
// ---------------------------------------------------------------------------
constexpr char kDifferentiable[] = "rms_norm, router_logits and route_tokens";  // (in messages)

std::optional<at::Tensor> if_defined(const at::Tensor &t) { return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt; }

// (y, sum); without a residual the sum is empty
using Normed = std::tuple<at::Tensor, at::Tensor>;
Normed normed_rows_op(const at::Tensor &x, const at::Tensor &weight, opt_tensor residual, double eps) {
  TORCH_CHECK(x.is_cuda(), "Tensor x must be on GPU");
  TORCH_CHECK(x.dim() == 2, "Tensor x must be 2 dimensional");
  const at::Tensor y = fresh(x.sizes(), x, x.scalar_type());
  const at::Tensor sum = residual ? fresh(x.sizes(), x, x.scalar_type()) : fresh({0}, x, x.scalar_type());
  rms_norm(&y, residual ? &sum : nullptr, nullptr, nullptr, x, weight, opt(residual), eps);
  return {y, sum};
}
Normed normed_rows_meta(const at::Tensor &x, const at::Tensor &, opt_tensor residual, double) {
  TORCH_CHECK(x.dim() == 2, "Tensor x must be 2 dimensional");
  return {fresh_traced(x.sym_sizes(), x, x.scalar_type()),
          residual ? fresh_traced(x.sym_sizes(), x, x.scalar_type()) : fresh({0}, x, x.scalar_type())};
}

// (y, sum, q, scale): rows in int8, or else e4m3; without a residual there is no sum (of the registered op: it is empty)
using Quantized = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;
Quantized empty_quantized(const at::Tensor &x, bool add, bool int8) {
  TORCH_CHECK(x.dim() == 2, "Tensor x must be 2 dimensional");
  const c10::SymInt m = x.sym_size(0), h = x.sym_size(1);
  return {fresh_traced({m, h}, x, x.scalar_type()), add ? fresh_traced({m, h}, x, x.scalar_type()) : at::Tensor(),
          fresh_traced({m, h}, x, int8 ? at::kChar : at::kFloat8_e4m3fn),
          int8 ? fresh_traced({m}, x, at::kFloat) : fresh_traced({m, (h + (kBlock - 1)) / kBlock}, x, at::kFloat)};
}
Quantized quantized_rows_op(const at::Tensor &x, const at::Tensor &weight, opt_tensor residual, double eps, bool int8) {
  TORCH_CHECK(x.is_cuda(), "Tensor x must be on GPU");
  Quantized made = empty_quantized(x, residual.has_value(), int8);
  auto &[y, sum, q, scale] = made;
  rms_norm(&y, defined(sum), &q, &scale, x, weight, opt(residual), eps);
  if (!residual) sum = fresh({0}, x, x.scalar_type());
  return made;
}
Quantized quantized_rows_meta(const at::Tensor &x, const at::Tensor &, opt_tensor residual, double, bool int8) {
  Quantized made = empty_quantized(x, residual.has_value(), int8);
  if (!residual) std::get<1>(made) = fresh({0}, x, x.scalar_type());
  return made;
}

// Of both: `format` is pplx_a2a_row_format, and with rows in 8 bits these and their scales, which have no gradient, come behind y and sum.
struct NormFunction : torch::autograd::Function<NormFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight,
                                                const std::optional<at::Tensor> &residual, double eps, int64_t format) {
    at::AutoDispatchBelowADInplaceOrView below;
    torch::autograd::variable_list made, fixed;
    if (format == PPLX_A2A_ROWS_PLAIN) {
      static auto op = op_handle<decltype(normed_rows_op)>("pplx_kernels::normed_rows");
      auto [y, sum] = op.call(x, weight, residual, eps);
      made = {y, sum};
    } else {
      static auto op = op_handle<decltype(quantized_rows_op)>("pplx_kernels::quantized_rows");
      auto [y, sum, q, scale] = op.call(x, weight, residual, eps, format == PPLX_A2A_ROWS_INT8);
      made = {y, sum, q, scale};
      fixed = {q, scale};
    }
    if (!residual) fixed.push_back(made[1]);
    ctx->save_for_backward({residual ? made[1] : x, weight});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["add"] = residual.has_value();
    ctx->mark_non_differentiable(fixed);
    ctx->set_materialize_grads(false);
    return made;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &h = saved[0], &weight = saved[1];
    const bool for_x = ctx->needs_input_grad(0), for_residual = ctx->saved_data["add"].toBool() && ctx->needs_input_grad(2);
    check_no_tangent({&grads[0], &grads[1], &h, &weight}, kDifferentiable);
    at::Tensor grad_h, grad_weight;
    if (grads[0].defined()) {
      at::NoGradGuard plain;
      static auto op = op_handle<decltype(rms_norm_backward_op)>("pplx_kernels::rms_norm_backward");
      if (for_x || for_residual) grad_h = fresh_traced(h.sym_sizes(), h, h.scalar_type());
      if (ctx->needs_input_grad(1)) grad_weight = fresh_traced(weight.sym_sizes(), weight, weight.scalar_type());
      op.call(if_defined(grad_h), if_defined(grad_weight), as_rows(grads[0]),
              grads[1].defined() ? std::optional<at::Tensor>(as_rows(grads[1])) : std::nullopt, h, weight,
              ctx->saved_data["eps"].toDouble(), std::nullopt);
    } else if (grads[1].defined()) {
      grad_h = grads[1];  // (of the sum alone)
    }
    return differentiable_once(
        {for_x ? grad_h : at::Tensor(), grad_weight, for_residual ? grad_h : at::Tensor(), at::Tensor(), at::Tensor()}, kDifferentiable);
  }
};
Normed normed_rows_autograd(const at::Tensor &x, const at::Tensor &weight, opt_tensor residual, double eps) {
  check_no_tangent({&x, &weight, opt(residual)}, kDifferentiable);
  auto made = NormFunction::apply(x, weight, residual, eps, (int64_t)PPLX_A2A_ROWS_PLAIN);
  return {made[0], made[1]};
}
Quantized quantized_rows_autograd(const at::Tensor &x, const at::Tensor &weight, opt_tensor residual, double eps, bool int8) {
  check_no_tangent({&x, &weight, opt(residual)}, kDifferentiable);
  auto made = NormFunction::apply(x, weight, residual, eps, (int64_t)(int8 ? PPLX_A2A_ROWS_INT8 : PPLX_A2A_ROWS_E4M3));
  return {made[0], made[1], made[2], made[3]};
}

at::Tensor new_logits_op(const at::Tensor &x, const at::Tensor &weight) {
  TORCH_CHECK(x.is_cuda(), "Tensor x must be on GPU");
  TORCH_CHECK(x.dim() == 2, "Tensor x must be 2 dimensional");
  TORCH_CHECK(weight.dim() == 2, "Tensor weight must be 2 dimensional");
  const at::Tensor logits = fresh({x.sizes()[0], weight.sizes()[0]}, x, at::kFloat);
  router_logits(logits, x, weight, nullptr);
  return logits;
}
at::Tensor new_logits_meta(const at::Tensor &x, const at::Tensor &weight) {
  TORCH_CHECK(x.dim() == 2, "Tensor x must be 2 dimensional");
  TORCH_CHECK(weight.dim() == 2, "Tensor weight must be 2 dimensional");
  return fresh_traced({x.sym_size(0), weight.sym_size(0)}, x, at::kFloat);
}

// Gradients come in any layout (that of a sum is one element, expanded); those of a traced step have none that is known.
at::Tensor as_lines(const at::Tensor &g) {
  if (g.is_meta() || g.key_set().has(c10::DispatchKey::Python) || g.key_set().has(c10::DispatchKey::Functionalize)) return g.contiguous();
  return g.sizes()[1] <= 1 || g.strides()[1] == 1 ? g : g.contiguous();
}

struct LogitsFunction : torch::autograd::Function<LogitsFunction> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = op_handle<at::Tensor(const at::Tensor &, const at::Tensor &)>("pplx_kernels::new_logits");
    at::Tensor logits = op.call(x, weight);
    ctx->save_for_backward({x, weight});
    return logits;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &weight = saved[1];
    check_no_tangent({&grads[0], &x, &weight}, kDifferentiable);
    at::Tensor grad_x, grad_weight;
    {
      at::NoGradGuard plain;
      static auto op = op_handle<decltype(router_logits_backward_op)>("pplx_kernels::router_logits_backward");
      if (ctx->needs_input_grad(0)) grad_x = fresh_traced(x.sym_sizes(), x, x.scalar_type());
      if (ctx->needs_input_grad(1)) grad_weight = fresh_traced(weight.sym_sizes(), weight, weight.scalar_type());
      op.call(if_defined(grad_x), if_defined(grad_weight), as_lines(grads[0]), x, weight, std::nullopt);
    }
    return differentiable_once({grad_x, grad_weight}, kDifferentiable);
  }
};
at::Tensor new_logits_autograd(const at::Tensor &x, const at::Tensor &weight) {
  check_no_tangent({&x, &weight}, kDifferentiable);
  return LogitsFunction::apply(x, weight);
}

using Routed = std::tuple<at::Tensor, at::Tensor>;
Routed routed_tokens(const at::Tensor &logits, int64_t picks, const at::Tensor *bias, const at::Tensor *bound_m, const Choice &c) {
  TORCH_CHECK(logits.is_cuda(), "Tensor logits must be on GPU");
  TORCH_CHECK(logits.dim() == 2, "Tensor logits must be 2 dimensional");
  TORCH_CHECK(picks >= 1 && picks <= 64, "pplx_kernels: invalid argument: experts_per_token must be in [1, 64]");
  const at::Tensor indices = fresh({logits.sizes()[0], picks}, logits, at::kUInt32);
  const at::Tensor weights = fresh({logits.sizes()[0], picks}, logits, at::kFloat);
  route_tokens(indices, weights, logits, bias, bound_m, c);
  return {indices, weights};
}
Routed routed_tokens_op(const at::Tensor &logits, int64_t picks, opt_tensor bias, opt_tensor bound_m, int64_t num_groups,
                        int64_t top_groups, int64_t group_top, bool sigmoid, bool renormalize, double scale) {
  return routed_tokens(logits, picks, opt(bias), opt(bound_m), {num_groups, top_groups, group_top, sigmoid, renormalize, scale});
}
Routed routed_tokens_meta(const at::Tensor &logits, int64_t picks, opt_tensor, opt_tensor, int64_t, int64_t, int64_t, bool, bool, double) {
  TORCH_CHECK(logits.dim() == 2, "Tensor logits must be 2 dimensional");
  TORCH_CHECK(picks >= 1 && picks <= 64, "pplx_kernels: invalid argument: experts_per_token must be in [1, 64]");
  const c10::SymInt m = logits.sym_size(0);
  return {fresh_traced({m, c10::SymInt(picks)}, logits, at::kUInt32), fresh_traced({m, c10::SymInt(picks)}, logits, at::kFloat)};
}

struct RouteFunction : torch::autograd::Function<RouteFunction> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext *ctx, const at::Tensor &logits, int64_t picks,
                                                const std::optional<at::Tensor> &bias, const std::optional<at::Tensor> &bound_m,
                                                int64_t num_groups, int64_t top_groups, int64_t group_top, bool sigmoid,
                                                bool renormalize, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    static auto op = op_handle<decltype(routed_tokens_op)>("pplx_kernels::routed_tokens");
    auto [indices, weights] = op.call(logits, picks, bias, bound_m, num_groups, top_groups, group_top, sigmoid, renormalize, scale);
    ctx->save_for_backward({logits, indices});
    ctx->saved_data["sigmoid"] = sigmoid;
    ctx->saved_data["renormalize"] = renormalize;
    ctx->saved_data["scale"] = scale;
    ctx->mark_non_differentiable({indices});
    ctx->set_materialize_grads(false);
    return {indices, weights};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &logits = saved[0], &indices = saved[1];
    at::Tensor grad_logits;
    check_no_tangent({&grads[1], &logits}, kDifferentiable);
    if (grads[1].defined()) {
      at::NoGradGuard plain;
      static auto op = op_handle<decltype(route_tokens_backward_op)>("pplx_kernels::route_tokens_backward");
      grad_logits = fresh_traced(logits.sym_sizes(), logits, logits.scalar_type());
      op.call(grad_logits, grads[1].contiguous(), logits, indices, ctx->saved_data["sigmoid"].toBool(),
              ctx->saved_data["renormalize"].toBool(), ctx->saved_data["scale"].toDouble());
    }
    torch::autograd::variable_list out = differentiable_once({grad_logits}, kDifferentiable);
    out.resize(10);
    return out;
  }
};
Routed routed_tokens_autograd(const at::Tensor &logits, int64_t picks, opt_tensor bias, opt_tensor bound_m, int64_t num_groups,
                              int64_t top_groups, int64_t group_top, bool sigmoid, bool renormalize, double scale) {
  check_no_tangent({&logits}, kDifferentiable);
  auto made = RouteFunction::apply(logits, picks, bias, bound_m, num_groups, top_groups, group_top, sigmoid, renormalize, scale);
  return {made[0], made[1]};
}

template <class Op, class Meta, class Autograd>
void define_differentiable(torch::Library &m, const char *name, const char *schema, Op op, Meta meta, Autograd autograd) {
  m.def((std::string(name) + schema).c_str());
  m.impl(name, c10::kCUDA, op);
  m.impl(name, c10::kMeta, meta);
  m.impl(name, c10::DispatchKey::Autograd, autograd);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(pplx_kernels, m) {
  define(m, "rms_norm",
         "(Tensor!? y, Tensor!? sum, Tensor!? q, Tensor!? scale, Tensor x, Tensor weight, Tensor? residual, float eps) -> ()",
         &rms_norm_op);
  define(m, "rms_norm_backward",
         "(Tensor!? grad_h, Tensor!? grad_weight, Tensor grad_y, Tensor? grad_sum, Tensor h, Tensor weight, float eps, "
         "Tensor!? workspace) -> ()",
         &rms_norm_backward_op);
  define(m, "router_logits", "(Tensor! logits, Tensor x, Tensor weight, Tensor!? workspace) -> ()", &router_logits_op);
  define(m, "router_logits_backward",
         "(Tensor!? grad_x, Tensor!? grad_weight, Tensor grad_logits, Tensor x, Tensor weight, Tensor!? workspace) -> ()",
         &router_logits_backward_op);
  define(m, "route_tokens",
         "(Tensor! indices, Tensor! weights, Tensor logits, Tensor? bias, Tensor? bound_m, int num_groups, int top_groups, "
         "int group_top, bool sigmoid, bool renormalize, float scale) -> ()",
         &route_tokens_op);
  define(m, "route_tokens_backward",
         "(Tensor! grad_logits, Tensor grad_weights, Tensor logits, Tensor indices, bool sigmoid, bool renormalize, float scale) "
         "-> ()",
         &route_tokens_backward_op);
  define_differentiable(m, "normed_rows", "(Tensor x, Tensor weight, Tensor? residual, float eps) -> (Tensor, Tensor)",
                        &normed_rows_op, &normed_rows_meta, &normed_rows_autograd);
  define_differentiable(m, "quantized_rows",
                        "(Tensor x, Tensor weight, Tensor? residual, float eps, bool int8) -> (Tensor, Tensor, Tensor, Tensor)",
                        &quantized_rows_op, &quantized_rows_meta, &quantized_rows_autograd);
  define_differentiable(m, "new_logits", "(Tensor x, Tensor weight) -> Tensor", &new_logits_op, &new_logits_meta, &new_logits_autograd);
  define_differentiable(m, "routed_tokens",
                        "(Tensor logits, int experts_per_token, Tensor? bias, Tensor? bound_m, int num_groups, int top_groups, "
                        "int group_top, bool sigmoid, bool renormalize, float scale) -> (Tensor, Tensor)",
                        &routed_tokens_op, &routed_tokens_meta, &routed_tokens_autograd);
}

// ---------------------------------------------------------------------------
// Functions of pplx_kernels._C
// ---------------------------------------------------------------------------
namespace {

double float_arg(PyObject *obj, const char *name) {
  const double v = PyFloat_AsDouble(obj);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, name, " must be a float, not ", Py_TYPE(obj)->tp_name);
  }
  return v;
}
uint64_t count_arg(PyObject *obj, const char *name) {
  const int64_t v = int_arg(obj, name);
  TORCH_CHECK(v >= 0 && v < (1ll << 31), "pplx_kernels: invalid argument: ", name, " out of range");
  return (uint64_t)v;
}

PyObject *pair(const at::Tensor &a, const at::Tensor &b) {
  PyObject *out = PyTuple_New(2);
  if (!out) throw python_error();
  PyTuple_SET_ITEM(out, 0, wrap_or_none(a));
  PyTuple_SET_ITEM(out, 1, wrap_or_none(b));
  return out;
}

// rms_norm(y, sum, q, scale, x, weight, residual, eps)
PyObject *py_rms_norm(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("rms_norm", nargs, 8);
  const at::Tensor *y = optional_tensor_arg(args[0], "y"), *sum = optional_tensor_arg(args[1], "sum"),
                   *q = optional_tensor_arg(args[2], "q"), *scale = optional_tensor_arg(args[3], "scale"),
                   *residual = optional_tensor_arg(args[6], "residual");
  const at::Tensor &x = tensor_arg(args[4], "x"), &weight = tensor_arg(args[5], "weight");
  const double eps = float_arg(args[7], "eps");
  if (straight({y, sum, q, scale, &x, &weight, residual})) {
    rms_norm(y, sum, q, scale, x, weight, residual, eps);
  } else {
    static auto op = op_handle<decltype(rms_norm_op)>("pplx_kernels::rms_norm");
    op.call(maybe(y), maybe(sum), maybe(q), maybe(scale), x, weight, maybe(residual), eps);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// The four fields of NormedRows.
PyObject *normed(const at::Tensor &y, const at::Tensor &sum, const at::Tensor &q, const at::Tensor &scale) {
  PyObject *out = PyTuple_New(4);
  if (!out) throw python_error();
  PyTuple_SET_ITEM(out, 0, wrap_or_none(y));
  PyTuple_SET_ITEM(out, 1, wrap_or_none(sum));
  PyTuple_SET_ITEM(out, 2, wrap_or_none(q));
  PyTuple_SET_ITEM(out, 3, wrap_or_none(scale));
  return out;
}

// normed_rows(x, weight, residual, eps, record) -> (y, sum, None, None): differentiable if `record`
PyObject *py_normed_rows(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("normed_rows", nargs, 5);
  const at::Tensor &x = tensor_arg(args[0], "x"), &weight = tensor_arg(args[1], "weight");
  const at::Tensor *residual = optional_tensor_arg(args[2], "residual");
  const double eps = float_arg(args[3], "eps");
  Normed made;
  if (bool_arg(args[4])) {
    made = normed_rows_autograd(x, weight, maybe(residual), eps);
  } else if (straight({&x, &weight, residual})) {
    check_matrix(x, "x");
    const at::Tensor y = fresh(x.sizes(), x, x.scalar_type()), sum = residual ? fresh(x.sizes(), x, x.scalar_type()) : at::Tensor();
    rms_norm(&y, defined(sum), nullptr, nullptr, x, weight, residual, eps);
    return normed(y, sum, at::Tensor(), at::Tensor());
  } else {
    static auto op = op_handle<decltype(normed_rows_op)>("pplx_kernels::normed_rows");
    made = op.call(x, weight, maybe(residual), eps);
  }
  return normed(std::get<0>(made), residual ? std::get<1>(made) : at::Tensor(), at::Tensor(), at::Tensor());
  END_HANDLE_TH_ERRORS
}

// quantized_rows(x, weight, residual, eps, int8, record) -> (y, sum, q, scale): rows in int8, or else e4m3; y and sum are
// differentiable if `record`
PyObject *py_quantized_rows(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("quantized_rows", nargs, 6);
  const at::Tensor &x = tensor_arg(args[0], "x"), &weight = tensor_arg(args[1], "weight");
  const at::Tensor *residual = optional_tensor_arg(args[2], "residual");
  const double eps = float_arg(args[3], "eps");
  const bool int8 = bool_arg(args[4]), record = bool_arg(args[5]);
  if (record) {
    const auto [y, sum, q, scale] = quantized_rows_autograd(x, weight, maybe(residual), eps, int8);
    return normed(y, residual ? sum : at::Tensor(), q, scale);
  }
  const auto [y, sum, q, scale] = empty_quantized(x, residual, int8);
  if (straight({&x, &weight, residual})) {
    rms_norm(&y, defined(sum), &q, &scale, x, weight, residual, eps);
  } else {
    static auto op = op_handle<decltype(rms_norm_op)>("pplx_kernels::rms_norm");
    op.call(y, if_defined(sum), q, scale, x, weight, maybe(residual), eps);
  }
  return normed(y, sum, q, scale);
  END_HANDLE_TH_ERRORS
}

// rms_norm_backward(grad_h, grad_weight, grad_y, grad_sum, h, weight, eps, workspace)
PyObject *py_rms_norm_backward(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("rms_norm_backward", nargs, 8);
  const at::Tensor *grad_h = optional_tensor_arg(args[0], "grad_h"), *grad_weight = optional_tensor_arg(args[1], "grad_weight"),
                   *grad_sum = optional_tensor_arg(args[3], "grad_sum"), *workspace = optional_tensor_arg(args[7], "workspace");
  const at::Tensor &grad_y = tensor_arg(args[2], "grad_y"), &h = tensor_arg(args[4], "h"), &weight = tensor_arg(args[5], "weight");
  const double eps = float_arg(args[6], "eps");
  if (straight({grad_h, grad_weight, &grad_y, grad_sum, &h, &weight, workspace})) {
    rms_norm_backward(grad_h, grad_weight, grad_y, grad_sum, h, weight, eps, workspace);
  } else {
    static auto op = op_handle<decltype(rms_norm_backward_op)>("pplx_kernels::rms_norm_backward");
    op.call(maybe(grad_h), maybe(grad_weight), grad_y, maybe(grad_sum), h, weight, eps, maybe(workspace));
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// router_logits(logits, x, weight, workspace)
PyObject *py_router_logits(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("router_logits", nargs, 4);
  const at::Tensor &logits = tensor_arg(args[0], "logits"), &x = tensor_arg(args[1], "x"), &weight = tensor_arg(args[2], "weight");
  const at::Tensor *workspace = optional_tensor_arg(args[3], "workspace");
  if (straight({&logits, &x, &weight, workspace})) {
    router_logits(logits, x, weight, workspace);
  } else {
    static auto op = op_handle<decltype(router_logits_op)>("pplx_kernels::router_logits");
    at::Tensor to = logits;
    op.call(to, x, weight, maybe(workspace));
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// new_logits(x, weight, record) -> logits: differentiable if `record`
PyObject *py_new_logits(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("new_logits", nargs, 3);
  const at::Tensor &x = tensor_arg(args[0], "x"), &weight = tensor_arg(args[1], "weight");
  if (bool_arg(args[2])) return THPVariable_Wrap(new_logits_autograd(x, weight));
  if (straight({&x, &weight})) return THPVariable_Wrap(new_logits_op(x, weight));
  static auto op = op_handle<decltype(new_logits_op)>("pplx_kernels::new_logits");
  return THPVariable_Wrap(op.call(x, weight));
  END_HANDLE_TH_ERRORS
}

// router_logits_backward(grad_x, grad_weight, grad_logits, x, weight, workspace)
PyObject *py_router_logits_backward(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("router_logits_backward", nargs, 6);
  const at::Tensor *grad_x = optional_tensor_arg(args[0], "grad_x"), *grad_weight = optional_tensor_arg(args[1], "grad_weight"),
                   *workspace = optional_tensor_arg(args[5], "workspace");
  const at::Tensor &grad_logits = tensor_arg(args[2], "grad_logits"), &x = tensor_arg(args[3], "x"), &weight = tensor_arg(args[4], "weight");
  if (straight({grad_x, grad_weight, &grad_logits, &x, &weight, workspace})) {
    router_logits_backward(grad_x, grad_weight, grad_logits, x, weight, workspace);
  } else {
    static auto op = op_handle<decltype(router_logits_backward_op)>("pplx_kernels::router_logits_backward");
    op.call(maybe(grad_x), maybe(grad_weight), grad_logits, x, weight, maybe(workspace));
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// rms_norm_workspace(tokens, width) -> bytes that its gradients take
PyObject *py_rms_norm_workspace(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("rms_norm_workspace", nargs, 2);
  uint64_t bytes = 0;
  A2A_CHECK(pplx_a2a_rms_norm_workspace((uint32_t)count_arg(args[0], "tokens"), count_arg(args[1], "width"), &bytes));
  return PyLong_FromUnsignedLongLong(bytes);
  END_HANDLE_TH_ERRORS
}

// router_workspace(x, weight, backward) -> bytes
PyObject *py_router_workspace(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("router_workspace", nargs, 3);
  const at::Tensor &x = tensor_arg(args[0], "x"), &weight = tensor_arg(args[1], "weight");
  const bool backward = bool_arg(args[2]);
  check_router(x, weight);
  uint64_t bytes = 0;
  A2A_CHECK(pplx_a2a_router_workspace(tokens_of(x), (uint32_t)weight.sizes()[0], (uint64_t)x.sizes()[1], dtype_code(x.scalar_type()),
                                      dtype_code(weight.scalar_type()), backward, &bytes));
  return PyLong_FromUnsignedLongLong(bytes);
  END_HANDLE_TH_ERRORS
}

// route_tokens(indices, weights, logits, bias, bound_m, num_groups, top_groups, group_top, sigmoid, renormalize, scale)
PyObject *py_route_tokens(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("route_tokens", nargs, 11);
  const at::Tensor &indices = tensor_arg(args[0], "indices"), &weights = tensor_arg(args[1], "weights"), &logits = tensor_arg(args[2], "logits");
  const at::Tensor *bias = optional_tensor_arg(args[3], "bias"), *bound_m = optional_tensor_arg(args[4], "bound_m");
  const Choice c{int_arg(args[5], "num_groups"), int_arg(args[6], "top_groups"), int_arg(args[7], "group_top"), bool_arg(args[8]),
                 bool_arg(args[9]), float_arg(args[10], "scale")};
  if (straight({&indices, &weights, &logits, bias, bound_m})) {
    route_tokens(indices, weights, logits, bias, bound_m, c);
  } else {
    static auto op = op_handle<decltype(route_tokens_op)>("pplx_kernels::route_tokens");
    at::Tensor to_indices = indices, to_weights = weights;
    op.call(to_indices, to_weights, logits, maybe(bias), maybe(bound_m), c.num_groups, c.top_groups, c.group_top, c.sigmoid,
            c.renormalize, c.scale);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// routed_tokens(logits, experts_per_token, bias, bound_m, num_groups, top_groups, group_top, sigmoid, renormalize, scale, record)
// -> (indices, weights): differentiable if `record`
PyObject *py_routed_tokens(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("routed_tokens", nargs, 11);
  const at::Tensor &logits = tensor_arg(args[0], "logits");
  const int64_t picks = int_arg(args[1], "experts_per_token");
  const at::Tensor *bias = optional_tensor_arg(args[2], "bias"), *bound_m = optional_tensor_arg(args[3], "bound_m");
  const Choice c{int_arg(args[4], "num_groups"), int_arg(args[5], "top_groups"), int_arg(args[6], "group_top"), bool_arg(args[7]),
                 bool_arg(args[8]), float_arg(args[9], "scale")};
  Routed made;
  if (bool_arg(args[10])) {
    made = routed_tokens_autograd(logits, picks, maybe(bias), maybe(bound_m), c.num_groups, c.top_groups, c.group_top, c.sigmoid,
                                  c.renormalize, c.scale);
  } else if (straight({&logits, bias, bound_m})) {
    made = routed_tokens(logits, picks, bias, bound_m, c);
  } else {
    static auto op = op_handle<decltype(routed_tokens_op)>("pplx_kernels::routed_tokens");
    made = op.call(logits, picks, maybe(bias), maybe(bound_m), c.num_groups, c.top_groups, c.group_top, c.sigmoid, c.renormalize,
                   c.scale);
  }
  return pair(std::get<0>(made), std::get<1>(made));
  END_HANDLE_TH_ERRORS
}

// route_tokens_backward(grad_logits, grad_weights, logits, indices, sigmoid, renormalize, scale)
PyObject *py_route_tokens_backward(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arity("route_tokens_backward", nargs, 7);
  const at::Tensor &grad_logits = tensor_arg(args[0], "grad_logits"), &grad_weights = tensor_arg(args[1], "grad_weights"),
                   &logits = tensor_arg(args[2], "logits"), &indices = tensor_arg(args[3], "indices");
  const bool sigmoid = bool_arg(args[4]), renormalize = bool_arg(args[5]);
  const double scale = float_arg(args[6], "scale");
  if (straight({&grad_logits, &grad_weights, &logits, &indices})) {
    route_tokens_backward(grad_logits, grad_weights, logits, indices, sigmoid, renormalize, scale);
  } else {
    static auto op = op_handle<decltype(route_tokens_backward_op)>("pplx_kernels::route_tokens_backward");
    at::Tensor to = grad_logits;
    op.call(to, grad_weights, logits, indices, sigmoid, renormalize, scale);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#ifndef PPLX_ROUTER_SOURCE_ID
#define PPLX_ROUTER_SOURCE_ID "unknown"
#endif
PyObject *py_router_build_id(PyObject *, PyObject *) { return PyUnicode_FromString(PPLX_ROUTER_SOURCE_ID); }

#define PPLX_FASTCALL(fn) (PyCFunction)(void (*)(void))fn, METH_FASTCALL
PyMethodDef kRouterMethods[] = {
    {"rms_norm", PPLX_FASTCALL(py_rms_norm), "rms_norm(y, sum, q, scale, x, weight, residual, eps)"},
    {"normed_rows", PPLX_FASTCALL(py_normed_rows), "normed_rows(x, weight, residual, eps, record) -> (y, sum, None, None)"},
    {"quantized_rows", PPLX_FASTCALL(py_quantized_rows), "quantized_rows(x, weight, residual, eps, int8, record) -> (y, sum, q, scale)"},
    {"rms_norm_backward", PPLX_FASTCALL(py_rms_norm_backward),
     "rms_norm_backward(grad_h, grad_weight, grad_y, grad_sum, h, weight, eps, workspace)"},
    {"rms_norm_workspace", PPLX_FASTCALL(py_rms_norm_workspace), "rms_norm_workspace(tokens, width) -> bytes that its gradients take"},
    {"router_logits", PPLX_FASTCALL(py_router_logits), "router_logits(logits, x, weight, workspace)"},
    {"new_logits", PPLX_FASTCALL(py_new_logits), "new_logits(x, weight, record) -> logits"},
    {"router_logits_backward", PPLX_FASTCALL(py_router_logits_backward),
     "router_logits_backward(grad_x, grad_weight, grad_logits, x, weight, workspace)"},
    {"router_workspace", PPLX_FASTCALL(py_router_workspace), "router_workspace(x, weight, backward) -> bytes"},
    {"route_tokens", PPLX_FASTCALL(py_route_tokens),
     "route_tokens(indices, weights, logits, bias, bound_m, num_groups, top_groups, group_top, sigmoid, renormalize, scale)"},
    {"routed_tokens", PPLX_FASTCALL(py_routed_tokens),
     "routed_tokens(logits, experts_per_token, bias, bound_m, num_groups, top_groups, group_top, sigmoid, renormalize, scale, "
     "record) -> (indices, weights)"},
    {"route_tokens_backward", PPLX_FASTCALL(py_route_tokens_backward),
     "route_tokens_backward(grad_logits, grad_weights, logits, indices, sigmoid, renormalize, scale)"},
    {"router_build_id", py_router_build_id, METH_NOARGS, "hash of the sources that these functions were built from"},
    {nullptr, nullptr, 0, nullptr},
};

}  // namespace

PyMethodDef *router_methods() { return kRouterMethods; }
