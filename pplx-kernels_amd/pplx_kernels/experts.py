"""What stands between dispatch and combine: the experts' products in 8-bit integers, and tokens sorted by expert and
back for a rank that holds its experts itself, with the gradients of both.

    s = sort_tokens(x, indices, num_experts)                      # rows by expert, as the routing says
    h = experts(s.rows, s.offsets)
    y = unsort_tokens(h, s.slots, s.offsets, weights)             # differentiable in x, h and weights

    s = sort_tokens(x, indices, num_experts, int8=True)           # the same for 8-bit experts
    h = int8_matmul(s.rows, s.scale, w13, w13_scale, offsets=s.offsets)
    q, scale = quantize_rows(h, offsets=s.offsets, swiglu=True)
    y = unsort_tokens(int8_matmul(q, scale, w2, w2_scale, offsets=s.offsets), s.slots, s.offsets, weights)

``quantize_rows`` and ``int8_matmul`` take the buffers that ``AllToAll.dispatch`` fills as well, with its
``out_expert_num_tokens`` as ``num_tokens``.  All of it runs on the current stream of the tensors' device and keeps
nothing between calls.  Gradients are those of reverse mode; forward mode is refused.  With ``out=`` a call allocates nothing, so it can be captured as it is; without, the results are
new tensors.  Under capture gradients go through ``unsort_tokens_backward`` and ``sort_tokens_backward``: a capture that
autograd recorded would depend on graphs of the same leaves that live outside.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from .ops import _C, _ops

_is_compiling = torch.compiler.is_compiling


class SortedTokens(NamedTuple):
    """What :func:`sort_tokens` makes."""

    rows: torch.Tensor  # [m * K, H], expert by expert; zeros behind the last row
    scale: torch.Tensor | None  # [m * K] float32: of quantised rows
    slots: torch.Tensor  # [m, K] int32: the row of each pick, -1 where it has none
    offsets: torch.Tensor  # [num_experts + 1] int32: the first row of each expert, and the number of rows
    workspace: torch.Tensor | None  # int32, for steps of many picks; of use for `out=` only

    @classmethod
    def empty(
        cls,
        num_tokens: int,
        hidden_dim: int,
        num_experts: int,
        experts_per_token: int,
        dtype: torch.dtype,
        device: torch.device | str = "cuda",
        int8: bool = False,
    ) -> "SortedTokens":
        """Buffers for ``sort_tokens(..., out=)``, which belong to one step at a time."""
        rows = num_tokens * experts_per_token
        words = _ops.sort_workspace(num_tokens, experts_per_token, num_experts)
        return cls(
            torch.empty(rows, hidden_dim, dtype=torch.int8 if int8 else dtype, device=device),
            torch.empty(rows, dtype=torch.float32, device=device) if int8 else None,
            torch.empty(num_tokens, experts_per_token, dtype=torch.int32, device=device),
            torch.empty(num_experts + 1, dtype=torch.int32, device=device),
            torch.empty(words, dtype=torch.int32, device=device) if words else None,
        )


def _wants_grad(*tensors: torch.Tensor | None) -> bool:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        return True
    # (a tensor with a tangent need not require a gradient)
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors
    )


def _check_recording(x: torch.Tensor) -> None:
    if x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(
            "pplx_kernels: gradients are not recorded under stream capture: capture the _backward functions, under torch.no_grad()"
        )


def sort_tokens(
    x: torch.Tensor,
    indices: torch.Tensor,
    num_experts: int,
    bound_m: torch.Tensor | None = None,
    *,
    int8: bool = False,
    out: SortedTokens | None = None,
) -> SortedTokens:
    """Copies of ``x[t]`` for the ``K`` experts in ``indices[t]`` (uint32) for ``t < bound_m``, ordered by (expert,
    token, pick).  Picks with an index of ``num_experts`` or more have no row here (their experts are elsewhere).

    ``x`` is ``[m, H]`` of float32, bfloat16 or float16, its rows multiples of 16 bytes that lie in one piece.  With
    ``int8`` the rows are quantised as by :func:`quantize_rows` (``H`` a multiple of 16).  Differentiable in ``x`` unless
    ``int8`` or ``out`` is given."""
    if out is not None:
        if out.scale is None and int8 or out.scale is not None and not int8:
            raise RuntimeError("pplx_kernels: out.scale goes with int8=True")
        if out.offsets.dim() != 1 or out.offsets.size(0) != num_experts + 1:
            raise RuntimeError("pplx_kernels: out.offsets must be [num_experts + 1]")
        fn = _ops.sort_tokens if _is_compiling() else _C.sort_tokens_out
        fn(out.rows, out.scale, out.slots, out.offsets, out.workspace, x, indices, bound_m)
        return out
    if _is_compiling():
        rows, scale, slots, offsets = _ops.sorted_tokens(x, indices, num_experts, bound_m, int8)
        return SortedTokens(rows, scale if int8 else None, slots, offsets, None)
    if not int8 and _wants_grad(x):
        _check_recording(x)
        rows, slots, offsets = _C.sorted_tokens(x, indices, num_experts, bound_m)
        return SortedTokens(rows, None, slots, offsets, None)
    return SortedTokens._make(_C.sort_tokens(x, indices, num_experts, bound_m, int8))


def sort_tokens_backward(
    grad_rows: torch.Tensor, slots: torch.Tensor, *, out: torch.Tensor | None = None
) -> torch.Tensor:
    """The gradient of ``sort_tokens(x, ...).rows`` with respect to ``x``: the sum of the gradients of a token's rows."""
    return _unsort(grad_rows, slots, None, None, out)


def unsort_tokens(
    y: torch.Tensor,
    slots: torch.Tensor,
    offsets: torch.Tensor,
    weights: torch.Tensor | None = None,
    *,
    out_dtype: torch.dtype | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``out[t] = sum_k weights[t, k] * y[slots[t, k]]`` over the picks that have a row, fp32 accumulation in pick order;
    a token without one becomes zeros.  ``weights`` are float32 (None: ones).  ``y`` is ``[rows, H]`` of float32, bfloat16 or
    float16, ``H`` a multiple of 8.  Differentiable in ``y`` and ``weights`` unless ``out`` is given."""
    if out is None and _is_compiling():
        return _ops.unsorted_tokens(y, slots, offsets, weights, out_dtype)
    if out is None and _wants_grad(y, weights):
        _check_recording(y)
        return _C.unsorted_tokens(y, slots, offsets, weights, out_dtype)
    return _unsort(y, slots, weights, out_dtype, out)


def _unsort(y, slots, weights, out_dtype, out) -> torch.Tensor:
    if out is None:
        out = torch.empty(slots.shape[0], y.shape[-1], dtype=out_dtype or y.dtype, device=y.device)
    elif out_dtype is not None and out.dtype != out_dtype:
        raise RuntimeError("pplx_kernels: out has another dtype than out_dtype")
    fn = _ops.unsort_tokens if _is_compiling() else _C.unsort_tokens
    fn(out, y, slots, weights)
    return out


def unsort_tokens_backward(
    grad_out: torch.Tensor,
    y: torch.Tensor,
    slots: torch.Tensor,
    offsets: torch.Tensor,
    weights: torch.Tensor | None = None,
    *,
    out: tuple[torch.Tensor | None, torch.Tensor | None] | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """The gradients of :func:`unsort_tokens`: ``grad_y[slots[t, k]] = weights[t, k] * grad_out[t]``, zeros in rows that no
    pick has, and ``grad_weights[t, k] = <grad_out[t], y[slots[t, k]]>`` (None without weights).  ``slots`` are a sort's, of
    all its tokens or of some, with any of them taken out (-1); no two name one row.  In ``out`` either may be None, which
    leaves it out."""
    if out is None:
        out = torch.empty_like(y, memory_format=torch.contiguous_format), None if weights is None else torch.empty_like(weights)
    fn = _ops.unsort_tokens_backward if _is_compiling() else _C.unsort_tokens_backward
    fn(out[0], out[1], grad_out, y, slots, offsets, weights)
    return out


def quantize_rows(
    x: torch.Tensor,
    *,
    num_tokens: torch.Tensor | None = None,
    offsets: torch.Tensor | None = None,
    swiglu: bool = False,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows to int8 with one float32 scale each: ``a = max(max |x[r]|, 2**-100)``, ``q = round(x[r] * (127 / a))`` (ties to
    even), ``scale = a / 127``.  With ``swiglu`` of ``silu(x[r, :W]) * x[r, W:]``, computed in fp32.  A row that holds an
    infinity or a NaN becomes zeros with a scale of NaN, and so NaN in whatever is made from it.

    ``x`` is ``[rows, ..]``, of which with ``offsets`` (``SortedTokens.offsets``) the first ``offsets[-1]`` are there, or
    ``[experts, rows, ..]`` with ``num_tokens`` (``[experts]`` int32) of each expert's there, as ``dispatch`` leaves them.
    Rows that are not there are neither read nor written.  Quantised rows are multiples of 16 bytes.  Not differentiable."""
    if out is None:
        shape = x.shape[:-1]
        width = x.shape[-1] // 2 if swiglu else x.shape[-1]
        out = (
            torch.empty((*shape, width), dtype=torch.int8, device=x.device),
            torch.empty(shape, dtype=torch.float32, device=x.device),
        )
    fn = _ops.quantize_rows if _is_compiling() else _C.quantize_rows
    fn(out[0], out[1], x.detach() if x.requires_grad else x, num_tokens, offsets, swiglu)
    return out


def int8_matmul(
    x: torch.Tensor,
    x_scale: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    *,
    num_tokens: torch.Tensor | None = None,
    offsets: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.bfloat16,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``out[r, n] = x_scale[r] * weight_scale[e, n] * sum_k x[r, k] * weight[e, n, k]`` for the rows of each expert ``e``,
    with exact int32 sums.  The scaling is fp32: the sum, the product of the scales and their product are rounded to it, and the
    result once more to its type.  Not differentiable, in the scales neither.

    ``x`` is int8 ``[rows, K]``, ``weight`` int8 ``[experts, N, K]`` and ``weight_scale`` float32 ``[experts, N]``; the rows
    of expert ``e`` are those from ``offsets[e]`` to ``offsets[e + 1]``.  Or ``x`` is ``[experts, rows, K]`` with
    ``num_tokens`` of each expert's rows there, as ``dispatch`` leaves them (its scales with a stride:
    ``out_expert_x_scale[..., 0]``).  Without either all rows take one weight ``[N, K]``.  Rows that are not there are
    neither read nor written.  ``K`` is a multiple of 16, at most 131056.  ``out`` is float32, bfloat16 or float16."""
    if out is None:
        out = torch.empty((*x.shape[:-1], weight.shape[-2]), dtype=out_dtype, device=x.device)
    fn = _ops.int8_matmul if _is_compiling() else _C.int8_matmul
    fn(out, x, x_scale, weight, weight_scale, num_tokens, offsets)
    return out
