"""What stands before dispatch: the norm whose rows are sent, in 8 bits where asked to, the router's product, and the choice of
experts with its weights, with the gradients of all three.

    n = rms_norm(x, norm_weight, residual, quantize=torch.float8_e4m3fn)   # n.y, n.sum; n.q and n.scale are what dispatch sends
    logits = router_logits(n.y, router_weight)                              # float32
    indices, weights = route_tokens(logits, 8, bias=bias, scores="sigmoid", num_groups=8, top_groups=4, scale=2.5)
    ata.dispatch(..., dp_x=n.q, dp_x_scale=n.scale, indices=indices)        # and weights to combine

A rank that holds its experts itself gives ``indices`` and ``weights`` to ``sort_tokens`` and ``unsort_tokens``, with rows of ``n.y``.
``n.y``, ``n.sum``, the logits and the weights are differentiable, and so are the sorted rows and their sum, so that the same calls
make a training step; ``n.q`` and ``n.scale`` have no gradient, and ``dispatch`` and ``combine`` pass none on.  Calls run on the current
stream of the tensors' device and keep nothing between calls.  With ``out=``, and ``workspace=`` where there is one, a call allocates nothing and can be captured as it is; without
``workspace`` it takes that from torch's allocator, which keeps it for a graph that torch captures, not for one that
``LoopbackWorld.capture`` does.  Gradients are those of reverse mode; under capture they go through the ``_backward`` functions.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .experts import _check_recording, _is_compiling, _wants_grad
from .ops import _C, _ops

BLOCK = 128  # columns that share a scale of e4m3 rows


class NormedRows(NamedTuple):
    """What :func:`rms_norm` makes."""

    y: torch.Tensor | None  # [m, H] of the type of x
    sum: torch.Tensor | None = None  # [m, H] of the type of x: x + residual
    q: torch.Tensor | None = None  # [m, H] int8 or float8_e4m3fn
    scale: torch.Tensor | None = None  # float32: [m] of int8 rows, [m, ceil(H / 128)] of e4m3 rows

    @classmethod
    def empty(
        cls,
        num_tokens: int,
        hidden_dim: int,
        dtype: torch.dtype,
        device: torch.device | str = "cuda",
        *,
        residual: bool = False,
        quantize: torch.dtype | None = None,
    ) -> "NormedRows":
        """Buffers for ``rms_norm(..., out=)``."""
        shape = (num_tokens, hidden_dim)
        q, scale = _quantized(shape, device, quantize)
        return cls(
            torch.empty(shape, dtype=dtype, device=device),
            torch.empty(shape, dtype=dtype, device=device) if residual else None,
            q,
            scale,
        )


def _check_quantize(quantize):
    if quantize not in (torch.int8, torch.float8_e4m3fn):
        raise RuntimeError("pplx_kernels: quantize must be torch.int8 or torch.float8_e4m3fn")


def _quantized(shape, device, quantize):
    if quantize is None:
        return None, None
    _check_quantize(quantize)
    of_scale = shape[:1] if quantize == torch.int8 else (shape[0], (shape[1] + BLOCK - 1) // BLOCK)
    return (
        torch.empty(shape, dtype=quantize, device=device),
        torch.empty(of_scale, dtype=torch.float32, device=device),
    )


def rms_norm(
    x: torch.Tensor,
    weight: torch.Tensor,
    residual: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    quantize: torch.dtype | None = None,
    out: NormedRows | None = None,
) -> NormedRows:
    """``h = x + residual``, rounded to the type of ``x``, and ``v = h * weight / sqrt(mean(h**2) + eps)`` in fp32: ``sum`` is ``h``
    (None without ``residual``) and ``y`` is ``v``, rounded once.  With ``quantize`` also ``v`` in 8 bits: ``torch.int8`` with one scale
    a row, as by :func:`quantize_rows`, or ``torch.float8_e4m3fn`` with one scale for each 128 columns, ``a = max(max |v|, 2**-100)``,
    ``q = e4m3(v * (448 / a))``, ``scale = a / 448``, which is what ``dispatch`` takes as ``dp_x`` and ``dp_x_scale``.  (Where ``v`` lies in
    the middle between two codes, fp32's roundings decide: another order of its sums may take the other one.)  A row that holds an
    infinity or a NaN becomes NaN (``q`` zeros, its scales NaN).

    ``x`` is ``[m, H]`` of float32, bfloat16 or float16, its rows 16-byte aligned and ``H`` a multiple of 8 (with ``quantize`` of 16);
    ``weight`` is ``[H]`` of its type or float32.  Differentiable in ``x``, ``residual`` and ``weight``, through ``y`` and ``sum`` (``q`` and
    ``scale`` have no gradient), unless ``out`` is given.  ``out`` may leave ``y`` out (None) where it has ``q``, and ``y`` and ``sum`` may be ``x`` and
    ``residual`` themselves."""
    if out is not None:
        if quantize is not None and (out.q is None or out.q.dtype != quantize):
            raise RuntimeError("pplx_kernels: out.q goes with quantize")
        fn = _ops.rms_norm if _is_compiling() else _C.rms_norm
        fn(out.y, out.sum, out.q, out.scale, x, weight, residual, eps)
        return out
    if quantize is not None:
        _check_quantize(quantize)
        if _is_compiling():
            y, total, q, scale = _ops.quantized_rows(x, weight, residual, eps, quantize == torch.int8)
            return NormedRows(y, None if residual is None else total, q, scale)
        record = _wants_grad(x, weight, residual)
        if record:
            _check_recording(x)
        return NormedRows._make(_C.quantized_rows(x, weight, residual, eps, quantize == torch.int8, record))
    if _is_compiling():
        y, total = _ops.normed_rows(x, weight, residual, eps)
        return NormedRows(y, None if residual is None else total)
    record = _wants_grad(x, weight, residual)
    if record:
        _check_recording(x)
    return NormedRows._make(_C.normed_rows(x, weight, residual, eps, record))


def rms_norm_backward(
    grad_y: torch.Tensor,
    h: torch.Tensor,
    weight: torch.Tensor,
    *,
    grad_sum: torch.Tensor | None = None,
    eps: float = 1e-6,
    out: tuple[torch.Tensor | None, torch.Tensor | None] | None = None,
    workspace: torch.Tensor | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """The gradients of :func:`rms_norm`: that of ``h`` (``NormedRows.sum``, or ``x`` where there was no residual), which is that of
    ``x`` and of ``residual``, and that of ``weight``.  ``grad_sum`` is the gradient that came for ``sum`` itself.  In ``out`` either
    may be None, which leaves it out; the first may be ``grad_y`` or ``grad_sum`` itself.  ``workspace`` is of
    :func:`rms_norm_workspace`."""
    if out is None:
        out = torch.empty_like(h, memory_format=torch.contiguous_format), torch.empty_like(weight)
    fn = _ops.rms_norm_backward if _is_compiling() else _C.rms_norm_backward
    fn(out[0], out[1], grad_y, grad_sum, h, weight, eps, workspace)
    return out


def rms_norm_workspace(h: torch.Tensor) -> torch.Tensor:
    """What :func:`rms_norm_backward` of ``h`` writes besides its results: for one call at a time."""
    return torch.empty(_C.rms_norm_workspace(*h.shape), dtype=torch.uint8, device=h.device)


def router_logits(
    x: torch.Tensor, weight: torch.Tensor, *, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None
) -> torch.Tensor:
    """``x @ weight.T`` in float32: products of 16-bit elements are exact, those of float32 count to 24 bits, and sums are float32.

    ``x`` is ``[m, H]`` of float32, bfloat16 or float16 and ``weight`` ``[experts, H]`` of its type or float32, both with rows that
    are 16-byte aligned and ``H`` a multiple of 8.  Differentiable in both unless ``out`` is given, with which ``workspace`` may be
    given too, of :func:`router_workspace`."""
    if out is not None:
        fn = _ops.router_logits if _is_compiling() else _C.router_logits
        fn(out, x, weight, workspace)
        return out
    if workspace is not None:
        raise RuntimeError("pplx_kernels: workspace goes with out")
    if _is_compiling():
        return _ops.new_logits(x, weight)
    record = _wants_grad(x, weight)
    if record:
        _check_recording(x)
    return _C.new_logits(x, weight, record)


def router_logits_backward(
    grad_logits: torch.Tensor,
    x: torch.Tensor,
    weight: torch.Tensor,
    *,
    out: tuple[torch.Tensor | None, torch.Tensor | None] | None = None,
    workspace: torch.Tensor | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """The gradients of :func:`router_logits`: ``grad_logits @ weight`` and ``grad_logits.T @ x``, added up in float32 and rounded
    once; operands count to 24 bits whatever the results' type.  In ``out`` either may be None, which leaves it out.  ``workspace`` is of :func:`router_workspace`."""
    if out is None:
        out = (
            torch.empty_like(x, memory_format=torch.contiguous_format),
            torch.empty_like(weight, memory_format=torch.contiguous_format),
        )
    fn = _ops.router_logits_backward if _is_compiling() else _C.router_logits_backward
    fn(out[0], out[1], grad_logits, x, weight, workspace)
    return out


def router_workspace(x: torch.Tensor, weight: torch.Tensor, *, backward: bool = False) -> torch.Tensor:
    """What :func:`router_logits`, or its gradients, write besides their results (nothing for some sizes): for one call at a time."""
    return torch.empty(_C.router_workspace(x, weight, backward), dtype=torch.uint8, device=x.device)


def _is_sigmoid(scores: str) -> bool:
    if scores not in ("softmax", "sigmoid"):
        raise RuntimeError('pplx_kernels: scores must be "softmax" or "sigmoid"')
    return scores == "sigmoid"


def route_tokens(
    logits: torch.Tensor,
    experts_per_token: int,
    *,
    bias: torch.Tensor | None = None,
    scores: str = "softmax",
    num_groups: int = 1,
    top_groups: int = 1,
    group_top: int = 2,
    renormalize: bool = True,
    scale: float = 1.0,
    bound_m: torch.Tensor | None = None,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Each token's experts and their weights: ``(indices, weights)``, ``[m, K]`` uint32 and float32, largest first, as ``dispatch``
    / ``combine`` and ``sort_tokens`` / ``unsort_tokens`` take them.

    ``s`` is the softmax of a token's logits or the sigmoid of each.  Chosen are the ``experts_per_token`` experts with the largest
    ``s + bias`` (``bias`` ``[experts]`` float32), out of the ``top_groups`` of ``num_groups`` groups of consecutive experts whose
    ``group_top`` (1 or 2) best have the largest sums.  The order is that of 64-bit arithmetic, equal ones by number.  Weights are ``s``
    at the choice (without the bias), divided by their sum with ``renormalize``, times ``scale``.

    An expert whose logit or ``s + bias`` is -inf is not there.  Picks that no expert is left for, and those of tokens from ``bound_m``
    on, have the index ``experts`` and weight 0, which ``sort_tokens`` takes for no row.  A token with a NaN or +inf among them gets
    the first experts, with weights of NaN.  ``logits`` are ``[m, experts]`` of float32, bfloat16 or float16.  The weights are
    differentiable in the logits unless ``out`` is given, the bias has no gradient."""
    sigmoid = _is_sigmoid(scores)
    choice = num_groups, top_groups, group_top, sigmoid, renormalize, scale
    if out is not None:
        if out[0].dim() != 2 or out[0].shape[1] != experts_per_token:
            raise RuntimeError("pplx_kernels: out must be [tokens, experts_per_token]")
        fn = _ops.route_tokens if _is_compiling() else _C.route_tokens
        fn(out[0], out[1], logits, bias, bound_m, *choice)
        return out
    if _is_compiling():
        return _ops.routed_tokens(logits, experts_per_token, bias, bound_m, *choice)
    record = _wants_grad(logits)
    if record:
        _check_recording(logits)
    return _C.routed_tokens(logits, experts_per_token, bias, bound_m, *choice, record)


def route_tokens_backward(
    grad_weights: torch.Tensor,
    logits: torch.Tensor,
    indices: torch.Tensor,
    *,
    scores: str = "softmax",
    renormalize: bool = True,
    scale: float = 1.0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """The gradient of the weights of :func:`route_tokens` with respect to ``logits``, for the picks in ``indices`` that it made (no
    expert twice in a token).  Every logit's is written, zeros where there is none, and NaN for a token that has picks and a NaN or
    +inf among its logits.  The bias has no part in it: where only the bias made the weights NaN, the gradient is that of the scores."""
    if out is None:
        out = torch.empty_like(logits, memory_format=torch.contiguous_format)
    fn = _ops.route_tokens_backward if _is_compiling() else _C.route_tokens_backward
    fn(out, grad_weights, logits, indices, _is_sigmoid(scores), renormalize, scale)
    return out
