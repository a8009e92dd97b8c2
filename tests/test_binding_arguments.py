"""What the functions of the binding take for a truth value."""

from __future__ import annotations

import pytest
import torch

from pplx_kernels import quantize_rows, route_tokens, route_tokens_backward
from pplx_kernels.ops import _C


class Undecided:
    def __bool__(self):
        raise ValueError("neither true nor false")


NO = Undecided()
x, i8, idx = torch.zeros(2, 16), torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2, 2, dtype=torch.uint32)
scale, w, bound = torch.zeros(2), torch.zeros(2, 2), torch.zeros(1, dtype=torch.uint32)


@pytest.mark.parametrize("call", [
    lambda: route_tokens(x, 2, renormalize=NO),
    lambda: route_tokens(x, 2, renormalize=NO, out=(idx, w)),
    lambda: route_tokens_backward(w, x, idx, renormalize=NO),
    lambda: quantize_rows(x, out=(i8, scale), swiglu=NO),
    lambda: _C.quantized_rows(x, x[0], None, 1e-6, NO, False),
    lambda: _C.quantized_rows(x, x[0], None, 1e-6, False, NO),
    lambda: _C.normed_rows(x, x[0], None, 1e-6, NO),
    lambda: _C.new_logits(x, x, NO),
    lambda: _C.router_workspace(x, x, NO),
    lambda: _C.sort_tokens(x, idx, 4, None, NO),
    lambda: _C.dispatch(0, idx, x, None, x, None, idx, None, NO, True),
    lambda: _C.dispatch(0, idx, x, None, x, None, idx, None, True, NO),
    lambda: _C.combine(0, x, idx, w, x, None, NO, True),
    lambda: _C.combine(0, x, idx, w, x, None, True, NO),
])  # fmt: skip
def test_an_error_of_a_truth_value_is_raised(call):
    """The error is the caller's own, and none is left behind for the next call.  (Without a device: it is found before the tensors are
    looked at.)"""
    with pytest.raises(ValueError, match="neither true nor false"):
        call()
    assert len(_C.build_id()) == 16


def test_truth_values_are_those_of_python():
    for yes, no in ((1, 0), ("a", ""), ([0], []), (torch.ones(1), torch.zeros(1))):
        for value in (yes, no):
            with pytest.raises(RuntimeError, match="must be on GPU"):
                route_tokens(x, 2, renormalize=value)
