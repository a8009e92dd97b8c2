"""The operators between dispatch and combine as they are used: in graphs."""

from __future__ import annotations

import pytest
import torch

from pplx_kernels import sort_tokens, sort_tokens_backward, unsort_tokens, unsort_tokens_backward
from tests.test_experts import BF16, make_indices

gpu = pytest.mark.gpu


@gpu
def test_gradients_in_a_graph(device):
    """The gradients' own forms are captured while an eager graph of the same leaves lives; autograd is refused there."""
    m, k, experts, hidden = 60, 3, 8, 96
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(m, hidden, generator=gen).to(device).requires_grad_(True)
    weights = torch.rand(m, k, generator=gen).to(device).requires_grad_(True)
    indices = to_u32(make_indices(m, k, experts, gen, "mixed"), device)
    s = sort_tokens(x, indices, experts)
    out = unsort_tokens(s.rows, s.slots, s.offsets, weights)
    grad = torch.randn(m, hidden, generator=gen).to(device)
    want_x, want_w = torch.autograd.grad(out, [x, weights], grad, retain_graph=True)
    grad_y, grad_w, grad_x = torch.empty_like(s.rows), torch.empty_like(weights), torch.empty_like(x)
    rows = s.rows.detach()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream), torch.no_grad():
        unsort_tokens_backward(grad, rows, s.slots, s.offsets, weights, out=(grad_y, grad_w))
        sort_tokens_backward(grad_y, s.slots, out=grad_x)
        with torch.enable_grad():
            for record in (lambda: sort_tokens(x, indices, experts),
                           lambda: unsort_tokens(rows, s.slots, s.offsets, weights)):  # fmt: skip
                with pytest.raises(RuntimeError, match="not recorded under stream capture"):
                    record()
    for _ in range(3):
        grad_x.zero_(), grad_w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad_x, want_x) and torch.equal(grad_w, want_w)
        (rows * 2).sum()
    again_x, _ = torch.autograd.grad(out, [x, weights], grad)
    assert torch.equal(again_x, want_x)
