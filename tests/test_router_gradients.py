"""Gradients of the operators before dispatch that come by less common ways: beside rows in 8 bits, of tokens whose logits are
no numbers, of more experts than a workgroup holds at once, of sums that cancel.  Tolerances count roundings, as in test_router.py."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from pplx_kernels import rms_norm, route_tokens, route_tokens_backward, router_logits, router_logits_backward
from tests.test_experts import BF16, F16, F32, assert_within, rounded
from tests.test_router import E4M3, gradient, product, router
from tests.test_router_path import make_step, same

gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Rows in 8 bits: y and sum beside them are differentiable
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("quantize", [torch.int8, E4M3])
@pytest.mark.parametrize("which", ["x", "weight", "residual"])
def test_quantised_norms_are_recorded(quantize, which):
    """Without a device: tensors that have none of their data."""
    made = {name: torch.empty(*shape, device="meta") for name, shape in (("x", (6, 256)), ("weight", (256,)), ("residual", (6, 256)))}
    made[which].requires_grad_(True)
    for residual in (made["residual"], None) if which != "residual" else (made["residual"],):
        n = rms_norm(made["x"], made["weight"], residual, quantize=quantize)
        assert n.y.requires_grad and not n.q.requires_grad and not n.scale.requires_grad
        assert n.q.dtype == quantize and n.scale.shape == ((6,) if quantize == torch.int8 else (6, 2))
        assert n.sum is None if residual is None else n.sum.requires_grad
        with torch.no_grad(), pytest.raises(RuntimeError, match="must be on GPU"):  # (nothing to record: the call itself)
            rms_norm(made["x"], made["weight"], residual, quantize=quantize)


def check_tangents_of_quantised_norms(device):
    x, weight = torch.ones(4, 16, device=device), torch.ones(16, device=device)
    with forward_ad.dual_level():
        dx, dw = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, weight))
        for quantize in (torch.int8, E4M3):
            for args in ((dx, weight), (x, dw), (x, weight, dx)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    rms_norm(*args, quantize=quantize)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    rms_norm(*args, quantize=quantize)


def test_tangents_of_quantised_norms_are_refused_before_the_device_is_looked_at():
    check_tangents_of_quantised_norms("cpu")


@gpu
def test_tangents_of_quantised_norms_are_refused(device):
    check_tangents_of_quantised_norms(device)


@gpu
@pytest.mark.parametrize("quantize", [torch.int8, E4M3])
@pytest.mark.parametrize("m,hidden,dtype,weight_dtype", [
    (1, 16, F32, F32), (33, 528, F16, F16), (70, 2048, BF16, F32), (9, 7168, BF16, BF16), (3, 20000, F16, F32), (0, 64, BF16, BF16),
])  # fmt: skip
@pytest.mark.parametrize("add", [False, True])
def test_gradients_through_quantised_norms(device, m, hidden, dtype, weight_dtype, add, quantize):
    """The bits that the norm without rows in 8 bits gives, results and gradients."""
    gen = torch.Generator().manual_seed(hidden)
    x, residual, weight, *_ = make_step(device, gen, m, hidden, 4, dtype, weight_dtype)
    grads = [torch.randn(m, hidden, generator=gen).to(dtype).to(device) for _ in range(1 + add)]
    got = []
    for more in (dict(), dict(quantize=quantize)):
        leaves = [t.detach().requires_grad_(True) for t in ((x, weight, residual) if add else (x, weight))]
        n = rms_norm(*leaves, **more)
        outs = [n.y, n.sum] if add else [n.y]
        got.append([t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, grads, retain_graph=True)))
        if add:  # of the sum alone
            got[-1] += torch.autograd.grad(n.sum, leaves[::2], grads[1])
    assert all(same(a, b) for a, b in zip(*got))
    assert not n.q.requires_grad and not n.scale.requires_grad
    with torch.no_grad():  # and the rows themselves are those of a call that records nothing
        plain = rms_norm(x, weight, residual if add else None, quantize=quantize)
        assert same(plain.q, n.q) and same(plain.scale, n.scale) and not plain.y.requires_grad


@gpu
def test_quantised_norms_under_autograd(device):
    """Differentiable once, told of what changed, refused under capture."""
    gen = torch.Generator().manual_seed(4)
    x, residual, weight, *_ = make_step(device, gen, 9, 64, 8, F32)
    leaf = x.clone().requires_grad_(True)
    (got,) = torch.autograd.grad(rms_norm(leaf, weight, quantize=torch.int8).y.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        got.sum().backward()
    n = rms_norm(leaf * 1.0, weight, residual, quantize=E4M3)
    with torch.no_grad():
        n.sum.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        n.y.sum().backward()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        with pytest.raises(RuntimeError, match="not recorded under stream capture"):
            rms_norm(leaf, weight, quantize=torch.int8)
        with torch.no_grad():
            captured = rms_norm(leaf, weight, quantize=torch.int8)
    for _ in range(3):
        captured.y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = rms_norm(x, weight, quantize=torch.int8)
        assert same(captured.y, eager.y) and same(captured.q, eager.q) and same(captured.scale, eager.scale)


@gpu
@pytest.mark.parametrize("quantize", [torch.int8, E4M3])
def test_a_step_whose_rows_are_sent_in_8_bits_trains_its_router(device, quantize):
    """The norm that makes the rows for dispatch makes the router's rows too: gradients reach x, the residual and the norm's weight."""
    gen = torch.Generator().manual_seed(5)
    x, residual, norm_weight, gate, bias = make_step(device, gen, 40, 256, 16, BF16, F32)
    results = []
    for more in (dict(), dict(quantize=quantize)):
        leaves = [t.detach().requires_grad_(True) for t in (x, residual, norm_weight, gate)]
        n = rms_norm(leaves[0], leaves[2], leaves[1], **more)
        _, weights = route_tokens(router_logits(n.y, leaves[3]), 4, bias=bias, scores="sigmoid")
        results.append(torch.autograd.grad(weights.square().sum() + n.sum.float().sum(), leaves))
    assert all(same(a, b) and a.abs().sum() > 0 for a, b in zip(*results))


@gpu
def test_quantised_norms_are_traced_with_their_gradients(device):
    gen = torch.Generator().manual_seed(6)

    def step(x, weight, residual):
        n = rms_norm(x * 1.0, weight, residual, quantize=torch.int8)
        e = rms_norm(n.y, weight, quantize=E4M3)
        return n.y, n.sum, n.q, n.scale, e.y, e.scale

    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    x, residual, weight, *_ = make_step(device, gen, 30, 256, 8, F32)
    for record in (True, False):
        leaves = [t.detach().requires_grad_(record) for t in (x, weight, residual)]
        want, got = step(*leaves), compiled(*leaves)
        assert all(same(a, b) and a.requires_grad == b.requires_grad for a, b in zip(got, want))
        if record:
            grads = [torch.autograd.grad(out[0].sum() + out[4].square().sum(), leaves) for out in (want, got)]
            assert all(torch.allclose(a, b, rtol=1e-5, atol=1e-6) for a, b in zip(*grads))


# ---------------------------------------------------------------------------
# Tokens whose logits are no numbers
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("experts,dtype", [(40, F32), (64, F16), (130, BF16), (256, F32), (500, F16), (700, F32), (1500, BF16)])
def test_tokens_of_bad_logits_have_gradients_of_nan(device, experts, dtype, scores, renormalize, bad):
    """Their weights are NaN, and so is what depends on them: at any expert, one of the picks or not.  The other tokens have the bits
    that they have without them."""
    gen = torch.Generator().manual_seed(experts)
    m, k = 13, 3
    logits = (2 * torch.randn(m, experts, generator=gen)).to(dtype)
    logits[::2, experts // 3] = float("-inf")
    grad = torch.randn(m, k, generator=gen).to(device)
    more = dict(scores=scores, renormalize=renormalize, scale=1.5)
    spoiled = {1: 0, 4: k - 1, 5: k, 8: experts // 2, 12: experts - 1}
    mixed = logits.clone()
    for t, e in spoiled.items():
        mixed[t, e] = bad
    leaf, clean = mixed.to(device).requires_grad_(True), logits.to(device).requires_grad_(True)
    indices, weights = route_tokens(leaf, k, **more)
    (got,) = torch.autograd.grad(weights, leaf, grad)
    (want,) = torch.autograd.grad(route_tokens(clean, k, **more)[1], clean, grad)
    rest = [t for t in range(m) if t not in spoiled]
    assert torch.isnan(weights[list(spoiled)]).all() and torch.isnan(got[list(spoiled)]).all()
    assert torch.isfinite(got[rest]).all() and same(got[rest], want[rest])
    # a token whose picks are all taken out has no part in anything, another one's pick that is taken out leaves it what it is
    at = indices.view(torch.int32).clone()
    at[1], at[8, 1], at[2] = experts, experts, experts
    got = route_tokens_backward(grad, mixed.to(device), at.view(torch.uint32), **more)
    assert (got[[1, 2]] == 0).all() and torch.isnan(got[[4, 5, 8, 12]]).all()


@gpu
@pytest.mark.parametrize("renormalize", [False, True])
def test_tokens_behind_the_last_have_no_gradient_whatever_their_logits(device, renormalize):
    logits = torch.randn(12, 256, generator=torch.Generator().manual_seed(1))
    logits[8:] = float("nan")
    leaf = logits.to(device).requires_grad_(True)
    bound = torch.tensor([8], dtype=torch.int32, device=device).view(torch.uint32)
    _, weights = route_tokens(leaf, 4, bound_m=bound, renormalize=renormalize)
    (got,) = torch.autograd.grad(weights.square().sum(), leaf)
    assert (got[8:] == 0).all() and torch.isfinite(got).all() and got[:8].abs().sum() > 0


# ---------------------------------------------------------------------------
# The router's product
# ---------------------------------------------------------------------------
MANY_EXPERTS = [
    # more experts than a workgroup of grad_x holds of the weight at once (256 to 512, by their types), and than one of grad_weight
    # takes; tokens that leave waves of the last round without rows
    (300, 257, 264, F16, F32), (37, 300, 136, BF16, F32), (515, 330, 136, F32, F32), (700, 520, 520, BF16, BF16), (290, 384, 72, F16, F16),
    (1, 513, 2056, BF16, BF16), (530, 1100, 64, BF16, F32), (70, 1333, 328, F32, F32), (20, 5461, 40, F16, F16), (33, 5461, 64, BF16, BF16),
]  # fmt: skip


@gpu
@pytest.mark.parametrize("m,experts,hidden,dtype,weight_dtype", MANY_EXPERTS)
def test_gradients_of_router_logits_of_many_experts(device, m, experts, hidden, dtype, weight_dtype):
    gen = torch.Generator().manual_seed(m + hidden)
    x, weight = router(m, experts, hidden, dtype, weight_dtype, gen)
    grad = 1e-2 * torch.randn(m, experts, generator=gen)
    leaves = [t.to(device).requires_grad_(True) for t in (x, weight)]
    gx, gw = torch.autograd.grad(router_logits(*leaves), leaves, grad.to(device))
    want, off = gradient(grad, weight, experts, dtype)
    want_w, off_w = gradient(grad.t(), x, m, weight_dtype)
    assert_within(gx, want, rounded(want, dtype, off))
    assert_within(gw, want_w, rounded(want_w, weight_dtype, off_w))
    dev = [t.to(device) for t in (grad, x, weight)]
    room = torch.full((m, hidden + 16), 7.0, dtype=dtype, device=device), torch.full((experts, hidden + 16), 7.0, dtype=weight_dtype, device=device)
    inner = [t[:, 8 : 8 + hidden] for t in room]
    router_logits_backward(*dev, out=(inner[0], None))
    router_logits_backward(*dev, out=(None, inner[1]))
    assert same(inner[0], gx) and same(inner[1], gw)
    assert all((t[:, :8] == 7).all() and (t[:, 8 + hidden :] == 7).all() for t in room)


@gpu
@pytest.mark.parametrize("dtype,weight_dtype,bits", [(F16, F16, 9), (F16, F32, 9), (BF16, BF16, 13), (BF16, F32, 13), (F32, F32, 16)])
def test_gradients_of_products_that_cancel(device, dtype, weight_dtype, bits):
    """Two products that cancel to 2^-bits of them: what is left shows the bits of grad_logits far behind those that a result of 16 bits
    has.  Only fp32's roundings are allowed for."""
    gen = torch.Generator().manual_seed(12)

    def two(n):  # n pairs of fp32 numbers whose sum is 2^-bits to twice that of them
        a = 1 + torch.rand(n, 1, generator=gen)
        return torch.cat([a, -a * (1 + 2.0**-bits * (1 + torch.rand(n, 1, generator=gen)))], 1)

    # of the rows: 64 tokens, two experts with one weight
    weight = (1 + torch.rand(1, 512, generator=gen)).to(weight_dtype).expand(2, 512).contiguous()
    x, grad = torch.randn(64, 512, generator=gen).to(dtype), two(64)
    got, _ = router_logits_backward(grad.to(device), x.to(device), weight.to(device))
    want, off = product(grad, weight, 2)
    assert_within(got, want, rounded(want, dtype, off))
    # of the weight: 64 experts, two tokens with one row
    x, grad = (1 + torch.rand(1, 512, generator=gen)).to(dtype).expand(2, 512).contiguous(), two(64).t().contiguous()
    weight = torch.randn(64, 512, generator=gen).to(weight_dtype)
    _, got = router_logits_backward(grad.to(device), x.to(device), weight.to(device))
    want, off = product(grad.t(), x, 2)
    assert_within(got, want, rounded(want, weight_dtype, off))
