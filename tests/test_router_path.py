"""The operators before dispatch as they are used: in a run, in graphs, on other streams, from two threads, traced; and what the C
entry points refuse, which needs no GPU."""

from __future__ import annotations

import ctypes
import threading

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from pplx_kernels import (
    LoopbackWorld,
    NormedRows,
    SortedTokens,
    int8_matmul,
    ops,
    quantize_rows,
    rms_norm,
    rms_norm_backward,
    rms_norm_workspace,
    route_tokens,
    route_tokens_backward,
    router_logits,
    router_logits_backward,
    router_workspace,
    sort_tokens,
    sort_tokens_backward,
    unsort_tokens,
    unsort_tokens_backward,
)
from pplx_kernels.workloads import DeviceStep, WorkloadSpec, generate, make_world
from tests.test_experts import BF16, F16, F32, U32, assert_within, rounded, to_u32
from tests.test_router import E4M3, ref_route, weight_error

gpu = pytest.mark.gpu


def signed(t):
    return t.view(torch.int32) if t.dtype == torch.uint32 else t


def same(a, b):
    """The same bits, also of NaN."""
    if a.dtype == E4M3 or a.dtype.is_floating_point:
        a, b = (t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]) for t in (a, b))
    return torch.equal(signed(a), signed(b))


# ---------------------------------------------------------------------------
# Runs
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("ranks,experts,k,hidden,tokens", [(2, 8, 2, 512, 20), (4, 32, 4, 1024, 65)])
def test_norm_router_dispatch_combine(device, ranks, experts, k, hidden, tokens):
    """A step whose rows, scales, picks and weights the operators make: experts that multiply their rows by a number of their own."""
    spec = WorkloadSpec("fp8", 90, ranks, experts, k, hidden, tokens, E4M3, tokens="uniform")
    step = DeviceStep(spec, generate(spec, seed=4))
    gen = torch.Generator().manual_seed(5)
    norm_weight = (1 + 0.1 * torch.randn(hidden, generator=gen)).to(BF16).to(device)
    gate = (torch.randn(experts, hidden, generator=gen) / hidden**0.5).to(device)
    bias = (0.05 * torch.randn(experts, generator=gen)).to(device)
    choice = dict(scores="sigmoid", num_groups=4, top_groups=2, scale=2.5)
    made = []
    for r in range(ranks):
        x, residual = (torch.randn(tokens, hidden, generator=gen).to(BF16).to(device) for _ in range(2))
        n = rms_norm(x, norm_weight, residual, quantize=E4M3)
        logits = router_logits(n.y, gate)
        indices, weights = route_tokens(logits, k, bias=bias, bound_m=step.bound_m[r], **choice)
        want, _ = ref_route(logits.cpu(), k, bias.cpu(), bound=step.groups[r].n, **choice)
        assert torch.equal(signed(indices).cpu(), want)
        step.dp_x[r], step.dp_x_scale[r], step.indices[r], step.weights[r] = n.q, n.scale, indices, weights
        made.append(n)
    world = make_world(spec, group_name=f"router-{ranks}-{hidden}")
    step.dispatch_world(world)
    for r in range(ranks):
        local = experts // ranks
        of_block = step.expert_x_scale[r].repeat_interleave(128, dim=2)[..., :hidden]
        factor = torch.arange(r * local + 1, (r + 1) * local + 1, device=device).view(-1, 1, 1)
        step.expert_y[r].copy_(step.expert_x[r].float() * of_block * factor)
    step.combine_world(world)
    assert world.faults() == 0
    for r in range(ranks):
        n, idx, w = step.groups[r].n, signed(step.indices[r]).cpu().long(), step.weights[r].cpu().double()
        q = made[r].q.float().cpu().double() * made[r].scale.cpu().double().repeat_interleave(128, dim=1)[:, :hidden]
        ref, size = torch.zeros(tokens, hidden, dtype=torch.float64), torch.zeros(tokens, hidden, dtype=torch.float64)
        for p in range(k):
            y = (q[:n] * (idx[:n, p : p + 1] + 1)).float().to(spec.expert_y_dtype).double()
            part = y * w[:n, p : p + 1]
            ref[:n] += part
            # (the copy above rounds its products in fp32 before it rounds to the experts' type, this one may round the other way)
            size[:n] += part.abs() * ((k + 1) * U32 + torch.finfo(spec.expert_y_dtype).eps)
        assert_within(step.out_tokens[r][:n], ref[:n], rounded(ref[:n], BF16, size[:n]))
    world.destroy()


def make_step(device, gen, m, hidden=256, experts=16, dtype=BF16, weight_dtype=None):
    """x, residual, the norm's weight, the router's weight, its bias"""
    weight_dtype = weight_dtype or dtype
    made = [torch.randn(m, hidden, generator=gen).to(dtype), torch.randn(m, hidden, generator=gen).to(dtype),
            (1 + 0.1 * torch.randn(hidden, generator=gen)).to(weight_dtype),
            (torch.randn(experts, hidden, generator=gen) / hidden**0.5).to(weight_dtype), 0.05 * torch.randn(experts, generator=gen)]  # fmt: skip
    return [t.to(device) for t in made]


CHOICE = dict(scores="sigmoid", num_groups=4, top_groups=2, scale=2.5)


@gpu
@pytest.mark.parametrize("m", [1, 70, 2100])
def test_a_layer_of_own_experts(device, m):
    """From the norm to the sum of the experts, on one rank: the picks and weights are what sort and unsort take."""
    gen = torch.Generator().manual_seed(m)
    k, experts, hidden, wide = 4, 16, 256, 96
    x, residual, norm_weight, gate, bias = make_step(device, gen, m, hidden, experts)
    w1, w2 = (torch.randint(-127, 128, shape, generator=gen, dtype=torch.int32).to(torch.int8).to(device)
              for shape in ((experts, 2 * wide, hidden), (experts, hidden, wide)))  # fmt: skip
    s1, s2 = (torch.rand(shape, generator=gen).div(73 * 16).to(device) for shape in ((experts, 2 * wide), (experts, hidden)))
    bound = to_u32(torch.tensor([max(1, m - 3)], dtype=torch.int32), device)

    def layer(indices, weights, y):
        s = sort_tokens(y, indices, experts, bound, int8=True)
        h = int8_matmul(s.rows, s.scale, w1, s1, offsets=s.offsets)
        q, scale = quantize_rows(h, offsets=s.offsets, swiglu=True)
        rows = int8_matmul(q, scale, w2, s2, offsets=s.offsets)
        return unsort_tokens(rows, s.slots, s.offsets, weights), unsort_tokens(rows.abs(), s.slots, s.offsets, weights, out_dtype=F32)

    n = rms_norm(x, norm_weight, residual)
    logits = router_logits(n.y, gate)
    indices, weights = route_tokens(logits, k, bias=bias, bound_m=bound, **CHOICE)
    got, _ = layer(indices, weights, n.y)
    # the choice by the oracle: the same picks, and weights that differ by their rounding
    want, want_weights = ref_route(logits.cpu(), k, bias.cpu(), bound=max(1, m - 3), **CHOICE)
    assert torch.equal(signed(indices).cpu(), want)
    other, size = (t.double().cpu() for t in layer(indices, want_weights.float().to(device), n.y))
    assert (got[max(1, m - 3):] == 0).all()
    # two sums of k products each, of weights that differ by weight_error and a rounding: d apart.  Both are rounded to bf16, each by
    # half a step, eps / 2 of its value, which is at most (|other| + d) (1 + eps).
    d, eps = size * (weight_error(experts) + U32 + 2 * (k + 1) * U32), torch.finfo(BF16).eps
    assert_within(got, other, d + (other.abs() + d) * eps * (1 + eps))


@gpu
@pytest.mark.parametrize("dtype,weight_dtype", [(F32, F32), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("m", [1, 60, 1500])
def test_a_training_step(device, m, dtype, weight_dtype):
    """Through the whole layer gradients come out that are the chain of the operators' own, which are held against the formulas one by
    one; the residual stream passes by the experts."""
    gen = torch.Generator().manual_seed(m)
    k, experts, hidden = 3, 12, 192
    x, residual, norm_weight, gate, bias = make_step(device, gen, m, hidden, experts, dtype, weight_dtype)
    leaves = [t.requires_grad_(True) for t in (x, residual, norm_weight, gate)]
    grad = torch.randn(m, hidden, generator=gen).to(dtype).to(device)
    more = dict(scores="sigmoid", renormalize=False)
    n = rms_norm(x, norm_weight, residual)
    logits = router_logits(n.y, gate)
    indices, weights = route_tokens(logits, k, bias=bias, **more)
    s = sort_tokens(n.y, indices, experts)
    out = n.sum + unsort_tokens(s.rows, s.slots, s.offsets, weights, out_dtype=dtype)
    got = torch.autograd.grad(out, leaves, grad)
    with torch.no_grad():
        y, total = n.y.detach(), n.sum.detach()
        grad_rows, grad_weights = unsort_tokens_backward(grad, s.rows, s.slots, s.offsets, weights)
        grad_y = sort_tokens_backward(grad_rows, s.slots)
        grad_logits = route_tokens_backward(grad_weights, logits, indices, **more)
        grad_y2, grad_gate = router_logits_backward(grad_logits, y, gate)
        for order in ((grad_y, grad_y2), (grad_y2, grad_y)):  # (which of the two is added to the other is autograd's affair)
            grad_h, grad_norm = rms_norm_backward(order[0] + order[1], total, norm_weight, grad_sum=grad)
        assert all(same(a, b) for a, b in zip(got, (grad_h, grad_h, grad_norm, grad_gate)))
        # and the choice itself has no gradient through the indices: all that the router learns came through the weights
        assert grad_gate.abs().sum() > 0


# ---------------------------------------------------------------------------
# Graphs, streams, threads
# ---------------------------------------------------------------------------
class Buffers:
    """All that a step of the operators writes, forwards and backwards."""

    def __init__(self, m, k, experts, hidden, dtype, args, quantize=None):
        device = args[0].device
        self.normed = NormedRows.empty(m, hidden, dtype, device, residual=True, quantize=quantize)
        self.logits = torch.zeros(m, experts, device=device)
        self.routed = torch.zeros(m, k, dtype=torch.uint32, device=device), torch.zeros(m, k, device=device)
        self.grad_logits = torch.zeros(m, experts, device=device)
        self.grad_router = torch.zeros_like(args[0]), torch.zeros_like(args[3])
        self.grad_norm = torch.zeros_like(args[0]), torch.zeros_like(args[2])
        self.spaces = (router_workspace(args[0], args[3]), router_workspace(args[0], args[3], backward=True),
                       rms_norm_workspace(args[0]))  # fmt: skip

    def all(self):
        return [t for part in (self.normed, [self.logits], self.routed, [self.grad_logits], self.grad_router, self.grad_norm)
                for t in part if t is not None]  # fmt: skip


def run_step(args, grad_weights, b, k, bound=None, spaces=True):
    x, residual, norm_weight, gate, bias = args
    s = b.spaces if spaces else (None, None, None)
    rms_norm(x, norm_weight, residual, out=b.normed)
    router_logits(b.normed.y, gate, out=b.logits, workspace=s[0])
    route_tokens(b.logits, k, bias=bias, bound_m=bound, out=b.routed, **CHOICE)
    route_tokens_backward(grad_weights, b.logits, b.routed[0], scores="sigmoid", scale=2.5, out=b.grad_logits)
    router_logits_backward(b.grad_logits, b.normed.y, gate, out=b.grad_router, workspace=s[1])
    rms_norm_backward(b.grad_router[0], b.normed.sum, norm_weight, out=b.grad_norm, workspace=s[2])


@gpu
@pytest.mark.parametrize("m,hidden,experts,dtype", [(1, 64, 16, F32), (40, 256, 64, BF16), (64, 2048, 256, F16), (2500, 512, 64, BF16)])
@pytest.mark.parametrize("raw", [False, True])
def test_a_captured_step_follows_its_inputs(device, m, hidden, experts, dtype, raw):
    k = 4
    gen = torch.Generator().manual_seed(7)
    args, grad_weights = make_step(device, gen, m, hidden, experts, dtype), torch.randn(m, k, generator=gen).to(device)
    bound = to_u32(torch.tensor([m], dtype=torch.int32), device)
    quantize = E4M3 if raw else torch.int8
    b, eager = (Buffers(m, k, experts, hidden, dtype, args, quantize) for _ in range(2))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run_step(args, grad_weights, b, k, bound)
        if raw:  # the library's own capture
            world = LoopbackWorld(16, 8, 2, 1, 1, 64, 128, 0, group_name=f"router-capture-{m}")
            with world.capture() as captured:
                run_step(args, grad_weights, b, k, bound)
            replay = captured.graph.replay
        else:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                run_step(args, grad_weights, b, k, bound, spaces=False)
            replay = graph.replay
        for i in range(4):
            for old, fresh in zip((*args, grad_weights), (*make_step(device, gen, m, hidden, experts, dtype),
                                                          torch.randn(m, k, generator=gen).to(device))):  # fmt: skip
                old.copy_(fresh)
            bound.view(torch.int32).fill_(max(0, m - 3 * i))
            for t in (b.logits, b.grad_logits, *b.grad_router, *b.grad_norm):
                t.fill_(float("nan"))
            replay()
            torch.cuda.synchronize()
            run_step(args, grad_weights, eager, k, bound)
            junk = torch.full((1 << 22,), float("nan"), device=device)  # (eager work between the replays)
            for got, want in zip(b.all(), eager.all()):
                assert same(got, want)
            del junk
        if raw:
            world.destroy()


@gpu
def test_two_graphs_of_one_workspace_follow_each_other(device):
    """Two captured steps that were given the same workspace, replayed in turn on one stream."""
    gen = torch.Generator().manual_seed(8)
    m, k, experts, hidden = 300, 4, 64, 1024
    steps = []
    stream = torch.cuda.Stream()
    for _ in range(2):
        args, grad_weights = make_step(device, gen, m, hidden, experts), torch.randn(m, k, generator=gen).to(device)
        steps.append((args, grad_weights, Buffers(m, k, experts, hidden, BF16, args), Buffers(m, k, experts, hidden, BF16, args)))
    steps[1][2].spaces = steps[0][2].spaces
    graphs = []
    torch.cuda.synchronize()
    for args, grad_weights, b, _ in steps:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run_step(args, grad_weights, b, k)
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for args, grad_weights, b, eager in steps:
        run_step(args, grad_weights, eager, k)
        assert all(same(x, y) for x, y in zip(b.all(), eager.all()))


@gpu
def test_gradients_are_not_recorded_under_capture(device):
    """The gradients' own forms are captured while an eager graph of the same leaves lives; autograd is refused there."""
    gen = torch.Generator().manual_seed(2)
    m, k, experts, hidden = 60, 3, 16, 128
    args = make_step(device, gen, m, hidden, experts, F32)
    leaves = [t.requires_grad_(True) for t in args[:4]]
    grad_weights = torch.randn(m, k, generator=gen).to(device)

    def loss():
        n = rms_norm(leaves[0], leaves[2], leaves[1])
        logits = router_logits(n.y, leaves[3])
        return route_tokens(logits, k, bias=args[4], **CHOICE)[1]

    weights = loss()
    want = torch.autograd.grad(weights, leaves, grad_weights, retain_graph=True)
    plain = [t.detach() for t in args]
    b = Buffers(m, k, experts, hidden, F32, plain)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream), torch.no_grad():
        run_step(plain, grad_weights, b, k)
        with torch.enable_grad():
            for record in (lambda: rms_norm(leaves[0], leaves[2]), lambda: router_logits(leaves[0], leaves[3]),
                           lambda: route_tokens(b.logits.requires_grad_(True), k)):  # fmt: skip
                with pytest.raises(RuntimeError, match="not recorded under stream capture"):
                    record()
        b.logits.requires_grad_(False)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got = (b.grad_norm[0], b.grad_norm[0], b.grad_norm[1], b.grad_router[1])
        assert all(same(x, y) for x, y in zip(got, want))
        (plain[0] * 2).sum()
    assert all(same(x, y) for x, y in zip(torch.autograd.grad(weights, leaves, grad_weights), want))


@gpu
def test_calls_follow_the_current_stream(device):
    gen = torch.Generator().manual_seed(3)
    m, k, experts, hidden = 300, 4, 64, 1024
    args, grad_weights = make_step(device, gen, m, hidden, experts), torch.randn(m, k, generator=gen).to(device)
    want, b = (Buffers(m, k, experts, hidden, BF16, args, E4M3) for _ in range(2))
    run_step(args, grad_weights, want, k)
    late = torch.zeros_like(args[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)  # (what runs on another stream would read zeros)
        late.copy_(args[0])
        run_step((late, *args[1:]), grad_weights, b, k, spaces=False)
    stream.synchronize()
    assert all(same(x, y) for x, y in zip(b.all(), want.all()))


@gpu
def test_two_threads_on_streams_of_their_own(device):
    gen = torch.Generator().manual_seed(6)
    steps = []
    for m, hidden, experts in ((500, 256, 64), (90, 4096, 256)):
        args, grad_weights = make_step(device, gen, m, hidden, experts), torch.randn(m, 4, generator=gen).to(device)
        b, want = (Buffers(m, 4, experts, hidden, BF16, args, torch.int8) for _ in range(2))
        run_step(args, grad_weights, want, 4)
        steps.append((args, grad_weights, b, want))
    torch.cuda.synchronize()
    failures: list = []

    def work(args, grad_weights, b, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i in range(30):
                    run_step(args, grad_weights, b, 4, spaces=i % 2 == 0)
                    torch.cuda.current_stream().synchronize()
                    if not all(same(x, y) for x, y in zip(b.all(), want.all())):
                        failures.append("other results")
        except Exception as exc:
            failures.append(exc)

    threads = [threading.Thread(target=work, args=step) for step in steps]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


@gpu
@pytest.mark.parametrize("m,hidden,experts,dtype", [(4000, 1024, 128, BF16), (700, 17008, 60, F32), (64, 4096, 256, F16)])
def test_the_same_inputs_give_the_same_bits(device, m, hidden, experts, dtype):
    gen = torch.Generator().manual_seed(8)
    args, grad_weights = make_step(device, gen, m, hidden, experts, dtype), torch.randn(m, 4, generator=gen).to(device)
    first = None
    for _ in range(4):
        b = Buffers(m, 4, experts, hidden, dtype, args, E4M3)
        run_step(args, grad_weights, b, 4)
        if first is not None:
            assert all(same(x, y) for x, y in zip(b.all(), first.all()))
        first = b


# ---------------------------------------------------------------------------
# Autograd's edges
# ---------------------------------------------------------------------------
@gpu
def test_gradients_of_some_inputs_and_some_outputs(device):
    gen = torch.Generator().manual_seed(4)
    x, residual, norm_weight, gate, _ = make_step(device, gen, 33, 128, 16, F32)
    grad = torch.randn(33, 128, generator=gen).to(device)
    want_h, want_w = rms_norm_backward(grad, x + residual, norm_weight)
    for needs in ((True, False, False), (False, True, False), (False, False, True), (True, True, True)):
        leaves = [t.detach().requires_grad_(n) for t, n in zip((x, residual, norm_weight), needs)]
        n = rms_norm(leaves[0], leaves[2], leaves[1])
        got = torch.autograd.grad(n.y, [t for t in leaves if t.requires_grad], grad, retain_graph=True)
        assert all(same(a, b) for a, b in zip(got, [g for g, need in zip((want_h, want_h, want_w), needs) if need]))
        if needs[0]:  # of the sum alone, which the weight has no part in
            (got,) = torch.autograd.grad(n.sum, leaves[:1], grad, retain_graph=True)
            assert torch.equal(got, grad)
    # x is its own residual; gradients that are one element, or rows that lie apart
    leaf = x.detach().requires_grad_(True)
    n = rms_norm(leaf, norm_weight, leaf)
    (got,) = torch.autograd.grad(n.y.sum(), leaf)
    assert torch.equal(got, 2 * rms_norm_backward(torch.ones_like(x), x + x, norm_weight)[0])
    leaf, weight = x.detach().requires_grad_(True), gate.detach().requires_grad_(True)
    logits = router_logits(leaf, weight)
    apart = torch.randn(33, 40, generator=gen).to(device)[:, 7:23]
    for g in (torch.ones((), device=device).expand(33, 16), apart, apart.t().contiguous().t()):
        got = torch.autograd.grad(logits, [leaf, weight], g, retain_graph=True)
        assert all(same(a, b) for a, b in zip(got, router_logits_backward(g.contiguous(), x, gate)))
    plain = torch.randn(33, 16, generator=gen).to(device)
    leaf = plain.clone().requires_grad_(True)
    indices, weights = route_tokens(leaf, 4)
    assert not indices.requires_grad
    (got,) = torch.autograd.grad(weights, leaf, torch.ones((), device=device).expand(33, 4))
    assert same(got, route_tokens_backward(torch.ones(33, 4, device=device), plain, indices))
    leaf.grad = None
    route_tokens(leaf * 1.0, 4)[1].square().sum().backward()
    assert leaf.grad.shape == leaf.shape


@gpu
def test_gradients_are_differentiable_once(device):
    gen = torch.Generator().manual_seed(4)
    x, _, norm_weight, gate, _ = make_step(device, gen, 9, 64, 8, F32)
    leaf = x.requires_grad_(True)
    for out in (rms_norm(leaf, norm_weight).y, router_logits(leaf, gate), route_tokens(leaf, 3)[1]):
        (got,) = torch.autograd.grad(out.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            got.sum().backward()


@gpu
def test_inputs_that_change_before_the_gradient_are_told(device):
    gen = torch.Generator().manual_seed(4)
    x, residual, norm_weight, gate, _ = make_step(device, gen, 9, 64, 8, F32)
    for make, change in (
        (lambda a: rms_norm(a * 1.0, norm_weight, residual), lambda n: rms_norm(x, norm_weight, residual, out=NormedRows(n.sum, torch.empty_like(x)))),
        (lambda a: rms_norm(a * 1.0, norm_weight, residual), lambda n: n.sum.zero_()),
    ):
        n = make(x.detach().requires_grad_(True))
        with torch.no_grad():
            change(n)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            n.y.sum().backward()
    a = x.detach().requires_grad_(True) * 1.0
    logits = router_logits(a, gate)
    with torch.no_grad():
        rms_norm(x.detach(), norm_weight, out=NormedRows(a))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        logits.sum().backward()
    a = torch.randn(9, 8, device=device, requires_grad=True) * 1.0
    weights = route_tokens(a, 3)[1]
    with torch.no_grad():
        router_logits(x.detach(), gate, out=a)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        weights.sum().backward()


def check_tangents_are_refused(device):
    """No derivative is lost: a tensor with a tangent, which need not require a gradient, is refused wherever it comes in."""
    x, weight, gate, logits = (torch.ones(*shape, device=device) for shape in ((4, 16), (16,), (8, 16), (4, 8)))
    with forward_ad.dual_level():
        dx, dw, dg, dl = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, weight, gate, logits))
        for call in (
            lambda: rms_norm(dx, weight), lambda: rms_norm(x, dw), lambda: rms_norm(x, weight, dx), lambda: router_logits(dx, gate),
            lambda: router_logits(x, dg), lambda: route_tokens(dl, 2),
            lambda: torch.ops.pplx_kernels.normed_rows(dx, weight, None, 1e-6), lambda: torch.ops.pplx_kernels.new_logits(x, dg),
            lambda: torch.ops.pplx_kernels.routed_tokens(dl, 2, None, None, 1, 1, 2, False, True, 1.0),
        ):  # fmt: skip
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_tangents_are_refused_before_the_device_is_looked_at():
    check_tangents_are_refused("cpu")


@gpu
def test_tangents_are_refused(device):
    check_tangents_are_refused(device)


@gpu
def test_steps_without_tokens(device):
    for dtype in (F32, BF16):
        x = torch.empty(0, 64, dtype=dtype, device=device, requires_grad=True)
        weight, gate = (torch.ones(*shape, dtype=dtype, device=device, requires_grad=True) for shape in ((64,), (8, 64)))
        n = rms_norm(x, weight, x)
        logits = router_logits(n.y, gate)
        indices, weights = route_tokens(logits, 2, num_groups=2, top_groups=1)
        assert n.y.shape == (0, 64) and logits.shape == (0, 8) and indices.shape == weights.shape == (0, 2)
        gx, gw, gg = torch.autograd.grad(weights.sum() + n.sum.sum(), [x, weight, gate])
        assert gx.shape == (0, 64) and (gw == 0).all() and (gg == 0).all()
        for code in (torch.int8, E4M3):
            q = rms_norm(x.detach(), weight, quantize=code)
            assert q.q.shape == (0, 64) and q.scale.shape[0] == 0


# ---------------------------------------------------------------------------
# Modes, tracers and tensors that are more than their data
# ---------------------------------------------------------------------------
def every_call(x, residual, norm_weight, gate, bias, logits, grad):
    """Each call of the operators, with results of its own and in the caller's."""
    n = rms_norm(x, norm_weight, residual)
    q = rms_norm(x, norm_weight, residual, quantize=torch.int8)
    e = rms_norm(x, norm_weight, quantize=E4M3)
    into = rms_norm(x, norm_weight, residual, out=NormedRows(torch.empty_like(x), torch.empty_like(x)))
    made = router_logits(n.y, gate)
    room = router_logits(n.y, gate, out=torch.empty_like(made))
    indices, weights = route_tokens(logits, 3, bias=bias, **CHOICE)
    again = route_tokens(made, 3, out=(torch.empty_like(indices), torch.empty_like(weights)))
    gl = route_tokens_backward(weights, logits, indices, scores="sigmoid", scale=2.5)
    gx, gg = router_logits_backward(made, n.y, gate)
    gh, gw = rms_norm_backward(grad, n.sum, norm_weight)
    return (n.y, n.sum, q.y, q.sum, q.q, q.scale, e.y, e.q, e.scale, into.y, into.sum, made, room, indices, weights, *again, gl, gx, gg, gh, gw)


CALLED = {"normed_rows": 1, "rms_norm": 3, "rms_norm_backward": 1, "new_logits": 1, "router_logits": 1, "router_logits_backward": 1,
          "routed_tokens": 1, "route_tokens": 1, "route_tokens_backward": 1}  # fmt: skip


def inputs_of_every_call(device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    made = make_step(device, gen, 6, 256, 16, F32)
    return [*made, torch.randn(6, 16, generator=gen).to(device), torch.randn(6, 256, generator=gen).to(device)]


def ops_called(graph) -> dict:
    names = [str(n.target).split(".")[1] for n in graph.graph.nodes if str(n.target).startswith("pplx_kernels.")]
    return {name: names.count(name) for name in set(names)}


def test_modes_and_traces_see_the_calls():
    """Without a device: tensors that have none of their data, and a trace of a graph that needs no compiler."""
    with FakeTensorMode():
        args = [torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in inputs_of_every_call("cpu")]
        got = every_call(*args)
        assert got[0].shape == (6, 256) and got[8].shape == (6, 2) and got[13].dtype == torch.uint32
        assert ops_called(make_fx(every_call)(*args)) == CALLED


@gpu
def test_traced_graphs_hold_the_calls(device):
    """What make_fx traces on real tensors computes the same on others."""
    graph = make_fx(every_call)(*inputs_of_every_call(device))
    assert ops_called(graph) == CALLED
    for seed in (1, 2):
        args = inputs_of_every_call(device, seed)
        want = every_call(*args)
        torch.full((1 << 20,), float("nan"), device=device)  # (memory that the results may get)
        assert all(same(a, b) for a, b in zip(graph(*args), want))


@gpu
def test_a_mode_sees_the_calls(device):
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.name())
            return func(*args, **(kwargs or {}))

    args = inputs_of_every_call(device)
    want = every_call(*args)
    with Mode():
        got = every_call(*args)
    assert all(same(a, b) for a, b in zip(got, want))
    assert {name: seen.count(f"pplx_kernels::{name}") for name in CALLED} == CALLED


@gpu
def test_traced_calls(device):
    """Under torch.compile the calls are the registered ops, traced once for any number of tokens; gradients flow through them."""
    gen = torch.Generator().manual_seed(9)
    traces, first = [], None

    def backend(graph, inputs):
        traces.append(len(inputs))
        return torch._dynamo.lookup_backend("aot_eager")(graph, inputs)

    def layer(x, residual, norm_weight, gate, bias):
        n = rms_norm(x * 1.0, norm_weight, residual)
        q = rms_norm(x, norm_weight, residual, quantize=E4M3)
        logits = router_logits(n.y, gate)
        indices, weights = route_tokens(logits, 3, bias=bias, **CHOICE)
        s = sort_tokens(n.y, indices, 16)
        return n.sum + unsort_tokens(s.rows * 2.0, s.slots, s.offsets, weights), q.scale, logits

    compiled = torch.compile(layer, backend=backend, fullgraph=True, dynamic=True)
    for m in (30, 41, 7):
        args = make_step(device, gen, m, 128, 16, F32)
        leaves = [t.requires_grad_(True) for t in args[:4]]
        want, got = layer(*args), compiled(*args)
        first = first or len(traces)  # (torch begins again where a size of the first call, here the blocks of a row, is one)
        assert len(traces) == first and all(same(a, b) for a, b in zip(got, want))
        grads = [torch.autograd.grad(out[0].sum(), leaves) for out in (want, got)]
        assert all(torch.allclose(a, b, rtol=1e-5, atol=1e-6) for a, b in zip(*grads))


@gpu
def test_every_call_compiled(device):
    args = inputs_of_every_call(device)
    got = torch.compile(every_call, backend="aot_eager", fullgraph=True)(*args)
    assert all(same(a, b) for a, b in zip(got, every_call(*args)))


# ---------------------------------------------------------------------------
# The C entry points refuse before anything reaches a device
# ---------------------------------------------------------------------------
P, U, I, L, Q, FL = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float


def struct(*fields):
    return type("Args", (ctypes.Structure,), {"_fields_": list(fields)})


NormArgs = struct(
    ("x", P), ("x_stride_row", L), ("residual", P), ("residual_stride_row", L), ("weight", P), ("dtype", I), ("weight_dtype", I),
    ("eps", FL), ("m", U), ("hidden_dim", Q), ("y", P), ("y_stride_row", L), ("sum", P), ("sum_stride_row", L), ("q", P),
    ("q_stride_row", L), ("scale", P), ("scale_stride_row", L), ("scale_stride_block", L), ("format", I),
)  # fmt: skip
NormBackwardArgs = struct(
    ("grad_y", P), ("grad_y_stride_row", L), ("grad_sum", P), ("grad_sum_stride_row", L), ("h", P), ("h_stride_row", L), ("weight", P),
    ("dtype", I), ("weight_dtype", I), ("eps", FL), ("m", U), ("hidden_dim", Q), ("grad_h", P), ("grad_h_stride_row", L),
    ("grad_weight", P), ("workspace", P),
)  # fmt: skip
LogitsArgs = struct(
    ("x", P), ("x_stride_row", L), ("weight", P), ("weight_stride_row", L), ("dtype", I), ("weight_dtype", I), ("m", U),
    ("num_experts", U), ("hidden_dim", Q), ("logits", P), ("logits_stride_row", L), ("workspace", P),
)  # fmt: skip
LogitsBackwardArgs = struct(
    ("grad_logits", P), ("grad_logits_stride_row", L), ("x", P), ("x_stride_row", L), ("weight", P), ("weight_stride_row", L),
    ("dtype", I), ("weight_dtype", I), ("m", U), ("num_experts", U), ("hidden_dim", Q), ("grad_x", P), ("grad_x_stride_row", L),
    ("grad_weight", P), ("grad_weight_stride_row", L), ("workspace", P),
)  # fmt: skip
RouteArgs = struct(
    ("logits", P), ("logits_stride_row", L), ("dtype", I), ("m", U), ("num_experts", U), ("experts_per_token", U), ("bias", P),
    ("bound_m", P), ("num_groups", U), ("top_groups", U), ("group_top", U), ("scores", I), ("renormalize", I), ("weight_scale", FL),
    ("indices", P), ("weights", P),
)  # fmt: skip
RouteBackwardArgs = struct(
    ("grad_weights", P), ("logits", P), ("logits_stride_row", L), ("indices", P), ("dtype", I), ("m", U), ("num_experts", U),
    ("experts_per_token", U), ("scores", I), ("renormalize", I), ("weight_scale", FL), ("grad_logits", P),
    ("grad_logits_stride_row", L),
)  # fmt: skip
A = 0x10000  # an address that nobody reads
GOOD = {
    "rms_norm": (NormArgs, dict(x=A, x_stride_row=64, weight=A, dtype=1, weight_dtype=1, eps=1e-6, m=4, hidden_dim=32, y=A,
                                y_stride_row=64)),
    "rms_norm_backward": (NormBackwardArgs, dict(grad_y=A, grad_y_stride_row=64, h=A, h_stride_row=64, weight=A, dtype=1,
                                                 weight_dtype=1, eps=1e-6, m=4, hidden_dim=32, grad_h=A, grad_h_stride_row=64,
                                                 grad_weight=A, workspace=A)),
    "router_logits": (LogitsArgs, dict(x=A, x_stride_row=64, weight=A, weight_stride_row=64, dtype=1, weight_dtype=1, m=4,
                                       num_experts=8, hidden_dim=32, logits=A, logits_stride_row=8, workspace=A)),
    "router_logits_backward": (LogitsBackwardArgs, dict(grad_logits=A, grad_logits_stride_row=8, x=A, x_stride_row=64, weight=A,
                                                        weight_stride_row=64, dtype=1, weight_dtype=1, m=4, num_experts=8,
                                                        hidden_dim=32, grad_x=A, grad_x_stride_row=64, grad_weight=A,
                                                        grad_weight_stride_row=64, workspace=A)),
    "route_tokens": (RouteArgs, dict(logits=A, logits_stride_row=8, dtype=0, m=4, num_experts=8, experts_per_token=2, num_groups=1,
                                     top_groups=1, group_top=2, weight_scale=1.0, indices=A, weights=A)),
    "route_tokens_backward": (RouteBackwardArgs, dict(grad_weights=A, logits=A, logits_stride_row=8, indices=A, dtype=0, m=4,
                                                      num_experts=8, experts_per_token=2, weight_scale=1.0, grad_logits=A,
                                                      grad_logits_stride_row=8)),
}  # fmt: skip


def c_call(name, device=0, **changed):
    kind, good = GOOD[name]
    lib = ops.load_library()
    fn = getattr(lib, f"pplx_a2a_{name}")
    fn.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
    args = kind(**{**good, **changed})
    return fn(device, ctypes.addressof(args), None), lib.pplx_a2a_last_error().decode()


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("name,changed,status,message", [
    ("rms_norm", dict(x=None), 1, "x is NULL"),
    ("rms_norm", dict(x=A + 8), 1, "16-byte"),
    ("rms_norm", dict(x_stride_row=72), 1, "16-byte"),
    ("rms_norm", dict(weight=None), 1, "weight"),
    ("rms_norm", dict(weight=A + 4), 1, "weight"),
    ("rms_norm", dict(dtype=3), 1, "dtype"),
    ("rms_norm", dict(weight_dtype=2), 1, "weight_dtype"),
    ("rms_norm", dict(eps=0.0), 1, "eps"),
    ("rms_norm", dict(eps=-1.0), 1, "eps"),
    ("rms_norm", dict(eps=NAN), 1, "eps"),
    ("rms_norm", dict(eps=INF), 1, "eps"),
    ("rms_norm", dict(hidden_dim=0), 1, "hidden_dim"),
    ("rms_norm", dict(hidden_dim=36), 1, "hidden_dim"),
    ("rms_norm", dict(hidden_dim=1 << 27), 1, "hidden_dim"),
    ("rms_norm", dict(y=None), 1, "neither y nor q"),
    ("rms_norm", dict(y=A + 8), 1, "16-byte"),
    ("rms_norm", dict(residual=A, residual_stride_row=64), 1, "sum"),
    ("rms_norm", dict(sum=A, sum_stride_row=64), 1, "sum"),
    ("rms_norm", dict(residual=A, residual_stride_row=40, sum=A, sum_stride_row=64), 1, "16-byte"),
    ("rms_norm", dict(format=3), 1, "format"),
    ("rms_norm", dict(format=1, q=A, q_stride_row=32), 1, "scale"),
    ("rms_norm", dict(format=1, q=A, q_stride_row=40, scale=A, scale_stride_row=1), 1, "16-byte"),
    ("rms_norm", dict(format=2, q=A, q_stride_row=32, scale=A, scale_stride_row=1, hidden_dim=24), 1, "16"),
    ("rms_norm", dict(m=1 << 31), 4, "2^31"),
    ("rms_norm_backward", dict(h=None), 1, "h is NULL"),
    ("rms_norm_backward", dict(grad_y=A + 4), 1, "16-byte"),
    ("rms_norm_backward", dict(grad_sum=A, grad_sum_stride_row=24), 1, "16-byte"),
    ("rms_norm_backward", dict(grad_h_stride_row=56), 1, "16-byte"),
    ("rms_norm_backward", dict(grad_weight=A + 4), 1, "grad_weight"),
    ("rms_norm_backward", dict(workspace=None), 1, "workspace"),
    ("rms_norm_backward", dict(workspace=A + 4), 1, "workspace"),
    ("rms_norm_backward", dict(m=0), 1, "tokens"),
    ("rms_norm_backward", dict(eps=0.0), 1, "eps"),
    ("rms_norm_backward", dict(m=1 << 31), 4, "2^31"),
    ("router_logits", dict(x=None), 1, "x is NULL"),
    ("router_logits", dict(weight=A + 8), 1, "16-byte"),
    ("router_logits", dict(weight_stride_row=72), 1, "16-byte"),
    ("router_logits", dict(dtype=1, weight_dtype=2), 1, "weight_dtype"),
    ("router_logits", dict(hidden_dim=12), 1, "hidden_dim"),
    ("router_logits", dict(hidden_dim=0), 1, "hidden_dim"),
    ("router_logits", dict(num_experts=0), 1, "num_experts"),
    ("router_logits", dict(num_experts=5462), 1, "num_experts"),
    ("router_logits", dict(logits=None), 1, "logits"),
    ("router_logits", dict(logits=A + 2), 1, "logits"),
    ("router_logits", dict(m=64, num_experts=256, hidden_dim=7168, x_stride_row=14336, weight_stride_row=14336, workspace=None), 1, "workspace"),
    ("router_logits", dict(m=1 << 31), 4, "2^31"),
    ("router_logits_backward", dict(grad_logits=None), 1, "grad_logits"),
    ("router_logits_backward", dict(x=None), 1, "x is NULL"),
    ("router_logits_backward", dict(weight=None), 1, "weight is NULL"),
    ("router_logits_backward", dict(grad_x_stride_row=72), 1, "16-byte"),
    ("router_logits_backward", dict(grad_weight=A + 8), 1, "16-byte"),
    ("router_logits_backward", dict(workspace=None), 1, "workspace"),
    ("router_logits_backward", dict(m=0), 1, "tokens"),
    ("route_tokens", dict(logits=None), 1, "NULL"),
    ("route_tokens", dict(indices=None), 1, "NULL"),
    ("route_tokens", dict(weights=None), 1, "NULL"),
    ("route_tokens", dict(logits=A + 2), 1, "aligned"),
    ("route_tokens", dict(bias=A + 2), 1, "aligned"),
    ("route_tokens", dict(bound_m=A + 2), 1, "aligned"),
    ("route_tokens", dict(dtype=7), 1, "dtype"),
    ("route_tokens", dict(num_experts=0), 1, "num_experts"),
    ("route_tokens", dict(num_experts=5462), 1, "num_experts"),
    ("route_tokens", dict(experts_per_token=0), 1, "experts_per_token"),
    ("route_tokens", dict(experts_per_token=9), 1, "experts_per_token"),
    ("route_tokens", dict(num_experts=100, experts_per_token=65), 1, "experts_per_token"),
    ("route_tokens", dict(num_groups=0), 1, "num_groups"),
    ("route_tokens", dict(num_groups=3), 1, "num_groups"),
    ("route_tokens", dict(num_groups=4, top_groups=0), 1, "top_groups"),
    ("route_tokens", dict(num_groups=4, top_groups=5), 1, "top_groups"),
    ("route_tokens", dict(num_groups=4, top_groups=2, group_top=0), 1, "group_top"),
    ("route_tokens", dict(num_groups=4, top_groups=2, group_top=3), 1, "group_top"),
    ("route_tokens", dict(num_groups=8, top_groups=2, group_top=2), 1, "group_top"),
    ("route_tokens", dict(num_groups=8, top_groups=1, group_top=1), 1, "fewer than"),
    ("route_tokens", dict(scores=2), 1, "scores"),
    ("route_tokens", dict(weight_scale=NAN), 1, "weight_scale"),
    ("route_tokens", dict(weight_scale=INF), 1, "weight_scale"),
    ("route_tokens", dict(m=1 << 31), 4, "2^31"),
    ("route_tokens_backward", dict(m=1 << 31), 4, "2^31"),
    ("route_tokens_backward", dict(grad_weights=None), 1, "NULL"),
    ("route_tokens_backward", dict(grad_logits=A + 1), 1, "aligned"),
    ("route_tokens_backward", dict(experts_per_token=9), 1, "experts_per_token"),
    ("route_tokens_backward", dict(scores=-1), 1, "scores"),
])  # fmt: skip
def test_c_entry_points_refuse(name, changed, status, message):
    got, said = c_call(name, **changed)
    assert got == status and message in said, (got, said)


@pytest.mark.parametrize("name", list(GOOD))
def test_c_entry_points_take_null_and_unknown_devices_for_errors(name):
    lib = ops.load_library()
    fn = getattr(lib, f"pplx_a2a_{name}")
    fn.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
    assert fn(0, None, None) == 1 and "args is NULL" in lib.pplx_a2a_last_error().decode()
    got, said = c_call(name, device=99)
    assert got == 3 and "99" in said


@pytest.mark.parametrize("name", ["rms_norm", "router_logits", "route_tokens", "route_tokens_backward"])
def test_c_entry_points_of_steps_without_tokens_touch_no_device(name):
    assert c_call(name, device=99, m=0)[0] == 0


def test_workspaces():
    lib = ops.load_library()
    norm, router = lib.pplx_a2a_rms_norm_workspace, lib.pplx_a2a_router_workspace
    norm.argtypes, router.argtypes = [U, Q, ctypes.c_void_p], [U, U, Q, I, I, I, ctypes.c_void_p]
    out = ctypes.c_uint64(7)
    at = ctypes.addressof(out)
    for m, hidden in ((1, 8), (100, 2048), (100000, 2048), (8192, 7168), (8192, 20000), (3, (1 << 27) - 8)):
        assert norm(m, hidden, at) == 0 and 0 < out.value <= 512 * 4 * hidden and out.value % 4 == 0
    assert norm(1, 12, at) == 1 and norm(1 << 31, 64, at) == 4 and norm(1, 8, None) == 1
    for dtype in (0, 1, 2):
        for weight_dtype in {dtype, 0}:
            for m, experts, hidden in ((1, 1, 8), (64, 256, 7168), (8192, 256, 7168), (100000, 5461, 64), (2**31 - 1, 4, 8)):
                assert router(m, experts, hidden, dtype, weight_dtype, 0, at) == 0 and out.value <= 512 << 20
                assert router(m, experts, hidden, dtype, weight_dtype, 1, at) == 0 and out.value > 0
    assert router(4, 256, 64, 1, 1, 0, at) == 0 and out.value == 0
    assert router(4, 256, 64, 1, 2, 0, at) == 1 and router(4, 0, 64, 1, 1, 0, at) == 1 and router(4, 4, 64, 1, 1, 0, None) == 1
