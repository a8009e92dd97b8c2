"""The operators between dispatch and combine where their callers may reach and the other tests do not: parts of a sort's slots,
sizes beyond a form's limits, ways of calling that see through the calls.

Tolerances count roundings as in test_experts.py."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from pplx_kernels import (
    SortedTokens,
    int8_matmul,
    ops,
    quantize_rows,
    sort_tokens,
    sort_tokens_backward,
    unsort_tokens,
    unsort_tokens_backward,
)
from tests import test_experts
from tests.test_capi_cpu import _gpu_kernels_of
from tests.test_experts import (
    BF16,
    F16,
    F32,
    U32,
    assert_within,
    check_quantized,
    make_indices,
    make_sorted,
    ref_unsort,
    rounded,
    swiglu64,
    to_u32,
)
from tests.test_experts_path import make_layer, product64, random_int8, run_layer

gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Rows of the gradient that no slot names
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("m,k,more,hidden,dtype", [
    (3, 2, 0, 8, F32), (40, 3, 5, 520, BF16), (700, 4, 0, 1032, F16), (9000, 5, 0, 64, F32), (9000, 5, 0, 16, BF16), (9000, 5, 300, 1040, BF16),
    (60001, 5, 7, 8, F16),
])  # fmt: skip
@pytest.mark.parametrize("part", ["first", "middle", "none", "taken out"])
def test_rows_of_the_gradient_without_a_name(device, m, k, more, hidden, dtype, part):
    """Slots of some of a sort's tokens, or with picks taken out: rows in front of the last live one that nobody names."""
    gen = torch.Generator().manual_seed(m + hidden)
    slots, offsets = make_sorted(m, k, 13, gen, device)
    if part == "taken out":
        slots[torch.rand(m, k, generator=gen) < 0.3] = -1
        tokens = slice(0, m)
    else:
        tokens = {"first": slice(0, m // 3 + 1), "middle": slice(m // 3, m - 1), "none": slice(0, m)}[part]
        if part == "none":
            slots[:] = -1
    slots = slots[tokens].contiguous()
    rows, n = m * k + more, slots.shape[0]
    y = torch.randn(rows, hidden, generator=gen).to(dtype)
    weights, grad_out = torch.rand(n, k, generator=gen), torch.randn(n, hidden, generator=gen).to(dtype)
    grad_y = torch.full((rows, hidden), float("nan"), dtype=dtype, device=device)
    grad_w = torch.full((n, k), float("nan"), device=device)
    unsort_tokens_backward(*(t.to(device) for t in (grad_out, y, slots, offsets, weights)), out=(grad_y, grad_w))
    ref_y = torch.zeros(rows, hidden, dtype=torch.float64)
    t, p = torch.nonzero(slots >= 0, as_tuple=True)
    ref_y[slots[t, p].long()] = grad_out.double()[t] * weights.double()[t, p][:, None]
    assert_within(grad_y, ref_y, rounded(ref_y, dtype, U32 * ref_y.abs()))
    named = torch.zeros(rows, dtype=torch.bool)
    named[slots[t, p].long()] = True
    assert (grad_y.cpu()[~named] == 0).all()
    assert torch.isfinite(grad_w).all() and (grad_w.cpu()[slots < 0] == 0).all()


@gpu
def test_gradients_of_tokens_in_parts(device):
    """A step whose tokens go back in parts, each through a call of its own, has the gradients of the whole step."""
    m, k, experts, hidden = 300, 3, 8, 264
    gen = torch.Generator().manual_seed(11)
    x = torch.randn(m, hidden, generator=gen).to(device)
    indices = to_u32(make_indices(m, k, experts, gen, "mixed"), device)
    weights = torch.rand(m, k, generator=gen).to(device).requires_grad_(True)
    grad = torch.randn(m, hidden, generator=gen).to(device)
    s = sort_tokens(x, indices, experts)
    y = s.rows.clone().requires_grad_(True)
    whole = torch.autograd.grad(unsort_tokens(y, s.slots, s.offsets, weights), [y, weights], grad)
    torch.full((4, *y.shape), float("nan"), device=device)  # (memory that the gradients may get holds no zeros)
    parts = [unsort_tokens(y, s.slots[a : a + 70], s.offsets, weights[a : a + 70]) for a in range(0, m, 70)]
    got = torch.autograd.grad(torch.cat(parts), [y, weights], grad)
    # (a row's gradient is one part's; the others add zeros)
    assert all(torch.equal(a, b) for a, b in zip(got, whole))


# ---------------------------------------------------------------------------
# Forward-mode differentiation
# ---------------------------------------------------------------------------
def check_tangents_are_refused(device):
    """No derivative is lost: a tensor with a tangent, which need not require a gradient, is refused wherever it comes in."""
    idx, offsets = torch.zeros(4, 2, dtype=torch.uint32, device=device), torch.tensor([0, 8], dtype=torch.int32, device=device)
    slots = torch.arange(8, dtype=torch.int32, device=device).view(4, 2)
    x, y, weights = (torch.ones(*shape, device=device) for shape in ((4, 16), (8, 16), (4, 2)))
    with forward_ad.dual_level():
        dx, dy, dw = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, y, weights))
        assert not dx.requires_grad
        for call in (
            lambda: sort_tokens(dx, idx, 1),
            lambda: unsort_tokens(dy, slots, offsets),
            lambda: unsort_tokens(dy, slots, offsets, weights),
            lambda: unsort_tokens(y, slots, offsets, dw),
            lambda: torch.ops.pplx_kernels.sorted_tokens(dx, idx, 1, None, False),
            lambda: torch.ops.pplx_kernels.unsorted_tokens(y, slots, offsets, dw, None),
        ):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_tangents_are_refused_before_the_device_is_looked_at():
    check_tangents_are_refused("cpu")


@gpu
def test_tangents_are_refused(device):
    check_tangents_are_refused(device)
    idx = torch.zeros(4, 2, dtype=torch.uint32, device=device)
    x, y, weights = (torch.randn(*shape, device=device, requires_grad=True) for shape in ((4, 16), (8, 16), (4, 2)))
    s = sort_tokens(x, idx, 1)
    out = unsort_tokens(y, s.slots, s.offsets, weights)
    with forward_ad.dual_level():  # (forward over reverse)
        for made, leaf in ((s.rows, x), (out, y), (out, weights)):
            grad = forward_ad.make_dual(torch.ones_like(made), torch.ones_like(made))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(made, leaf, grad, retain_graph=True)
        # what is not differentiable takes the values
        d = forward_ad.make_dual(x.detach(), torch.ones_like(x))
        assert torch.equal(sort_tokens(d, idx, 1, int8=True).rows, sort_tokens(x.detach(), idx, 1, int8=True).rows)
    assert torch.equal(torch.autograd.grad(s.rows.sum(), x)[0], torch.full_like(x, 2))


# ---------------------------------------------------------------------------
# Modes, tracers and tensors that are more than their data
# ---------------------------------------------------------------------------
def every_call(x, idx, q, scale, weight, weight_scale, w):
    """Each call of the operators, with results of its own and in the caller's."""
    s = sort_tokens(x, idx, 3)
    t = sort_tokens(x, idx, 3, int8=True)
    room = SortedTokens(*(None if a is None else torch.empty_like(a) for a in (s.rows, None, s.slots, s.offsets, None)))
    r = sort_tokens(x, idx, 3, out=room)
    out = unsort_tokens(s.rows, s.slots, s.offsets, w)
    gx = sort_tokens_backward(r.rows, r.slots)
    gy, gw = unsort_tokens_backward(out, s.rows, s.slots, s.offsets, w)
    into = unsort_tokens(s.rows, s.slots, s.offsets, w, out=torch.empty_like(x))
    v, vs = quantize_rows(x)
    y = int8_matmul(q, scale, weight, weight_scale)
    return (*s[:1], *s[2:4], *t[:4], *r[:1], *r[2:4], out, gx, gy, gw, into, v, vs, y)


CALLED = {"sorted_tokens": 2, "sort_tokens": 1, "unsort_tokens": 3, "unsort_tokens_backward": 1, "quantize_rows": 1, "int8_matmul": 1}


def inputs_of_every_call(device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    made = (torch.randn(6, 32, generator=gen), make_indices(6, 2, 3, gen, "mixed"),
            torch.randint(-127, 128, (5, 48), generator=gen, dtype=torch.int8), torch.rand(5, generator=gen),
            torch.randint(-127, 128, (7, 48), generator=gen, dtype=torch.int8), torch.rand(7, generator=gen),
            torch.rand(6, 2, generator=gen))  # fmt: skip
    return [t.to(device).view(torch.uint32) if i == 1 else t.to(device) for i, t in enumerate(made)]


def ops_called(graph) -> dict:
    names = [str(n.target).split(".")[1] for n in graph.graph.nodes if str(n.target).startswith("pplx_kernels.")]
    return {name: names.count(name) for name in set(names)}


def test_modes_and_traces_see_the_calls():
    """Without a device: tensors that have none of their data, and a trace of a graph that needs no compiler."""
    with FakeTensorMode():
        args = [torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in inputs_of_every_call("cpu")]
        got = every_call(*args)
        assert got[0].shape == (12, 32) and got[-1].shape == (5, 7) and got[-1].dtype == BF16
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
        got = graph(*args)
        n = int(want[2][-1])
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), i
        assert n == int(got[2][-1])


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
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert {name: seen.count(f"pplx_kernels::{name}") for name in CALLED} == CALLED


def test_rows_without_a_gradient_need_no_multiple_of_eight():
    """Rows of 12 fp32 elements have a sort and no gradient of it: the registered op takes them unless one is recorded."""
    def call(x):
        return torch.ops.pplx_kernels.sorted_tokens(x, torch.empty(4, 2, dtype=torch.uint32, device="meta"), 3, None, False)

    x = torch.empty(4, 12, device="meta")
    assert call(x)[0].shape == (8, 12)
    x.requires_grad_(True)
    with torch.no_grad():
        assert call(x)[0].shape == (8, 12)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        call(x)


@gpu
def test_traced_rows_without_a_gradient_need_no_multiple_of_eight(device):
    x, idx = torch.randn(4, 12, device=device), torch.zeros(4, 2, dtype=torch.uint32, device=device)
    call = torch.compile(lambda a: sort_tokens(a, idx, 3).rows, backend="aot_eager", fullgraph=True)
    assert torch.equal(call(x), sort_tokens(x, idx, 3).rows)
    x.requires_grad_(True)
    with torch.no_grad():
        assert torch.equal(call(x), sort_tokens(x, idx, 3).rows)
    with pytest.raises(Exception, match="multiple of 8"):
        call(x)


@gpu
def test_compiled_calls(device):
    """torch.compile with its own backend, which turns what surrounds the calls into kernels of its own."""
    pytest.importorskip("triton")
    import torch._inductor.config as inductor

    k, experts, hidden = 2, 4, 64

    def layer(x, weights, indices):
        s = sort_tokens(x, indices, experts)
        return unsort_tokens(s.rows * 2.0, s.slots, s.offsets, weights)

    gen = torch.Generator().manual_seed(9)
    with inductor.patch(compile_threads=1):
        compiled = torch.compile(layer, fullgraph=True, dynamic=True)
        for m in (30, 41):
            x = torch.randn(m, hidden, generator=gen).to(device).requires_grad_(True)
            weights = torch.rand(m, k, generator=gen).to(device).requires_grad_(True)
            indices = to_u32(make_indices(m, k, experts, gen, "mixed"), device)
            want, got = layer(x, weights, indices), compiled(x, weights, indices)
            assert torch.equal(got, want)
            grads = [torch.autograd.grad(out.sum(), [x, weights]) for out in (want, got)]
            assert all(torch.equal(a, b) for a, b in zip(*grads))
        args = make_layer(device, gen, 40, 2, 4, 64, 48)
        assert torch.equal(torch.compile(lambda *a: run_layer(a)[0], fullgraph=True)(*args), run_layer(args)[0])


# ---------------------------------------------------------------------------
# More workgroups than a launch takes threads for along one dimension
# ---------------------------------------------------------------------------
@gpu
def test_more_tokens_than_one_line_of_workgroups(device):
    """2^26 tokens and a few, four to a workgroup of 256 threads: sorted, back again, and the gradient of that."""
    m, experts = (1 << 26) + 5, 8
    gen = torch.Generator(device).manual_seed(1)
    x = torch.randint(-(1 << 15), 1 << 15, (m, 8), dtype=torch.int16, device=device, generator=gen).view(BF16)
    idx = torch.randint(0, experts, (m, 1), dtype=torch.int32, device=device, generator=gen)
    s = sort_tokens(x, idx.view(torch.uint32), experts)
    order = torch.argsort(idx[:, 0], stable=True)
    assert torch.equal(s.slots[:, 0][order], torch.arange(m, dtype=torch.int32, device=device))
    # (in pieces: torch's own gather of 2^26 rows of 16 bytes at once leaves the last ones as zeros)
    for rows, picked in zip(s.rows.view(torch.int16).split(1 << 22), order.split(1 << 22)):
        assert torch.equal(rows, x.view(torch.int16)[picked])
    del order, rows, picked
    x = torch.randn(m, 8, dtype=F32, device=device, generator=gen).to(BF16)
    sort_tokens(x, idx.view(torch.uint32), experts, out=s)
    assert torch.equal(unsort_tokens(s.rows, s.slots, s.offsets), x)
    grad_y, grad_w = torch.empty_like(s.rows), torch.empty(m, 1, device=device)
    unsort_tokens_backward(x, s.rows, s.slots, s.offsets, out=(grad_y, grad_w))
    assert torch.equal(grad_y, s.rows)
    for a in (0, m - 1000):
        size = (x[a : a + 1000].double() ** 2).sum(1, keepdim=True).cpu()
        assert_within(grad_w[a : a + 1000], size, 9 * U32 * size)


@gpu
def test_more_tokens_than_one_line_of_workgroups_one_to_each(device):
    """2^24 tokens and a few, one to a workgroup."""
    m, hidden = (1 << 24) + 3, 1032
    gen = torch.Generator().manual_seed(2)
    y, grad = torch.randn(64, hidden, generator=gen).to(BF16).to(device), torch.randn(1, hidden, generator=gen).to(BF16).to(device)
    slots = (torch.arange(m, dtype=torch.int32, device=device) % 64)[:, None]
    offsets = torch.tensor([0, 64], dtype=torch.int32, device=device)
    got, few = torch.empty(m, 1, device=device), torch.empty(64, 1, device=device)
    unsort_tokens_backward(grad.expand(m, hidden), y, slots, offsets, out=(None, got))
    unsort_tokens_backward(grad.expand(64, hidden), y, slots[:64], offsets, out=(None, few))
    assert all(torch.equal(part, few.repeat(1 << 14, 1)[: part.shape[0]]) for part in got.split(64 << 14))
    # the sort, of rows in 8 bits
    wide = torch.randn(1, 2064, generator=gen).to(BF16).to(device)
    s = sort_tokens(wide.expand(m, 2064), torch.zeros(m, 1, dtype=torch.uint32, device=device), 1, int8=True)
    q, scale = quantize_rows(wide)
    assert all(bool((part == q).all()) for part in s.rows.split(1 << 20)) and bool((s.scale == scale).all())


@gpu
def test_more_rows_than_one_line_of_workgroups(device):
    rows = (1 << 26) + 7
    x = torch.empty(rows, 16, dtype=BF16, device=device).normal_(generator=torch.Generator(device).manual_seed(3))
    q, scale = quantize_rows(x)
    for part, q_part, scale_part in zip(x.split(1 << 22), q.split(1 << 22), scale.split(1 << 22)):
        want, want_scale = quantize_rows(part)
        assert torch.equal(q_part, want) and torch.equal(scale_part, want_scale)


# ---------------------------------------------------------------------------
# Rows that go past the caches, and rows longer than registers hold
# ---------------------------------------------------------------------------
def large_step(device, m, k, hidden, y_dtype, grad_dtype):
    gen = torch.Generator(device).manual_seed(m + hidden)
    idx = torch.randint(0, 10, (m, k), dtype=torch.int32, generator=gen, device=device)  # (two of ten experts are elsewhere)
    s = sort_tokens(torch.zeros(m, 8, dtype=BF16, device=device), idx.view(torch.uint32), 8)
    y = torch.randn(m * k, hidden, generator=gen, device=device).to(y_dtype)
    y[int(s.offsets[-1]) :] = float("nan")
    weights = torch.where(s.slots >= 0, torch.rand(m, k, generator=gen, device=device), float("nan"))
    grad = torch.randn(m, hidden, generator=gen, device=device).to(grad_dtype)
    return s.slots, s.offsets, y, weights, grad


@gpu
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k,hidden,y_dtype", [(9001, 6, 1000, BF16), (9001, 6, 1000, F16), (9001, 3, 1000, F32)])
def test_large_gathers(device, m, k, hidden, y_dtype, out_dtype):
    """More than the 96 MiB from which on rows are read past the caches: as in parts, which are read through them."""
    assert m * k * hidden * y_dtype.itemsize > 96 << 20 > 3000 * k * hidden * y_dtype.itemsize
    slots, offsets, y, weights, _ = large_step(device, m, k, hidden, y_dtype, F32)
    got = unsort_tokens(y, slots, offsets, weights, out_dtype=out_dtype)
    for a in range(0, m, 3000):
        assert torch.equal(got[a : a + 3000], unsort_tokens(y, slots[a : a + 3000], offsets, weights[a : a + 3000], out_dtype=out_dtype))
    few = slice(m - 40, m)
    ref, size = ref_unsort(y.cpu(), slots[few].cpu(), weights[few].cpu())
    assert_within(got[few], ref, rounded(ref, out_dtype, (k + 1) * U32 * size))


@gpu
@pytest.mark.parametrize("grad_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k,hidden,y_dtype", [
    (9001, 4, 1000, BF16), (9001, 4, 1000, F16), (9001, 2, 1000, F32), (6001, 4, 1544, BF16), (6001, 4, 1544, F16), (6001, 2, 1544, F32),
])  # fmt: skip
def test_large_gradients(device, m, k, hidden, y_dtype, grad_dtype):
    """The same of the gradient, from 56 MiB on, with a wave to a token and with a workgroup."""
    part = 2500
    assert m * k * hidden * y_dtype.itemsize > 56 << 20 > part * k * hidden * y_dtype.itemsize
    slots, offsets, y, weights, grad = large_step(device, m, k, hidden, y_dtype, grad_dtype)
    grad_y, grad_w = unsort_tokens_backward(grad, y, slots, offsets, weights)
    assert (grad_y[int(offsets[-1]) :] == 0).all()
    for a in range(0, m, part):
        some = slots[a : a + part]
        part_y, part_w = unsort_tokens_backward(grad[a : a + part], y, some, offsets, weights[a : a + part])
        rows = some[some >= 0].long()
        assert torch.equal(grad_y[rows], part_y[rows]) and torch.equal(grad_w[a : a + part], part_w)
    few = torch.arange(m - 40, m)
    live, at = slots[few].cpu() >= 0, slots[few].cpu().clamp_min(0).long()
    picked = torch.where(live[:, :, None], y.cpu().double()[at], 0.0) * grad[few].cpu().double()[:, None]
    assert_within(grad_w[few], picked.sum(2), (hidden + 1) * U32 * picked.abs().sum(2))
    t, p = torch.nonzero(live, as_tuple=True)
    ref = grad[few].cpu().double()[t] * weights[few].cpu().double()[t, p][:, None]
    assert_within(grad_y[at[t, p].to(device)], ref, rounded(ref, y_dtype, U32 * ref.abs()))


@gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("m,k,experts,hidden,dtype,bound,routing", [
    (33, 3, 7, 8208, BF16, 30, "mixed"), (40, 2, 5, 8208, F32, None, "any"), (40, 2, 5, 5000, F32, None, "mixed"), (7, 3, 4, 20000, F16, 6, "mixed"),
    (4200, 2, 5, 8208, BF16, 4199, "mixed"), (2100, 4, 9, 8208, F32, None, "mixed"),
])  # fmt: skip
def test_sort_tokens_of_long_rows(device, m, k, experts, hidden, dtype, bound, routing, int8):
    """Copies of more than 16 KiB and quantised rows of more than 8192 elements take more than one turn, in one launch and in
    three."""
    test_experts.test_sort_tokens(device, m, k, experts, hidden, dtype, bound, routing, int8)


@gpu
def test_the_activation_to_the_end_of_its_range(device):
    """Gates down to -88.7, whose sigmoid is subnormal, with values that bring the result back to ordinary sizes."""
    gate = torch.linspace(-88.7, -80.0, 256)[:, None].expand(256, 48)
    x = torch.cat([gate, torch.full((256, 48), 1e36)], dim=1).contiguous()
    q, scale = quantize_rows(x.to(device), swiglu=True)
    v, off = swiglu64(x)
    assert float(v.abs().min()) > 0.1
    check_quantized(q, scale, v, off)


# ---------------------------------------------------------------------------
# Products whose workgroups take several tiles
# ---------------------------------------------------------------------------
SEVERAL_TILES = [
    # tile, layout, experts, rows (padded: of each expert), n, k: odd and even n, k that fills the steps of its form and k that does not
    ((32, 128), "dense", 1, 9, 65544, 128),
    ((32, 128), "dense", 1, 9, 65537, 64),
    ((32, 128), "sorted", 32, 33, 2057, 128),
    ((32, 128), "sorted", 32, 33, 2056, 64),
    ((32, 128), "padded", 4, 40, 8201, 64),
    ((64, 128), "sorted", 16, 33, 2056, 2064),
    ((64, 128), "sorted", 16, 33, 2057, 2064),
    ((64, 128), "sorted", 8, 700, 2056, 1024),
    ((64, 128), "sorted", 8, 700, 2057, 1024),
    ((64, 128), "padded", 32, 257, 520, 272),
    ((64, 256), "sorted", 4, 200, 16392, 528),
    ((64, 256), "sorted", 4, 200, 16385, 528),
    ((64, 256), "sorted", 32, 1500, 2056, 1024),
    ((64, 256), "sorted", 32, 1500, 2057, 1024),
    ((64, 256), "padded", 32, 520, 1000, 528),
    ((128, 128), "dense", 1, 70, 65544, 64),
    ((128, 128), "dense", 1, 70, 65537, 80),
    ((128, 128), "sorted", 32, 1500, 2056, 80),
    ((128, 128), "sorted", 32, 1500, 2057, 64),
    ((128, 128), "padded", 4, 2000, 2057, 64),
    ((128, 256), "sorted", 4, 257, 16392, 528),
    ((128, 256), "sorted", 4, 257, 16385, 528),
    ((128, 256), "sorted", 32, 2049, 2056, 1024),
    ((128, 256), "sorted", 32, 2049, 2057, 1024),
    ((128, 256), "padded", 16, 520, 2057, 272),
    ((256, 256), "dense", 1, 700, 32776, 272),
    ((256, 256), "dense", 1, 700, 32777, 512),
    ((256, 256), "sorted", 16, 4999, 2056, 512),
    ((256, 256), "sorted", 16, 4999, 2057, 528),
    ((256, 256), "padded", 8, 2000, 4104, 64),
]


def rows_of_experts(layout, experts, rows):
    if layout == "padded":
        return [rows - e % 5 for e in range(experts)]
    return [rows // experts + (e < rows % experts) for e in range(experts)]


@pytest.mark.parametrize("tile,layout,experts,rows,n,k", SEVERAL_TILES)
def test_the_products_of_several_tiles_are_that(tile, layout, experts, rows, n, k):
    """Each size of the test below takes the form that it is there for, and more of its tiles than there are workgroups."""
    plan = ops.product_plan_of(rows, n, k, experts, layout)
    assert (plan.tile_rows, plan.tile_columns) == tile and not plan.split
    columns = -(-n // tile[1])
    tiles = sum(-(-c // tile[0]) for c in rows_of_experts(layout, experts, rows)) * columns
    assert plan.workgroups < tiles <= plan.tiles


@gpu
def test_products_record_no_gradient(device):
    """Neither the products nor the quantisation are differentiable: their results say so, whatever the scales require."""
    q, scale = quantize_rows(torch.randn(4, 32, device=device, requires_grad=True))
    assert not q.requires_grad and not scale.requires_grad
    got = int8_matmul(q, scale.requires_grad_(True), q, scale)
    assert not got.requires_grad


def test_plans_of_products():
    assert ops.product_plan_of(1, 1408, 2048).split == 1
    nothing = ops.product_plan_of(0, 8, 16)
    assert (nothing.tile_rows, nothing.workgroups, nothing.tiles) == (0, 0, 0)
    for bad, message in (
        (dict(rows=4, n=8, k=24), "multiple of 16"),
        (dict(rows=4, n=8, k=131072), "131056"),
        (dict(rows=4, n=1 << 31, k=16), "2\\^31"),
        (dict(rows=4, n=8, k=16, experts=0, layout="sorted"), "num_experts"),
        (dict(rows=4, n=8, k=16, experts=2), "one expert"),
        (dict(rows=1 << 30, n=8, k=16, experts=2, layout="padded"), "2\\^31"),
    ):
        with pytest.raises(RuntimeError, match=message):
            ops.product_plan_of(**bad)
    lib = ops.load_library()
    assert lib.pplx_a2a_int8_matmul_plan(None, 8, 16, None) == 1


def test_the_products_of_several_tiles_are_of_every_kind():
    steps = {(32, 128): 128, (64, 128): 128, (64, 256): 128, (128, 128): 64, (128, 256): 64, (256, 256): 64}
    for tile, step in steps.items():
        here = [(n % 2, k % step == 0) for t, _, _, _, n, k in SEVERAL_TILES if t == tile]
        assert {odd for odd, _ in here} == {0, 1} and {full for _, full in here} == {True, False}
        assert any(t == tile and layout == "padded" for t, layout, *_ in SEVERAL_TILES)


def assert_product(got, ref):
    """The sum becomes fp32, the scales are multiplied, and their product with the sum; then the result is rounded to its type.
    (fp16 has no more than multiples of 2^-24 below 2^-14: off by 2^-25 there, which `rounded` counts.)"""
    off = (got.double() - ref).abs() - rounded(ref, got.dtype, 3 * U32 * ref.abs())
    assert float(off.max()) <= 0


@gpu
@pytest.mark.parametrize("tile,layout,experts,rows,n,k", SEVERAL_TILES)
def test_products_of_several_tiles(device, tile, layout, experts, rows, n, k):
    """A workgroup's second tile, whose first loads go out in front of the stores of the tile before, in every form and type."""
    gen = torch.Generator(device).manual_seed(rows + n + k)
    counts = rows_of_experts(layout, experts, rows)
    shape = (experts, rows) if layout == "padded" else (rows,)
    x, xs = random_int8((*shape, k), gen, device), torch.rand(shape, generator=gen, device=device) * 1e-2
    lead = () if layout == "dense" else (experts,)
    w, ws = random_int8((*lead, n, k), gen, device), torch.rand((*lead, n), generator=gen, device=device) * 1e-2
    where = {}
    if layout == "padded":
        where["num_tokens"] = torch.tensor(counts, dtype=torch.int32, device=device)
    elif layout == "sorted":
        where["offsets"] = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=device)
    outs = [torch.full((*shape, n), 7.0, dtype=t, device=device) for t in (BF16, F16, F32)]
    for out in outs:
        int8_matmul(x, xs, w, ws, **where, out=out)
    first = 0
    for e, c in enumerate(counts):
        at = (e, slice(0, c)) if layout == "padded" else (slice(first, first + c),)
        first += c
        ref = product64(x[at], xs[at], w[e] if lead else w, ws[e] if lead else ws)
        for out in outs:
            assert_product(out[at], ref)
            if layout == "padded":
                assert (out[e, c:] == 7).all()


# ---------------------------------------------------------------------------
# What the kernels take of a workgroup
# ---------------------------------------------------------------------------
def test_product_tiles_begin_at_the_first_byte_of_lds():
    """The steps of a tile, which loads write to LDS directly, lie in front of everything else that a workgroup has there, and
    no kernel of the products spills."""
    kernels = [k for k in _gpu_kernels_of(ops._LIB_PATH) if "matmul_tiles" in k[".name"]]
    assert len(kernels) == 6 * 2 * 3  # forms, k that fills the steps or not, types
    assert {k[".group_segment_fixed_size"] for k in kernels} == {0}
    assert {k[".vgpr_spill_count"] for k in kernels} == {0} and {k[".sgpr_spill_count"] for k in kernels} == {0}
