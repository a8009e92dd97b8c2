"""The operators between dispatch and combine against their definitions in 64 bits on the CPU.

Tolerances count roundings: one to nearest is off by at most ``finfo(t).eps / 2`` of the value (half the step of the
subnormals where it is below those), and a chain of n fp32 additions or fused multiply-adds by n * 2**-24 of the sum of the
magnitudes (to first order; the second is far below the slack that counting the longest chain leaves)."""

from __future__ import annotations

import pytest
import torch

from pplx_kernels import (
    AllToAll,
    LoopbackWorld,
    SortedTokens,
    int8_matmul,
    quantize_rows,
    sort_tokens,
    sort_tokens_backward,
    unsort_tokens,
    unsort_tokens_backward,
)

U32 = 2.0**-24  # a rounding to fp32
TINY = 2.0**-100
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
gpu = pytest.mark.gpu


def rounded(ref: torch.Tensor, dtype: torch.dtype, before: torch.Tensor) -> torch.Tensor:
    """How far a value may be from ``ref`` that was off by ``before`` and then rounded to ``dtype``."""
    info = torch.finfo(dtype)
    half = info.eps / 2
    return before + half * (ref.abs() + before) + info.smallest_normal * half


def assert_within(got: torch.Tensor, ref: torch.Tensor, tolerance: torch.Tensor) -> None:
    got = got.detach().cpu().double()
    off = (got - ref).abs() - tolerance
    assert torch.isfinite(got).all()
    assert (off <= 0).all(), f"off by {off.max().item()} more than allowed at {off.argmax().item()}"


# ---------------------------------------------------------------------------
# Definitions
# ---------------------------------------------------------------------------
def ref_sort(indices: torch.Tensor, experts: int, bound: int):
    """slots, offsets and the pick of each row, by walking through experts, tokens and picks."""
    ids = indices.long()
    ids[bound:] = experts
    m, k = ids.shape
    picks = torch.nonzero(ids.reshape(-1) < experts)[:, 0]
    by_expert = ids.reshape(-1)[picks].sort(stable=True)
    order = picks[by_expert.indices]
    slots = torch.full((m * k,), -1, dtype=torch.int32)
    slots[order] = torch.arange(order.numel(), dtype=torch.int32)
    counts = torch.bincount(by_expert.values, minlength=experts)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).to(torch.int32)
    return slots.view(m, k), offsets, order


def ref_quantize(v: torch.Tensor):
    """fp32 rows to whole numbers and scales, in fp32 (each operation is rounded once, here as there; quotients of two
    tensors, because torch takes a number over a tensor for the number times a rounded reciprocal)."""
    a, most = v.abs().amax(1).clamp_min(TINY), torch.full((v.shape[0],), 127.0)
    return torch.round(v * torch.div(most, a)[:, None]).to(torch.int8), torch.div(a, most)


def make_indices(m: int, k: int, experts: int, gen: torch.Generator, kind: str) -> torch.Tensor:
    if kind == "one":  # all to one expert, as often as there are picks
        return torch.full((m, k), experts - 1, dtype=torch.int32)
    if kind == "none":  # all experts are elsewhere
        return torch.where(torch.rand(m, k, generator=gen) < 0.5, -1, experts).to(torch.int32)
    if kind == "mixed":  # some elsewhere, experts repeat inside tokens
        return torch.randint(0, 2 * experts, (m, k), generator=gen, dtype=torch.int32)
    return torch.randint(0, experts, (m, k), generator=gen, dtype=torch.int32)


def to_u32(t: torch.Tensor, device) -> torch.Tensor:
    return t.to(device).view(torch.uint32)


SORTS = [
    # tokens, picks, experts, hidden, dtype, bound, routing
    (1, 1, 1, 8, BF16, None, "any"),
    (1, 8, 256, 7168, BF16, None, "any"),
    (4, 6, 64, 2048, F16, 3, "any"),
    (5, 64, 64, 16, F16, None, "mixed"),
    (33, 3, 7, 520, BF16, 0, "any"),
    (100, 10, 128, 4328, BF16, 77, "mixed"),
    (127, 8, 5461, 24, BF16, None, "any"),
    (512, 8, 256, 264, F32, None, "mixed"),
    (513, 8, 256, 264, F32, 500, "mixed"),
    (1024, 8, 256, 264, F16, None, "mixed"),  # the most picks that take one launch
    (8192, 1, 5461, 16, BF16, 8191, "any"),
    (1025, 8, 256, 264, F16, 1000, "mixed"),  # few more: three
    (1500, 7, 5461, 40, BF16, 1499, "any"),
    (1500, 7, 1700, 40, BF16, None, "mixed"),
    (9001, 9, 33, 136, F16, 8000, "mixed"),
    (2000, 5, 3, 2880, BF16, None, "one"),
    (700, 6, 16, 2056, BF16, None, "none"),
    (70000, 2, 8, 8, BF16, 100000, "any"),  # a bound beyond the tokens
]


@gpu
@pytest.mark.parametrize("m,k,experts,hidden,dtype,bound,routing", SORTS)
@pytest.mark.parametrize("int8", [False, True])
def test_sort_tokens(device, m, k, experts, hidden, dtype, bound, routing, int8):
    gen = torch.Generator().manual_seed(m * 31 + k)
    if int8:
        hidden = (hidden + 15) // 16 * 16
    x = (torch.randn(m, hidden, generator=gen) * torch.exp(torch.randn(m, 1, generator=gen))).to(dtype)
    indices = make_indices(m, k, experts, gen, routing)
    there = m if bound is None else min(m, bound)
    slots, offsets, order = ref_sort(torch.where(indices < 0, experts, indices), experts, there)
    bound_m = None if bound is None else to_u32(torch.tensor([bound], dtype=torch.int32), device)
    got = sort_tokens(x.to(device), to_u32(indices, device), experts, bound_m, int8=int8)
    assert torch.equal(got.slots.cpu(), slots)
    assert torch.equal(got.offsets.cpu(), offsets)
    source, scale = ref_quantize(x.float()) if int8 else (x, None)
    rows = torch.zeros(m * k, hidden, dtype=source.dtype)
    rows[: order.numel()] = source[order // k]
    assert torch.equal(got.rows.cpu(), rows)
    if int8:
        scales = torch.zeros(m * k)
        scales[: order.numel()] = scale[order // k]
        assert torch.equal(got.scale.cpu(), scales)
    else:
        assert got.scale is None


@gpu
def test_sort_tokens_of_no_tokens(device):
    got = sort_tokens(torch.empty(0, 16, dtype=BF16, device=device), torch.empty(0, 4, dtype=torch.uint32, device=device), 9)
    assert got.rows.shape == (0, 16) and got.slots.shape == (0, 4)
    assert torch.equal(got.offsets.cpu(), torch.zeros(10, dtype=torch.int32))
    y = torch.empty(0, 16, dtype=BF16, device=device)
    assert unsort_tokens(y, got.slots, got.offsets).shape == (0, 16)
    grad_y, grad_w = unsort_tokens_backward(y, y, got.slots, got.offsets, torch.empty(0, 4, device=device))
    assert grad_y.shape == (0, 16) and grad_w.shape == (0, 4)


@gpu
def test_sort_tokens_takes_strided_rows_and_buffers(device):
    m, k, experts, hidden = 40, 4, 16, 64
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(m, 2 * hidden, generator=gen).to(BF16).to(device)
    x = wide[:, hidden:]  # every other half row
    indices = to_u32(make_indices(m, k, experts, gen, "mixed"), device)
    buffers = SortedTokens.empty(m, hidden, experts, k, BF16, device)
    room = torch.full((m * k, hidden + 32), 7.0, dtype=BF16, device=device)
    buffers = buffers._replace(rows=room[:, 16 : 16 + hidden])
    got = sort_tokens(x, indices, experts, out=buffers)
    want = sort_tokens(x.contiguous(), indices, experts)
    assert got is buffers and torch.equal(got.rows, want.rows) and torch.equal(got.slots, want.slots)
    assert (room[:, :16] == 7).all() and (room[:, 16 + hidden :] == 7).all()
    expanded = x[:1].expand(m, hidden)
    assert torch.equal(sort_tokens(expanded, indices, experts).rows, sort_tokens(expanded.contiguous(), indices, experts).rows)


UNSORTS = [
    # tokens, picks, rows behind the picks, hidden, y, out, weights
    (1, 1, 0, 8, BF16, BF16, True),
    (1, 64, 0, 520, F16, F16, True),
    (7, 8, 0, 7168, BF16, BF16, True),
    (33, 5, 0, 2880, F32, F16, True),
    (33, 6, 3, 2048, F32, BF16, False),
    (200, 3, 0, 1032, F16, F32, True),
    (301, 10, 500, 512, BF16, BF16, False),
    (64, 9, 0, 504, BF16, F32, True),
]


def make_sorted(m, k, experts, gen, device, bound=None, routing="mixed"):
    indices = make_indices(m, k, experts, gen, routing)
    slots, offsets, order = ref_sort(torch.where(indices < 0, experts, indices), experts, m if bound is None else bound)
    return slots, offsets


def ref_unsort(y, slots, weights):
    live = slots >= 0
    picked = torch.where(live[:, :, None], y.double()[slots.clamp_min(0).long()], 0.0)
    w = torch.where(live, weights.double(), 0.0) if weights is not None else live.double()
    return (picked * w[:, :, None]).sum(1), (picked * w[:, :, None]).abs().sum(1)


@gpu
@pytest.mark.parametrize("m,k,more,hidden,y_dtype,out_dtype,weighted", UNSORTS)
def test_unsort_tokens_and_its_gradients(device, m, k, more, hidden, y_dtype, out_dtype, weighted):
    gen = torch.Generator().manual_seed(m + 7 * k)
    slots, offsets = make_sorted(m, k, 13, gen, device, bound=max(1, m - 2))
    rows = m * k + more
    y = torch.randn(rows, hidden, generator=gen).to(y_dtype)
    weights = torch.randn(m, k, generator=gen) if weighted else None
    grad_out = torch.randn(m, hidden, generator=gen).to(out_dtype)
    # what no pick names is not looked at
    live = slots >= 0
    y[int(offsets[-1]) :] = float("nan")
    if weighted:
        weights[~live] = float("nan")
    dev = [t if t is None else t.to(device) for t in (y, slots, offsets, weights)]
    out = unsort_tokens(*dev, out_dtype=out_dtype)
    assert out.dtype == out_dtype
    ref, size = ref_unsort(y, slots, weights)
    assert_within(out, ref, rounded(ref, out_dtype, (k + 1) * U32 * size))

    grad_y, grad_w = unsort_tokens_backward(grad_out.to(device), *dev)
    w = torch.where(live, weights, 0.0) if weighted else live.float()
    ref_y = torch.zeros(rows, hidden, dtype=torch.float64)
    t, p = torch.nonzero(live, as_tuple=True)
    ref_y[slots[t, p].long()] = grad_out.double()[t] * w.double()[t, p][:, None]
    assert_within(grad_y, ref_y, rounded(ref_y, y_dtype, U32 * ref_y.abs()))
    if not weighted:
        assert grad_w is None
        return
    picked = torch.where(live[:, :, None], y.double()[slots.clamp_min(0).long()], 0.0) * grad_out.double()[:, None]
    assert_within(grad_w, picked.sum(2), (hidden + 1) * U32 * picked.abs().sum(2))
    assert (grad_w.cpu()[~live] == 0).all()
    # each of the two alone
    only_y, none = torch.empty_like(dev[0]), None
    unsort_tokens_backward(grad_out.to(device), *dev, out=(only_y, none))
    assert torch.equal(only_y.cpu(), grad_y.cpu())
    only_w = torch.empty_like(dev[3])
    unsort_tokens_backward(grad_out.to(device), *dev, out=(none, only_w))
    assert torch.equal(only_w.cpu(), grad_w.cpu())


@gpu
def test_unsort_keeps_infinities_of_live_rows_and_ignores_others(device):
    slots = torch.tensor([[0, -1], [-1, -1], [1, 2], [9, 0]], dtype=torch.int32, device=device)  # 9: behind the rows
    offsets = torch.tensor([0, 3], dtype=torch.int32, device=device)
    y = torch.tensor([1.0, float("inf"), 2.0], device=device)[:, None].expand(3, 8).to(BF16).contiguous()
    weights = torch.tensor([[2.0, float("inf")], [float("nan"), 1.0], [1.0, 1.0], [float("nan"), 3.0]], device=device)
    out = unsort_tokens(y, slots, offsets, weights)
    assert torch.equal(out[:, 0].cpu().float(), torch.tensor([2.0, 0.0, float("inf"), 3.0]))


@gpu
@pytest.mark.parametrize("hidden,k", [(64, 3), (2048, 2), (7168, 8)])
def test_autograd_of_sort_and_unsort(device, hidden, k):
    m, experts = 50, 6
    gen = torch.Generator().manual_seed(hidden)
    x = torch.randn(m, hidden, generator=gen)
    weights = torch.rand(m, k, generator=gen)
    indices = make_indices(m, k, experts, gen, "mixed")
    bound = 45
    scale = torch.rand(experts, generator=gen) + 0.5
    slots, offsets, order = ref_sort(torch.where(indices < 0, experts, indices), experts, bound)
    expert_of = torch.zeros(m * k, dtype=torch.long)
    expert_of[: order.numel()] = torch.bucketize(torch.arange(order.numel()), offsets[1:].long(), right=True)

    def leaves(dtype, dev):
        return [t.to(dev, dtype).requires_grad_(True) for t in (x, weights)]

    ref_x, ref_w = leaves(torch.float64, "cpu")
    rows = torch.zeros(m * k, hidden, dtype=torch.float64).index_add(0, torch.arange(order.numel()), ref_x[order // k])
    y = rows * scale.double()[expert_of][:, None]
    live = slots >= 0
    picked = y[slots.clamp_min(0).long()] * (live * ref_w)[:, :, None]
    grad = torch.randn(m, hidden, generator=gen)
    ref_gx, ref_gw = torch.autograd.grad(picked.sum(1), [ref_x, ref_w], grad.double())

    got_x, got_w = leaves(F32, device)
    s = sort_tokens(got_x, to_u32(indices, device), experts, to_u32(torch.tensor([bound], dtype=torch.int32), device))
    out = unsort_tokens(s.rows * scale.to(device)[expert_of.to(device)][:, None], s.slots, s.offsets, got_w)
    gx, gw = torch.autograd.grad(out, [got_x, got_w], grad.to(device))
    # x: the weight, the scale and a sum over the picks; w: a product with the scale and a sum over the row
    size_x = (live * weights).double().abs() @ torch.ones(k, dtype=torch.float64)
    assert_within(gx, ref_gx, (k + 3) * U32 * 1.5 * size_x[:, None] * grad.double().abs())
    size_w = torch.where(live, (x.double().abs() * grad.double().abs()).sum(1)[:, None] * 1.5, 0.0)
    assert_within(gw, ref_gw, (hidden + 3) * U32 * size_w)
    # against differences along one direction: the output is bilinear in x and w
    step_x, step_w = torch.randn(m, hidden, generator=gen).to(device), torch.randn(m, k, generator=gen).to(device)

    def value(a):
        with torch.no_grad():
            r = sort_tokens(got_x + a * step_x, to_u32(indices, device), experts,
                            to_u32(torch.tensor([bound], dtype=torch.int32), device))  # fmt: skip
            o = unsort_tokens(r.rows * scale.to(device)[expert_of.to(device)][:, None], r.slots, r.offsets, got_w + a * step_w)
            return (o.double() * grad.to(device).double()).sum().item()

    along = ((gx.double() * step_x.double()).sum() + (gw.double() * step_w.double()).sum()).item()
    # (a central difference of a quadratic is exact; each value's fp32 sums are off by (k + 3) * 2^-24 of their magnitudes)
    a = 0.5
    noise = sum((k + 3) * U32 * ((abs(got_x) + a * abs(step_x)).double().amax(1, True).expand(m, hidden).cpu() *
                ((live * (weights + a * step_w.abs().cpu())).double().sum(1) * 1.5)[:, None] * grad.double().abs()).sum().item()
                for _ in range(2)) / (2 * a)  # fmt: skip
    noise += ((gx.double().abs() * step_x.double().abs()).sum() + (gw.double().abs() * step_w.double().abs()).sum()).item() * 1e-5
    assert abs((value(a) - value(-a)) / (2 * a) - along) <= noise


@gpu
def test_autograd_layouts_of_gradients(device):
    """Gradients that come expanded, transposed or from part of the outputs; leaves that want none."""
    m, k, experts, hidden = 20, 2, 4, 32
    gen = torch.Generator().manual_seed(1)
    indices = to_u32(make_indices(m, k, experts, gen, "any"), device)
    x = torch.randn(m, hidden, generator=gen).to(device).requires_grad_(True)
    s = sort_tokens(x, indices, experts)
    s.rows.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, k))
    x.grad = None
    s = sort_tokens(x, indices, experts)
    (s.rows.t() * 2.0).t().sum(0).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2 * k))
    weights = torch.ones(m, k, device=device, requires_grad=True)
    out = unsort_tokens(s.rows.detach(), s.slots, s.offsets, weights)
    out.sum().backward()
    want = (k * 0 + x.detach().double().sum(1, keepdim=True)).expand(m, k)
    size = x.detach().double().abs().sum(1, keepdim=True).expand(m, k).cpu()
    assert_within(weights.grad, want.cpu(), (hidden + 1) * U32 * size)
    assert not sort_tokens(x, indices, experts, int8=True).scale.requires_grad
    with torch.no_grad():
        assert not sort_tokens(x, indices, experts).rows.requires_grad


@gpu
def test_gradients_are_differentiable_once(device):
    m, k, experts, hidden = 8, 2, 4, 32
    indices = to_u32(make_indices(m, k, experts, torch.Generator().manual_seed(1), "any"), device)
    x = torch.randn(m, hidden, device=device, requires_grad=True)
    weights = torch.rand(m, k, device=device, requires_grad=True)
    s = sort_tokens(x, indices, experts)
    out = unsort_tokens(s.rows, s.slots, s.offsets, weights)
    gx, gw = torch.autograd.grad(out.sum(), [x, weights], create_graph=True)
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all()
    with pytest.raises(RuntimeError, match="differentiable once"):
        (gx.sum() + gw.sum()).backward()


@gpu
def test_a_saved_tensor_that_is_written_over_is_noticed(device):
    m, k, experts, hidden = 8, 2, 4, 32
    gen = torch.Generator().manual_seed(1)
    indices = to_u32(make_indices(m, k, experts, gen, "any"), device)
    x = torch.randn(m, hidden, generator=gen).to(device).requires_grad_(True)
    s = sort_tokens(x, indices, experts)
    buffers = SortedTokens.empty(m, hidden, experts, k, F32, device)._replace(slots=s.slots)
    sort_tokens(x.detach(), to_u32(make_indices(m, k, experts, gen, "any"), device), experts, out=buffers)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        s.rows.sum().backward()


# ---------------------------------------------------------------------------
# Quantised rows
# ---------------------------------------------------------------------------
def swiglu64(x: torch.Tensor):
    gate, up = x.double().chunk(2, dim=-1)
    v = gate / (1 + torch.exp(-gate)) * up
    # exp2 of a product that was rounded: off by |g| log2(e) 2^-24, and two ulps of its own; the sum, the quotient (a reciprocal of one
    # ulp and a product), and the product with up are further roundings
    return v, v.abs() * (1.5 * gate.abs() + 12) * U32


def check_quantized(q, scale, v, off):
    """Rows of q * scale against v, of which the kernel had values up to `off` away."""
    a = v.abs().amax(1).clamp_min(TINY)
    slack = off.amax(1)
    assert_within(scale, a / 127, slack / 127 + 2 * U32 * a / 127)
    s = scale.detach().cpu().double()[:, None]
    # half a step, by the kernel's own scale; the product with 127 / a is off by three roundings of at most 127
    assert_within(q.cpu().double() * s, v, s * (0.5 + 127 * 4 * U32) + off)
    assert q.abs().max() <= 127


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,width", [(1, 16), (3, 1024), (130, 1040), (9, 8192), (5, 8208), (4, 20000), (0, 64)])
def test_quantize_rows(device, dtype, rows, width):
    gen = torch.Generator().manual_seed(width)
    x = (torch.randn(rows, width, generator=gen) * torch.exp(2 * torch.randn(rows, 1, generator=gen))).to(dtype)
    if rows > 2:
        x[1] = 0
        x[2, -1] = torch.finfo(dtype).max
    q, scale = quantize_rows(x.to(device))
    want_q, want_scale = ref_quantize(x.float()) if rows else (x.to(torch.int8), x.float().sum(1))
    assert torch.equal(q.cpu(), want_q) and torch.equal(scale.cpu(), want_scale)
    y = (torch.randn(rows, 2 * width, generator=gen) * 2).to(dtype)
    if rows > 1:
        y[1, :width] = -80  # (the activation all but vanishes)
        y[0, :8] = 60
    q, scale = quantize_rows(y.to(device), swiglu=True)
    if rows:
        check_quantized(q, scale, *swiglu64(y))


@gpu
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("width", [48, 2048])
def test_quantize_rows_of_buffers_leaves_other_rows_alone(device, swiglu, width):
    gen = torch.Generator().manual_seed(5)
    counts = [0, 3, 17, 1, 0, 40, -2]  # (17 rows at most: 40 and -2 are taken for 17 and 0)
    there = [0, 3, 17, 1, 0, 17, 0]
    x = torch.randn(7, 17, (2 if swiglu else 1) * width, generator=gen).to(BF16)
    for e, n in enumerate(there):
        x[e, n:] = float("nan")
    q = torch.full((7, 17, width), 99, dtype=torch.int8, device=device)
    scales = torch.full((7, 17, 4), 5.0, device=device)
    quantize_rows(x.to(device), num_tokens=torch.tensor(counts, dtype=torch.int32, device=device), swiglu=swiglu,
                  out=(q, scales[..., 0]))  # fmt: skip
    for e, n in enumerate(there):
        assert (q[e, n:] == 99).all() and (scales[e, n:, 0] == 5).all()
        if n:
            v, off = swiglu64(x[e, :n]) if swiglu else (x[e, :n].double(), torch.zeros(n, width, dtype=torch.float64))
            check_quantized(q[e, :n], scales[e, :n, 0], v, off)
    assert (scales[..., 1:] == 5).all()
    # sorted rows: those behind the last offset
    offsets = torch.tensor([0, 4, 4, 9], dtype=torch.int32, device=device)
    flat = torch.randn(17, (2 if swiglu else 1) * width, generator=gen).to(BF16)
    flat[9:] = float("inf")
    q, scale = q[0], scales[0, :, 0].contiguous()
    quantize_rows(flat.to(device), offsets=offsets, swiglu=swiglu, out=(q, scale))
    v, off = swiglu64(flat[:9]) if swiglu else (flat[:9].double(), torch.zeros(9, width, dtype=torch.float64))
    check_quantized(q[:9], scale[:9], v, off)
    assert (q[9:] == 99).all() and (scale[9:] == 5).all()


@gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_rows_with_infinities_and_nans_become_nan(device, bad):
    x = torch.ones(3, 2048, dtype=BF16, device=device)
    x[1, 77] = bad
    for q, scale in (quantize_rows(x), (lambda s: (s.rows, s.scale))(
            sort_tokens(x, to_u32(torch.zeros(3, 1, dtype=torch.int32), device), 1, int8=True))):  # fmt: skip
        assert torch.isnan(scale[1]) and (q[1] == 0).all()
        assert torch.isfinite(scale[[0, 2]]).all() and (q[[0, 2]] == 127).all()
    weight = torch.ones(8, 2048, dtype=torch.int8, device=device)
    y = int8_matmul(q, scale, weight, torch.ones(8, device=device))
    assert torch.isnan(y[1]).all() and torch.isfinite(y[[0, 2]]).all()


# ---------------------------------------------------------------------------
# Products
# ---------------------------------------------------------------------------
def make_int8(shape, gen, extreme=False):
    q = torch.randint(-127, 128, shape, generator=gen, dtype=torch.int32)
    return (torch.where(q < 0, -128, 127) if extreme else q).to(torch.int8)


def ref_product(x, xs, w, ws):
    sums = (x.double() @ w.double().t())  # (whole numbers below 2^53)
    return sums * xs.double()[:, None] * ws.double()


def check_product(got, x, xs, w, ws, dtype):
    ref = ref_product(x, xs, w, ws)
    # the sum becomes fp32, the scales are multiplied, and their product with the sum
    assert_within(got, ref, rounded(ref, dtype, 3 * U32 * ref.abs()))


@gpu
@pytest.mark.parametrize("out_dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,n,k", [
    (1, 1, 16), (1, 1408, 2048), (2, 130, 48), (16, 257, 144), (31, 128, 128), (33, 515, 1040), (70, 96, 272),
    (130, 1000, 400), (300, 600, 1136), (513, 259, 64), (17, 7, 4112),
])  # fmt: skip
def test_int8_matmul_dense(device, rows, n, k, out_dtype):
    gen = torch.Generator().manual_seed(rows * n + k)
    x, w = make_int8((rows, k), gen), make_int8((n, k), gen)
    xs, ws = torch.rand(rows, generator=gen) * 1e-2, torch.rand(n, generator=gen) * 1e-2
    got = int8_matmul(x.to(device), xs.to(device), w.to(device), ws.to(device), out_dtype=out_dtype)
    assert got.dtype == out_dtype
    check_product(got, x, xs, w, ws, out_dtype)


@gpu
@pytest.mark.parametrize("k", [16, 131056])
def test_int8_matmul_holds_the_largest_sums(device, k):
    gen = torch.Generator().manual_seed(2)
    x = torch.full((3, k), -128, dtype=torch.int8)
    w = make_int8((20, k), gen, extreme=True)
    w[0] = -128
    xs, ws = torch.ones(3), torch.full((20,), 2.0**-12)
    got = int8_matmul(x.to(device), xs.to(device), w.to(device), ws.to(device), out_dtype=F32)
    check_product(got, x, xs, w, ws, F32)


@gpu
@pytest.mark.parametrize("counts", [
    [1, 0, 2, 0, 0, 1], [0, 0, 0], [5, 40, 0, 129, 1, 64], [300, 0, 513, 7], [16] * 40, [0] * 300 + [3], [1000],
])  # fmt: skip
@pytest.mark.parametrize("n,k", [(200, 160), (129, 2064)])
def test_int8_matmul_of_experts(device, counts, n, k):
    experts, total, cap = len(counts), sum(counts), max(max(counts), 1)
    gen = torch.Generator().manual_seed(total + n)
    w, ws = make_int8((experts, n, k), gen), torch.rand(experts, n, generator=gen) * 1e-2
    spare = 9
    x, xs = make_int8((total + spare, k), gen), torch.rand(total + spare, generator=gen) * 1e-2
    xs[total:] = float("nan")
    offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)
    out = torch.full((total + spare, n + 8), 3.0, dtype=BF16, device=device)
    wd, wsd, xd, xsd = (t.to(device) for t in (w, ws, x, xs))
    got = int8_matmul(xd, xsd, wd, wsd, offsets=offsets.to(device), out=out[:, 4 : 4 + n])
    assert got.data_ptr() == out[:, 4:].data_ptr()
    for e, c in enumerate(counts):
        if c:
            a = int(offsets[e])
            check_product(out[a : a + c, 4 : 4 + n], x[a : a + c], xs[a : a + c], w[e], ws[e], BF16)
    assert (out[total:] == 3).all() and (out[:, :4] == 3).all() and (out[:, 4 + n :] == 3).all()
    # the same rows in buffers, with scales as dispatch leaves them
    xp, xsp = torch.zeros(experts, cap, k, dtype=torch.int8), torch.full((experts, cap, 4), float("nan"))
    for e, c in enumerate(counts):
        a = int(offsets[e])
        xp[e, :c], xsp[e, :c, 0] = x[a : a + c], xs[a : a + c]
    padded = torch.full((experts, cap, n), 3.0, dtype=BF16, device=device)
    num = torch.tensor(counts, dtype=torch.int32, device=device)
    int8_matmul(xp.to(device), xsp.to(device)[..., 0], wd, wsd, num_tokens=num, out=padded)
    for e, c in enumerate(counts):
        a = int(offsets[e])
        assert torch.equal(padded[e, :c], out[a : a + c, 4 : 4 + n])
        assert (padded[e, c:] == 3).all()


@gpu
def test_int8_matmul_of_long_weights(device):
    """Weights whose bytes pass 2^32, of which the last are used."""
    n, k, experts = 4096, 16384, 65
    w = torch.zeros(experts, n, k, dtype=torch.int8, device=device)
    gen = torch.Generator().manual_seed(9)
    last = make_int8((n, k), gen)
    w[-1] = last.to(device)
    ws = torch.full((experts, n), 2.0**-10, device=device)
    x, xs = make_int8((5, k), gen), torch.rand(5, generator=gen)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=device)
    offsets[-1] = 5
    got = int8_matmul(x.to(device), xs.to(device), w, ws, offsets=offsets)
    check_product(got, x, xs, last, ws[0].cpu(), BF16)


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def test_tensors_on_the_cpu_are_refused():
    x, idx = torch.zeros(2, 16, dtype=BF16), torch.zeros(2, 2, dtype=torch.uint32)
    slots, offsets = torch.zeros(2, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    q, s = torch.zeros(2, 16, dtype=torch.int8), torch.ones(2)
    for call in (
        lambda: sort_tokens(x, idx, 2),
        lambda: unsort_tokens(x, slots, offsets),
        lambda: unsort_tokens_backward(x, x, slots, offsets),
        lambda: sort_tokens_backward(x, slots),
        lambda: quantize_rows(x),
        lambda: int8_matmul(q, s, q, s),
    ):
        with pytest.raises(RuntimeError, match="must be on GPU"):
            call()


@gpu
def test_refused_tensors(device):
    def t(*shape, dtype=BF16):
        return torch.zeros(*shape, dtype=dtype, device=device)

    i32, u32, i8 = torch.int32, torch.uint32, torch.int8
    x, idx = t(4, 32), t(4, 2, dtype=u32)
    s = sort_tokens(x, idx, 3)
    w = t(4, 2, dtype=F32)
    y = s.rows
    bad = [
        (lambda: sort_tokens(x.double(), idx, 3), "dtype for x"),
        (lambda: sort_tokens(x[:3], idx, 3), "indices.size"),
        (lambda: sort_tokens(x, idx.view(i32), 3), "indices must be of type"),
        (lambda: sort_tokens(x, idx, 0), "num_experts"),
        (lambda: sort_tokens(x, idx, 5462), "num_experts"),
        (lambda: sort_tokens(x, t(4, 65, dtype=u32), 3), "experts_per_token"),
        (lambda: sort_tokens(x, t(4, 0, dtype=u32), 3), "experts_per_token"),
        (lambda: sort_tokens(t(4, 12), idx, 3), "16"),
        (lambda: sort_tokens(t(4, 8), idx, 3, int8=True), "16"),
        (lambda: sort_tokens(t(32, 4).t(), idx, 3), "contiguous"),
        (lambda: sort_tokens(t(4, 40)[:, 1:33], idx, 3), "aligned"),
        (lambda: sort_tokens(x.cpu(), idx, 3), "GPU"),
        (lambda: sort_tokens(x, idx.cpu(), 3), "GPU"),
        (lambda: sort_tokens(x, idx, 3, t(2, dtype=u32)), "scalar"),
        (lambda: sort_tokens(x, idx, 3, t(1, dtype=i32)), "UInt32"),
        (lambda: sort_tokens(x, idx, 4, out=s), "num_experts"),
        (lambda: sort_tokens(x, idx, 3, out=s, int8=True), "int8"),
        (lambda: sort_tokens(x[:2], idx[:2], 3, out=s), "slots"),
        (lambda: sort_tokens(y[:4], idx, 3, out=s), "overlaps"),
        (lambda: sort_tokens(t(9000, 8), t(9000, 2, dtype=u32), 3, out=SortedTokens.empty(
            9000, 8, 3, 2, BF16, device)._replace(workspace=None)), "workspace"),
        (lambda: unsort_tokens(y, s.slots, s.offsets, w.to(BF16)), "weights must be of type"),
        (lambda: unsort_tokens(y, s.slots, s.offsets, w[:, :1]), "weights"),
        (lambda: unsort_tokens(y, s.slots.long(), s.offsets), "slots must be of type"),
        (lambda: unsort_tokens(t(8, 12)[:, :8], s.slots, s.offsets), "aligned"),
        (lambda: unsort_tokens(y, s.slots, s.offsets, out=t(5, 32)), "slots must have a row"),
        (lambda: unsort_tokens(y, s.slots, s.offsets, out=y[:4]), "overlaps"),
        (lambda: unsort_tokens(y, s.slots, s.offsets, out=t(1, 32).expand(4, 32)), "more than once"),
        (lambda: unsort_tokens_backward(x, y, s.slots, s.offsets, w, out=(t(7, 32), None)), "grad_y"),
        (lambda: unsort_tokens_backward(x, y, s.slots, s.offsets, w, out=(y, None)), "overlaps"),
        (lambda: unsort_tokens_backward(x, y, s.slots, s.offsets.float(), w), "offsets"),
        (lambda: quantize_rows(t(4, 24)), "16"),
        (lambda: quantize_rows(t(4, 33), swiglu=True), "halves|aligned"),
        (lambda: quantize_rows(t(2, 4, 32)), "num_tokens"),
        (lambda: quantize_rows(t(2, 4, 32), num_tokens=t(3, dtype=i32)), "num_tokens"),
        (lambda: quantize_rows(x, offsets=t(1, dtype=i32)), "offsets"),
        (lambda: quantize_rows(x, num_tokens=t(4, dtype=i32)), "num_tokens"),
        (lambda: quantize_rows(x, out=(t(4, 16, dtype=i8), t(4, dtype=F32))), "out must"),
        (lambda: quantize_rows(t(4, 32, dtype=i32)), "dtype for x"),
        (lambda: int8_matmul(x, w[:, 0], x, w[:, 0]), "Char"),
        (lambda: int8_matmul(t(4, 32, dtype=i8), t(4, dtype=F32), t(5, 48, dtype=i8), t(5, dtype=F32)), "length"),
        (lambda: int8_matmul(t(4, 24, dtype=i8), t(4, dtype=F32), t(5, 24, dtype=i8), t(5, dtype=F32)), "16"),
        (lambda: int8_matmul(t(4, 32, dtype=i8), t(3, dtype=F32), t(5, 32, dtype=i8), t(5, dtype=F32)), "x_scale"),
        (lambda: int8_matmul(t(4, 32, dtype=i8), t(4, dtype=F32), t(5, 32, dtype=i8), t(4, dtype=F32)), "weight_scale"),
        (lambda: int8_matmul(t(4, 32, dtype=i8), t(4, dtype=F32), t(2, 5, 32, dtype=i8), t(2, 5, dtype=F32),
                             offsets=t(4, dtype=i32)), "experts"),
        (lambda: int8_matmul(t(4, 32, dtype=i8), t(4, dtype=F32), t(5, 32, dtype=i8), t(5, dtype=F32), out=t(4, 6)), "out"),
        (lambda: int8_matmul(t(1, 131072, dtype=i8), t(1, dtype=F32), t(1, 131072, dtype=i8), t(1, dtype=F32)), "131056"),
    ]  # fmt: skip
    for call, message in bad:
        with pytest.raises(RuntimeError, match=message):
            call()
    # and the device still works
    assert torch.equal(sort_tokens(x, idx, 3).offsets.cpu(), s.offsets.cpu())


def test_the_layer_is_built_from_the_sources_in_the_tree():
    import hashlib
    import os

    from pplx_kernels import ops

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    h = hashlib.sha256()
    for path in ("pplx-kernels_amd/csrc/torch_common.h", "pplx-kernels_amd/csrc/torch_experts.cpp", "include/pplx_a2a.h"):
        h.update(open(os.path.join(root, path), "rb").read())
    assert ops._C.experts_build_id() == h.hexdigest()[:16], "pplx_kernels/_C.so is stale: run `make -C pplx-kernels_amd/csrc`"
