"""The operators before dispatch at their ends: more workgroups than a launch takes threads for, rows past 32-bit offsets and far apart,
workspaces that do not fit, parts of the results, inference mode, bounds of tokens."""

from __future__ import annotations

import pytest
import torch

from pplx_kernels import (
    NormedRows,
    rms_norm,
    rms_norm_backward,
    rms_norm_workspace,
    route_tokens,
    route_tokens_backward,
    router_logits,
    router_logits_backward,
    router_workspace,
)
from tests.test_experts import BF16, F16, F32, U32, assert_within, rounded
from tests.test_router import E4M3, product, ref_route, router
from tests.test_router_path import CHOICE, same

gpu = pytest.mark.gpu


def rows_on(device, m, hidden, dtype, seed):
    """Made on the device, in pieces."""
    gen = torch.Generator(device).manual_seed(seed)
    x = torch.empty(m, hidden, dtype=dtype, device=device)
    for part in x.split(max(1, (1 << 26) // hidden)):
        part.copy_(torch.randn(part.shape, device=device, generator=gen))
    return x


# ---------------------------------------------------------------------------
# More workgroups than a launch takes threads for along one dimension
# ---------------------------------------------------------------------------
@gpu
def test_norms_of_more_rows_than_one_line_of_workgroups(device):
    """2^26 rows and a few, four to a workgroup."""
    m, hidden = (1 << 26) + 5, 16
    x, weight = rows_on(device, m, hidden, BF16, 1), torch.full((hidden,), 1.5, dtype=BF16, device=device)
    n = rms_norm(x, weight, x, quantize=torch.int8)
    for part in zip(x.split(1 << 24), n.y.split(1 << 24), n.sum.split(1 << 24), n.q.split(1 << 24), n.scale.split(1 << 24)):
        want = rms_norm(part[0], weight, part[0], quantize=torch.int8)
        assert all(same(a, b) for a, b in zip(part[1:], want))
    grad, _ = rms_norm_backward(n.y, n.sum, weight, out=(n.q.new_empty(m, hidden, dtype=BF16), None))
    for y, h, got in zip(n.y.split(1 << 24), n.sum.split(1 << 24), grad.split(1 << 24)):
        assert same(got, rms_norm_backward(y, h, weight, out=(torch.empty_like(h), None))[0])


@gpu
def test_norms_of_more_rows_than_one_line_of_workgroups_one_to_each(device):
    """2^23 rows and a few of more than 2048 elements: 512 threads to a row.  All of them are one row, or two."""
    m, hidden = (1 << 23) + 3, 2064
    two = rows_on(device, 2, hidden, BF16, 2)
    weight = torch.ones(hidden, dtype=F32, device=device)
    x = two[:1].expand(m, hidden)
    q, scale = torch.empty(m, hidden, dtype=torch.int8, device=device), torch.empty(m, device=device)
    rms_norm(x, weight, out=NormedRows(None, None, q, scale))
    want = rms_norm(two, weight, quantize=torch.int8)
    assert all(bool((part == want.q[0]).all()) for part in q.split(1 << 20)) and bool((scale == want.scale[0]).all())


@gpu
def test_choices_of_more_tokens_than_one_line_of_workgroups(device):
    m, experts = (1 << 26) + 5, 3
    logits = rows_on(device, m, experts, BF16, 3)
    indices, weights = route_tokens(logits, 1, renormalize=False)
    grad = route_tokens_backward(weights, logits, indices, renormalize=False)
    for part in zip(logits.split(1 << 24), indices.view(torch.int32).split(1 << 24), weights.split(1 << 24), grad.split(1 << 24)):
        at, w = route_tokens(part[0], 1, renormalize=False)
        assert torch.equal(at.view(torch.int32), part[1]) and torch.equal(w, part[2])
        assert same(route_tokens_backward(w, part[0], at, renormalize=False), part[3])
    # a workgroup to a token, where a lane does not hold the experts of several groups
    m, experts = (1 << 26) + 5, 1030
    one = rows_on(device, 1, experts, F32, 4)
    indices, weights = route_tokens(one.expand(m, experts), 1)
    at, w = route_tokens(one, 1)
    assert bool((indices.view(torch.int32) == at.view(torch.int32)).all()) and bool((weights == w).all())


@gpu
def test_products_of_more_rows_than_one_launch(device):
    """2^28 rows and a few: more blocks of 64 rows than a launch takes."""
    m, hidden, experts = (1 << 28) + 77, 8, 8
    x, weight = rows_on(device, m, hidden, BF16, 5), rows_on(device, experts, hidden, BF16, 6)
    got = router_logits(x, weight)
    for a in (0, (1 << 28) - 200, m - 300):
        want, off = product(x[a : a + 300].cpu(), weight.t().cpu(), hidden)
        assert_within(got[a : a + 300], want, off)
    for part, rows in zip(got.split(1 << 24), x.split(1 << 24)):  # (products of 16-bit elements are exact, eight to a sum)
        assert torch.allclose(part, rows.float() @ weight.float().t(), rtol=0, atol=1e-3)


# ---------------------------------------------------------------------------
# Rows past 32-bit offsets, and far apart
# ---------------------------------------------------------------------------
@gpu
def test_rows_past_four_gigabytes(device):
    m, hidden, experts, k = 560000, 4096, 16, 3
    x = rows_on(device, m, hidden, BF16, 7)  # 4.6 GB
    weight, gate = torch.ones(hidden, dtype=BF16, device=device), rows_on(device, experts, hidden, BF16, 8)
    n = rms_norm(x, weight)
    logits = router_logits(n.y, gate)
    tail = slice(m - 50, m)
    assert same(n.y[tail], rms_norm(x[tail], weight).y)
    want, off = product(n.y[tail].cpu(), gate.t().cpu(), hidden)
    assert_within(logits[tail], want, off)
    grad = 1e-2 * torch.randn(m, experts, device=device)
    gx, gw = router_logits_backward(grad, n.y, gate)
    few, _ = router_logits_backward(grad[tail].contiguous(), n.y[tail], gate)
    assert same(gx[tail], few)
    # the weight's gradient: all rows, in 64 bits
    ref, size = torch.zeros(experts, hidden, dtype=torch.float64, device=device), torch.zeros(experts, hidden, device=device)
    for g, y in zip(grad.split(20000), n.y.split(20000)):
        ref += g.double().t() @ y.double()
        size += g.abs().t() @ y.abs().float()
    # (two pieces of grad: 2^-18 of each product; sums of fp32 in 64 chains and more)
    assert_within(gw, ref.cpu(), rounded(ref.cpu(), BF16, size.double().cpu() * 1.01 * (2.0**-18 + (m / 16 + 40) * U32)))
    gh, _ = rms_norm_backward(gx, n.y, weight, out=(torch.empty_like(x), None))
    assert same(gh[tail], rms_norm_backward(gx[tail], n.y[tail], weight, out=(torch.empty_like(x[tail]), None))[0])
    indices, weights = route_tokens(logits, k)
    want, _ = ref_route(logits[tail].cpu(), k)
    assert torch.equal(indices.view(torch.int32)[tail].cpu(), want)


@gpu
@pytest.mark.parametrize("dtype,weight_dtype", [(BF16, BF16), (F32, F32), (F16, F32)])
def test_rows_eight_megabytes_apart(device, dtype, weight_dtype):
    """Strides that a tile's 32-bit offsets do not reach."""
    gen = torch.Generator().manual_seed(9)
    m, experts, hidden = 40, 33, 520
    x, weight = router(m, experts, hidden, dtype, weight_dtype, gen)

    def apart(t):
        step = (1 << 23) // t.element_size()
        room = torch.zeros(t.shape[0] * step, dtype=t.dtype, device=device)
        view = room.as_strided(t.shape, (step, 1), 8)
        view.copy_(t)
        return view

    want, off = product(x, weight.t(), hidden)
    xs, ws = apart(x), apart(weight)
    for a, b in ((xs, weight.to(device)), (x.to(device), ws), (xs, ws)):
        assert_within(router_logits(a, b), want, off)
    grad = 1e-2 * torch.randn(m, experts, generator=gen).to(device)
    out = apart(torch.zeros_like(x)), apart(torch.zeros_like(weight))
    got = router_logits_backward(grad, xs, ws, out=out)
    assert all(same(a, b) for a, b in zip(got, router_logits_backward(grad, x.to(device), weight.to(device))))
    w = torch.ones(hidden, dtype=weight_dtype, device=device)
    n = rms_norm(xs, w, xs, out=NormedRows(apart(torch.zeros_like(x)), apart(torch.zeros_like(x))))
    plain = rms_norm(x.to(device), w, x.to(device))
    assert same(n.y, plain.y) and same(n.sum, plain.sum)
    assert same(rms_norm_backward(xs, n.sum, w)[0], rms_norm_backward(x.to(device), plain.sum, w)[0])


# ---------------------------------------------------------------------------
# Parts of the results, workspaces, modes, bounds
# ---------------------------------------------------------------------------
@gpu
def test_parts_of_the_results(device):
    x, weight, gate = rows_on(device, 37, 256, F16, 10), torch.ones(256, dtype=F16, device=device), rows_on(device, 9, 256, F16, 11)
    for code in (torch.int8, E4M3):
        all_of_it = rms_norm(x, weight, x, quantize=code)
        some = NormedRows(None, torch.empty_like(x), torch.empty_like(all_of_it.q), torch.empty_like(all_of_it.scale))
        assert rms_norm(x, weight, x, out=some) is some
        assert same(some.sum, all_of_it.sum) and same(some.q, all_of_it.q) and same(some.scale, all_of_it.scale)
        assert same(rms_norm(x, weight, x).y, all_of_it.y)
    # scales that lie apart, in both directions
    room = torch.zeros(4, 37, device=device)
    into = NormedRows(None, None, torch.empty_like(all_of_it.q), room.t()[:, 1:3])
    assert same(rms_norm(x, weight, out=into).scale, rms_norm(x, weight, quantize=E4M3).scale) and (room[[0, 3]] == 0).all()
    grad = rows_on(device, 37, 256, F16, 12)
    gh, gw = rms_norm_backward(grad, x, weight)
    assert same(rms_norm_backward(grad, x, weight, out=(None, torch.empty_like(weight)))[1], gw)
    assert same(rms_norm_backward(grad, x, weight, out=(torch.empty_like(x), None))[0], gh)
    assert rms_norm_backward(grad, x, weight, out=(None, None)) == (None, None)
    into = grad.clone()
    assert same(rms_norm_backward(into, x, weight, out=(into, None))[0], gh)
    g = torch.randn(37, 9, device=device)
    gx, gg = router_logits_backward(g, x, gate)
    assert same(router_logits_backward(g, x, gate, out=(None, torch.empty_like(gate)))[1], gg)
    assert same(router_logits_backward(g, x, gate, out=(torch.empty_like(x), None))[0], gx)
    assert router_logits_backward(g, x, gate, out=(None, None)) == (None, None)


@gpu
def test_workspaces_that_do_not_fit(device):
    x, gate = rows_on(device, 64, 4096, BF16, 13), rows_on(device, 256, 4096, BF16, 14)
    weight, logits = torch.ones(4096, dtype=BF16, device=device), torch.zeros(64, 256, device=device)
    spaces = router_workspace(x, gate), router_workspace(x, gate, backward=True), rms_norm_workspace(x)
    assert all(s.dtype == torch.uint8 and s.is_cuda and s.numel() for s in spaces)
    out = torch.empty_like(x), torch.empty_like(gate)
    calls = (
        lambda s: router_logits(x, gate, out=logits, workspace=s),
        lambda s: router_logits_backward(logits, x, gate, out=out, workspace=s),
        lambda s: rms_norm_backward(x, x, weight, out=(out[0], torch.empty_like(weight)), workspace=s),
    )
    for call, space in zip(calls, spaces):
        call(space)
        call(torch.empty(space.numel() + 5, dtype=torch.uint8, device=device))
        wide = torch.empty(space.numel() + 16, dtype=torch.uint8, device=device)
        for wrong, message in ((space[:-1], "fewer than"), (space.view(torch.int32), "workspace"), (space.cpu(), "GPU"),
                               (wide[1:], "16-byte aligned"), (x.view(torch.uint8).view(-1), "overlaps|fewer")):  # fmt: skip
            with pytest.raises(RuntimeError, match=message):
                call(wrong)
    with pytest.raises(RuntimeError, match="goes with out"):
        router_logits(x, gate, workspace=spaces[0])
    # a step that needs none takes any
    few = rows_on(device, 2, 4096, BF16, 15)
    small = rows_on(device, 16, 64, BF16, 16)
    assert router_workspace(small, small).numel() == 0
    assert same(router_logits(small, small, out=torch.empty(16, 16, device=device), workspace=spaces[0]), router_logits(small, small))
    assert rms_norm_backward(few, few, weight, out=(torch.empty_like(few), None), workspace=spaces[0])[1] is None


@gpu
def test_inference_mode(device):
    x, weight, gate = rows_on(device, 9, 64, F32, 17), torch.ones(64, device=device), rows_on(device, 8, 64, F32, 18)
    n = rms_norm(x, weight, x)
    logits = router_logits(n.y, gate)
    want = [*n[:2], logits, *route_tokens(logits, 2, **CHOICE)]
    with torch.inference_mode():
        for leaf in (x, x.clone().requires_grad_(True)):
            n = rms_norm(leaf, weight, leaf)
            logits = router_logits(n.y, gate)
            got = [*n[:2], logits, *route_tokens(logits, 2, **CHOICE)]
            assert all(same(a, b) for a, b in zip(got, want)) and not logits.requires_grad
            router_logits(n.y, gate, out=logits)
            rms_norm(n.y, weight, out=NormedRows(n.y))
    y = rms_norm(x.clone().requires_grad_(True), weight).y
    assert y.requires_grad


@gpu
@pytest.mark.parametrize("experts", [48, 1200])
def test_bounds_of_tokens(device, experts):
    logits = rows_on(device, 30, experts, F32, 19)
    bias = rows_on(device, 1, experts, F32, 20)[0]
    for b in (None, bias):
        full = route_tokens(logits, 4, bias=b)
        for bound in (0, 1, 29, 30, 31, 2**32 - 1):
            t = torch.tensor([bound], dtype=torch.int64, device=device).to(torch.uint32)
            at, w = route_tokens(logits, 4, bias=b, bound_m=t)
            n = min(bound, 30)
            assert torch.equal(at.view(torch.int32)[:n], full[0].view(torch.int32)[:n]) and torch.equal(w[:n], full[1][:n])
            assert (at.view(torch.int32)[n:] == experts).all() and (w[n:] == 0).all()
            grad = route_tokens_backward(torch.ones_like(w), logits, at)
            assert (grad[n:] == 0).all()


@gpu
def test_gradients_with_picks_taken_out(device):
    """Picks without an expert have no part, whatever gradient they bring."""
    logits = rows_on(device, 12, 20, F32, 21)
    indices, _ = route_tokens(logits, 4, renormalize=False)
    at = indices.view(torch.int32).clone()
    at[:, 2] = 20
    at[5] = 2**31 - 1
    grad = torch.randn(12, 4, device=device)
    grad[:, 2], grad[5] = float("nan"), float("inf")
    got = route_tokens_backward(grad, logits, at.view(torch.uint32), renormalize=False)
    few = at[:, [0, 1, 3]].contiguous().view(torch.uint32)
    want = route_tokens_backward(grad[:, [0, 1, 3]].contiguous(), logits, few, renormalize=False)
    assert torch.isfinite(got).all() and same(got, want) and (got[5] == 0).all()


@gpu
@pytest.mark.parametrize("hidden", [256, 2048, 7168, 16384, 20000])
@pytest.mark.parametrize("over_sum", [False, True])
def test_the_gradient_of_a_norm_over_its_own_operand(device, hidden, over_sum):
    """Into grad_y or grad_sum, beside the weight's gradient: the bits that buffers of their own get."""
    gen = torch.Generator().manual_seed(hidden)
    h, grad, grad_sum = (torch.randn(37, hidden, generator=gen).to(torch.bfloat16).to(device) for _ in range(3))
    weight = torch.randn(hidden, generator=gen).to(device)
    want, want_weight = rms_norm_backward(grad, h, weight, grad_sum=grad_sum)
    over, of_weight = (grad_sum if over_sum else grad), torch.empty_like(weight)
    rms_norm_backward(grad, h, weight, grad_sum=grad_sum, out=(over, of_weight))
    assert torch.equal(over, want) and torch.equal(of_weight, want_weight)


def groups_by_sums(logits, bias, groups, top, k):
    """Choices of `k` in 64 bits, by the two best keys of each group."""
    keys = torch.sigmoid(logits.double()) + bias.double()
    sums = keys.view(len(keys), groups, -1).topk(2, 2).values.sum(2)
    inside = torch.zeros(sums.shape, dtype=torch.bool).scatter_(1, sums.sort(dim=1, descending=True, stable=True).indices[:, :top], True)
    keys = torch.where(inside.repeat_interleave(keys.shape[1] // groups, 1), keys, float("-inf"))
    return keys.sort(dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32)


@gpu
@pytest.mark.parametrize("experts,groups", [(32, 4), (256, 8), (250, 5), (512, 64)])
def test_groups_whose_sums_fp32_holds_for_nothing(device, experts, groups):
    """Two biases around -3e38 leave fp32 at its lower end: the group is there all the same."""
    gen = torch.Generator().manual_seed(experts)
    logits = torch.randn(20, experts, generator=gen)
    bias = -3e38 + 1e38 * torch.rand(experts, generator=gen)
    got, _ = route_tokens(logits.to(device), 3, bias=bias.to(device), scores="sigmoid", num_groups=groups, top_groups=2)
    assert torch.equal(got.view(torch.int32).cpu(), groups_by_sums(logits, bias, groups, 2, 3))


@gpu
@pytest.mark.parametrize("experts,groups", [(32, 4), (256, 8), (250, 5), (512, 64)])
@pytest.mark.parametrize("size", [100.0, 3e4])
def test_groups_whose_best_two_cancel(device, experts, groups, size):
    """Keys are rounded by their size, which the sum of two does not show."""
    gen = torch.Generator().manual_seed(experts)
    logits = torch.randn(2000, experts, generator=gen)
    bias = torch.full((groups, experts // groups), -1e6)
    bias[:, 0], bias[:, 1] = -size, size
    bias = bias.flatten()
    got, _ = route_tokens(logits.to(device), 3, bias=bias.to(device), scores="sigmoid", num_groups=groups, top_groups=2)
    assert torch.equal(got.view(torch.int32).cpu(), groups_by_sums(logits, bias, groups, 2, 3))


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups", [(32, 4), (128, 2), (250, 5), (512, 64), (1000, 4), (1200, 6), (1320, 330)])
def test_groups_by_their_best_expert_where_scores_meet(device, scores, experts, groups):
    """Scores of different logits that are one in 64 bits: near 1, near 0, of logits near 0, and beside ones that are not."""
    gen = torch.Generator().manual_seed(experts)
    size = experts // groups
    logits = torch.randn(120, experts, generator=gen) - 40
    best = torch.randn(120, groups, generator=gen)
    best[:30] = 10 + 40 * torch.rand(30, groups, generator=gen)  # sigmoids that meet, and ones that do not
    best[30:60] = 1e-30 * best[30:60].round()  # 0.5, or one exponential
    best[60:90] = best[60:90].round() * (1 + 2.0**-23 * torch.randint(0, 2, (30, groups), generator=gen))  # a last bit apart
    logits.view(120, groups, size)[:, :, size // 2] = best
    logits[90:105] = logits[90:105] * 30 - 800  # sigmoids of 0
    for top in (1, groups // 2):
        more = dict(scores=scores, num_groups=groups, top_groups=top, group_top=1)
        got, weights = route_tokens(logits.to(device), 2, **more)
        want, want_weights = ref_route(logits, 2, **more)
        assert torch.equal(got.view(torch.int32).cpu(), want)
        assert torch.isfinite(weights).all()
