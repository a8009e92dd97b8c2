"""The operators before dispatch against their definitions in 64 bits on the CPU.

Tolerances count roundings, as in test_experts.py: one to nearest is off by at most ``finfo(t).eps / 2`` of the value, a chain of n fp32
additions by n * 2**-24 of the sum of the magnitudes."""

from __future__ import annotations

import hashlib
import os

import pytest
import torch

from pplx_kernels import (
    NormedRows,
    ops,
    rms_norm,
    rms_norm_backward,
    route_tokens,
    route_tokens_backward,
    router_logits,
    router_logits_backward,
)
from tests.test_experts import BF16, F16, F32, TINY, U32, assert_within, check_quantized, rounded, to_u32

E4M3 = torch.float8_e4m3fn
EPS = 1e-6
F64 = torch.float64
gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------
# The norm
# ---------------------------------------------------------------------------
def rows(m, h, dtype, gen, size=1.0):
    return (size * torch.randn(m, h, generator=gen) * torch.exp(torch.randn(m, 1, generator=gen))).to(dtype)


def norm_weight(h, dtype, gen):
    return (1 + 0.3 * torch.randn(h, generator=gen)).to(dtype)


def root_error(h: int) -> float:
    """Of 1 / sqrt(mean(h^2) + eps), relative: the sum of squares is a chain of at most h / 64 + 20 (a row has 64 threads or more),
    which the root halves; the product with 1 / h (itself rounded), the sum with eps and a root of one ulp."""
    return ((h / 64 + 20) / 2 + 4) * U32


def ref_norm(h, weight, eps=EPS):
    root = 1 / torch.sqrt(h.double().square().mean(1, keepdim=True) + eps)
    v = h.double() * root * weight.double()
    return v, root, v.abs() * (root_error(h.shape[1]) + 2 * U32)


def check_e4m3(q, scale, v, off):
    """Rows of q times their blocks' scales against v, of which the kernel had values up to `off` away."""
    m, h = v.shape
    blocks = scale.shape[1]
    assert blocks == (h + 127) // 128
    q, scale = q.cpu().float(), scale.detach().cpu().double()
    assert torch.isfinite(q).all()
    of = torch.arange(h) // 128
    for b in range(blocks):
        part = v[:, of == b]
        a = part.abs().amax(1).clamp_min(TINY)
        slack = off[:, of == b].amax(1)
        assert_within(scale[:, b], a / 448, slack / 448 + 2 * U32 * a / 448)
        # the largest value of a block comes out as the largest code
        assert (q[:, of == b].abs().amax(1)[a > TINY] == 448).all()
    s = scale[:, of]
    # half a step of three bits, or of the subnormals (2^-9); the product with 448 / a is off by three roundings
    tolerance = (v.abs() + off) * (2.0**-4 + 4 * U32) + s * 2.0**-10 + off
    assert_within(q.double() * s, v, tolerance)


NORMS = [
    # tokens, hidden, dtype, weight
    (1, 2048, BF16, BF16),
    (3, 16, F32, F32),
    (5, 7168, BF16, F32),
    (130, 1040, F16, F16),
    (2, 8208, BF16, BF16),
    (3, 16384, F16, F32),
    (2, 20000, BF16, BF16),
    (2, 40016, F32, F32),
    (9, 528, F16, F32),
    (7, 512, BF16, BF16),
    (6, 4096, F32, F32),
    (5, 4112, BF16, F32),
    (4, 8192, F16, F16),
    (2051, 128, BF16, BF16),
    (0, 64, BF16, BF16),
]


@gpu
@pytest.mark.parametrize("m,hidden,dtype,weight_dtype", NORMS)
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("quantize", [None, torch.int8, E4M3])
def test_rms_norm(device, m, hidden, dtype, weight_dtype, add, quantize):
    gen = torch.Generator().manual_seed(hidden + m)
    x, weight = rows(m, hidden, dtype, gen), norm_weight(hidden, weight_dtype, gen)
    residual = rows(m, hidden, dtype, gen) if add else None
    if m > 2:
        x[1] = 0
        if add:
            residual[1] = 0
    got = rms_norm(x.to(device), weight.to(device), residual.to(device) if add else None, quantize=quantize)
    h = (x.float() + residual.float()).to(dtype) if add else x
    if add:
        assert torch.equal(got.sum.cpu(), h)
    else:
        assert got.sum is None
    assert got.y.dtype == dtype and got.y.shape == (m, hidden)
    if m == 0:
        return
    v, _, off = ref_norm(h, weight)
    assert_within(got.y, v, rounded(v, dtype, off))
    if quantize is None:
        assert got.q is None and got.scale is None
    elif quantize == torch.int8:
        check_quantized(got.q, got.scale, v, off)
    else:
        assert got.q.dtype == E4M3
        check_e4m3(got.q, got.scale, v, off)


@gpu
def test_rms_norm_of_width_eight(device):
    gen = torch.Generator().manual_seed(8)
    for dtype in (BF16, F32):
        x, weight = rows(700, 8, dtype, gen), norm_weight(8, dtype, gen)
        v, _, off = ref_norm(x, weight, 1e-5)
        assert_within(rms_norm(x.to(device), weight.to(device), eps=1e-5).y, v, rounded(v, dtype, off))


@gpu
@pytest.mark.parametrize("hidden", [64, 4096, 12288, 20000])
def test_rms_norm_of_huge_and_tiny_rows(device, hidden):
    """Values whose squares fp32 does not hold, and values beside which eps is everything."""
    gen = torch.Generator().manual_seed(hidden)
    x = torch.randn(4, hidden, generator=gen)
    x = (x * torch.tensor([1e37, 1e30, 1e-30, 1e-12])[:, None]).to(BF16)
    weight = norm_weight(hidden, BF16, gen)
    v, _, off = ref_norm(x, weight)
    # (the factor 2^-70 is exact, the rows' r is that of values without eps)
    off = off + v.abs() * 4 * U32
    got = rms_norm(x.to(device), weight.to(device), quantize=torch.int8)
    assert_within(got.y, v, rounded(v, BF16, off))
    grad = torch.randn(4, hidden, generator=gen).to(BF16)
    gx, gw = rms_norm_backward(grad.to(device), x.to(device), weight.to(device))
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all()


@gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("hidden", [256, 7168, 20000])
def test_rms_norm_of_rows_with_infinities_and_nans(device, bad, hidden):
    x = torch.ones(3, hidden, dtype=BF16, device=device)
    x[1, 77] = bad
    weight = torch.ones(hidden, dtype=BF16, device=device)
    for quantize in (torch.int8, E4M3):
        got = rms_norm(x, weight, torch.zeros_like(x), quantize=quantize)
        assert torch.isnan(got.y[1]).all() and torch.isfinite(got.y[[0, 2]]).all()
        assert torch.isnan(got.scale[1]).all() and torch.isfinite(got.scale[[0, 2]]).all()
        assert (got.q[1].float() == 0).all() and (got.q[[0, 2]].float() == (127 if quantize == torch.int8 else 448)).all()


@gpu
@pytest.mark.parametrize("hidden", [512, 7168, 20000])
@pytest.mark.parametrize("quantize", [None, torch.int8, E4M3])
def test_rms_norm_in_place_and_into_strided_buffers(device, hidden, quantize):
    gen = torch.Generator().manual_seed(hidden)
    m = 6
    wide = rows(m, 2 * hidden, BF16, gen).to(device)
    x, residual = wide[:, hidden:], rows(m, hidden, BF16, gen).to(device)
    weight = norm_weight(hidden, F32, gen).to(device)
    want = rms_norm(x.contiguous(), weight, residual, quantize=quantize)
    room = torch.full((m, hidden + 32), 7.0, dtype=BF16, device=device)
    of_scale = torch.full((m, 3, 200), 5.0, device=device)
    q = None if quantize is None else torch.empty(m, hidden, dtype=quantize, device=device)
    scale = None
    if quantize is not None:
        scale = of_scale[:, 1, 0] if quantize == torch.int8 else of_scale[:, 1, : want.scale.shape[1]]
    got = rms_norm(x, weight, residual, out=NormedRows(room[:, 16 : 16 + hidden], torch.empty_like(residual), q, scale))
    assert torch.equal(got.y, want.y) and torch.equal(got.sum, want.sum)
    assert (room[:, :16] == 7).all() and (room[:, 16 + hidden :] == 7).all()
    if quantize is not None:
        assert torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(got.scale, want.scale)
        assert (of_scale[:, [0, 2]] == 5).all()
    # the sum over the residual, the result over the rows
    a, b = x.contiguous(), residual.clone()
    got = rms_norm(a, weight, b, out=NormedRows(a, b, q, scale))
    assert got.y is a and torch.equal(a, want.y) and torch.equal(b, want.sum)
    # the sum over the rows, the result over the residual
    a, b = x.contiguous(), residual.clone()
    rms_norm(a, weight, b, out=NormedRows(b, a, q, scale))
    assert torch.equal(b, want.y) and torch.equal(a, want.sum)
    # only the quantised rows
    if quantize is not None:
        q.view(torch.uint8).fill_(99)
        rms_norm(x, weight, residual, out=NormedRows(None, torch.empty_like(residual), q, scale))
        assert torch.equal(q.view(torch.uint8), want.q.view(torch.uint8))
    # rows that are one
    one = x[:1].expand(m, hidden)
    assert torch.equal(rms_norm(one, weight).y, rms_norm(one.contiguous(), weight).y)


NORM_GRADIENTS = [
    (1, 8, F32, F32), (1, 2048, BF16, BF16), (33, 520, F16, F16), (600, 264, F32, F32), (1100, 64, BF16, F32), (40, 7168, BF16, F32),
    (7, 16384, BF16, BF16), (5, 20000, F16, F32), (3, 17000, F32, F32),
    (4100, 128, BF16, F32),
    (2100, 512, F16, F16),
    (300, 4096, F32, F32),
    (513, 4104, BF16, BF16),
    (261, 8192, F32, F32),
    (30, 8200, F16, F32),
]  # fmt: skip


def ref_norm_gradients(grad, grad_sum, h, weight, eps=EPS):
    """By autograd in 64 bits, and how far the kernel may be off before its results are rounded."""
    leaf, w = h.double().requires_grad_(True), weight.double().requires_grad_(True)
    unit = leaf / torch.sqrt(leaf.square().mean(1, keepdim=True) + eps)
    (unit * w * grad.double()).sum().backward()
    with torch.no_grad():
        root = 1 / torch.sqrt(h.double().square().mean(1, keepdim=True) + eps)
        width, m = h.shape[1], h.shape[0]
        e = root_error(width)
        unit, g = h.double() * root, grad.double() * w
        along = (g * unit).mean(1, keepdim=True).abs()
        size = (g * unit).abs().mean(1, keepdim=True)
        off_along = size * ((width / 64 + 20 + 6) * U32 + e)
        off = root * (g.abs() * (4 * U32 + e) + unit.abs() * (off_along + along * (2 * e + 6 * U32)))
        out = leaf.grad if grad_sum is None else leaf.grad + grad_sum.double()
        if grad_sum is not None:
            off = off + U32 * (leaf.grad.abs() + grad_sum.double().abs())
        off_w = (grad.double() * unit).abs().sum(0) * ((m + 4) * U32 + e)
    return out, off, w.grad, off_w


@gpu
@pytest.mark.parametrize("m,hidden,dtype,weight_dtype", NORM_GRADIENTS)
@pytest.mark.parametrize("add", [False, True])
def test_gradients_of_rms_norm(device, m, hidden, dtype, weight_dtype, add):
    gen = torch.Generator().manual_seed(hidden + m)
    x, weight = rows(m, hidden, dtype, gen), norm_weight(hidden, weight_dtype, gen)
    residual = rows(m, hidden, dtype, gen) if add else None
    grad = torch.randn(m, hidden, generator=gen).to(dtype)
    grad_sum = torch.randn(m, hidden, generator=gen).to(dtype) if add else None
    h = (x.float() + residual.float()).to(dtype) if add else x
    want, off, want_w, off_w = ref_norm_gradients(grad, grad_sum, h, weight)
    leaves = [t.to(device).requires_grad_(True) for t in ((x, weight, residual) if add else (x, weight))]
    got = rms_norm(*leaves)
    outs, grads = ([got.y, got.sum], [grad, grad_sum]) if add else ([got.y], [grad])
    made = torch.autograd.grad(outs, leaves, [g.to(device) for g in grads])
    assert_within(made[0], want, rounded(want, dtype, off))
    assert_within(made[1], want_w, rounded(want_w, weight_dtype, off_w))
    if add:
        assert torch.equal(made[2], made[0])
    # the call itself, and each of the two alone
    dev = [t.to(device) for t in (grad, h, weight)]
    more = dict(grad_sum=None if grad_sum is None else grad_sum.to(device))
    both = rms_norm_backward(*dev, **more)
    assert torch.equal(both[0], made[0]) and torch.equal(both[1], made[1])
    only_h, only_w = torch.empty_like(both[0]), torch.empty_like(both[1])
    rms_norm_backward(*dev, **more, out=(only_h, None))
    rms_norm_backward(*dev, **more, out=(None, only_w))
    assert torch.equal(only_h, both[0]) and torch.equal(only_w, both[1])
    # over the gradient that came
    over = dev[0].clone()
    rms_norm_backward(over, *dev[1:], **more, out=(over, None))
    assert torch.equal(over, both[0])
    if add:
        # of the sum alone: it goes through
        (through,) = torch.autograd.grad(rms_norm(*leaves).sum, leaves[0], grad_sum.to(device))
        assert torch.equal(through.cpu(), grad_sum)


@gpu
def test_gradients_of_rms_norm_against_differences(device):
    m, hidden = 6, 264
    gen = torch.Generator().manual_seed(4)
    x, weight = rows(m, hidden, F32, gen), norm_weight(hidden, F32, gen)
    step_x, step_w, grad = (torch.randn(*s, generator=gen) for s in ((m, hidden), (hidden,), (m, hidden)))
    leaves = [t.to(device).requires_grad_(True) for t in (x, weight)]
    gx, gw = torch.autograd.grad(rms_norm(*leaves).y, leaves, grad.to(device))
    along = ((gx.cpu().double() * step_x.double()).sum() + (gw.cpu().double() * step_w.double()).sum()).item()
    a = 2.0**-6

    def value(s, exact):
        if exact:
            h, w = x.double() + s * step_x.double(), weight.double() + s * step_w.double()
            return (h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * w * grad.double()).sum().item()
        y = rms_norm((x + s * step_x).to(device), (weight + s * step_w).to(device)).y
        return (y.cpu().double() * grad.double()).sum().item()

    difference = (value(a, False) - value(-a, False)) / (2 * a)
    exact = (value(a, True) - value(-a, True)) / (2 * a)
    # values: the points themselves are rounded twice, an element's relative error is that of the norm
    reach = (x.double().abs() + a * step_x.abs()) / torch.sqrt(x.double().square().mean(1, keepdim=True)) * 1.5
    size = (reach * (weight.double().abs() + a * step_w.abs()) * grad.double().abs()).sum().item()
    noise = size * (root_error(hidden) + 8 * U32) / a
    assert abs(difference - exact) <= noise
    # the gradient along the step, against the same difference without its noise: what is left is the third derivative's part,
    # which the exact difference at half the step bounds (it falls by four)
    half = (value(a / 2, True) - value(-a / 2, True)) / a
    want, off, want_w, off_w = ref_norm_gradients(grad, None, x, weight)
    slack = ((rounded(want, F32, off) * step_x.abs()).sum() + (rounded(want_w, F32, off_w) * step_w.abs()).sum()).item()
    assert abs(difference - along) <= noise + slack + 2 * abs(exact - half)


# ---------------------------------------------------------------------------
# The router's product
# ---------------------------------------------------------------------------
LOGITS = [
    # tokens, experts, hidden, dtype, weight
    (1, 1, 8, BF16, BF16),
    (1, 64, 2048, BF16, F32),
    (4, 60, 16, F32, F32),
    (3, 33, 8, F16, F32),
    (5, 7, 24, BF16, F32),
    (17, 256, 520, F16, F16),
    (64, 256, 7168, BF16, F32),
    (33, 5461, 40, BF16, BF16),
    (130, 61, 1032, F32, F32),
    (300, 257, 264, F16, F32),
    (515, 128, 328, BF16, BF16),
    (2050, 72, 136, F16, F16),
    (4100, 256, 200, BF16, BF16),
    (16400, 300, 200, F16, F16),
    (5000, 30, 4104, BF16, F32),
    (5000, 8, 4096, F32, F32),
    (16384, 30, 1032, F16, F32),
    (3001, 384, 7168, BF16, BF16),
    (8200, 300, 2048, BF16, BF16),
    (1000, 300, 1024, BF16, F32),
    (0, 8, 64, BF16, BF16),
]


def router(m, experts, hidden, dtype, weight_dtype, gen):
    return rows(m, hidden, dtype, gen), (torch.randn(experts, hidden, generator=gen) * hidden**-0.5).to(weight_dtype)


def product(a, b, chain):
    """a @ b and how far sums of so many terms may be off: every addition rounds, in the matrix cores down at worst, and products of
    pieces leave out 2^-24."""
    return a.double() @ b.double(), (a.double().abs() @ b.double().abs()) * (2 * (chain + 8) * U32)


def gradient(a, b, chain, dtype):
    """The same of gradients, whose 16-bit results are sums of operands that count to two pieces of eight bits.  A value less its
    nearest piece p is at most 2^-9 of it, and that less its own nearest piece at most 2^-9 of the rest: two pieces leave out 2^-18
    of a value.  bf16 is one piece; where both operands are cut, both leave that out, and the product of the two second pieces,
    2^-9 of each value, is left out too."""
    want, off = product(a, b, chain)
    if dtype != F32:
        off = off + (a.double().abs() @ b.double().abs()) * 2.0**-18 * (1 if b.dtype == BF16 else 3)
    return want, off


@gpu
@pytest.mark.parametrize("m,experts,hidden,dtype,weight_dtype", LOGITS)
def test_router_logits(device, m, experts, hidden, dtype, weight_dtype):
    gen = torch.Generator().manual_seed(m + experts)
    x, weight = router(m, experts, hidden, dtype, weight_dtype, gen)
    got = router_logits(x.to(device), weight.to(device))
    assert got.dtype == F32 and got.shape == (m, experts)
    want, off = product(x, weight.t(), hidden)
    assert_within(got, want, off)
    room = torch.full((m, experts + 5), 7.0, device=device)
    router_logits(x.to(device), weight.to(device), out=room[:, 3 : 3 + experts])
    assert torch.equal(room[:, 3 : 3 + experts], got)
    assert (room[:, :3] == 7).all() and (room[:, 3 + experts :] == 7).all()


EVERY_TILE = {
    # what a product's sizes choose: each tile, with a multiple of 64 to add up and not, split and not
    (F32, F32): [
        (40, 5, 4096), (40, 5, 4104), (257, 5, 4096), (1000, 5, 4104), (1500, 200, 1032), (2050, 384, 72), (2050, 384, 128),
        (4100, 70, 1024), (4100, 200, 136), (8200, 384, 72), (8200, 384, 128), (12000, 150, 64),
    ],
    (BF16, F32): [
        (40, 5, 4096), (40, 5, 4104), (1000, 5, 4096), (1000, 130, 2048), (2050, 150, 520), (2050, 384, 72), (2050, 384, 128),
        (3000, 70, 1032), (4100, 200, 136), (8200, 384, 64), (12000, 150, 64), (16400, 100, 72),
    ],
    (BF16, BF16): [
        (40, 5, 4096), (40, 5, 4104), (1030, 384, 72), (1500, 200, 2056), (2050, 300, 64), (3000, 70, 2048), (3000, 70, 2056),
        (4100, 130, 4096), (4100, 130, 4104), (4100, 200, 64), (8200, 70, 72), (12000, 384, 256), (12000, 384, 264),
        (16400, 70, 64), (16400, 70, 72),
    ],
    (F16, F32): [
        (40, 5, 4096), (40, 5, 4104), (65, 200, 4104), (520, 5, 4096), (700, 384, 2048), (1000, 384, 1032), (2050, 384, 136),
        (4100, 200, 136), (8200, 300, 64), (8200, 384, 64), (8200, 384, 72), (16400, 150, 64),
    ],
    (F16, F16): [
        (40, 5, 4096), (40, 5, 4104), (1030, 384, 72), (1500, 200, 2056), (2050, 300, 64), (3000, 70, 2048), (3000, 70, 2056),
        (4100, 130, 4096), (4100, 130, 4104), (4100, 200, 64), (8200, 70, 72), (12000, 384, 256), (12000, 384, 264),
        (16400, 70, 64), (16400, 70, 72),
    ],
}  # fmt: skip


@gpu
@pytest.mark.parametrize("dtype,weight_dtype,m,experts,hidden", [(*types, *size) for types, sizes in EVERY_TILE.items() for size in sizes])
def test_router_logits_of_every_tile(device, dtype, weight_dtype, m, experts, hidden):
    gen = torch.Generator().manual_seed(m + hidden)
    x, weight = (t.to(device) for t in router(m, experts, hidden, dtype, weight_dtype, gen))
    want, off = product(x, weight.t(), hidden)
    room = torch.full((m, experts + 3), 7.0, device=device)
    router_logits(x, weight, out=room[:, 1 : 1 + experts])
    assert_within(room[:, 1 : 1 + experts], want.cpu(), off.cpu())
    assert (room[:, 0] == 7).all() and (room[:, 1 + experts :] == 7).all()


@gpu
@pytest.mark.parametrize("dtype,weight_dtype", [(F32, F32), (BF16, F32), (F16, F32), (F16, F16), (BF16, BF16)])
def test_router_logits_hold_every_bit(device, dtype, weight_dtype):
    """One product to a sum: fp32 operands count to 24 bits, from the smallest normal values on."""
    gen = torch.Generator().manual_seed(11)
    for m, experts in ((33, 70), (400, 256)):
        x, weight = torch.zeros(m, 16), torch.zeros(experts, 16)
        at = torch.randint(0, 16, (1,), generator=gen).item()
        x[:, at], weight[:, at] = torch.randn(m, generator=gen), torch.randn(experts, generator=gen)
        x, weight = x.to(dtype), weight.to(weight_dtype)
        want = x.double() @ weight.double().t()
        # (a sum of up to six products of pieces, of which what is left out is 2^-24 of the whole)
        assert_within(router_logits(x.to(device), weight.to(device)), want, want.abs() * 8 * U32)


@gpu
@pytest.mark.parametrize("m", [2, 600])
def test_router_logits_of_strided_rows_and_nans(device, m):
    gen = torch.Generator().manual_seed(m)
    x, weight = router(m, 40, 128, BF16, BF16, gen)
    wide, wide_weight = torch.zeros(m, 256, dtype=BF16), torch.zeros(40, 136, dtype=BF16)
    wide[:, 128:], wide_weight[:, :128] = x, weight
    got = router_logits(wide.to(device)[:, 128:], wide_weight.to(device)[:, :128])
    want = router_logits(x.to(device), weight.to(device))
    assert torch.equal(got, want)
    one = x[:1].to(device).expand(m, 128)
    assert torch.equal(router_logits(one, weight.to(device)), router_logits(one.contiguous(), weight.to(device)))
    bad, bad_weight = x.clone(), weight.clone()
    bad[1, 5], bad_weight[3, 9] = float("nan"), float("inf")
    got = router_logits(bad.to(device), bad_weight.to(device))
    assert torch.isnan(got[1]).all()
    assert not torch.isfinite(got[:, 3]).any()
    keep = torch.ones(m, 40, dtype=torch.bool, device=device)
    keep[1], keep[:, 3] = False, False
    assert torch.equal(got[keep], want[keep])


LOGIT_GRADIENTS = [
    (1, 1, 8, F32, F32), (3, 60, 16, BF16, BF16), (5, 33, 264, F16, F32), (65, 64, 520, F16, F16), (130, 256, 1032, BF16, F32),
    (515, 61, 328, F32, F32), (1031, 256, 512, BF16, BF16), (700, 9, 2056, F16, F16), (2500, 128, 136, BF16, BF16),
]  # fmt: skip


@gpu
@pytest.mark.parametrize("m,experts,hidden,dtype,weight_dtype", LOGIT_GRADIENTS)
def test_gradients_of_router_logits(device, m, experts, hidden, dtype, weight_dtype):
    gen = torch.Generator().manual_seed(m + hidden)
    x, weight = router(m, experts, hidden, dtype, weight_dtype, gen)
    grad = 1e-2 * torch.randn(m, experts, generator=gen)
    leaves = [t.to(device).requires_grad_(True) for t in (x, weight)]
    gx, gw = torch.autograd.grad(router_logits(*leaves), leaves, grad.to(device))
    want, off = gradient(grad, weight, experts, dtype)
    want_w, off_w = gradient(grad.t(), x, m, weight_dtype)
    assert_within(gx, want, rounded(want, dtype, off))
    assert_within(gw, want_w, rounded(want_w, weight_dtype, off_w))
    # the call itself, with rows that lie apart, and each of the two alone
    dev = [t.to(device) for t in (x, weight)]
    apart = torch.full((m, experts + 3), float("nan"), device=device)
    apart[:, 1 : 1 + experts] = grad.to(device)
    both = router_logits_backward(apart[:, 1 : 1 + experts], *dev)
    assert torch.equal(both[0], gx) and torch.equal(both[1], gw)
    only_x, only_w = torch.empty_like(gx), torch.empty_like(gw)
    router_logits_backward(grad.to(device), *dev, out=(only_x, None))
    router_logits_backward(grad.to(device), *dev, out=(None, only_w))
    assert torch.equal(only_x, gx) and torch.equal(only_w, gw)


@gpu
def test_gradients_of_router_logits_against_differences(device):
    m, experts, hidden = 20, 12, 64
    gen = torch.Generator().manual_seed(3)
    x, weight = router(m, experts, hidden, F32, F32, gen)
    step_x, step_w, grad = (torch.randn(*s, generator=gen) for s in ((m, hidden), (experts, hidden), (m, experts)))
    leaves = [t.to(device).requires_grad_(True) for t in (x, weight)]
    gx, gw = torch.autograd.grad(router_logits(*leaves), leaves, grad.to(device))
    along = ((gx.cpu().double() * step_x).sum() + (gw.cpu().double() * step_w).sum()).item()
    a = 0.5

    def value(s):
        return (router_logits((x + s * step_x).to(device), (weight + s * step_w).to(device)).cpu().double() * grad.double()).sum().item()

    # (a central difference of a bilinear function is exact; the points are rounded, and the sums)
    size = ((x.abs() + a * step_x.abs()).double() @ (weight.abs() + a * step_w.abs()).double().t() * grad.double().abs()).sum().item()
    noise = size * (2 * (hidden + 8) + 4) * U32 / a
    off = (product(grad, weight, experts)[1] * step_x.abs()).sum() + (product(grad.t(), x, m)[1] * step_w.abs()).sum()
    assert abs((value(a) - value(-a)) / (2 * a) - along) <= noise + off.item()


# ---------------------------------------------------------------------------
# The choice of experts
# ---------------------------------------------------------------------------
def ref_scores(logits, scores):
    l64 = logits.double()
    if scores == "sigmoid":
        return 1 / (1 + torch.exp(-l64))
    shifted = torch.exp(l64 - l64.amax(1, keepdim=True).nan_to_num(0.0, neginf=0.0))
    return shifted / shifted.sum(1, keepdim=True).clamp_min(1e-300)


def ref_route(logits, k, bias=None, scores="softmax", num_groups=1, top_groups=1, group_top=2, renormalize=True, scale=1.0, bound=None):
    """Token by token, pick by pick."""
    m, experts = logits.shape
    s = ref_scores(logits, scores)
    chance = s + (0 if bias is None else bias.double())
    chance[logits == float("-inf")] = float("-inf")
    keys = (logits.double() if bias is None else chance).clone()
    indices, weights = torch.full((m, k), experts, dtype=torch.int32), torch.zeros(m, k, dtype=F64)
    for t in range(m if bound is None else min(m, bound)):
        row = keys[t]
        if not (row < float("inf")).all() or not (logits[t].double() < float("inf")).all():
            indices[t], weights[t] = torch.arange(k), float("nan")
            continue
        if top_groups < num_groups:
            sums = chance[t].view(num_groups, -1).sort(1, descending=True).values[:, :group_top].sum(1)
            inside = torch.zeros(num_groups, dtype=torch.bool)
            inside[sums.sort(stable=True, descending=True).indices[:top_groups]] = True
            row = torch.where(inside.repeat_interleave(experts // num_groups), row, float("-inf"))
        value, order = row.sort(stable=True, descending=True)
        n = int((value[:k] > float("-inf")).sum())
        indices[t, :n] = order[:n].to(torch.int32)
        picked = s[t, order[:n]]
        if renormalize and n:
            l64 = logits[t, order[:n]].double()
            top = l64.max()
            if scores == "softmax":
                part = torch.exp(l64 - top)
            else:
                up = (-top).clamp_min(0)
                part = 1 / (torch.exp(-up) + torch.exp(-l64 - up))
            picked = part / part.sum()
        weights[t, :n] = picked * scale
    return indices, weights


def weight_error(experts: int) -> float:
    """Relative, of a score or its share in fp32: an exponential of four ulps, a sum of at most experts / 64 + 6 and the products."""
    return (experts / 64 + 24) * U32


def make_logits(m, experts, dtype, gen, kind="any"):
    logits = torch.randn(m, experts, generator=gen) * 1.5
    if kind == "tied":  # few different values
        logits = torch.round(logits)
    elif kind == "masked":  # most experts are not there, in some rows none
        logits[torch.rand(m, experts, generator=gen) < 0.8] = float("-inf")
        logits[::5] = float("-inf")
    elif kind == "lowest":  # masks of the type's lowest value, in some rows everywhere
        logits[torch.rand(m, experts, generator=gen) < 0.8] = torch.finfo(dtype).min
        logits[::5] = torch.finfo(dtype).min
    elif kind == "far":  # scores that vanish in fp32, in some rows all of them
        logits = logits * 100 - 300
    return logits.to(dtype)


ROUTES = [
    # tokens, experts, picks, dtype, kind, bound, the rest
    (1, 1, 1, F32, "any", None, {}),
    (4, 64, 6, BF16, "any", 3, dict(renormalize=False)),
    (33, 256, 8, F32, "any", None, dict(scores="sigmoid", bias=True, num_groups=8, top_groups=4, scale=2.5)),
    (33, 256, 8, BF16, "tied", None, dict(scores="sigmoid", bias=True, num_groups=8, top_groups=3, group_top=1)),
    (50, 160, 6, F32, "any", 49, dict(num_groups=8, top_groups=3, group_top=1, renormalize=False, scale=16.0)),
    (65, 8, 2, F16, "tied", None, {}),
    (30, 60, 4, F32, "masked", None, dict(num_groups=4, top_groups=2)),
    (31, 61, 10, BF16, "masked", 29, dict(scores="sigmoid", bias=True)),
    (31, 61, 61, F32, "masked", None, dict(renormalize=False)),
    (40, 128, 64, F32, "lowest", None, {}),
    (40, 130, 9, BF16, "lowest", None, dict(scores="sigmoid", bias=True, num_groups=5, top_groups=2)),
    (40, 33, 5, F32, "far", None, dict(scores="sigmoid")),
    (40, 33, 5, F32, "far", None, dict(bias=True)),
    (7, 513, 3, F16, "any", None, dict(bias=True, num_groups=3, top_groups=2)),
    (9, 1000, 12, F32, "any", None, dict(scores="sigmoid", bias=True)),
    (5, 2000, 8, BF16, "tied", None, dict(num_groups=1000, top_groups=10)),
    (3, 5461, 64, F32, "masked", None, dict(scores="sigmoid", bias=True, num_groups=5461, top_groups=100, group_top=1)),
    (3, 5461, 10, F16, "any", None, dict(renormalize=False)),
    (20, 12, 3, F32, "any", 0, {}),
    (20, 12, 3, F32, "tied", 1000, dict(bias="tied")),
    (500, 384, 8, F32, "any", None, dict(scores="sigmoid", bias=True)),
    (300, 72, 6, BF16, "any", None, dict(bias=True, num_groups=2, top_groups=1)),
    (0, 16, 2, F32, "any", None, {}),
]  # fmt: skip


def route_case(m, experts, k, dtype, kind, bound, rest, device):
    gen = torch.Generator().manual_seed(m * 7 + experts)
    logits = make_logits(m, experts, dtype, gen, kind)
    bias = None
    if rest.get("bias"):
        bias = 0.2 * torch.randn(experts, generator=gen)
        if rest["bias"] == "tied":
            bias = torch.round(bias * 4) / 4
    rest = {key: value for key, value in rest.items() if key != "bias"}
    more = dict(rest, bias=None if bias is None else bias.to(device))
    if bound is not None:
        more["bound_m"] = to_u32(torch.tensor([bound], dtype=torch.int32), device)
    return logits, bias, rest, more


@gpu
@pytest.mark.parametrize("m,experts,k,dtype,kind,bound,rest", ROUTES)
def test_route_tokens(device, m, experts, k, dtype, kind, bound, rest):
    logits, bias, rest, more = route_case(m, experts, k, dtype, kind, bound, rest, device)
    indices, weights = route_tokens(logits.to(device), k, **more)
    assert indices.dtype == torch.uint32 and weights.dtype == F32 and indices.shape == weights.shape == (m, k)
    want, want_weights = ref_route(logits, k, bias, bound=bound, **rest)
    assert torch.equal(indices.view(torch.int32).cpu(), want)
    assert_within(weights, want_weights, rounded(want_weights, F32, want_weights.abs() * weight_error(experts)))
    # rows that lie apart, and into buffers
    apart = torch.full((m, experts + 3), float("nan"), dtype=dtype, device=device)
    apart[:, 1 : 1 + experts] = logits.to(device)
    out = torch.full_like(indices.view(torch.int32), 77).view(torch.uint32), torch.full_like(weights, 7.0)
    assert route_tokens(apart[:, 1 : 1 + experts], k, out=out, **more) is out
    assert torch.equal(out[0].view(torch.int32), indices.view(torch.int32)) and torch.equal(out[1], weights)


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_route_tokens_tells_close_experts_apart(device, scores, groups):
    """Keys that fp32 holds for equal, in both orders: logits next to each other, and biases that differ in their last bit."""
    gen = torch.Generator().manual_seed(2)
    m, experts, k = 64, 64, 6
    logits = torch.randn(m, 1, generator=gen).expand(m, experts).clone()
    up = torch.randint(-2, 3, (m, experts), generator=gen)
    for step in (1, 2):
        logits = torch.where(up >= step, torch.nextafter(logits, torch.tensor(9.0)), logits)
        logits = torch.where(up <= -step, torch.nextafter(logits, torch.tensor(-9.0)), logits)
    bias = torch.full((experts,), 0.37)
    bias[::3] = torch.nextafter(bias[::3], torch.tensor(1.0))
    more = dict(scores=scores, num_groups=groups, top_groups=max(1, groups // 2))
    for b in (None, bias):
        got, _ = route_tokens(logits.to(device), k, bias=None if b is None else b.to(device), **more)
        want, _ = ref_route(logits, k, b, **more)
        assert torch.equal(got.view(torch.int32).cpu(), want)


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups", [(64, 1), (66, 2), (104, 8), (128, 1), (256, 8), (500, 4), (500, 1), (520, 40), (1000, 1), (1200, 6)])
def test_route_tokens_tells_picks_from_runners_up(device, scores, experts, groups):
    """Every pick is close to the next one and the last to what comes after it, in each layout of experts over lanes.  Logits are a few
    last bits apart, by the marks of a ruler on which no two distances are alike: sums of two differ unless their logits are the same."""
    gen = torch.Generator().manual_seed(experts)
    marks = torch.tensor([0.0, 1, 4, 9, 15, 22, 32, 34])
    for k in (1, 7, 8):
        logits = 2 + marks[torch.randint(0, 8, (200, experts), generator=gen)] * 2.0**-22
        bias = torch.full((experts,), 0.25)
        more = dict(scores=scores, num_groups=groups, top_groups=max(1, groups // 2))
        got, _ = route_tokens(logits.to(device), k, bias=bias.to(device), **more)
        want, _ = ref_route(logits, k, bias, **more)
        assert torch.equal(got.view(torch.int32).cpu(), want)


@gpu
@pytest.mark.parametrize("experts,groups", [(64, 8), (128, 4), (250, 5), (1200, 6)])
def test_route_tokens_without_a_bias_keeps_the_logits_order(device, experts, groups):
    """Logits whose sigmoid is 1 in 64 bits too: groups are equal then, experts are not."""
    gen = torch.Generator().manual_seed(experts)
    logits = 38 + 60 * torch.rand(50, experts, generator=gen)
    logits[:, ::3] -= 40
    more = dict(scores="sigmoid", num_groups=groups, top_groups=2)
    got, weights = route_tokens(logits.to(device), 6, **more)
    want, want_weights = ref_route(logits, 6, **more)
    assert torch.equal(got.view(torch.int32).cpu(), want)
    assert_within(weights, want_weights, rounded(want_weights, F32, want_weights * weight_error(experts)))


@gpu
def test_route_tokens_with_biases_whose_sums_leave_fp32(device):
    gen = torch.Generator().manual_seed(4)
    logits, bias = torch.randn(20, 64, generator=gen), torch.full((64,), -3e38)
    bias[:32] = 2e38 + 1e38 * torch.rand(32, generator=gen)
    more = dict(scores="sigmoid", num_groups=8, top_groups=2)
    got, _ = route_tokens(logits.to(device), 5, bias=bias.to(device), **more)
    want, _ = ref_route(logits, 5, bias, **more)
    assert torch.equal(got.view(torch.int32).cpu(), want)


@gpu
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("bias", [False, True])
def test_route_tokens_of_logits_that_are_no_numbers(device, bad, bias):
    gen = torch.Generator().manual_seed(1)
    for experts in (40, 1500):
        logits = torch.randn(5, experts, generator=gen)
        logits[1, 39], logits[3] = bad, float("-inf")
        b = torch.randn(experts, generator=gen) if bias else None
        for more in (dict(), dict(scores="sigmoid", renormalize=False), dict(num_groups=10, top_groups=5)):
            indices, weights = route_tokens(logits.to(device), 3, bias=None if b is None else b.to(device), **more)
            want, want_weights = ref_route(logits, 3, b, **more)
            assert torch.equal(indices.view(torch.int32).cpu(), want)
            assert torch.isnan(weights[1]).all() and (weights[3] == 0).all() and (want[3] == experts).all()
            assert torch.isfinite(weights[[0, 2, 4]]).all()
        if bias:  # of the bias itself: all tokens; -inf takes the expert out
            b[2] = bad
            indices, weights = route_tokens(logits.to(device), 3, bias=b.to(device))
            assert torch.isnan(weights[[0, 1, 2, 4]]).all() and torch.equal(indices[0].view(torch.int32).cpu(), torch.arange(3, dtype=torch.int32))
            b[2] = float("-inf")
            logits[:, 2] = 50
            indices, weights = route_tokens(logits.to(device), 3, bias=b.to(device))
            assert not (indices.view(torch.int32)[[0, 2, 4]] == 2).any() and torch.isfinite(weights[[0, 2, 4]]).all()


def ref_route_gradient(logits, indices, grad, scores, renormalize, scale):
    """By autograd in 64 bits through the choice, and how far the kernel may be off before its result is rounded."""
    m, experts = logits.shape
    leaf = logits.double().requires_grad_(True)
    out, off = torch.zeros(m, experts, dtype=F64), torch.zeros(m, experts, dtype=F64)
    rel = weight_error(experts) + 80 * U32
    for t in range(m):
        at = indices[t][indices[t] < experts].long()
        if not at.numel():
            continue
        g = grad[t][indices[t] < experts].double()
        l64 = leaf[t]
        if renormalize:
            log = l64 if scores == "softmax" else -torch.nn.functional.softplus(-l64)
            w = torch.softmax(log[at], 0)
        else:
            w = (torch.softmax(l64, 0) if scores == "softmax" else torch.sigmoid(l64))[at]
        (d,) = torch.autograd.grad((w * g).sum() * scale, leaf)
        out[t] = d[t]
        # every part of the sums, by its magnitude
        with torch.no_grad():
            size = torch.zeros(experts, dtype=F64)
            size[at] = w * g.abs()
            inner = (w * g.abs()).sum()
            if renormalize:
                size[at] += w * inner
            elif scores == "softmax":
                size += torch.softmax(l64, 0) * inner
            off[t] = size * abs(scale) * rel
    return out, off


ROUTE_GRADIENTS = [case for case in ROUTES if case[0] and case[4] != "lowest"]


@gpu
@pytest.mark.parametrize("m,experts,k,dtype,kind,bound,rest", ROUTE_GRADIENTS)
def test_gradients_of_route_tokens(device, m, experts, k, dtype, kind, bound, rest):
    logits, bias, rest, more = route_case(m, experts, k, dtype, kind, bound, rest, device)
    grad = torch.randn(m, k, generator=torch.Generator().manual_seed(experts))
    leaf = logits.to(device).requires_grad_(True)
    indices, weights = route_tokens(leaf, k, **more)
    assert not indices.requires_grad and weights.requires_grad
    (got,) = torch.autograd.grad(weights, leaf, grad.to(device))
    form = dict(scores=rest.get("scores", "softmax"), renormalize=rest.get("renormalize", True), scale=rest.get("scale", 1.0))
    want, off = ref_route_gradient(logits, indices.view(torch.int32).cpu(), grad, **form)
    assert got.dtype == dtype
    assert_within(got, want, rounded(want, dtype, off))
    room = torch.full((m, experts + 3), 7.0, dtype=dtype, device=device)
    route_tokens_backward(grad.to(device), logits.to(device), indices, **form, out=room[:, 1 : 1 + experts])
    assert torch.equal(room[:, 1 : 1 + experts], got)
    assert (room[:, 0] == 7).all() and (room[:, 1 + experts :] == 7).all()


@gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradients_of_route_tokens_against_differences(device, scores, renormalize):
    m, experts, k = 10, 40, 5
    gen = torch.Generator().manual_seed(6)
    # (experts far apart, so that the steps change no choice)
    logits = torch.stack([torch.randperm(experts, generator=gen) for _ in range(m)]) * 0.2 - 4
    step, grad = torch.randn(m, experts, generator=gen).clamp(-2, 2), torch.randn(m, k, generator=gen)
    more = dict(scores=scores, renormalize=renormalize, scale=1.5)
    leaf = logits.to(device).requires_grad_(True)
    indices, weights = route_tokens(leaf, k, **more)
    (d,) = torch.autograd.grad(weights, leaf, grad.to(device))
    along = (d.cpu().double() * step).sum().item()
    a = 2.0**-6

    def value(s, exact):
        if exact:
            at, w = ref_route(logits.double() + s * step.double(), k, **more)
        else:
            at, w = route_tokens((logits + s * step).to(device), k, **more)
            at, w = at.view(torch.int32).cpu(), w.cpu().double()
        assert torch.equal(at, indices.view(torch.int32).cpu())
        return (w * grad.double()).sum().item()

    difference = (value(a, False) - value(-a, False)) / (2 * a)
    exact, half = ((value(s, True) - value(-s, True)) / (2 * s) for s in (a, a / 2))
    # weights of at most 1.5; a logit of up to 4 that is rounded moves one by less than 4 * 2^-24 of it, twice in a share
    noise = 1.5 * grad.double().abs().sum().item() * (weight_error(experts) + 12 * U32) / a
    assert abs(difference - exact) <= noise
    _, off = ref_route_gradient(logits, indices.view(torch.int32).cpu(), grad, **more)
    slack = (rounded(d.cpu().double(), F32, off) * step.abs()).sum().item()
    assert abs(difference - along) <= noise + slack + 2 * abs(exact - half)


# ---------------------------------------------------------------------------
# Refusals
# ---------------------------------------------------------------------------
def test_tensors_on_the_cpu_are_refused():
    x, weight, square = torch.zeros(2, 16, dtype=BF16), torch.zeros(16, dtype=BF16), torch.zeros(3, 16, dtype=BF16)
    logits, idx, w = torch.zeros(2, 3), torch.zeros(2, 2, dtype=torch.uint32), torch.zeros(2, 2)
    for call in (
        lambda: rms_norm(x, weight),
        lambda: rms_norm(x, weight, x, quantize=torch.int8),
        lambda: rms_norm_backward(x, x, weight),
        lambda: router_logits(x, square),
        lambda: router_logits_backward(logits, x, square),
        lambda: route_tokens(logits, 2),
        lambda: route_tokens_backward(w, logits, idx),
    ):
        with pytest.raises(RuntimeError, match="must be on GPU"):
            call()


@gpu
def test_refused_tensors(device):
    def t(*shape, dtype=BF16):
        return torch.zeros(*shape, dtype=dtype, device=device)

    i32, u32, i8 = torch.int32, torch.uint32, torch.int8
    x, w, router_weight = t(4, 32), t(32), t(6, 32)
    logits, idx, picked = t(4, 6, dtype=F32), t(4, 2, dtype=u32), t(4, 2, dtype=F32)
    bad = [
        (lambda: rms_norm(x.double(), w), "dtype for x"),
        (lambda: rms_norm(x, w.to(F16)), "weight must have the dtype"),
        (lambda: rms_norm(x, t(16)), "weight must be"),
        (lambda: rms_norm(x, t(64)[::2]), "contiguous"),
        (lambda: rms_norm(x, w.cpu()), "GPU"),
        (lambda: rms_norm(t(4, 12), t(12)), "aligned|multiple of 8"),
        (lambda: rms_norm(t(4, 24), t(24), quantize=i8), "multiple of 16|aligned"),
        (lambda: rms_norm(t(4, 40)[:, 1:33], w), "aligned"),
        (lambda: rms_norm(t(32, 4).t(), t(32)), "contiguous"),
        (lambda: rms_norm(x, w, t(3, 32)), "residual must have"),
        (lambda: rms_norm(x, w, x.to(F16)), "residual must have"),
        (lambda: rms_norm(x, w, eps=0.0), "eps"),
        (lambda: rms_norm(x, w, eps=-1.0), "eps"),
        (lambda: rms_norm(x, w, eps=float("nan")), "eps"),
        (lambda: rms_norm(x, w, eps=1e-45), "eps"),
        (lambda: rms_norm(x, w, quantize=torch.uint8), "quantize must be"),
        (lambda: rms_norm(x, w, out=NormedRows(None)), "neither"),
        (lambda: rms_norm(x, w, x, out=NormedRows(t(4, 32))), "sum goes with"),
        (lambda: rms_norm(x, w, out=NormedRows(t(4, 32), t(4, 32))), "sum goes with"),
        (lambda: rms_norm(x, w, out=NormedRows(t(4, 16))), "y must have"),
        (lambda: rms_norm(x, w, out=NormedRows(t(1, 32).expand(4, 32))), "more than once"),
        (lambda: rms_norm(x, w, out=NormedRows(None, None, t(4, 32, dtype=i8))), "scale goes with"),
        (lambda: rms_norm(x, w, out=NormedRows(None, None, t(4, 32, dtype=i8), t(3, dtype=F32))), "scale must be"),
        (lambda: rms_norm(x, w, out=NormedRows(None, None, t(4, 32, dtype=E4M3), t(4, dtype=F32))), "scale must be"),
        (lambda: rms_norm(x, w, out=NormedRows(None, None, t(4, 32, dtype=torch.uint8), t(4, dtype=F32))), "q must be"),
        (lambda: rms_norm(x, w, quantize=i8, out=NormedRows(t(4, 32))), "out.q"),
        (lambda: (lambda both: rms_norm(both[:4], w, out=NormedRows(both[1:5])))(t(5, 32)), "overlaps"),
        (lambda: (lambda one: rms_norm(x, w, x, out=NormedRows(one, one)))(t(4, 32)), "overlaps"),
        (lambda: rms_norm_backward(t(3, 32), x, w), "grad_y must have"),
        (lambda: rms_norm_backward(x, x, w, grad_sum=t(4, 16)), "grad_sum must have"),
        (lambda: rms_norm_backward(t(4, 32), x, w, out=(x, None)), "overlaps"),
        (lambda: rms_norm_backward(t(4, 32), x, w, out=(None, t(32, dtype=F32))), "grad_weight"),
        (lambda: router_logits(x, t(6, 16)), "length"),
        (lambda: router_logits(x, router_weight.to(F16)), "weight must have the dtype"),
        (lambda: router_logits(x, t(0, 32)), "num_experts"),
        (lambda: router_logits(x, t(5462, 32)), "num_experts"),
        (lambda: router_logits(t(4, 12), t(6, 12)), "aligned|multiple of 8"),
        (lambda: router_logits(x, router_weight.cpu()), "GPU"),
        (lambda: router_logits(x, router_weight, out=t(4, 5, dtype=F32)), "logits must be"),
        (lambda: router_logits(x, router_weight, out=t(4, 6)), "Float"),
        (lambda: router_logits(x, router_weight, out=t(6, 4, dtype=F32).t()), "contiguous"),
        (lambda: router_logits(x, router_weight, out=t(1, 6, dtype=F32).expand(4, 6)), "more than once"),
        (lambda: router_logits_backward(t(4, 5, dtype=F32), x, router_weight), "grad_logits must be"),
        (lambda: router_logits_backward(t(4, 6), x, router_weight), "Float"),
        (lambda: router_logits_backward(logits, x, router_weight, out=(t(4, 16), None)), "grad_x"),
        (lambda: router_logits_backward(logits, x, router_weight, out=(x, None)), "overlaps"),
        (lambda: route_tokens(logits.double(), 2), "dtype for logits"),
        (lambda: route_tokens(logits[0], 2), "2 dimensional"),
        (lambda: route_tokens(logits, 0), "experts_per_token"),
        (lambda: route_tokens(logits, 7), "experts_per_token"),
        (lambda: route_tokens(t(4, 100, dtype=F32), 65), "experts_per_token"),
        (lambda: route_tokens(t(4, 0, dtype=F32), 1), "num_experts"),
        (lambda: route_tokens(t(4, 5462, dtype=F32), 1), "num_experts"),
        (lambda: route_tokens(logits, 2, scores="tanh"), "scores"),
        (lambda: route_tokens(logits, 2, num_groups=4), "num_groups"),
        (lambda: route_tokens(logits, 2, num_groups=0), "num_groups"),
        (lambda: route_tokens(logits, 2, num_groups=-1), "out of range"),
        (lambda: route_tokens(logits, 2, num_groups=3, top_groups=4), "top_groups"),
        (lambda: route_tokens(logits, 2, num_groups=3, top_groups=0), "top_groups"),
        (lambda: route_tokens(logits, 2, num_groups=6, top_groups=3), "group_top"),
        (lambda: route_tokens(logits, 2, num_groups=2, top_groups=1, group_top=3), "group_top"),
        (lambda: route_tokens(logits, 5, num_groups=3, top_groups=2), "fewer than"),
        (lambda: route_tokens(logits, 2, bias=t(5, dtype=F32)), "bias must be"),
        (lambda: route_tokens(logits, 2, bias=t(6)), "bias must be of type"),
        (lambda: route_tokens(logits, 2, bound_m=t(1, dtype=i32)), "UInt32"),
        (lambda: route_tokens(logits, 2, bound_m=t(2, dtype=u32)), "scalar"),
        (lambda: route_tokens(logits, 2, scale=float("inf")), "weight_scale"),
        (lambda: route_tokens(t(6, 4, dtype=F32).t(), 2), "contiguous"),
        (lambda: route_tokens(logits, 3, out=(idx, picked)), "experts_per_token"),
        (lambda: route_tokens(logits, 2, out=(idx.view(i32), picked)), "indices must be of type"),
        (lambda: route_tokens(logits, 2, out=(idx, picked.to(BF16))), "weights must be of type"),
        (lambda: route_tokens(logits, 2, out=(idx[:3], picked[:3])), "indices.size"),
        (lambda: route_tokens(logits, 2, out=(idx, idx.view(F32))), "overlaps"),
        (lambda: route_tokens_backward(picked[:, :1], logits, idx), "contiguous|grad_weights"),
        (lambda: route_tokens_backward(picked, logits, idx.view(i32)), "indices must be of type"),
        (lambda: route_tokens_backward(picked, logits, idx, out=t(4, 6)), "grad_logits must have"),
        (lambda: route_tokens_backward(picked, logits, idx, out=logits), "overlaps"),
        (lambda: route_tokens_backward(picked, logits, idx, scores="none"), "scores"),
    ]  # fmt: skip
    for i, (call, message) in enumerate(bad):
        with pytest.raises(RuntimeError, match=message):
            call()
            raise AssertionError(f"call {i} was taken")
    assert rms_norm(x, w).y.shape == x.shape  # and the device still works


def test_the_layer_is_built_from_the_sources_in_the_tree():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    h = hashlib.sha256()
    for name in ("torch_common.h", "torch_tensors.h", "torch_router.cpp", "../../include/pplx_a2a.h"):
        h.update(open(os.path.join(root, "pplx-kernels_amd", "csrc", name), "rb").read())
    assert ops._C.router_build_id() == h.hexdigest()[:16], "pplx_kernels/_C.so is stale: run `make -C pplx-kernels_amd/csrc`"
