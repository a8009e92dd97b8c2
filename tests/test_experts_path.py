"""The operators between dispatch and combine as they are used: in a run, in graphs, on other streams, from two threads,
traced; and what the C entry points refuse, which needs no GPU."""

from __future__ import annotations

import ctypes
import threading

import pytest
import torch

from pplx_kernels import (
    LoopbackWorld,
    SortedTokens,
    int8_matmul,
    ops,
    quantize_rows,
    sort_tokens,
    sort_tokens_backward,
    unsort_tokens,
    unsort_tokens_backward,
)
from pplx_kernels.workloads import DeviceStep, Int8Experts, WorkloadSpec, generate, make_world
from tests.test_experts import (
    BF16,
    F32,
    U32,
    assert_within,
    check_product,
    check_quantized,
    make_indices,
    ref_sort,
    rounded,
    swiglu64,
    to_u32,
)

gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Runs
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("ranks,experts,k,hidden,tokens,wide", [(2, 8, 2, 256, 20, 96), (4, 32, 4, 1024, 65, 352)])
def test_dispatch_experts_combine(device, ranks, experts, k, hidden, tokens, wide):
    """A step of int8 rows: what dispatch leaves goes through the experts of 8-bit weights to combine."""
    spec = WorkloadSpec("int8", 90, ranks, experts, k, hidden, tokens, torch.int8, tokens="uniform")
    step = DeviceStep(spec, generate(spec, seed=4))
    step.expert_y_all.fill_(float("nan"))
    layer = Int8Experts(step, wide, seed=1)
    layer.h.fill_(float("nan"))
    world = make_world(spec, group_name=f"experts-{ranks}-{hidden}")
    step.dispatch_world(world)
    layer.run()
    step.combine_world(world)
    assert world.faults() == 0
    counts = layer.num_tokens.tolist()
    assert sum(counts) == sum(g.n for g in step.groups) * k
    cpu = {name: getattr(layer, name).cpu() for name in ("x", "x_scale", "h", "q", "q_scale", "y", "gate_up", "gate_up_scale",
                                                          "down", "down_scale")}  # fmt: skip
    for e, n in enumerate(counts):
        assert torch.isnan(cpu["h"][e, n:]).all() and torch.isnan(cpu["y"][e, n:]).all()
        if n:
            check_product(cpu["h"][e, :n], cpu["x"][e, :n], cpu["x_scale"][e, :n], cpu["gate_up"][e], cpu["gate_up_scale"][e], BF16)
            check_quantized(cpu["q"][e, :n], cpu["q_scale"][e, :n], *swiglu64(cpu["h"][e, :n]))
            check_product(cpu["y"][e, :n], cpu["q"][e, :n], cpu["q_scale"][e, :n], cpu["down"][e], cpu["down_scale"][e], BF16)
    # combine: rows of an expert are ordered by (group, token)
    place = [0] * experts
    for g, group in enumerate(step.groups):
        for t in range(group.n):
            ref, size = torch.zeros(hidden, dtype=torch.float64), torch.zeros(hidden, dtype=torch.float64)
            for p in range(k):
                e = int(group.indices[t, p])
                row = cpu["y"][e, place[e]].double() * float(group.weights[t, p])
                place[e] += 1
                ref, size = ref + row, size + row.abs()
            assert_within(step.out_tokens[g][t], ref, rounded(ref, BF16, (k + 1) * U32 * size))
    world.destroy()


def make_layer(device, gen, m, k, experts, hidden, wide):
    x = torch.randn(m, hidden, generator=gen).to(BF16).to(device)
    indices = to_u32(make_indices(m, k, experts, gen, "mixed"), device)
    weights = torch.rand(m, k, generator=gen).to(device)
    w1 = torch.randint(-127, 128, (experts, 2 * wide, hidden), generator=gen, dtype=torch.int32).to(torch.int8).to(device)
    w2 = torch.randint(-127, 128, (experts, hidden, wide), generator=gen, dtype=torch.int32).to(torch.int8).to(device)
    s1 = (torch.rand(experts, 2 * wide, generator=gen) / (73 * hidden**0.5)).to(device)
    s2 = (torch.rand(experts, hidden, generator=gen) / (73 * wide**0.5)).to(device)
    return x, indices, weights, w1, s1, w2, s2


class Buffers:
    """All that a step of sorted 8-bit experts writes."""

    def __init__(self, m, k, experts, hidden, wide, device):
        self.sorted = SortedTokens.empty(m, hidden, experts, k, BF16, device, int8=True)
        self.h = torch.zeros(m * k, 2 * wide, dtype=BF16, device=device)
        self.q = torch.zeros(m * k, wide, dtype=torch.int8, device=device), torch.zeros(m * k, device=device)
        self.y = torch.zeros(m * k, hidden, dtype=BF16, device=device)
        self.out = torch.zeros(m, hidden, dtype=BF16, device=device)


def run_layer(args, bound_m=None, b=None):
    x, indices, weights, w1, s1, w2, s2 = args
    s = sort_tokens(x, indices, w1.shape[0], bound_m, int8=True, out=b and b.sorted)
    h = int8_matmul(s.rows, s.scale, w1, s1, offsets=s.offsets, out=b and b.h)
    q, scale = quantize_rows(h, offsets=s.offsets, swiglu=True, out=b and b.q)
    y = int8_matmul(q, scale, w2, s2, offsets=s.offsets, out=b and b.y)
    return unsort_tokens(y, s.slots, s.offsets, weights, out=b and b.out), s, h, (q, scale), y


@gpu
@pytest.mark.parametrize("m,k,experts,hidden,wide", [(1, 2, 4, 64, 48), (70, 4, 16, 528, 144), (2100, 4, 8, 256, 128)])
def test_sorted_experts_layer(device, m, k, experts, hidden, wide):
    gen = torch.Generator().manual_seed(m)
    args = make_layer(device, gen, m, k, experts, hidden, wide)
    out, s, h, (q, scale), y = run_layer(args)
    x, indices, weights, w1, s1, w2, s2 = (a.cpu() if a.dtype != torch.uint32 else a.view(torch.int32).cpu() for a in args)
    slots, offsets, _ = ref_sort(torch.where(indices < 0, experts, indices), experts, m)
    assert torch.equal(s.slots.cpu(), slots) and torch.equal(s.offsets.cpu(), offsets)
    s_rows, s_scale, h, q, scale, y = (a.cpu() for a in (s.rows, s.scale, h, q, scale, y))
    for e in range(experts):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if b > a:
            check_product(h[a:b], s_rows[a:b], s_scale[a:b], w1[e], s1[e], BF16)
            check_quantized(q[a:b], scale[a:b], *swiglu64(h[a:b]))
            check_product(y[a:b], q[a:b], scale[a:b], w2[e], s2[e], BF16)
    live = slots >= 0
    picked = torch.where(live[:, :, None], y.double()[slots.clamp_min(0).long()], 0.0) * weights.double()[:, :, None]
    ref = picked.sum(1)
    assert_within(out, ref, rounded(ref, BF16, (k + 1) * U32 * picked.abs().sum(1)))


# ---------------------------------------------------------------------------
# Graphs, streams, threads
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("m", [40, 2500])  # (one launch of the sort, and three with a workspace)
@pytest.mark.parametrize("raw", [False, True])
def test_a_captured_layer_follows_its_inputs(device, m, raw):
    k, experts, hidden, wide = 4, 8, 128, 64
    gen = torch.Generator().manual_seed(7)
    args = make_layer(device, gen, m, k, experts, hidden, wide)
    bound = to_u32(torch.tensor([m], dtype=torch.int32), device)
    b, eager = Buffers(m, k, experts, hidden, wide, device), Buffers(m, k, experts, hidden, wide, device)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        run_layer(args, bound, b)
        if raw:  # the library's own capture
            world = LoopbackWorld(16, 8, 2, 1, 1, 64, 128, 0, group_name=f"capture-{m}")
            with world.capture() as captured:
                run_layer(args, bound, b)
            replay = captured.graph.replay
        else:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                run_layer(args, bound, b)
            replay = graph.replay
        for i in range(4):
            new = make_layer(device, gen, m, k, experts, hidden, wide)
            for old, fresh in zip(args[:3], new[:3]):
                old.copy_(fresh)
            bound.view(torch.int32).fill_(m - 3 * i)
            b.out.fill_(float("nan"))
            replay()
            torch.cuda.synchronize()
            run_layer(args, bound, eager)
            n = int(eager.sorted.offsets[-1])
            for got, want in ((b.out, eager.out), (b.sorted.rows, eager.sorted.rows), (b.sorted.slots, eager.sorted.slots),
                              (b.y[:n], eager.y[:n]), (b.q[0][:n], eager.q[0][:n])):  # fmt: skip
                assert torch.equal(got, want)
        if raw:
            world.destroy()


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


@gpu
def test_calls_follow_the_current_stream(device):
    gen = torch.Generator().manual_seed(3)
    args = make_layer(device, gen, 300, 4, 16, 256, 128)
    want = run_layer(args)[0]
    stream = torch.cuda.Stream()
    x = torch.zeros_like(args[0])
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)  # (what runs on another stream would read zeros)
        x.copy_(args[0])
        got = run_layer((x, *args[1:]))[0]
    stream.synchronize()
    assert torch.equal(got, want)


@gpu
def test_two_threads_on_streams_of_their_own(device):
    gen = torch.Generator().manual_seed(6)
    sizes = [(500, 4, 16, 256, 128), (3000, 4, 8, 128, 64)]
    layers = [make_layer(device, gen, *size) for size in sizes]
    want = [run_layer(args)[0] for args in layers]
    torch.cuda.synchronize()
    failures: list = []

    def work(args, expected):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got = run_layer(args)[0]
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(got, expected):
                        failures.append("other results")
        except Exception as exc:
            failures.append(exc)

    threads = [threading.Thread(target=work, args=pair) for pair in zip(layers, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


@gpu
def test_the_same_inputs_give_the_same_bits(device):
    gen = torch.Generator().manual_seed(8)
    m, k, experts, hidden = 4000, 4, 8, 512
    x = torch.randn(m, hidden, generator=gen).to(BF16).to(device)
    indices = to_u32(make_indices(m, k, experts, gen, "any"), device)
    weights = torch.rand(m, k, generator=gen).to(device)
    first = None
    for _ in range(5):
        s = sort_tokens(x, indices, experts)
        out = unsort_tokens(s.rows, s.slots, s.offsets, weights)
        gy, gw = unsort_tokens_backward(x, s.rows, s.slots, s.offsets, weights)
        now = [s.rows, s.slots, s.offsets, out, gy, gw, sort_tokens_backward(gy, s.slots)]
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(first, now))
        first = now


@gpu
@pytest.mark.parametrize("rows,width", [(12800, 2032), (3500, 14352), (3000, 17008)])
def test_large_rows_are_quantised_as_small_ones(device, rows, width):
    """More than the last-level cache may hold: read another way, with the same results."""
    x = torch.empty(rows, 2 * width, dtype=torch.float32, device=device).normal_(generator=torch.Generator(device).manual_seed(9))
    q, scale = quantize_rows(x, swiglu=True)
    for r in range(0, rows, 1000):
        part, part_scale = quantize_rows(x[r : r + 1000], swiglu=True)
        assert torch.equal(q[r : r + 1000], part) and torch.equal(scale[r : r + 1000], part_scale)
    check_quantized(q[:20], scale[:20], *swiglu64(x[:20].cpu()))


def product64(x, xs, w, ws):
    sums = x.double() @ w.double().t()  # (whole numbers below 2^53)
    return sums * xs.double()[:, None] * ws.double()


def random_int8(shape, gen, device):
    return torch.randint(-128, 128, shape, generator=gen, dtype=torch.int8, device=device)


def assert_product(got, ref):
    # as in check_product, on the device
    bound = ref.abs() * ((torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0) * (1 + 3 * U32) + 3 * U32) + 2.0**-130
    assert bool(((got.double() - ref).abs() <= bound).all())


@gpu
@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("rows,n,k", [
    (700, 136, 272), (1025, 136, 272), (401, 1160, 256), (401, 1159, 272), (5000, 136, 256), (4999, 133, 272),
    (2049, 1000, 128), (2049, 1000, 272), (400, 8200, 128), (397, 8193, 272), (3000, 4104, 128), (2049, 4101, 272),
    (400, 8200, 1024), (399, 8199, 528),
])  # fmt: skip
def test_products_of_every_tile(device, rows, n, k, out_dtype):
    """Sizes for which each form of the product is chosen, with k that fills its steps and k that does not."""
    gen = torch.Generator(device).manual_seed(rows)
    x, w = random_int8((rows, k), gen, device), random_int8((n, k), gen, device)
    xs, ws = (torch.rand(size, generator=gen, device=device) * 1e-2 for size in (rows, n))
    out = torch.full((rows + 3, n), 7.0, dtype=out_dtype, device=device)
    int8_matmul(x, xs, w, ws, out=out[:rows])
    assert_product(out[:rows], product64(x, xs, w, ws))
    assert (out[rows:] == 7).all()


@gpu
@pytest.mark.parametrize("rows,n,k", [
    (9, 40, 64), (401, 1160, 256), (4999, 133, 272), (2049, 1000, 128), (397, 8193, 272), (2049, 4101, 272), (399, 8199, 528),
])  # fmt: skip
def test_products_into_rows_that_begin_anywhere(device, rows, n, k):
    """Rows of out at every address that a result may have, with what lies between them left as it is."""
    gen = torch.Generator(device).manual_seed(n)
    x, w = random_int8((rows, k), gen, device), random_int8((n + 9, k), gen, device)
    xs, ws = (torch.rand(size, generator=gen, device=device) * 1e-2 for size in (rows, n + 9))
    ref = product64(x, xs, w, ws)
    for first, pitch, less in ((0, n + 1, 0), (1, n + 8, -1), (3, n + 11, -2), (5, n + 17, -9), (2, n + 9, 1), (7, n + 16, 2), (1, n + 9, 3)):
        columns = n + less
        out = torch.full((rows, max(pitch, first + columns)), 7.0, dtype=BF16, device=device)
        int8_matmul(x, xs, w[:columns], ws[:columns], out=out[:, first : first + columns])
        assert_product(out[:, first : first + columns], ref[:, :columns])
        assert (out[:, :first] == 7).all() and (out[:, first + columns :] == 7).all()


@gpu
@pytest.mark.parametrize("k", [2064, 2176])
@pytest.mark.parametrize("counts", [
    [3] * 10 + [0] * 14, [0] * 5 + [1, 400, 0, 33] + [20] * 15, [65, 64, 1, 900, 0, 0] + [30] * 18, [100] * 24,
])  # fmt: skip
def test_products_of_weights_beyond_the_caches(device, counts, k):
    """Weights that some experts' rows read once, past the caches, and others' several times."""
    experts, n, total = len(counts), 2056, sum(counts)
    gen = torch.Generator(device).manual_seed(total)
    w, ws = random_int8((experts, n, k), gen, device), torch.rand(experts, n, generator=gen, device=device)
    x, xs = random_int8((total, k), gen, device), torch.rand(total, generator=gen, device=device)
    starts = [0, *torch.tensor(counts).cumsum(0).tolist()]
    got = int8_matmul(x, xs, w, ws, offsets=torch.tensor(starts, dtype=torch.int32, device=device), out_dtype=F32)
    for e, c in enumerate(counts):
        rows = slice(starts[e], starts[e] + c)
        assert_product(got[rows], product64(x[rows], xs[rows], w[e], ws[e]))


@gpu
def test_offsets_that_do_not_ascend(device):
    """What belongs to two experts is one's or the other's; everything else is as it should be."""
    gen = torch.Generator(device).manual_seed(3)
    for rows, n, k in ((30, 264, 512), (3000, 2056, 1024)):
        a, b = rows // 3, 2 * rows // 3
        starts = torch.tensor([0, b, a, rows + 5, rows, -3], dtype=torch.int32, device=device)  # [0, b), none, [a, rows), none, none
        x, xs = random_int8((rows, k), gen, device), torch.ones(rows, device=device)
        w, ws = random_int8((5, n, k), gen, device), torch.ones(5, n, device=device)
        got = int8_matmul(x, xs, w, ws, offsets=starts, out_dtype=F32)
        assert_product(got[:a], product64(x[:a], xs[:a], w[0], ws[0]))
        assert_product(got[b:], product64(x[b:], xs[b:], w[2], ws[2]))


@gpu
def test_traced_calls(device):
    """Under torch.compile the calls are the registered ops; gradients flow through them."""
    gen = torch.Generator().manual_seed(9)
    m, k, experts, hidden = 30, 2, 4, 64
    x = torch.randn(m, hidden, generator=gen).to(device).requires_grad_(True)
    weights = torch.rand(m, k, generator=gen).to(device).requires_grad_(True)
    indices = to_u32(make_indices(m, k, experts, gen, "mixed"), device)

    def layer(x, weights):
        s = sort_tokens(x, indices, experts)
        return unsort_tokens(s.rows * 2.0, s.slots, s.offsets, weights)

    want = layer(x, weights)
    want_grads = torch.autograd.grad(want.sum(), [x, weights])
    got = torch.compile(layer, backend="aot_eager", fullgraph=True)(x, weights)
    got_grads = torch.autograd.grad(got.sum(), [x, weights])
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(got_grads, want_grads))

    args = make_layer(device, gen, 40, 2, 4, 64, 48)
    want = run_layer(args)[0]
    got = torch.compile(lambda *a: run_layer(a)[0], backend="aot_eager", fullgraph=True)(*args)
    assert torch.equal(got, want)


@gpu
def test_traced_calls_of_unknown_sizes(device):
    """Traced once for any number of tokens."""
    gen = torch.Generator().manual_seed(10)
    k, experts, hidden, traces = 2, 4, 64, []

    def backend(graph, inputs):
        traces.append(len(inputs))
        return torch._dynamo.lookup_backend("aot_eager")(graph, inputs)

    def layer(x, weights, indices):
        s = sort_tokens(x, indices, experts)
        q = sort_tokens(x.detach(), indices, experts, int8=True)
        return unsort_tokens(s.rows * 2.0, s.slots, s.offsets, weights), q.rows, q.scale

    compiled = torch.compile(layer, backend=backend, fullgraph=True, dynamic=True)
    for m in (30, 41, 7):
        x = torch.randn(m, hidden, generator=gen).to(device).requires_grad_(True)
        weights = torch.rand(m, k, generator=gen).to(device).requires_grad_(True)
        indices = to_u32(make_indices(m, k, experts, gen, "mixed"), device)
        want = layer(x, weights, indices)
        want_grads = torch.autograd.grad(want[0].sum(), [x, weights])
        got = compiled(x, weights, indices)
        assert len(traces) == 1
        got_grads = torch.autograd.grad(got[0].sum(), [x, weights])
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(got_grads, want_grads))


@gpu
def test_gradients_at_the_edges(device):
    """What the gradient could not do is refused when it is recorded; without tokens it is zeros."""
    x = torch.randn(4, 12, device=device, requires_grad=True)
    indices = torch.zeros(4, 2, dtype=torch.int32, device=device).view(torch.uint32)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        sort_tokens(x, indices, 3)
    s = sort_tokens(x.detach(), indices, 3)
    assert torch.equal(s.rows[s.slots.long()], x.detach()[:, None].expand(-1, 2, -1))
    y = torch.randn(8, 16, device=device, requires_grad=True)
    for offsets in (s.offsets.float(), s.offsets[None], s.offsets[:0], s.offsets.cpu()):
        with pytest.raises(RuntimeError, match="offsets"):
            unsort_tokens(y, s.slots, offsets)
    none = torch.empty(0, 2, dtype=torch.int32, device=device)
    weights = torch.empty(0, 2, device=device, requires_grad=True)
    out = unsort_tokens(y, none, torch.zeros(4, dtype=torch.int32, device=device), weights)
    grad_y, grad_w = torch.autograd.grad(out.sum(), [y, weights])
    assert out.shape == (0, 16) and (grad_y == 0).all() and grad_w.shape == (0, 2)


@gpu
@pytest.mark.parametrize("experts", [963, 964, 1820, 1821, 5461])
def test_sort_of_many_picks_and_experts(device, experts):
    """The tables of the experts at the sizes where they fill a workgroup's share of the memory that it counts in."""
    m, k = 1100, 8
    gen = torch.Generator().manual_seed(experts)
    x = torch.randn(m, 8, generator=gen)
    indices = make_indices(m, k, experts, gen, "mixed")
    s = sort_tokens(x.to(device), to_u32(indices, device), experts)
    slots, offsets, order = ref_sort(indices, experts, m)
    rows = torch.zeros(m * k, 8)
    rows[: order.numel()] = x[order // k]
    assert torch.equal(s.slots.cpu(), slots) and torch.equal(s.offsets.cpu(), offsets) and torch.equal(s.rows.cpu(), rows)


# ---------------------------------------------------------------------------
# The C entry points refuse before anything reaches a device
# ---------------------------------------------------------------------------
P, U, I, L, Q = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64


def struct(*fields):
    return type("Args", (ctypes.Structure,), {"_fields_": list(fields)})


Rows = struct(("layout", I), ("num_experts", U), ("rows", Q), ("starts_or_counts", P))
SortArgs = struct(
    ("x", P), ("x_stride_row", L), ("dtype", I), ("m", U), ("experts_per_token", U), ("num_experts", U), ("hidden_dim", Q),
    ("indices", P), ("bound_m", P), ("out_rows", P), ("out_stride_row", L), ("out_scale", P), ("slots", P), ("offsets", P),
    ("workspace", P),
)  # fmt: skip
UnsortArgs = struct(
    ("out", P), ("out_stride_row", L), ("out_dtype", I), ("y_dtype", I), ("y", P), ("y_stride_row", L), ("y_rows", L),
    ("slots", P), ("weights", P), ("m", U), ("experts_per_token", U), ("hidden_dim", Q),
)  # fmt: skip
BackwardArgs = struct(
    ("grad_y", P), ("grad_y_stride_row", L), ("grad_weights", P), ("grad_out", P), ("grad_out_stride_row", L), ("grad_dtype", I),
    ("dtype", I), ("y", P), ("y_stride_row", L), ("y_rows", L), ("slots", P), ("num_rows", P), ("weights", P), ("m", U),
    ("experts_per_token", U), ("hidden_dim", Q),
)  # fmt: skip
QuantizeArgs = struct(
    ("rows", Rows), ("out", P), ("out_stride_row", L), ("out_stride_expert", L), ("out_scale", P), ("out_scale_stride_row", L),
    ("out_scale_stride_expert", L), ("x", P), ("x_stride_row", L), ("x_stride_expert", L), ("dtype", I), ("swiglu", I), ("width", Q),
)  # fmt: skip
MatmulArgs = struct(
    ("rows", Rows), ("out", P), ("out_stride_row", L), ("out_stride_expert", L), ("out_dtype", I), ("x", P), ("x_stride_row", L),
    ("x_stride_expert", L), ("x_scale", P), ("x_scale_stride_row", L), ("x_scale_stride_expert", L), ("weight", P),
    ("weight_scale", P), ("n", Q), ("k", Q),
)  # fmt: skip
A = 0x10000  # an address that nobody reads
GOOD = {
    "sort_tokens": (SortArgs, dict(x=A, x_stride_row=64, dtype=1, m=4, experts_per_token=2, num_experts=3, hidden_dim=32, indices=A,
                                   out_rows=A, out_stride_row=64, slots=A, offsets=A)),
    "unsort_tokens": (UnsortArgs, dict(out=A, out_stride_row=64, out_dtype=1, y_dtype=1, y=A, y_stride_row=64, y_rows=8, slots=A,
                                       weights=A, m=4, experts_per_token=2, hidden_dim=32)),
    "unsort_tokens_backward": (BackwardArgs, dict(grad_y=A, grad_y_stride_row=64, grad_weights=A, grad_out=A, grad_out_stride_row=64,
                                                  grad_dtype=1, dtype=1, y=A, y_stride_row=64, y_rows=8, slots=A, num_rows=A,
                                                  weights=A, m=4, experts_per_token=2, hidden_dim=32)),
    "quantize_rows": (QuantizeArgs, dict(rows=Rows(0, 1, 4, None), out=A, out_stride_row=32, out_scale=A, out_scale_stride_row=1,
                                         x=A, x_stride_row=64, dtype=1, width=32)),
    "int8_matmul": (MatmulArgs, dict(rows=Rows(0, 1, 4, None), out=A, out_stride_row=8, out_dtype=1, x=A, x_stride_row=32,
                                     x_scale=A, x_scale_stride_row=1, weight=A, weight_scale=A, n=8, k=32)),
}  # fmt: skip


def c_call(name, device=0, **changed):
    kind, good = GOOD[name]
    lib = ops.load_library()
    fn = getattr(lib, f"pplx_a2a_{name}")
    fn.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
    args = kind(**{**good, **changed})
    return fn(device, ctypes.addressof(args), None), lib.pplx_a2a_last_error().decode()


@pytest.mark.parametrize("name,changed,status,message", [
    ("sort_tokens", dict(x=None), 1, "NULL"),
    ("sort_tokens", dict(offsets=None), 1, "offsets"),
    ("sort_tokens", dict(offsets=A + 2), 1, "offsets"),
    ("sort_tokens", dict(x=A + 8), 1, "16-byte"),
    ("sort_tokens", dict(out_stride_row=72), 1, "16-byte"),
    ("sort_tokens", dict(indices=A + 1), 1, "aligned"),
    ("sort_tokens", dict(dtype=3), 1, "dtype"),
    ("sort_tokens", dict(experts_per_token=65), 1, "experts_per_token"),
    ("sort_tokens", dict(experts_per_token=0), 1, "experts_per_token"),
    ("sort_tokens", dict(num_experts=5462), 1, "num_experts"),
    ("sort_tokens", dict(hidden_dim=0), 1, "16 bytes"),
    ("sort_tokens", dict(hidden_dim=36), 1, "16 bytes"),
    ("sort_tokens", dict(hidden_dim=24, x_stride_row=48, out_scale=A), 1, "16 bytes"),
    ("sort_tokens", dict(m=1 << 31, experts_per_token=1), 4, "2^31"),
    ("sort_tokens", dict(m=10000), 1, "workspace"),
    ("unsort_tokens", dict(out=None), 1, "NULL"),
    ("unsort_tokens", dict(hidden_dim=36), 1, "hidden_dim"),
    ("unsort_tokens", dict(y_rows=-1), 1, "rows"),
    ("unsort_tokens", dict(out_dtype=7), 1, "dtype"),
    ("unsort_tokens", dict(y=A + 4), 1, "16-byte"),
    ("unsort_tokens", dict(m=1 << 31, experts_per_token=64), 4, "too many"),
    ("unsort_tokens_backward", dict(y=None), 1, "y is NULL"),
    ("unsort_tokens_backward", dict(num_rows=None), 1, "num_rows"),
    ("unsort_tokens_backward", dict(m=0), 1, "tokens"),
    ("unsort_tokens_backward", dict(grad_out=A + 8), 1, "16-byte"),
    ("quantize_rows", dict(rows=Rows(1, 1, 4, None)), 1, "starts_or_counts"),
    ("quantize_rows", dict(rows=Rows(0, 2, 4, None)), 1, "one expert"),
    ("quantize_rows", dict(rows=Rows(3, 1, 4, None)), 1, "layout"),
    ("quantize_rows", dict(rows=Rows(2, 2, 1 << 30, A)), 4, "2^31"),
    ("quantize_rows", dict(width=24), 1, "width"),
    ("quantize_rows", dict(out=None), 1, "NULL"),
    ("int8_matmul", dict(k=24), 1, "multiple of 16"),
    ("int8_matmul", dict(k=131072), 1, "131056"),
    ("int8_matmul", dict(weight=A + 8), 1, "weight"),
    ("int8_matmul", dict(x_stride_row=1 << 23), 4, "8 MiB"),
    ("int8_matmul", dict(out=A + 1), 1, "aligned"),
    ("int8_matmul", dict(n=1 << 31), 1, "2^31"),
    ("int8_matmul", dict(rows=Rows(0, 0, 4, None)), 1, "num_experts"),
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


def test_workspace_of_the_sort():
    lib = ops.load_library()
    fn = lib.pplx_a2a_sort_workspace
    fn.argtypes = [U, U, U, ctypes.c_void_p]
    out = ctypes.c_uint64(7)
    for m, k, experts, tiles in ((0, 8, 4, 0), (1024, 8, 256, 0), (1025, 8, 256, 9), (65536, 8, 256, 64), (5000, 2, 5461, 40)):
        assert fn(m, k, experts, ctypes.addressof(out)) == 0
        assert out.value <= 64 * 4 * experts and (out.value == 0) == (tiles == 0)
        assert out.value == 4 * experts * tiles, (m, k, experts, out.value / (4 * experts))
    assert fn(1, 1, 1, None) == 1
