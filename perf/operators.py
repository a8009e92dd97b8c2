"""The measured cases of the operators between dispatch and combine: tokens sorted by expert and back, the gradients of
both, rows quantised to 8 bits, and the experts' products in 8-bit integers.

Fields of a case:
  op        "sort"     a step's tokens to rows sorted by expert (with "int8" quantised on the way)
            "unsort"   the experts' rows back to tokens, weighted
            "train"    both, and the gradients of both
            "swiglu"   the gated activation of rows, quantised with one scale a row
            "product"  rows of 8-bit integers times the experts' weights
  tokens, experts, topk, hidden, type   the step; "experts" counts those that are here
  ranks     picks go to ranks * experts experts, and those of other ranks' experts get no row here
  present   "full": all tokens are there; "ragged": a count in device memory says how many
  routing   "uniform", "zipf" (s = 1.2) or "mix" (half uniform, half Zipf with s = 1.0)
  form      of the rows of "swiglu" and "product": "sorted" (one behind the other, with offsets), "padded" (a buffer for each
            expert, as dispatch leaves them, with counts), "dense" (one weight for all rows)
  width     of an activated row ("swiglu"), columns of the result ("product", whose rows are `hidden` long)
"""

from __future__ import annotations

import os
import sys

import torch

own = False  # False: plain forms out of elementary torch operations; True: the framework's kernels

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_TINY = 2.0**-100  # rows whose largest value is below this are quantised as if it were this


def _package():
    """The package, which lives in a folder of the repository that is the working directory."""
    folder = os.path.join(os.getcwd(), "pplx-kernels_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import pplx_kernels

    return pplx_kernels


def listed() -> list[dict]:
    return [
        # A decode step of four tokens in the smaller of the two model shapes of the latency table.
        _sort("sort-decode-4", tokens=4, experts=64, topk=6, hidden=2048),
        # A ragged chunk of a prefill, quantised on its way to the experts' products.
        _sort("sort-int8-chunk-509", tokens=509, experts=256, topk=8, hidden=7168, int8=True, present="ragged", routing="mix"),
        # The largest batch of one rank: 8192 tokens, 256 experts, top-8.
        _sort("sort-prefill-8192", tokens=8192, experts=256, topk=8, hidden=7168, routing="mix"),
        # Decode with a batch of 64, and back to tokens.
        _unsort("unsort-decode-64", tokens=64, experts=256, topk=8, hidden=7168),
        # Rows of no round size that the experts left in fp32, half of the picks served elsewhere.
        _unsort("unsort-ragged-f32", tokens=3001, experts=32, topk=5, hidden=2880, type="f32", out="f16", ranks=2, present="ragged"),
        # Training: a ragged micro-batch in half precision, some of whose experts live elsewhere.
        _train("train-ragged-f16", tokens=3001, experts=32, topk=5, hidden=2880, type="f16", ranks=2, present="ragged"),
        # Training: 8 experts, top-2, skewed.
        _train("train-8192-zipf", tokens=8192, experts=8, topk=2, hidden=4096, routing="zipf"),
        # The activation between the two products of a decode step, in dispatch's buffers: 64 tokens of a
        # deployment of 8 ranks, of which this one holds 32 experts.
        _swiglu("swiglu-decode-padded", tokens=64, experts=32, topk=8, ranks=8, form="padded", width=2048),
        # The same of a prefill, sorted, of no round width.
        _swiglu("swiglu-prefill", tokens=8192, experts=64, topk=6, form="sorted", width=1408),
        # One token through one weight: latency.
        _product("product-one-token", tokens=1, experts=1, topk=1, hidden=2048, width=1408, form="dense"),
        # The first product of the decode step above: the weights' bytes count.
        _product("product-decode-padded", tokens=64, experts=32, topk=8, ranks=8, hidden=7168, width=4096, form="padded"),
        # The first product of a skewed prefill with 8 experts: the operations count.
        _product("product-prefill-zipf", tokens=8192, experts=8, topk=2, hidden=4096, width=14336, form="sorted", routing="zipf"),
    ]  # fmt: skip


def _case(op, name, **fields) -> dict:
    case = dict(op=op, ranks=1, present="full", routing="uniform", type="bf16")
    case.update(fields)
    return {"name": name, **case} if name else case


def _sort(name="", **fields) -> dict:
    return _case("sort", name, **{"int8": False, **fields})


def _unsort(name="", **fields) -> dict:
    return _case("unsort", name, **{"out": "bf16", **fields})


def _train(name="", **fields) -> dict:
    return _case("train", name, **fields)


def _swiglu(name="", **fields) -> dict:
    return _case("swiglu", name, **fields)


def _product(name="", **fields) -> dict:
    return _case("product", name, **fields)


def _log_uniform(rng, low: int, high: int) -> int:
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng) -> dict:
    """One more case: sizes spread over their logarithm, types, forms and routing at random, no dearer than the dearest
    listed case of its operator."""
    while True:
        op = rng.choice(["sort", "unsort", "train", "swiglu", "product", "product"])
        experts = _log_uniform(rng, 4, 256)
        tokens = _log_uniform(rng, 1, 16384)
        topk = min(rng.randint(1, 10), experts)
        step = dict(
            tokens=tokens, experts=experts, topk=topk, ranks=rng.choice([1, 1, 2]), present=rng.choice(["full", "ragged"]),
            routing=rng.choice(["uniform", "zipf", "mix"]), type=rng.choice(["bf16", "bf16", "f16"]),
        )  # fmt: skip
        if op == "sort":
            # (16-byte multiples of 16-bit elements; quantised rows are multiples of 16 elements)
            int8 = rng.random() < 0.4
            unit = 16 if int8 else 8
            case = _sort(**step, int8=int8, hidden=unit * _log_uniform(rng, 256 // unit, 8192 // unit))
        elif op == "unsort":
            y = rng.choice(["bf16", "f16", "f32"])
            out = rng.choice(["bf16", "f16"]) if y == "f32" else y
            case = _unsort(**{**step, "type": y}, out=out, hidden=8 * _log_uniform(rng, 32, 1024))
        elif op == "train":
            case = _train(**step, hidden=8 * _log_uniform(rng, 32, 1024))
        else:
            form = rng.choice(["sorted", "padded", "dense"] if op == "product" else ["sorted", "padded"])
            step["present"] = "full"
            if form == "padded":
                step["tokens"] = _log_uniform(rng, 1, 1024)
                step["ranks"] = rng.choice([1, 2, 8])
            elif form == "sorted":
                step["ranks"] = 1
            else:
                step.update(experts=1, topk=1, ranks=1, routing="uniform")
            if op == "swiglu":
                case = _swiglu(**step, form=form, width=16 * _log_uniform(rng, 8, 512))
            else:
                step["experts"] = min(step["experts"], 64)
                step["topk"] = min(step["topk"], step["experts"])
                case = _product(**step, form=form, hidden=16 * _log_uniform(rng, 16, 512), width=_log_uniform(rng, 100, 16384))
        dearest = max(_cost(c) for c in listed() if c["op"] == op)
        if _cost(case) <= dearest and _state_bytes(case) <= 12e9:
            return case


# ---------------------------------------------------------------------------
# Sizes
# ---------------------------------------------------------------------------
def _present(case: dict) -> int:
    return case["tokens"] if case["present"] == "full" else max(1, case["tokens"] * 7 // 8)


def _expected_rows(case: dict) -> float:
    return _present(case) * case["topk"] / case["ranks"]


def _cost(case: dict) -> float:
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 2e15


def _state_bytes(case: dict) -> float:
    """The largest thing that a pass in plain form holds."""
    if case["op"] == "product":
        rows = case["experts"] * case["tokens"] if case["form"] == "padded" else _expected_rows(case)
        return 8 * case["experts"] * case["hidden"] * case["width"] + 4 * rows * (case["hidden"] + case["width"])
    if case["op"] == "swiglu":
        rows = case["experts"] * case["tokens"] if case["form"] == "padded" else _expected_rows(case)
        return 16 * rows * case["width"]
    return 16 * case["tokens"] * case["topk"] * case["hidden"]


def work(case: dict) -> dict:
    """Bytes: every input that a token, a pick or a row needs is read once and every output written once.  Flops: one
    multiply-add per gathered element, product or gradient."""
    op, m, k, e = case["op"], case["tokens"], case["topk"], case["experts"]
    rows, size = _expected_rows(case), _DTYPES[case["type"]].itemsize
    if op in ("sort", "unsort", "train"):
        h, present, picks = case["hidden"], _present(case), m * k
        sort = present * h * size + picks * (4 + 4) + 4 * (e + 1) + picks * (h + 4 if case.get("int8") else h * size)
        out = _DTYPES[case.get("out", case["type"])].itemsize
        unsort = rows * h * size + picks * (4 + 4) + m * h * out
        if op == "sort":
            return {"bytes": sort, "flops": 0}
        if op == "unsort":
            return {"bytes": unsort, "flops": 2 * rows * h}
        # the gradient of unsort writes a row for each that it reads, that of sort is an unsort without weights
        backward = (rows * h + m * h) * size + picks * 8 + picks * h * size + picks * 4 + rows * h * size + m * h * size
        return {"bytes": sort + unsort + backward, "flops": 2 * rows * h * 4}
    if case["form"] == "dense":
        rows, e = m, 1
    if op == "swiglu":
        return {"bytes": rows * (case["width"] * (2 * size + 1) + 4), "flops": 8 * rows * case["width"]}
    h, n = case["hidden"], case["width"]
    with_rows = e * (1 - (1 - 1 / e) ** rows) if e > 1 else 1
    return {"bytes": rows * (h + 4 + n * size) + with_rows * n * (h + 4), "flops": 2 * rows * h * n}


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _routing(case: dict, gen: torch.Generator) -> torch.Tensor:
    """[m, K] expert ids, distinct in each row, in no order; ids of experts on other ranks lie behind those here."""
    m, k, experts = case["tokens"], case["topk"], case["experts"] * case["ranks"]

    def top(log_pmf) -> torch.Tensor:
        # Gumbel top-k: sampling without replacement
        u = torch.rand(m, experts, generator=gen, device="cuda").clamp_min(1e-20)
        return (log_pmf - torch.log((-torch.log(u)).clamp_min(1e-20))).topk(k, dim=1).indices

    def zipf(s: float) -> torch.Tensor:
        # (which experts are the popular ones differs from seed to seed)
        order = torch.randperm(experts, generator=gen, device="cuda")
        return -s * torch.log(1.0 + order.float())

    if case["routing"] == "uniform":
        return top(0.0).to(torch.int32)
    if case["routing"] == "zipf":
        return top(zipf(1.2)).to(torch.int32)
    skewed = torch.rand(m, 1, generator=gen, device="cuda") < 0.5
    return torch.where(skewed, top(zipf(1.0)), top(0.0)).to(torch.int32)


def _activations(shape: tuple, dtype: torch.dtype, gen: torch.Generator) -> torch.Tensor:
    """Normal values, whose size differs from row to row, with a few columns of large ones."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((*shape[:-1], 1), generator=gen, device="cuda"))
    x *= torch.where(torch.rand(shape[-1], generator=gen, device="cuda") < 0.005, 6.0, 1.0)
    return x.to(dtype)


def _int8(shape: tuple, gen: torch.Generator) -> torch.Tensor:
    q = torch.empty(shape, dtype=torch.int8, device="cuda")
    for part in q.view(-1, shape[-1]).split(1 << 16):
        part.copy_((30.0 * torch.randn(part.shape, generator=gen, device="cuda")).round_().clamp_(-127, 127))
    return q


def _counts(indices: torch.Tensor, experts: int) -> torch.Tensor:
    ids = torch.where(indices < experts, indices, experts).reshape(-1).to(torch.int64)
    return torch.zeros(experts + 1, dtype=torch.int64, device="cuda").index_add_(0, ids, torch.ones_like(ids))[:experts]


def _offsets(counts: torch.Tensor) -> torch.Tensor:
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)


def prepare(case: dict, seed: int) -> dict:
    gen = _generator(seed)
    op, m, k, e, dtype = case["op"], case["tokens"], case["topk"], case["experts"], _DTYPES[case["type"]]
    s: dict = {"case": case}
    indices = _routing(case, gen)
    if op in ("sort", "unsort", "train"):
        h, picks = case["hidden"], m * k
        bound = torch.full((1,), _present(case), dtype=torch.int32, device="cuda")
        s["indices"] = indices.view(torch.uint32)
        s["bound_m"] = bound.view(torch.uint32) if case["present"] == "ragged" else None
        s["weights"] = torch.softmax(torch.randn(m, k, generator=gen, device="cuda"), dim=1)
        if op != "unsort":
            s["x"] = _activations((m, h), dtype, gen)
        if op != "sort":
            s["y"] = _activations((picks, h), dtype, gen)
        if op == "sort" and case["int8"]:
            s["values"] = torch.empty(picks, h, dtype=dtype, device="cuda")
        if op == "unsort":  # (the step's sort, which ran before the experts)
            s["slots"], s["offsets"], _ = _plain_routing(indices, e, s["bound_m"])
            s["out"] = torch.zeros(m, h, dtype=_DTYPES[case["out"]], device="cuda")
        if op == "train":
            s["grad_rows"] = (1e-2 * torch.randn(picks, h, generator=gen, device="cuda")).to(dtype)
            s["grad_out"] = (1e-2 * torch.randn(m, h, generator=gen, device="cuda")).to(dtype)
            for leaf in ("x", "y", "weights"):
                s[leaf].requires_grad_(True)
        return s
    if case["form"] == "padded":
        s["num_tokens"] = _counts(indices, e).to(torch.int32)
        shape: tuple = (e, m)
    elif case["form"] == "sorted":
        s["offsets"] = _offsets(_counts(indices, e))
        shape = (m * k,)
    else:
        shape = (m,)
    if op == "swiglu":
        width = case["width"]
        s["x"] = _activations((*shape, 2 * width), dtype, gen)
        s["q"] = torch.zeros((*shape, width), dtype=torch.int8, device="cuda")
        s["scale"] = torch.zeros(shape, dtype=torch.float32, device="cuda")
        s["values"] = torch.empty((*shape, width), dtype=dtype, device="cuda")
        return s
    weight = (case["width"], case["hidden"]) if case["form"] == "dense" else (e, case["width"], case["hidden"])
    s["x"] = _int8((*shape, case["hidden"]), gen)
    s["x_scale"] = 0.02 * torch.exp(0.5 * torch.randn(shape, generator=gen, device="cuda"))
    s["weight"] = _int8(weight, gen)
    s["weight_scale"] = 1e-3 * torch.exp(0.3 * torch.randn(weight[:-1], generator=gen, device="cuda"))
    s["y"] = torch.zeros((*shape, case["width"]), dtype=dtype, device="cuda")
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s: dict) -> dict:
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


def _run_own(s: dict) -> dict:
    pplx, case = _package(), s["case"]
    op, e = case["op"], case["experts"]
    if op == "sort":
        got = pplx.sort_tokens(s["x"], s["indices"], e, s["bound_m"], int8=case["int8"])
        if not case["int8"]:
            return {"rows": got.rows, "slots": got.slots, "offsets": got.offsets}
        values = torch.mul(got.rows, got.scale[:, None], out=s["values"])
        return {"values": values, "scale": got.scale, "slots": got.slots, "offsets": got.offsets}
    if op == "unsort":
        return {"out": pplx.unsort_tokens(s["y"], s["slots"], s["offsets"], s["weights"], out=s["out"])}
    if op == "train":
        got = pplx.sort_tokens(s["x"], s["indices"], e, s["bound_m"])
        out = pplx.unsort_tokens(s["y"], got.slots, got.offsets, s["weights"])
        gx, gy, gw = torch.autograd.grad([got.rows, out], [s["x"], s["y"], s["weights"]], [s["grad_rows"], s["grad_out"]])
        return {"rows": got.rows, "out": out, "grad_x": gx, "grad_y": gy, "grad_weights": gw}
    rows = {name: s[name] for name in ("num_tokens", "offsets") if name in s}
    if op == "swiglu":
        q, scale = pplx.quantize_rows(s["x"], **rows, swiglu=True, out=(s["q"], s["scale"]))
        return {"values": torch.mul(q, scale[..., None], out=s["values"]), "scale": scale}
    return {"y": pplx.int8_matmul(s["x"], s["x_scale"], s["weight"], s["weight_scale"], **rows, out=s["y"])}


def _plain_routing(indices: torch.Tensor, experts: int, bound_m: torch.Tensor | None):
    """Slots [m, K], offsets [E + 1] and the pick of each row [P] (P where there is none)."""
    m, k = indices.shape
    ids = indices.view(torch.int32).to(torch.int64)
    live = (ids >= 0) & (ids < experts)
    if bound_m is not None:
        live = live & (torch.arange(m, device=ids.device) < bound_m.view(torch.int32))[:, None]
    key = torch.where(live, ids, experts).reshape(-1)
    order = torch.argsort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(m * k, device=ids.device)
    slots = torch.where(live, position.view(m, k), -1).to(torch.int32)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device).index_add_(0, key, torch.ones_like(key))
    pick = torch.where(key[order] < experts, order, m * k)
    return slots, _offsets(counts[:experts]), pick


def _plain_quantize(v: torch.Tensor):
    """fp32 rows to whole numbers of at most 127 and their scales."""
    largest = v.abs().amax(dim=-1).clamp_min(_TINY)
    return torch.round(v * (127.0 / largest)[..., None]), largest / 127.0


def _run_plain(s: dict) -> dict:
    case = s["case"]
    op, k, e = case["op"], case["topk"], case["experts"]
    if op in ("sort", "train"):
        slots, offsets, pick = _plain_routing(s["indices"], e, s["bound_m"])
        here = (pick < pick.numel())[:, None]
        token = torch.where(here[:, 0], pick, 0) // k
        if op == "sort" and case["int8"]:
            q, scale = _plain_quantize(s["x"].float())
            scale = torch.where(here[:, 0], scale[token], 0.0)
            values = torch.where(here, q[token], 0.0) * scale[:, None]
            return {"values": values.to(s["x"].dtype), "scale": scale, "slots": slots, "offsets": offsets}
        rows = torch.where(here, s["x"][token], 0)
        if op == "sort":
            return {"rows": rows, "slots": slots, "offsets": offsets}
        row = slots.clamp_min(0).to(torch.int64)
        live = slots >= 0
        weights = torch.where(live, s["weights"], 0.0)
        gathered = torch.where(live[:, :, None], s["y"][row].float(), 0.0)
        out = (gathered * weights[:, :, None]).sum(1).to(s["x"].dtype)
        grad_out = s["grad_out"].float()
        grad_weights = torch.where(live, (gathered * grad_out[:, None, :]).sum(2), 0.0)
        weight_of_row = torch.where(here[:, 0], weights.reshape(-1)[torch.where(here[:, 0], pick, 0)], 0.0)
        grad_y = (grad_out[token] * weight_of_row[:, None]).to(s["y"].dtype)
        grad_x = torch.where(live[:, :, None], s["grad_rows"][row].float(), 0.0).sum(1).to(s["x"].dtype)
        return {"rows": rows, "out": out, "grad_x": grad_x, "grad_y": grad_y, "grad_weights": grad_weights}
    if op == "unsort":
        live = s["slots"] >= 0
        gathered = torch.where(live[:, :, None], s["y"][s["slots"].clamp_min(0).to(torch.int64)].float(), 0.0)
        out = (gathered * torch.where(live, s["weights"], 0.0)[:, :, None]).sum(1)
        return {"out": out.to(s["out"].dtype)}
    if op == "swiglu":
        gate, up = s["x"].float().chunk(2, dim=-1)
        q, scale = _plain_quantize(gate / (1.0 + torch.exp(-gate)) * up)
        if case["form"] == "padded":
            there = torch.arange(scale.shape[1], device=scale.device) < s["num_tokens"][:, None]
            q, scale = torch.where(there[..., None], q, 0.0), torch.where(there, scale, 0.0)
        return {"values": (q * scale[..., None]).to(s["x"].dtype), "scale": scale}
    scales = s["weight_scale"]
    if case["form"] == "padded":
        sums = torch.bmm(s["x"].float(), s["weight"].float().transpose(1, 2).contiguous())
        y = sums * s["x_scale"][..., None] * scales[:, None, :]
        there = torch.arange(y.shape[1], device=y.device) < s["num_tokens"][:, None]
        return {"y": torch.where(there[..., None], y, 0.0).to(s["y"].dtype)}
    if case["form"] == "dense":
        sums = torch.mm(s["x"].float(), s["weight"].float().t())
        return {"y": (sums * s["x_scale"][:, None] * scales).to(s["y"].dtype)}
    offsets, y = s["offsets"].tolist(), s["y"]
    for expert in range(e):
        a, b = offsets[expert], offsets[expert + 1]
        if b > a:
            sums = torch.mm(s["x"][a:b].float(), s["weight"][expert].float().t())
            y[a:b] = (sums * s["x_scale"][a:b, None] * scales[expert]).to(y.dtype)
    return {"y": y}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_quantize(v: torch.Tensor):
    a = torch.maximum(v.abs().max(dim=-1, keepdim=True).values, torch.full((), _TINY, dtype=torch.float64, device=v.device))
    return torch.round(v * 127.0 / a) * (a / 127.0), (a / 127.0).squeeze(-1)


def exact(case: dict, seed: int) -> dict:
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_step(case, s) if case["op"] in ("sort", "unsort", "train") else _exact_rows(case, s)


def _exact_step(case: dict, s: dict) -> dict:
    """Expert by expert and pick by pick, in the order of the definition."""
    op, m, k, e, h = case["op"], case["tokens"], case["topk"], case["experts"], case["hidden"]
    ids = s["indices"].view(torch.int32).cpu().long()
    ids[_present(case):] = -1
    token = torch.cat([torch.nonzero((ids == expert).any(1))[:, 0] for expert in range(e)]).cuda()
    expert_of = torch.cat([torch.full((int((ids == expert).sum()),), expert) for expert in range(e)]).cuda()
    pick = (ids.cuda()[token] == expert_of[:, None]).long().argmax(1)  # (a token's picks are distinct)
    n, f64 = token.numel(), torch.float64
    weight = s["weights"].to(f64)[token, pick]
    got: dict = {}
    if op != "unsort":
        rows = torch.zeros(m * k, h, dtype=f64, device="cuda")
        if op == "sort" and case["int8"]:
            values, scale = _exact_quantize(s["x"].to(f64))
            rows[:n] = values[token]
            scales = torch.zeros(m * k, dtype=f64, device="cuda")
            scales[:n] = scale[token]
            return {"values": rows, "scale": scales, "slots": None, "offsets": None}
        rows[:n] = s["x"].to(f64)[token]
        if op == "sort":
            return {"rows": rows, "slots": None, "offsets": None}
        got["rows"] = rows
    out = torch.zeros(m, h, dtype=f64, device="cuda")
    got["out"] = out.index_add_(0, token, s["y"][:n].to(f64) * weight[:, None])
    if op == "train":
        grad_x = torch.zeros(m, h, dtype=f64, device="cuda")
        got["grad_x"] = grad_x.index_add_(0, token, s["grad_rows"][:n].to(f64))
        got["grad_y"] = torch.zeros(m * k, h, dtype=f64, device="cuda")
        got["grad_weights"] = torch.zeros(m, k, dtype=f64, device="cuda")
        for a in range(0, n, 1 << 14):  # (a piece at a time: 8 bytes an element)
            t, p, g = token[a : a + (1 << 14)], pick[a : a + (1 << 14)], s["grad_out"].to(f64)
            got["grad_y"][a : a + t.numel()] = g[t] * weight[a : a + t.numel(), None]
            got["grad_weights"][t, p] = (g[t] * s["y"][a : a + t.numel()].to(f64)).sum(1)
    return got


def _exact_rows(case: dict, s: dict) -> dict:
    op, f64 = case["op"], torch.float64
    if case["form"] == "padded":
        spans = [((i, slice(0, n)), i) for i, n in enumerate(s["num_tokens"].tolist())]
    elif case["form"] == "sorted":
        ends = s["offsets"].tolist()
        spans = [((slice(a, b),), i) for i, (a, b) in enumerate(zip(ends, ends[1:]))]
    else:
        spans = [((slice(0, case["tokens"]),), None)]
    if op == "swiglu":
        values = torch.zeros(s["values"].shape, dtype=f64, device="cuda")
        scale = torch.zeros(s["scale"].shape, dtype=f64, device="cuda")
        for at, _ in spans:
            x = s["x"][at].to(f64)
            if x.shape[0]:
                gate, up = x[:, : case["width"]], x[:, case["width"] :]
                values[at], scale[at] = _exact_quantize(gate * torch.sigmoid(gate) * up)
        return {"values": values, "scale": scale}
    y = torch.zeros(s["y"].shape, dtype=f64, device="cuda")
    for at, expert in spans:
        weight = s["weight"] if expert is None else s["weight"][expert]
        scale = s["weight_scale"] if expert is None else s["weight_scale"][expert]
        x = s["x"][at].to(f64)
        if x.shape[0]:
            y[at] = (x * s["x_scale"][at].to(f64)[:, None]) @ (weight.to(f64) * scale.to(f64)[:, None]).t()
    return {"y": y}
