"""The measured cases of the operators before dispatch: the norm whose rows are sent, in 8 bits where asked to, the router's
product, the choice of experts with its weights, and the gradients of all three.

Fields of a case:
  op        "norm"          root-mean-square norm of rows, with the residual's addition and the rows in 8 bits where asked to
            "norm-train"    the norm with the residual's addition, and its gradients
            "logits"        the router's product, in fp32
            "logits-train"  the same and its gradients
            "route"         each token's experts and their weights
            "route-train"   the same and the gradient of the logits
  tokens, hidden, experts, topk   the step
  type      of the rows, and of the logits of "route"
  weight    "same": the norm's and the router's weights have the rows' type; "f32"
  add       whether "norm" adds a residual
  quantize  "none", "int8" (one scale a row) or "fp8" (e4m3, one scale for each 128 columns)
  scores    "softmax" or "sigmoid"
  bias      whether a bias for balance takes part in the choice
  groups, top_groups, group_top   experts come from the top_groups groups whose best group_top experts have the largest sums
  renormalize, scale              of the weights
  masked    share of a token's experts that are not there (logits of -inf)
  present   "full": all tokens are there; "ragged": a count in device memory says how many
"""

from __future__ import annotations

import os
import sys

import torch

own = False  # False: plain forms out of elementary torch operations; True: the framework's kernels

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_CODES = {"none": None, "int8": torch.int8, "fp8": torch.float8_e4m3fn}
_TINY = 2.0**-100  # what is quantised with a largest value below this is quantised as if it were this
_EPS = 1e-6
_BLOCK = 128


def _package():
    """The package, which lives in a folder of the repository that is the working directory."""
    folder = os.path.join(os.getcwd(), "pplx-kernels_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import pplx_kernels

    return pplx_kernels


def listed() -> list[dict]:
    return [
        # One decoded token in the smaller of the two model shapes of the latency table: latency.
        _norm("norm-decode-1", tokens=1, hidden=2048),
        # A chunk of a prefill, sent as int8 rows.
        _norm("norm-add-int8-509", tokens=509, hidden=7168, add=True, quantize="int8"),
        # The largest batch of one rank, sent as fp8 rows with block scales, which is how the benchmark's rows come.
        _norm("norm-add-fp8-8192", tokens=8192, hidden=7168, add=True, quantize="fp8"),
        # Training: a micro-batch of odd sizes in half precision.
        _norm_train("norm-train-f16-3001", tokens=3001, hidden=2880, type="f16"),
        # Training: weights kept in fp32.
        _norm_train("norm-train-8192", tokens=8192, hidden=4096, weight="f32"),
        # The router of a decode step of four tokens, small shape: latency.
        _logits("logits-decode-4", tokens=4, experts=64, hidden=2048),
        # Decode with a batch of 64, router kept in fp32: the weights' bytes count.
        _logits("logits-decode-64", tokens=64, experts=256, hidden=7168, weight="f32"),
        # The largest batch of one rank: the rows' bytes count, and the operations.
        _logits("logits-prefill-8192", tokens=8192, experts=256, hidden=7168),
        # Training: a micro-batch of odd length with both gradients.
        _logits_train("logits-train-3001", tokens=3001, experts=256, hidden=7168),
        # Decode with a batch of 64: sigmoid scores, a bias for balance, four of eight groups, renormalised weights.
        _route("route-decode-64", tokens=64, experts=256, topk=8, scores="sigmoid", bias=True, groups=8, top_groups=4, scale=2.5),
        # The largest batch of one rank, ragged: softmax, some experts switched off, weights as they are.
        _route("route-prefill-8192", tokens=8192, experts=256, topk=8, renormalize=False, masked=0.1, present="ragged"),
        # Training: softmax over 256 experts with the gradient of all logits.
        _route_train("route-train-16384", tokens=16384, experts=256, topk=8, renormalize=False),
    ]  # fmt: skip


def _case(op, name, **fields) -> dict:
    return {"name": name, "op": op, **fields} if name else {"op": op, **fields}


def _norm(name="", **fields) -> dict:
    return _case("norm", name, **{"type": "bf16", "weight": "same", "add": False, "quantize": "none", **fields})


def _norm_train(name="", **fields) -> dict:
    return _case("norm-train", name, **{"type": "bf16", "weight": "same", **fields})


def _logits(name="", **fields) -> dict:
    return _case("logits", name, **{"type": "bf16", "weight": "same", **fields})


def _logits_train(name="", **fields) -> dict:
    return _case("logits-train", name, **{"type": "bf16", "weight": "same", **fields})


_ROUTE = dict(
    type="f32", scores="softmax", bias=False, groups=1, top_groups=1, group_top=2, renormalize=True, scale=1.0, masked=0.0,
    present="full",
)  # fmt: skip


def _route(name="", **fields) -> dict:
    return _case("route", name, **{**_ROUTE, **fields})


def _route_train(name="", **fields) -> dict:
    return _case("route-train", name, **{**_ROUTE, **fields})


def _log_uniform(rng, low: int, high: int) -> int:
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng) -> dict:
    """One more case: sizes spread over their logarithm, types and forms at random, no dearer than the dearest listed case of its
    operator."""
    while True:
        op = rng.choice(["norm", "norm-train", "logits", "logits-train", "route", "route", "route-train"])
        step: dict = dict(tokens=_log_uniform(rng, 1, 16384))
        if op.startswith("norm"):
            step.update(type=rng.choice(["bf16", "bf16", "f16", "f32"]), weight=rng.choice(["same", "f32"]))
            if op == "norm":
                # (16-byte multiples of 16-bit elements; quantised rows are multiples of 16 elements)
                quantize = rng.choice(["none", "int8", "fp8"])
                unit = 8 if quantize == "none" else 16
                step.update(hidden=unit * _log_uniform(rng, 256 // unit, 16384 // unit), add=rng.random() < 0.7, quantize=quantize)
                case = _norm(**step)
            else:
                case = _norm_train(**step, hidden=8 * _log_uniform(rng, 32, 2048))
        elif op.startswith("logits"):
            step.update(type=rng.choice(["bf16", "bf16", "f16", "f32"]), weight=rng.choice(["same", "same", "f32"]))
            step.update(experts=_log_uniform(rng, 4, 512), hidden=8 * _log_uniform(rng, 32, 1024))
            case = _logits(**step) if op == "logits" else _logits_train(**step)
        else:
            per_group, groups = 1, 1
            if rng.random() < 0.4:
                groups = rng.choice([2, 4, 8])
                per_group = _log_uniform(rng, 2, 512 // groups)
            else:
                per_group = _log_uniform(rng, 4, 512)
            top_groups = rng.randint(1, groups)
            step.update(
                experts=groups * per_group, topk=min(rng.randint(1, 10), top_groups * per_group), groups=groups,
                top_groups=top_groups, group_top=rng.choice([1, 2]), type=rng.choice(["f32", "f32", "bf16", "f16"]),
                scores=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, renormalize=rng.random() < 0.6,
                scale=rng.choice([1.0, 2.5]), masked=rng.choice([0.0, 0.0, 0.1, 0.9]), present=rng.choice(["full", "ragged"]),
            )  # fmt: skip
            case = _route(**step) if op == "route" else _route_train(**step)
        if _cost(case) <= max(_cost(c) for c in listed() if c["op"] == op):
            return case


# ---------------------------------------------------------------------------
# Sizes
# ---------------------------------------------------------------------------
def _present(case: dict) -> int:
    return case["tokens"] if case["present"] == "full" else max(1, case["tokens"] * 7 // 8)


def _cost(case: dict) -> float:
    w = work(case)
    products = {"f32": 6.0, "f16": 3.0, "bf16": 1.5}[case["type"]] if case["op"].startswith("logits") else 1.0
    return w["bytes"] / 5e12 + products * w["flops"] / 1e15


def work(case: dict) -> dict:
    """Bytes: every input is read once and every output written once.  Flops: multiply-adds of the products, some ten operations
    an element elsewhere."""
    op, m, size = case["op"], case["tokens"], _DTYPES[case["type"]].itemsize
    if op.startswith("norm"):
        h = case["hidden"]
        weight = h * (4 if case["weight"] == "f32" else size)
        if op == "norm":
            sent = {"none": 0, "int8": h + 4, "fp8": h + 4 * -(-h // _BLOCK)}[case["quantize"]]
            return {"bytes": m * (h * size * (4 if case["add"] else 2) + sent) + weight, "flops": 6 * m * h}
        return {"bytes": m * h * size * (4 + 4) + 3 * weight, "flops": 16 * m * h}  # (both passes; x and residual share a gradient)
    if op.startswith("logits"):
        h, e = case["hidden"], case["experts"]
        weight = e * h * (4 if case["weight"] == "f32" else size)
        forward = {"bytes": m * h * size + weight + 4 * m * e, "flops": 2 * m * h * e}
        if op == "logits":
            return forward
        backward = 4 * m * e + 2 * m * h * size + 2 * weight
        return {"bytes": forward["bytes"] + backward, "flops": 3 * forward["flops"]}
    e, picks = case["experts"], m * case["topk"]
    forward = _present(case) * e * size + 8 * picks + (4 * e if case["bias"] else 0)
    if op == "route":
        return {"bytes": forward, "flops": 8 * m * e}
    return {"bytes": forward + 8 * picks + _present(case) * e * size + m * e * size, "flops": 16 * m * e}


# ---------------------------------------------------------------------------
# What a program has in hand
# ---------------------------------------------------------------------------
def _activations(shape: tuple, dtype: torch.dtype, gen: torch.Generator) -> torch.Tensor:
    """Normal values, whose size differs from row to row, with a few columns of large ones."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn((*shape[:-1], 1), generator=gen, device="cuda"))
    x *= torch.where(torch.rand(shape[-1], generator=gen, device="cuda") < 0.005, 6.0, 1.0)
    return x.to(dtype)


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, m, dtype = case["op"], case["tokens"], _DTYPES[case["type"]]
    s: dict = {"case": case}

    def normal(*shape, size=1.0) -> torch.Tensor:
        return size * torch.randn(shape, generator=gen, device="cuda")

    if op.startswith("norm"):
        h = case["hidden"]
        s["x"] = _activations((m, h), dtype, gen)
        s["weight"] = (1.0 + normal(h, size=0.1)).to(torch.float32 if case["weight"] == "f32" else dtype)
        s["residual"] = _activations((m, h), dtype, gen) if op == "norm-train" or case["add"] else None
        if op == "norm-train":
            s["grad_y"] = normal(m, h, size=1e-2).to(dtype)
            s["grad_sum"] = normal(m, h, size=1e-2).to(dtype)
            for leaf in ("x", "weight", "residual"):
                s[leaf].requires_grad_(True)
        elif case["quantize"] != "none":
            s["values"] = torch.empty(m, h, dtype=dtype, device="cuda")
        return s
    if op.startswith("logits"):
        h, e = case["hidden"], case["experts"]
        s["x"] = _activations((m, h), dtype, gen)
        s["weight"] = normal(e, h, size=h**-0.5).to(torch.float32 if case["weight"] == "f32" else dtype)
        if op == "logits-train":
            s["grad_logits"] = normal(m, e, size=1e-3)
            for leaf in ("x", "weight"):
                s[leaf].requires_grad_(True)
        return s
    e, k = case["experts"], case["topk"]
    # (some experts are liked by most tokens; which ones differs from seed to seed)
    logits = normal(m, e, size=1.5) + normal(e, size=0.7)
    if case["masked"]:
        logits.masked_fill_(torch.rand(m, e, generator=gen, device="cuda") < case["masked"], float("-inf"))
    s["logits"] = logits.to(dtype)
    s["bias"] = normal(e, size=0.1) if case["bias"] else None
    bound = torch.full((1,), _present(case), dtype=torch.int32, device="cuda")
    s["bound_m"] = bound.view(torch.uint32) if case["present"] == "ragged" else None
    if op == "route-train":
        s["grad_weights"] = normal(m, k, size=1e-2)
        s["logits"].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s: dict) -> dict:
    if own:
        return _run_own(s)
    with torch.no_grad():
        op = s["case"]["op"]
        return _plain_norm(s) if op.startswith("norm") else _plain_logits(s) if op.startswith("logits") else _plain_route(s)


def _run_own(s: dict) -> dict:
    pplx, case = _package(), s["case"]
    op = case["op"]
    if op == "norm":
        got = pplx.rms_norm(s["x"], s["weight"], s["residual"], eps=_EPS, quantize=_CODES[case["quantize"]])
        out = {"y": got.y}
        if case["add"]:
            out["sum"] = got.sum
        if case["quantize"] == "int8":
            out["values"] = torch.mul(got.q, got.scale[:, None], out=s["values"])
        elif case["quantize"] == "fp8":
            _blocks_of(got.q.to(s["values"].dtype), got.scale, out=s["values"])
            out["values"] = s["values"]
        return out if case["quantize"] == "none" else {**out, "scale": got.scale}
    if op == "norm-train":
        got = pplx.rms_norm(s["x"], s["weight"], s["residual"], eps=_EPS)
        leaves = [s["x"], s["residual"], s["weight"]]
        gx, gr, gw = torch.autograd.grad([got.y, got.sum], leaves, [s["grad_y"], s["grad_sum"]])
        return {"y": got.y, "sum": got.sum, "grad_x": gx, "grad_residual": gr, "grad_weight": gw}
    if op.startswith("logits"):
        logits = pplx.router_logits(s["x"], s["weight"])
        if op == "logits":
            return {"logits": logits}
        gx, gw = torch.autograd.grad(logits, [s["x"], s["weight"]], s["grad_logits"])
        return {"logits": logits, "grad_x": gx, "grad_weight": gw}
    indices, weights = pplx.route_tokens(
        s["logits"], case["topk"], bias=s["bias"], scores=case["scores"], num_groups=case["groups"], top_groups=case["top_groups"],
        group_top=case["group_top"], renormalize=case["renormalize"], scale=case["scale"], bound_m=s["bound_m"],
    )  # fmt: skip
    out = {"indices": indices.view(torch.int32), "weights": weights}
    if op == "route-train":
        (out["grad_logits"],) = torch.autograd.grad(weights, s["logits"], s["grad_weights"])
    return out


def _blocks_of(q: torch.Tensor, scale: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """[m, H] times [m, ceil(H / 128)], each for its 128 columns."""
    if q.shape[1] % _BLOCK:
        return torch.mul(q, scale.repeat_interleave(_BLOCK, dim=1)[:, : q.shape[1]], out=out)
    shape = (q.shape[0], -1, _BLOCK)
    product = torch.mul(q.view(shape), scale[:, :, None], out=None if out is None else out.view(shape))
    return product.view(q.shape)


def _plain_norm(s: dict) -> dict:
    case, dtype = s["case"], s["x"].dtype
    h = s["x"].float() if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(dtype).float()
    r = torch.rsqrt(h.square().mean(dim=1, keepdim=True) + _EPS)
    weight = s["weight"].float()
    v = h * r * weight
    out = {"y": v.to(dtype)}
    if s["residual"] is not None:
        out["sum"] = h.to(dtype)
    if case["op"] == "norm-train":
        normed, grad = h * r, s["grad_y"].float()
        g = grad * weight
        grad_h = r * (g - normed * (g * normed).mean(dim=1, keepdim=True)) + s["grad_sum"].float()
        grad_weight = (grad * normed).sum(dim=0).to(s["weight"].dtype)
        return {**out, "grad_x": grad_h.to(dtype), "grad_residual": grad_h.to(dtype), "grad_weight": grad_weight}
    if case["quantize"] == "int8":
        largest = v.abs().amax(dim=1).clamp_min(_TINY)
        scale = largest / 127.0
        out["values"] = (torch.round(v * (127.0 / largest)[:, None]) * scale[:, None]).to(dtype)
        out["scale"] = scale
    elif case["quantize"] == "fp8":
        short = -v.shape[1] % _BLOCK
        padded = torch.cat([v, v.new_zeros(v.shape[0], short)], dim=1) if short else v
        largest = padded.view(v.shape[0], -1, _BLOCK).abs().amax(dim=2).clamp_min(_TINY)
        scale = largest / 448.0
        q = _blocks_of(v, 448.0 / largest).to(torch.float8_e4m3fn)
        out["values"] = _blocks_of(q.float(), scale).to(dtype)
        out["scale"] = scale
    return out


def _plain_logits(s: dict) -> dict:
    x, weight = s["x"].float(), s["weight"].float()
    out = {"logits": torch.mm(x, weight.t())}
    if s["case"]["op"] == "logits-train":
        out["grad_x"] = torch.mm(s["grad_logits"], weight).to(s["x"].dtype)
        out["grad_weight"] = torch.mm(s["grad_logits"].t(), x).to(s["weight"].dtype)
    return out


def _plain_route(s: dict) -> dict:
    """In 64 bits: two experts may lie next to each other."""
    case, lowest = s["case"], float("-inf")
    logits = s["logits"].double()
    m, e = logits.shape
    k, groups = case["topk"], case["groups"]
    if case["scores"] == "softmax":
        shifted = torch.exp(logits - logits.amax(dim=1, keepdim=True))  # (NaN where nothing is there)
        total = shifted.sum(dim=1, keepdim=True)
        scores = torch.where(total > 0, shifted / total, 0.0)
    else:
        scores = 1.0 / (1.0 + torch.exp(-logits))
    live = logits > lowest
    if s["bound_m"] is not None:
        live = live & (torch.arange(m, device=live.device) < s["bound_m"].view(torch.int32))[:, None]
    biased = scores if s["bias"] is None else scores + s["bias"].double()
    # (without a bias the logits have the scores' order)
    keys = torch.where(live, logits if s["bias"] is None else biased, lowest)
    if case["top_groups"] < groups:
        by_group = torch.where(live, biased, lowest).view(m, groups, -1)
        best = by_group.sort(dim=2, descending=True).values[:, :, : case["group_top"]].sum(dim=2)
        chosen = best.sort(dim=1, descending=True, stable=True).indices[:, : case["top_groups"]]
        group_live = torch.zeros(m, groups, dtype=torch.bool, device=live.device).scatter_(1, chosen, True)
        keys = torch.where(group_live.repeat_interleave(e // groups, dim=1), keys, lowest)
    ordered, order = keys.sort(dim=1, descending=True, stable=True)
    there = ordered[:, :k] > lowest
    picks = order[:, :k]
    picked = torch.where(there, scores.gather(1, picks), 0.0)
    total = picked.sum(dim=1, keepdim=True)
    weights = torch.where(there, picked / total, 0.0) if case["renormalize"] else picked
    weights = weights * case["scale"]
    out = {"indices": torch.where(there, picks, e).to(torch.int32), "weights": weights.float()}
    if case["op"] == "route-train":
        g = torch.where(there, s["grad_weights"].double(), 0.0)
        inner = (g * weights).sum(dim=1, keepdim=True)
        if case["renormalize"]:
            grad = weights * (g - inner / case["scale"])
        else:
            grad = weights * g
        if case["scores"] == "sigmoid":
            grad = grad * (1.0 - picked)
        grad_logits = torch.zeros_like(logits).scatter_add_(1, picks, torch.where(there, grad, 0.0))
        if case["scores"] == "softmax" and not case["renormalize"]:
            grad_logits = grad_logits - torch.where(live, scores, 0.0) * inner
        out["grad_logits"] = grad_logits.to(s["logits"].dtype)
    return out


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case: dict, seed: int) -> dict:
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"].startswith("norm"):
            return _exact_norm(case, s)
        return _exact_logits(case, s) if case["op"].startswith("logits") else _exact_route(case, s)


def _e4m3(v: torch.Tensor) -> torch.Tensor:
    """The nearest values that four bits of exponent and three of mantissa stand for."""
    exponent = torch.frexp(v.abs()).exponent.clamp_min(-5).double()  # v = f * 2^exponent, 0.5 <= f < 1
    step = torch.exp2(exponent - 4.0)
    return torch.round(v / step) * step


def _exact_norm(case: dict, s: dict) -> dict:
    f64, dtype, width = torch.float64, s["x"].dtype, case["hidden"]
    names = ["y"] + (["sum"] if s["residual"] is not None else [])
    got: dict = {name: [] for name in names}
    grad_weight = torch.zeros(width, dtype=f64, device="cuda")
    for a in range(0, case["tokens"], 1024):  # (a piece at a time: 8 bytes an element)
        rows = slice(a, a + 1024)
        total = s["x"][rows].to(f64)
        if s["residual"] is not None:
            total = total + s["residual"][rows].to(f64)
            got["sum"].append(total)
            total = total.to(dtype).to(f64)  # (the norm is that of the sum as it is kept)
        length = torch.linalg.vector_norm(total, dim=1, keepdim=True)
        unit = total / torch.sqrt(length**2 / width + _EPS)
        v = unit * s["weight"].to(f64)
        got["y"].append(v)
        if case["op"] == "norm-train":
            g = s["grad_y"][rows].to(f64)
            grad_weight += torch.einsum("th,th->h", g, unit)
            along = torch.einsum("th,th->t", g * s["weight"].to(f64), unit)[:, None] / width
            grad = (g * s["weight"].to(f64) - unit * along) / torch.sqrt(length**2 / width + _EPS) + s["grad_sum"][rows].to(f64)
            got.setdefault("grad_x", []).append(grad)
            got.setdefault("grad_residual", []).append(grad)
        elif case["quantize"] == "int8":
            top = torch.clamp(v.abs().max(dim=1, keepdim=True).values, min=_TINY)
            got.setdefault("values", []).append(torch.round(127.0 * v / top) * top / 127.0)
            got.setdefault("scale", []).append(top[:, 0] / 127.0)
        elif case["quantize"] == "fp8":
            values, scales = [], []
            for part in v.split(_BLOCK, dim=1):
                top = torch.clamp(part.abs().max(dim=1, keepdim=True).values, min=_TINY)
                values.append(_e4m3(448.0 * part / top) * top / 448.0)
                scales.append(top / 448.0)
            got.setdefault("values", []).append(torch.cat(values, dim=1))
            got.setdefault("scale", []).append(torch.cat(scales, dim=1))
    out = {name: torch.cat(parts) for name, parts in got.items()}
    if case["op"] == "norm-train":
        out["grad_weight"] = grad_weight
    return out


def _exact_logits(case: dict, s: dict) -> dict:
    f64 = torch.float64
    weight = s["weight"].to(f64).t().contiguous()
    out = {"logits": torch.cat([part.to(f64) @ weight for part in s["x"].split(2048)])}
    if case["op"] == "logits-train":
        grad = s["grad_logits"].to(f64)
        out["grad_x"] = (weight @ grad.t().contiguous()).t().contiguous()
        out["grad_weight"] = (s["x"].to(f64).t().contiguous() @ grad).t().contiguous()
    return out


def _exact_route(case: dict, s: dict) -> dict:
    """Pick by pick, each the first of the largest keys that are left."""
    f64, lowest = torch.float64, float("-inf")
    logits, e, m, there = s["logits"].detach().to(f64), case["experts"], case["tokens"], _present(case)
    scores = torch.softmax(logits, dim=1).nan_to_num(0.0) if case["scores"] == "softmax" else torch.sigmoid(logits)
    chance = scores + (s["bias"].to(f64) if case["bias"] else 0.0)
    chance[logits == lowest] = lowest
    keys = chance.clone() if case["bias"] else logits.clone()
    ids = torch.arange(e, device="cuda")
    if case["top_groups"] < case["groups"]:
        parts = chance.view(m, case["groups"], -1)
        rank = parts.topk(case["group_top"], dim=2).values.sum(dim=2)
        out_of = torch.ones_like(rank, dtype=torch.bool)
        group_ids = torch.arange(case["groups"], device="cuda")
        for _ in range(case["top_groups"]):
            open_rank = torch.where(out_of, rank, float("nan"))
            best = open_rank.nan_to_num(lowest, neginf=lowest).amax(dim=1, keepdim=True)
            first = torch.where(out_of & (rank == best), group_ids, e).amin(dim=1, keepdim=True)
            out_of &= group_ids != first
        keys[out_of.repeat_interleave(e // case["groups"], dim=1)] = lowest
    keys[there:] = lowest
    picked = torch.zeros(m, case["topk"], dtype=f64, device="cuda")
    index = torch.full((m, case["topk"]), e, device="cuda")
    for k in range(case["topk"]):
        best = keys.amax(dim=1, keepdim=True)
        first = torch.where((keys == best) & (keys > lowest), ids, e).amin(dim=1, keepdim=True)
        index[:, k] = first[:, 0]
        picked[:, k] = torch.cat([scores, scores.new_zeros(m, 1)], dim=1).gather(1, first)[:, 0]
        keys[ids == first] = lowest
    total = picked.sum(dim=1, keepdim=True)
    share = (picked / total.where(total > 0, 1.0) if case["renormalize"] else picked) * case["scale"]
    out = {"indices": None, "weights": share}
    if case["op"] == "route-train":
        # (by the Jacobian of the weights in the picks' scores, then that of the scores in the logits)
        g = s["grad_weights"].to(f64) * (index < e) * case["scale"]
        if case["renormalize"]:
            safe = total.where(total > 0, 1.0)
            g = (g - (g * picked).sum(dim=1, keepdim=True) / safe) / safe * (index < e)
        to_scores = torch.zeros(m, e + 1, dtype=f64, device="cuda").scatter_add_(1, index, g)[:, :e]
        if case["scores"] == "softmax":
            out["grad_logits"] = scores * (to_scores - (to_scores * scores).sum(dim=1, keepdim=True))
        else:
            out["grad_logits"] = scores * (1.0 - scores) * to_scores
    return out
