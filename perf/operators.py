"""Measured cases of the 8-bit linear path: one scale per token for activations, one per channel for weights.

Three operators, each in a plain form (elementary torch operations) and as the calls of hearth_b200.api:

  norm    h = x + r;  t = weight * h;  q = rint(t * 127 / max|t|);  scale = max|t| / 127 / sqrt(mean(h^2) + eps)
          outputs h and the values q * scale
  silu    v = g / (1 + exp(-g)) * u, quantized per token; outputs the values q * scale
  matmul  x quantized per token, times int8 weights with a scale per row; outputs f32 [tokens, rows]

The 8-bit rows that norm and silu leave in an activation handle are returned as the f32 values they stand for.
What is rounded to 8 bits is an f32 number, and so is what it is multiplied by: h, t, v, 127 / max and the product with
it are each rounded to f32 (as in the Q8_0 quantizer beside them), so the whole numbers are determined to the last one.
"""
import math

import torch

own = False

EPS = 1e-6
SMALLEST = 2.0 ** -100  # a row whose largest magnitude is below this is stored as zeros


def listed():
    return [
        # the norm in front of a projection, one token of an 8B-sized model: latency
        {"name": "norm 1x4096", "op": "norm", "tokens": 1, "cols": 4096},
        # a ragged decode batch at the 27B width
        {"name": "norm 37x5120", "op": "norm", "tokens": 37, "cols": 5120},
        # a long prompt
        {"name": "norm 4096x4096", "op": "norm", "tokens": 4096, "cols": 4096},
        # the input of the down projection, one token
        {"name": "silu 1x12288", "op": "silu", "tokens": 1, "cols": 12288, "packed": True},
        # the same for a prompt; gate and up are the halves of one buffer, as one product of both leaves them
        {"name": "silu 512x17408", "op": "silu", "tokens": 512, "cols": 17408, "packed": True},
        # one token through a square projection: the smallest product
        {"name": "matmul 1x4096x4096", "op": "matmul", "tokens": 1, "cols": 4096, "rows": 4096},
        # one token through the output head (an odd number of rows)
        {"name": "matmul 1x2048x151669", "op": "matmul", "tokens": 1, "cols": 2048, "rows": 151669},
        # a few tokens through gate and up together
        {"name": "matmul 4x5120x34816", "op": "matmul", "tokens": 4, "cols": 5120, "rows": 34816},
        # batched decode through the down projection
        {"name": "matmul 32x17408x5120", "op": "matmul", "tokens": 32, "cols": 17408, "rows": 5120},
        # an odd-sized short prompt
        {"name": "matmul 77x12288x4096", "op": "matmul", "tokens": 77, "cols": 12288, "rows": 4096},
        # a prompt of 512 tokens through gate and up
        {"name": "matmul 512x4096x24576", "op": "matmul", "tokens": 512, "cols": 4096, "rows": 24576},
        # a long prompt: bound by the tensor cores
        {"name": "matmul 4096x5120x17408", "op": "matmul", "tokens": 4096, "cols": 5120, "rows": 17408},
    ]


def _spread(rng, low, high):
    """An integer of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "silu", "matmul", "matmul"])
    if op == "norm":
        cols = _spread(rng, 33, 16384)
        return {"op": op, "tokens": _spread(rng, 1, max(1, min(8192, (4096 * 4096) // cols))), "cols": cols}
    if op == "silu":
        cols = _spread(rng, 33, 20480)
        return {"op": op, "tokens": _spread(rng, 1, max(1, min(8192, (512 * 17408) // cols))), "cols": cols, "packed": rng.random() < 0.5}
    cols = _spread(rng, 40, 17408)
    rows = _spread(rng, 17, 34816)
    tokens = _spread(rng, 1, 4096)
    return {"op": op, "tokens": max(1, min(tokens, (4096 * 5120 * 17408) // (cols * rows))), "cols": cols, "rows": rows}


class _Held:
    """The handles a program keeps between calls, freed with the state."""

    def __init__(self, act, weight=None):
        self.act, self.weight = act, weight

    def __del__(self):
        for h in (self.act, self.weight):
            if h is not None:
                h.free()


def _inputs(case, seed):
    """Inputs from the seed alone: activations with a few outlying channels, as residual streams have them, weights that
    use the 8 bits the way a bell-shaped channel does."""
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    m, k = case["tokens"], case["cols"]

    def rows(spread, outlier=8.0):
        channel = torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, outlier, 1.0)
        return torch.randn(m, k, device="cuda", generator=g) * channel * spread

    if case["op"] == "norm":
        return {"x": rows(0.5), "residual": rows(2.0), "weight": 1.0 + 0.3 * torch.randn(k, device="cuda", generator=g)}
    if case["op"] == "silu":
        if case["packed"]:
            both = torch.cat([rows(1.5, 1.0), rows(1.0, 2.0)], dim=1)
            return {"gate": both[:, :k], "up": both[:, k:]}
        return {"gate": rows(1.5, 1.0), "up": rows(1.0, 2.0)}
    n = case["rows"]
    q = torch.empty(n, k, dtype=torch.int8, device="cuda")
    step = max(1, (1 << 26) // k)
    for i in range(0, n, step):
        part = torch.randn(min(step, n - i), k, device="cuda", generator=g)
        q[i:i + step] = (part * 36.0).round_().clamp_(-127, 127).to(torch.int8)
    scales = torch.rand(n, device="cuda", generator=g) * 1e-3 + 2e-4
    return {"x": rows(1.0), "q": q, "scales": scales}


def prepare(case, seed):
    state = {"case": case, **_inputs(case, seed)}
    if own:
        from hearth_b200 import api
        api.init(0)
        m, k = case["tokens"], case["cols"]
        weight = None
        if case["op"] == "matmul":
            weight = api.WeightI8.upload_dev(state.pop("q"), state.pop("scales"))
            state["out"] = torch.empty(m, case["rows"], device="cuda")
        else:
            state["values"] = torch.empty(m, k, device="cuda")
            state["sum"] = torch.empty(m, k, device="cuda")
        state["held"] = _Held(api.ActI8(m, k), weight)
    return state


def _quantized(v):
    """Rows of f32 -> whole numbers of -127 .. 127 (as f32) and a scale per row."""
    top = v.abs().amax(dim=1, keepdim=True)
    full = torch.full_like(top, 127.0)
    q = torch.where(top >= SMALLEST, v * (full / top), 0.0).round()
    return q, torch.where(top >= SMALLEST, top / full, 0.0)


def run(state):
    case = state["case"]
    m = case["tokens"]
    if own:
        from hearth_b200 import api
        act = state["held"].act
        if case["op"] == "norm":
            act.add_rms_norm(state["x"], state["weight"], EPS, m, residual_dev=state["residual"], sum_dev=state["sum"])
            act.dequantize(state["values"], m)
            return {"sum": state["sum"], "values": state["values"]}
        if case["op"] == "silu":
            act.silu_mul(state["gate"], state["up"], m)
            act.dequantize(state["values"], m)
            return {"values": state["values"]}
        act.quantize(state["x"], m)
        api.matmul_i8_dev(state["held"].weight, act, m, state["out"])
        return {"out": state["out"]}
    if case["op"] == "norm":
        h = state["x"] + state["residual"]
        q, scale = _quantized(h * state["weight"])
        factor = 1.0 / torch.sqrt((h * h).mean(dim=1, keepdim=True) + EPS)
        return {"sum": h, "values": q * (scale * factor)}
    if case["op"] == "silu":
        g = state["gate"]
        q, scale = _quantized(g / (1.0 + torch.exp(-g)) * state["up"])
        return {"values": q * scale}
    q, scale = _quantized(state["x"])
    return {"out": (q @ state["q"].float().t()) * state["scales"] * scale}


def work(case):
    m, k = case["tokens"], case["cols"]
    if case["op"] == "norm":  # x, r read; h and the values written; the weight read
        return {"bytes": 16 * m * k + 4 * k, "flops": 8 * m * k}
    if case["op"] == "silu":
        return {"bytes": 12 * m * k, "flops": 8 * m * k}
    n = case["rows"]
    return {"bytes": 4 * m * k + n * k + 4 * n + 4 * m * n, "flops": 2 * m * n * k}


def exact(case, seed):
    given = _inputs(case, seed)

    def rounded(v, single):
        """Whole numbers and steps of the rows `v` (f64).  A quotient within 1e-5 of a border between two whole numbers
        goes where f32 arithmetic puts it (`single`: v in f32), since the definition rounds f32 numbers."""
        top = v.abs().max(dim=1, keepdim=True).values
        live = top >= SMALLEST
        r = torch.where(live, v * 127 / torch.where(live, top, 1.0), 0.0)
        border = ((r - r.floor()) - 0.5).abs() < 1e-5 * (1 + r.abs())
        top32 = single.abs().max(dim=1, keepdim=True).values
        by32 = single * (torch.full_like(top32, 127.0) / torch.where(live, top32, 1.0))
        return torch.where(border & live, by32.double(), r).round(), torch.where(live, top / 127, 0.0)

    if case["op"] == "norm":
        h = given["x"].double() + given["residual"].double()
        stored = h.float()
        whole, step = rounded(h * given["weight"].double(), stored * given["weight"])
        return {"sum": h, "values": whole * step * torch.rsqrt(h.pow(2).sum(dim=1, keepdim=True) / case["cols"] + EPS)}
    if case["op"] == "silu":
        g, u = given["gate"], given["up"]
        whole, step = rounded(g.double() * torch.sigmoid(g.double()) * u.double(), g / (1 + torch.exp(-g)) * u)
        return {"values": whole * step}
    whole, step = rounded(given["x"].double(), given["x"])
    parts = [whole @ part.double().t() for part in given["q"].split(16384)]
    return {"out": torch.cat(parts, dim=1) * given["scales"].double() * step}
