"""Operators in microscaled 4-bit floats, and the router of experts: what is measured of them, and their plain forms.

Numbers in 4 bits: 32 neighbours along a row share a scale 2^(byte - 127), each is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  In
memory a matrix [n, k] is ``codes`` uint8 [n, k / 2], the earlier number of a pair in the low four bits (bit 3 the sign), and ``scales``
uint8 [n, k / 32].  A case is one call (or the calls that go together) of one operator:

* ``quantize``: a matrix into 4 bits and back into the values that it then stands for.
* ``linear``: rows quantised as they come, times weights in 4 bits.
* ``unit``: a gated feed-forward, down(silu(gate x) * (up x)), rows and inner rows quantised as they come.
* ``route``: from a token's logits to its experts and their weights.
* ``experts``: the same unit as chosen experts' weighted sum.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
BLOCK = 32
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases --------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the float32 rows of a step of 64 sequences, hidden size of the 1B preset
        {"name": "quantize step", "op": "quantize", "rows": 64, "k": 2048, "type": "f32"},
        # a layer's up projection of the 8B preset, as a model is loaded
        {"name": "quantize weights", "op": "quantize", "rows": 14336, "k": 4096, "type": "bf16"},
        # the smallest product: one row, the output projection of the 1B preset
        {"name": "linear one", "op": "linear", "rows": 1, "n": 2048, "k": 2048, "add": False, "type": "bf16"},
        # the down projection of a decode step of eight sequences, 8B preset, added to the float32 residual
        {"name": "linear step", "op": "linear", "rows": 8, "n": 4096, "k": 14336, "add": True, "type": "bf16"},
        # the up projection of a prompt step of 8,192 tokens
        {"name": "linear prompts", "op": "linear", "rows": 8192, "n": 14336, "k": 4096, "add": False, "type": "bf16"},
        # the feed-forward of a decode step of sixteen sequences, 1B preset
        {"name": "unit step", "op": "unit", "rows": 16, "k": 2048, "inter": 8192, "type": "bf16"},
        # the feed-forward of prompts of 2,011 tokens in all, 8B preset
        {"name": "unit prompts", "op": "unit", "rows": 2011, "k": 4096, "inter": 14336, "type": "bf16"},
        # a decode step's choice among 64 experts by softmax
        {"name": "route step", "op": "route", "rows": 8, "experts": 64, "top": 6, "scores": "softmax", "groups": 1, "keep": 1, "by": "max",
         "correct": False},
        # a prompt step's choice among 256 experts in 8 groups, by sigmoid scores with a correction for balance
        {"name": "route prompts", "op": "route", "rows": 8192, "experts": 256, "top": 8, "scores": "sigmoid", "groups": 8, "keep": 4,
         "by": "two", "correct": True},
        # one token's experts
        {"name": "experts one", "op": "experts", "rows": 1, "k": 2048, "inter": 1408, "experts": 64, "top": 6, "type": "bf16"},
        # a decode step of sixteen sequences: most experts have a token or two
        {"name": "experts step", "op": "experts", "rows": 16, "k": 2048, "inter": 1408, "experts": 64, "top": 6, "type": "bf16"},
        # a prompt step of 2,048 tokens, 192 rows an expert on average
        {"name": "experts prompts", "op": "experts", "rows": 2048, "k": 2048, "inter": 1408, "experts": 64, "top": 6, "type": "bf16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "linear", "unit", "unit", "route", "experts", "experts"])
    kind = rng.choice(["bf16", "bf16", "f32"])
    if op == "quantize":
        return {"op": op, "rows": _log_int(rng, 1, 14336), "k": 32 * _log_int(rng, 1, 128), "type": kind}
    if op == "linear":
        rows = _log_int(rng, 1, 8192)
        return {"op": op, "rows": rows, "n": 8 * _log_int(rng, 32, 1792), "k": 32 * _log_int(rng, 4, 128), "add": rng.random() < 0.4,
                "type": kind}
    if op == "unit":
        return {"op": op, "rows": _log_int(rng, 1, 2011), "k": 32 * _log_int(rng, 8, 128), "inter": 32 * _log_int(rng, 16, 448),
                "type": "bf16"}
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log_int(rng, 4, 256 // groups)
        keep = rng.randint(1, groups)
        return {"op": op, "rows": _log_int(rng, 1, 8192), "experts": experts, "top": rng.randint(1, min(8, keep * (experts // groups))),
                "scores": rng.choice(["softmax", "sigmoid"]), "groups": groups, "keep": keep, "by": rng.choice(["max", "two"]),
                "correct": rng.random() < 0.6}
    experts = _log_int(rng, 4, 64)
    return {"op": op, "rows": _log_int(rng, 1, 2048), "k": 32 * _log_int(rng, 8, 64), "inter": 32 * _log_int(rng, 8, 44),
            "experts": experts, "top": rng.randint(1, min(6, experts)), "type": "bf16"}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _weights(n, k, gen, spread=0.02):
    """Codes and scales of a normal matrix [n, k], drawn as such: each block's scale and its codes."""
    codes = torch.empty((n, k // 2), dtype=torch.uint8, device=DEVICE)
    scales = torch.empty((n, k // BLOCK), dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 26) // k)
    for lo in range(0, n, step):
        x = torch.randn((min(step, n - lo), k), generator=gen, device=DEVICE) * spread
        codes[lo:lo + step], scales[lo:lo + step] = _quantize(x)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    state = {"case": dict(case)}
    rows, op = case["rows"], case["op"]
    if op == "route":
        experts, top = case["experts"], case["top"]
        state["logits"] = torch.randn((rows, experts), generator=gen, device=DEVICE) * 1.5
        state["correction"] = torch.randn((experts,), generator=gen, device=DEVICE) * 0.05 if case["correct"] else None
        state["expert_of"] = torch.zeros((rows, top), dtype=torch.int32, device=DEVICE)
        state["weight"] = torch.zeros((rows, top), dtype=torch.float32, device=DEVICE)
        return state
    dtype, k = TYPES[case["type"]], case["k"]
    x = torch.randn((rows, k), generator=gen, device=DEVICE)
    if op == "quantize":
        state["x"] = (x * 0.02).to(dtype)
        state["out"] = torch.zeros_like(state["x"])
        if own:
            from supersonic_b200.weights import Fp4Matrix
            state["held"] = Fp4Matrix.empty(rows, k, device=DEVICE)
        return state
    x[:, :: 97] *= 8.0                                            # a few channels are much larger, as activations' are
    state["x"] = x.to(dtype)
    if op == "linear":
        state["w"] = _weights(case["n"], k, gen)
        out_type = torch.float32 if case["add"] else dtype
        state["out"] = torch.randn((rows, case["n"]), generator=gen, device=DEVICE).to(out_type)
    else:
        inter, experts = case["inter"], case.get("experts", 1)
        first = _weights(experts * 2 * inter, k, gen)             # gate rows, then up rows, of every expert
        second = _weights(experts * k, inter, gen)
        if op == "experts":
            first, second = ([t.view(experts, -1, t.shape[1]) for t in w] for w in (first, second))
            # experts of unlike popularity; a token has an expert once
            popular = torch.randn((experts,), generator=gen, device=DEVICE) * 0.5
            score = torch.randn((rows, experts), generator=gen, device=DEVICE) + popular
            best = torch.topk(score, case["top"], dim=-1)
            state["expert_of"] = best.indices.to(torch.int32)
            state["weight"] = torch.softmax(best.values, dim=-1)
        state["first"], state["second"] = tuple(first), tuple(second)
        state["out"] = torch.zeros((rows, k), dtype=dtype, device=DEVICE)
    if own:                                                       # laid out once, as a model is loaded
        from supersonic_b200.weights import Fp4Matrix
        if op == "linear":
            state["w"] = Fp4Matrix.from_parts(*state["w"])
        else:
            state["first"] = Fp4Matrix.from_parts(*state["first"], gated=True)
            state["second"] = Fp4Matrix.from_parts(*state["second"])
    return state


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _run_own(state):
    from supersonic_b200.csrc import fp4_ops, ops
    case = state["case"]
    if case["op"] == "quantize":
        fp4_ops.quantize(state["x"], state["held"])
        fp4_ops.values(state["held"], state["out"])
        return state["out"]
    if case["op"] == "linear":
        fp4_ops.linear(state["x"], state["w"], state["out"], accumulate=case["add"])
        return state["out"]
    if case["op"] == "unit":
        inner = fp4_ops.gate_up(state["x"], state["first"])
        fp4_ops.linear(inner, state["second"], state["out"])
        return state["out"]
    if case["op"] == "route":
        ops.route_scored(state["logits"], case["experts"], state["expert_of"], state["weight"], scores=case["scores"],
                         correction=state["correction"], groups=case["groups"], keep=case["keep"], group_score=case["by"],
                         renormalize=True)
        return {"expert_of": state["expert_of"], "weight": state["weight"]}
    fp4_ops.experts(state["x"], state["expert_of"], state["weight"], state["first"], state["second"], state["out"])
    return state["out"]


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _quantize(x):
    """(codes, scales) of a float32 matrix."""
    b = x.view(x.shape[0], -1, BLOCK)
    exponent = torch.frexp(b.abs().amax(-1)).exponent - 3         # floor(log2 max) - 2
    scale = torch.where(b.abs().amax(-1) > 0, exponent + 127, torch.zeros_like(exponent)).clamp_(0, 254)
    y = torch.ldexp(b, (127 - scale)[..., None])
    m = y.abs()
    # whole steps of 0.5, 1 and 2: codes 0..4, 4..6, 6..7
    code = torch.where(m < 2, (m * 2).round(), torch.where(m < 4, m.round() + 2, (m * 0.5).round().clamp(max=3) + 4)).to(torch.uint8)
    code |= (torch.signbit(y).to(torch.uint8) << 3)
    code = code.view(x.shape[0], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), scale.to(torch.uint8)


def _values(codes, scales):
    """float32 values of codes and scales, of any leading sizes"""
    four = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    size = (four & 7).float()
    size = torch.where(size < 4, size * 0.5, torch.where(size < 6, size - 2, size * 2 - 8))
    size = torch.where(four > 7, -size, size)
    return torch.ldexp(size.unflatten(-1, (-1, BLOCK)), scales.int()[..., None] - 127).flatten(-2)


def _rounded(x):
    return _values(*_quantize(x.float()))


def _plain_unit(x, first, second):
    """x: values; first, second: codes and scales"""
    g, u = torch.chunk(x @ _values(*first).t(), 2, dim=-1)
    return _rounded(g / (1 + torch.exp(-g)) * u) @ _values(*second).t()


def _plain_route(state):
    case = state["case"]
    z = state["logits"].double()
    if case["scores"] == "softmax":
        s = torch.exp(z - z.amax(-1, keepdim=True))
        s = s / s.sum(-1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-z))
    c = s if state["correction"] is None else s + state["correction"].double()
    if case["keep"] < case["groups"]:
        g = c.unflatten(-1, (case["groups"], -1))
        best = torch.sort(g, dim=-1, descending=True).values[..., : 1 if case["by"] == "max" else 2].sum(-1)
        order = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, : case["keep"]]
        stays = torch.zeros_like(best, dtype=torch.bool).scatter_(1, order, torch.ones_like(order, dtype=torch.bool))
        c = g.masked_fill(~stays[..., None], float("-inf")).flatten(-2)
    chosen = torch.sort(c, dim=-1, descending=True, stable=True).indices[:, : case["top"]]
    w = s.gather(1, chosen)
    state["expert_of"].copy_(chosen)
    state["weight"].copy_(w / (w.sum(-1, keepdim=True) + 1e-20))
    return {"expert_of": state["expert_of"], "weight": state["weight"]}


def _plain_experts(state):
    x, experts = _rounded(state["x"]), state["case"]["experts"]
    total = torch.zeros(state["out"].shape, dtype=torch.float32, device=DEVICE)
    chosen = state["expert_of"].long()
    for e in range(experts):
        token, choice = torch.nonzero(chosen == e, as_tuple=True)
        if token.numel():
            y = _plain_unit(x[token], [t[e] for t in state["first"]], [t[e] for t in state["second"]])
            total.index_add_(0, token, y * state["weight"][token, choice][:, None])
    state["out"].copy_(total)
    return state["out"]


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "route":
        return _plain_route(state)
    if case["op"] == "experts":
        return _plain_experts(state)
    if case["op"] == "quantize":
        state["out"].copy_(_rounded(state["x"]))
    elif case["op"] == "unit":
        state["out"].copy_(_plain_unit(_rounded(state["x"]), state["first"], state["second"]))
    else:
        y = _rounded(state["x"]) @ _values(*state["w"]).t()
        if case["add"]:
            state["out"].add_(y)
        else:
            state["out"].copy_(y)
    return state["out"]


# ---- work ---------------------------------------------------------------------------------------------------------
def work(case):
    rows = case["rows"]
    if case["op"] == "route":
        return {"bytes": rows * (4 * case["experts"] + 8 * case["top"]), "flops": 10.0 * rows * case["experts"]}
    size, k, held = (2 if case["type"] == "bf16" else 4), case["k"], 17 / 32
    if case["op"] == "quantize":
        # read, written in 4 bits, read again, written as values
        return {"bytes": rows * k * (2 * size + 2 * held), "flops": 4.0 * rows * k}
    if case["op"] == "linear":
        n = case["n"]
        return {"bytes": n * k * held + rows * k * size + rows * n * (8 if case["add"] else size), "flops": 2.0 * rows * n * k}
    inter = case["inter"]
    if case["op"] == "unit":
        return {"bytes": 3 * inter * k * held + 2 * rows * k * size, "flops": 6.0 * rows * inter * k}
    # experts that some token chose, on average, of choices spread evenly
    hit = case["experts"] * (1 - (1 - case["top"] / case["experts"]) ** rows)
    return {"bytes": hit * 3 * inter * k * held + rows * (2 * k * size + 8 * case["top"]), "flops": 6.0 * rows * case["top"] * inter * k}


# ---- the operators' definitions in 64 bits --------------------------------------------------------------------------
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_round(x):
    """The nearest of the format's numbers, of float64 x [rows, k]: between two, the one of the even code."""
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    out = torch.empty_like(x)
    for lo in range(0, x.shape[0], 4096):
        b = x[lo:lo + 4096].unflatten(-1, (-1, BLOCK))
        top = b.abs().amax(-1, keepdim=True)
        power = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
        # log2 may round to the next whole number: the power is the largest whose 2^power is not above the maximum
        power = power - (torch.exp2(power) > top).double() + (torch.exp2(power + 1) <= top).double()
        scale = torch.exp2(torch.clamp(power - 2, min=-127.0))
        m = (b / scale).abs()
        above = torch.bucketize(m, grid).clamp(1, 7)              # grid[above - 1] < m <= grid[above]
        low, high = grid[above - 1], grid[above]
        up = (m - low > high - m) | ((m - low == high - m) & (above % 2 == 0))
        out[lo:lo + 4096] = (torch.copysign(torch.where(up, high, low), b) * scale).flatten(-2)
    return out


def _exact_values(codes, scales):
    grid = torch.tensor(_GRID + tuple(-g for g in _GRID), dtype=torch.float64, device=codes.device)
    pairs = torch.stack([grid[(codes % 16).long()], grid[torch.div(codes, 16, rounding_mode="floor").long()]], dim=-1)
    return (pairs.view(*codes.shape[:-1], -1, BLOCK) * torch.exp2(scales.double() - 127)[..., None]).view(*codes.shape[:-1], -1)


def _exact_unit(x, first, second):
    both = torch.matmul(x, _exact_values(*first).t())
    inter = both.shape[1] // 2
    z = both[:, :inter] * torch.sigmoid(both[:, :inter]) * both[:, inter:]
    return torch.matmul(_exact_round(z), _exact_values(*second).t())


def _exact_route(state):
    case = state["case"]
    z = state["logits"].double()
    s = torch.softmax(z, dim=-1) if case["scores"] == "softmax" else torch.sigmoid(z)
    c = s + (0 if state["correction"] is None else state["correction"].double())
    per = case["experts"] // case["groups"]
    c, scores = c.cpu().tolist(), s.cpu().tolist()
    chosen, weight = [], []
    for row, own_scores in zip(c, scores):
        groups = range(case["groups"])
        if case["keep"] < case["groups"]:
            best = [sum(sorted(row[g * per:(g + 1) * per], reverse=True)[: 1 if case["by"] == "max" else 2]) for g in groups]
            groups = sorted(groups, key=lambda g: (-best[g], g))[: case["keep"]]
        live = sorted((e for g in groups for e in range(g * per, (g + 1) * per)), key=lambda e: (-row[e], e))[: case["top"]]
        total = math.fsum(own_scores[e] for e in live)
        chosen.append(live)
        weight.append([own_scores[e] / total for e in live])
    return {"expert_of": torch.tensor(chosen, dtype=torch.int32, device=DEVICE),
            "weight": torch.tensor(weight, dtype=torch.float64, device=DEVICE)}


def exact(case, seed):
    global own
    was, own = own, False                                         # weights as codes and scales
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "route":
        return _exact_route(state)
    x = _exact_round(state["x"].double())
    if case["op"] == "quantize":
        return x
    if case["op"] == "linear":
        y = torch.matmul(x, _exact_values(*state["w"]).t())
        return y + state["out"].double() if case["add"] else y
    if case["op"] == "unit":
        return _exact_unit(x, state["first"], state["second"])
    total = torch.zeros((case["rows"], case["k"]), dtype=torch.float64, device=DEVICE)
    chosen = state["expert_of"].tolist()
    for e in range(case["experts"]):
        tokens = [(t, row.index(e)) for t, row in enumerate(chosen) if e in row]
        if tokens:
            at = torch.tensor([t for t, _ in tokens], device=DEVICE)
            w = torch.stack([state["weight"][t, j] for t, j in tokens]).double()
            y = _exact_unit(x[at], [t[e] for t in state["first"]], [t[e] for t in state["second"]])
            total[at] += w[:, None] * y
    return total
