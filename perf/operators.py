"""The 8-bit serving operators: what is measured of them, and their plain forms.

A case is one call (or the calls that go together) of one operator:

* ``append``: the rotation of a step's queries and keys, and its keys and values into a cache of 8-bit codes with a scale for
  each block of tokens and kv head.
* ``attend``: a step's rows over that cache, causal, in packed sequences; with ``weigh`` the last rows of every sequence add
  what they attend to into a weight per cached token and kv head.
* ``evict``: a cache cut down to its first, its latest and its heaviest tokens, moved to new pages and read back.
* ``linear``: rows quantised to 8 bits as they come, times 8-bit weights with a scale per output channel.

A cache is paged: ``k``, ``v`` int8 [pages, n_kv, 64, dim], scales float32 [pages, n_kv, 64 / block], weights float32
[pages, n_kv, 64]; tokens 64 p .. 64 p + 63 of a sequence lie in page ``table[slot, p]``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
PAGE = 64
LEAST_SCALE = 2.0 ** -100
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---- cases --------------------------------------------------------------------------------------------------------
def listed():
    llama = {"n_q": 32, "n_kv": 8, "dim": 128, "block": 16, "type": "bf16"}          # heads of the 8B preset
    small = {"n_q": 32, "n_kv": 8, "dim": 64, "block": 32, "type": "bf16"}           # heads of the 1B preset
    return [
        # a decode step's keys and values, batch 8 at 520 tokens (the headline workload's step)
        {"name": "append step", "op": "append", "seqs": 8, "held": 520, "held_low": 500, "new": 1, "new_low": 1, **llama},
        # a step of sixteen prompts of 64 to 2,048 tokens
        {"name": "append prompts", "op": "append", "seqs": 16, "held": 0, "held_low": 0, "new": 2048, "new_low": 64, **llama},
        # the smallest decode step: one sequence of 512 tokens, where latency counts
        {"name": "attend one", "op": "attend", "seqs": 1, "held": 511, "held_low": 511, "new": 1, "new_low": 1, "window": 0,
         "weigh": 0, **llama},
        # a full batch of decode, sequences of very different lengths
        {"name": "attend step ragged", "op": "attend", "seqs": 64, "held": 8191, "held_low": 1, "new": 1, "new_low": 1, "window": 0,
         "weigh": 0, **llama},
        # decode of long sequences that keep account of what is attended to, in the float32 path
        {"name": "attend step weighed", "op": "attend", "seqs": 16, "held": 8191, "held_low": 8000, "new": 1, "new_low": 1,
         "window": 0, "weigh": 1, **dict(small, type="f32")},
        # a step of four whole prompts
        {"name": "attend prompts", "op": "attend", "seqs": 4, "held": 0, "held_low": 0, "new": 2048, "new_low": 2048, "window": 0,
         "weigh": 0, **llama},
        # the last chunk of a long prompt, whose last 32 rows decide what is evicted after it
        {"name": "attend chunk weighed", "op": "attend", "seqs": 1, "held": 16001, "held_low": 16001, "new": 500, "new_low": 500,
         "window": 0, "weigh": 32, **small},
        # eight sequences a little over their budget
        {"name": "evict short", "op": "evict", "seqs": 8, "held": 700, "held_low": 600, "keep": 512, "first": 4, "recent": 64, **small},
        # four sequences near the position limit cut to 4,096 tokens
        {"name": "evict long", "op": "evict", "seqs": 4, "held": 131000, "held_low": 60000, "keep": 4096, "first": 4, "recent": 256,
         **llama},
        # the smallest product: one row, 2,048 x 2,048 (output projection of the 1B preset)
        {"name": "linear one", "op": "linear", "rows": 1, "n": 2048, "k": 2048, "add": False, "type": "bf16"},
        # the down projection of a decode step of eight sequences, into the float32 residual
        {"name": "linear step", "op": "linear", "rows": 8, "n": 4096, "k": 14336, "add": True, "type": "bf16"},
        # the gate and up projections of a prompt step of 8,192 tokens
        {"name": "linear prompts", "op": "linear", "rows": 8192, "n": 28672, "k": 4096, "add": False, "type": "bf16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "evict", "linear"])
    kind = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "linear":
        rows = _log_int(rng, 1, 8192)
        n, k = 8 * _log_int(rng, 128, 3584), 16 * _log_int(rng, 64, 1024)
        return {"op": op, "rows": rows, "n": n, "k": k, "add": rng.random() < 0.4, "type": kind}
    n_kv = rng.choice([1, 2, 4, 8])
    heads = {"n_q": n_kv * rng.choice([1, 2, 3, 4, 8]), "n_kv": n_kv, "dim": rng.choice([64, 128]), "block": rng.choice([16, 32, 64]),
             "type": kind}
    if op == "append":
        if rng.random() < 0.5:
            held = _log_int(rng, 1, 4000)
            return {"op": op, "seqs": _log_int(rng, 1, 64), "held": held, "held_low": max(0, held // 3), "new": 1, "new_low": 1, **heads}
        new = _log_int(rng, 8, 2048)
        return {"op": op, "seqs": _log_int(rng, 1, 16), "held": rng.choice([0, _log_int(rng, 1, 500)]), "held_low": 0, "new": new,
                "new_low": 1, **heads}
    if op == "evict":
        keep = _log_int(rng, 64, 4096)
        held = _log_int(rng, keep, 32 * keep)
        return {"op": op, "seqs": _log_int(rng, 1, 8), "held": held, "held_low": max(1, held // 4), "keep": keep,
                "first": rng.choice([0, 1, 4, 16]), "recent": rng.choice([0, keep // 16, keep // 2]), **heads}
    window = rng.choice([0, 0, 0, _log_int(rng, 16, 2048)])
    if rng.random() < 0.6:                                       # decode
        held = _log_int(rng, 1, 16000)
        return {"op": op, "seqs": _log_int(rng, 1, 32), "held": held, "held_low": max(0, held // 8), "new": 1, "new_low": 1,
                "window": window, "weigh": rng.choice([0, 0, 1]), **heads}
    new = _log_int(rng, 2, 1024 if kind == "bf16" else 300)
    return {"op": op, "seqs": _log_int(rng, 1, 4), "held": rng.choice([0, _log_int(rng, 1, 4000)]), "held_low": 0, "new": new,
            "new_low": max(1, new // 4), "window": window, "weigh": rng.choice([0, 0, 1, 16]), **heads}


def _lengths(case):
    """(tokens held before, new tokens) of every sequence, from the case alone: the two ends of its ranges, the rest between."""
    rng = random.Random("%s %s %s" % (case["seqs"], case["held"], case.get("new")))
    held = [case["held"], case["held_low"]] + [rng.randint(case["held_low"], case["held"]) for _ in range(case["seqs"])]
    new = [rng.randint(case.get("new_low", 0), case.get("new", 0)) for _ in range(case["seqs"])]
    return held[: case["seqs"]], ([case.get("new", 0), case.get("new_low", 0)] + new)[: case["seqs"]]


# ---- inputs -------------------------------------------------------------------------------------------------------
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _cache(case, lengths, gen, spare=0):
    """A cache that holds ``lengths`` tokens: codes, scales, weights; pages in no order; ``spare`` pages a sequence beside them."""
    n_kv, dim, block = case["n_kv"], case["dim"], case["block"]
    per = max(1, -(-max(lengths) // PAGE))
    pages = sum(-(-n // PAGE) for n in lengths) + spare * len(lengths) + 1
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32).tolist()
    table = torch.zeros((len(lengths), per), dtype=torch.int32)
    for i, n in enumerate(lengths):
        for p in range(-(-n // PAGE)):
            table[i, p] = order.pop()
    more = _ints([[order.pop() for _ in range(spare)] for _ in lengths]) if spare else None
    codes = []
    for _ in range(2):
        c = torch.empty((pages, n_kv, PAGE, dim), dtype=torch.int8, device=DEVICE)
        for lo in range(0, pages, 1024):                          # codes of a normal distribution whose largest is 127
            x = torch.randn(c[lo:lo + 1024].shape, generator=gen, device=DEVICE)
            c[lo:lo + 1024] = (x * 36).round_().clamp_(-127, 127).to(torch.int8)
        codes.append(c)
    scales = [0.02 * torch.exp(0.4 * torch.randn((pages, n_kv, PAGE // block), generator=gen, device=DEVICE)) for _ in range(2)]
    weight = torch.exp(2.0 * torch.randn((pages, n_kv, PAGE), generator=gen, device=DEVICE) - 3.0)
    return {"k": codes[0], "v": codes[1], "k_scale": scales[0], "v_scale": scales[1], "weight": weight, "table": table.to(DEVICE)}, more


def _packed(case, held, new):
    """The integers of a step of packed sequences: row and sequence of every token."""
    slot = [i for i, n in enumerate(new) for _ in range(n)]
    place = [h + t for h, n in zip(held, new) for t in range(n)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return {"cu": _ints(cu), "start": _ints(held), "seq_slot": _ints(list(range(len(new)))), "slot": _ints(slot), "place": _ints(place),
            "max_new": max(new), "rows": cu[-1]}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    dtype = TYPES[case["type"]]
    state = {"case": dict(case)}
    if case["op"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        x = torch.randn((rows, k), generator=gen, device=DEVICE)
        x[:, :: 97] *= 8.0                                        # a few channels are much larger, as activations' are
        state["x"] = x.to(dtype)
        state["w"] = (torch.randn((n, k), generator=gen, device=DEVICE) * 36).round_().clamp_(-127, 127).to(torch.int8)
        state["w_scale"] = 0.0005 * torch.exp(0.2 * torch.randn((n,), generator=gen, device=DEVICE))
        out_type = torch.float32 if case["add"] else dtype
        state["out"] = torch.randn((rows, n), generator=gen, device=DEVICE).to(out_type)
        return state
    held, new = _lengths(case)
    n_q, n_kv, dim = case["n_q"], case["n_kv"], case["dim"]
    if case["op"] == "evict":
        keep = case["keep"]
        state["cache"], state["new_table"] = _cache(case, held, gen, spare=-(-keep // PAGE))
        state["lengths"], state["seq_slot"] = _ints(held), _ints(list(range(len(held))))
        state["kept"] = _ints([0]).expand(len(held), n_kv, keep).contiguous()
        state["values"] = [torch.zeros((len(held), keep, n_kv, dim), dtype=dtype, device=DEVICE) for _ in range(2)]
        state["new_lengths"] = _ints([min(n, keep) for n in held])
        return state
    state["cache"], _ = _cache(case, [h + n for h, n in zip(held, new)], gen)
    state["step"] = step = _packed(case, held, new)
    if case["op"] == "append":
        width = (n_q + 2 * n_kv) * dim
        state["qkv"] = torch.randn((step["rows"], width), generator=gen, device=DEVICE).to(dtype)
        angle = torch.arange(max(h + n for h, n in zip(held, new)), device=DEVICE)[:, None].double() \
            * 500000.0 ** (-torch.arange(0, dim, 2, device=DEVICE).double() / dim)
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        state["out"] = torch.zeros_like(state["qkv"])
        return state
    # queries spread their scores by about two, as a trained model's do
    state["q"] = (torch.randn((step["rows"], n_q * dim), generator=gen, device=DEVICE) * 2.0).to(dtype)
    state["out"] = torch.zeros_like(state["q"])
    state["lse"] = torch.zeros((step["rows"], n_q), dtype=torch.float32, device=DEVICE)
    return state


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _run_own(state):
    from supersonic_b200.cache import Int8Pages
    from supersonic_b200.csrc import int8_ops
    case = state["case"]
    if case["op"] == "linear":
        int8_ops.linear(state["x"], state["w"], state["w_scale"], state["out"], accumulate=case["add"])
        return state["out"]
    c = state["cache"]
    if case["op"] == "evict":
        pages = Int8Pages(c["k"], c["v"], c["k_scale"], c["v_scale"], c["weight"])
        int8_ops.evict(pages, c["table"], state["seq_slot"], state["lengths"], state["new_table"], case["keep"], case["first"],
                       case["recent"], state["kept"])
        int8_ops.read(pages, state["new_table"], state["seq_slot"], state["new_lengths"], *state["values"])
        return {"kept": state["kept"], "k": state["values"][0], "v": state["values"][1], "k_scale": c["k_scale"],
                "v_scale": c["v_scale"], "weight": c["weight"]}
    step = state["step"]
    if case["op"] == "append":
        pages = Int8Pages(c["k"], c["v"], c["k_scale"], c["v_scale"], c["weight"])
        int8_ops.append(state["qkv"], state["cos"], state["sin"], step["place"], step["place"], step["slot"], c["table"], pages,
                        state["out"], case["n_q"])
        return {"rows": state["out"], "k_scale": c["k_scale"], "v_scale": c["v_scale"], "weight": c["weight"]}
    pages = Int8Pages(c["k"], c["v"], c["k_scale"], c["v_scale"], c["weight"])
    int8_ops.attention(state["q"], pages, c["table"], step["cu"], step["start"], step["seq_slot"], step["max_new"], state["out"],
                       case["n_q"], case["dim"] ** -0.5, window=case["window"] or None, lse=state["lse"], weigh_last=case["weigh"])
    return {"out": state["out"], "lse": state["lse"], "weight": c["weight"]} if case["weigh"] else {"out": state["out"], "lse": state["lse"]}


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _plain_append(state):
    case, c, step = state["case"], state["cache"], state["step"]
    n_q, n_kv, dim, block = case["n_q"], case["n_kv"], case["dim"], case["block"]
    x = state["qkv"].float().view(-1, n_q + 2 * n_kv, dim)
    place, slot = step["place"].long(), step["slot"].long()
    cos, sin = state["cos"][place][:, None], state["sin"][place][:, None]
    turned, half = x[:, : n_q + n_kv], dim // 2
    lo, hi = turned[..., :half], turned[..., half:]
    turned = torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], dim=-1)
    rows = [turned[:, :n_q]]
    page = c["table"][slot, place // PAGE].long()
    per = PAGE // block
    at = page * per + place % PAGE // block                       # the token's block among all
    heads = torch.arange(n_kv, device=DEVICE)
    for new, codes, scale in ((turned[:, n_q:], c["k"], c["k_scale"]), (x[:, n_q + n_kv:], c["v"], c["v_scale"])):
        blocks = scale.shape[0] * per
        old = scale.transpose(1, 2).reshape(blocks, n_kv)
        # a block whose first token is new holds nothing yet
        fresh = torch.zeros(blocks, device=DEVICE).index_reduce(0, at, (place % block == 0).float(), "amax")
        begun = torch.where(fresh[:, None] > 0, torch.zeros_like(old), old)
        most = torch.zeros_like(old).index_reduce(0, at, new.abs().amax(-1), "amax")
        touched = torch.zeros(blocks, device=DEVICE).index_reduce(0, at, torch.ones_like(place, dtype=torch.float32), "amax")
        now = torch.maximum(torch.maximum(begun, most / 127.0), torch.full_like(old, LEAST_SCALE))
        now = torch.where(touched[:, None] > 0, now, old)
        ratio = torch.where(touched[:, None] > 0, begun / now, torch.ones_like(old))
        all_ratios = ratio.view(-1, per, n_kv).transpose(1, 2)
        wide = all_ratios[..., None].expand(-1, -1, -1, block).reshape(-1, n_kv, PAGE, 1)
        codes.copy_((codes.float() * wide).round().to(torch.int8))
        mine = now[at][..., None]
        put = (new / mine).round().clamp(-127, 127)
        codes[page[:, None], heads, (place % PAGE)[:, None]] = put.to(torch.int8)
        scale.copy_(now.view(-1, per, n_kv).transpose(1, 2))
        rows.append(put * mine)
    c["weight"][page[:, None], heads, (place % PAGE)[:, None]] = 0.0
    state["out"].copy_(torch.cat(rows, dim=1).reshape(state["out"].shape))
    return {"rows": state["out"], "k_scale": c["k_scale"], "v_scale": c["v_scale"], "weight": c["weight"]}


def _values(codes, scale, table, block):
    """float32 [sequences, n_kv, tokens of the table's pages, dim]"""
    x = codes[table.long()].float() * scale[table.long()].repeat_interleave(block, dim=-1)[..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(state):
    case, c, step = state["case"], state["cache"], state["step"]
    n_q, n_kv, dim = case["n_q"], case["n_kv"], case["dim"]
    table, seqs, most = c["table"][step["seq_slot"].long()], case["seqs"], step["max_new"]
    first, n_new, start = step["cu"][:-1, None], step["cu"].diff()[:, None], step["start"][:, None]
    i = torch.arange(most, device=DEVICE)[None]
    live = i < n_new
    row = torch.where(live, first + i, 0).long()
    q = state["q"].float().view(-1, n_kv, n_q // n_kv, dim)[row]                      # [seqs, most, n_kv, group, dim]
    k = _values(c["k"], c["k_scale"], table, case["block"])
    s = torch.einsum("btkgd,bkjd->bkgtj", q, k) * dim ** -0.5
    del k
    j = torch.arange(s.shape[-1], device=DEVICE)
    at = (start + i)[..., None]
    seen = (j <= at) & live[..., None]
    if case["window"]:
        seen &= j > at - case["window"]
    s = s.masked_fill_(~seen[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    s = s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    s = s.div_(torch.where(total > 0, total, torch.ones_like(total)))
    v = _values(c["v"], c["v_scale"], table, case["block"])
    o = torch.einsum("bkgtj,bkjd->btkgd", s, v).reshape(seqs, most, n_q * dim)
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(seqs, most, n_q)
    state["out"].copy_(o[live])
    state["lse"].copy_(lse[live])
    if not case["weigh"]:
        return {"out": state["out"], "lse": state["lse"]}
    weighs = live & (i >= n_new - case["weigh"])
    add = (s * weighs[:, None, None, :, None]).sum((2, 3))                            # [seqs, n_kv, keys]
    add = add.view(seqs, n_kv, -1, PAGE).transpose(1, 2).reshape(-1, n_kv, PAGE)
    held = (torch.arange(table.shape[1], device=DEVICE) * PAGE < start + n_new).reshape(-1)
    c["weight"].index_add_(0, torch.where(held, table.reshape(-1), 0).long(), add * held[:, None, None])
    return {"out": state["out"], "lse": state["lse"], "weight": c["weight"]}


def _gathered(x, table, place):
    """x [pages, n_kv, 64, ...] at places [sequences, n_kv, n] of the sequences' tables"""
    page = table.long()[torch.arange(place.shape[0], device=DEVICE)[:, None, None], place // PAGE]
    return x[page, torch.arange(place.shape[1], device=DEVICE)[:, None], place % PAGE]


def _plain_evict(state):
    case, c = state["case"], state["cache"]
    n_kv, keep, block = case["n_kv"], case["keep"], case["block"]
    table = c["table"][state["seq_slot"].long()]
    n = state["lengths"].long()[:, None, None]
    seqs, per = table.shape
    weight = c["weight"][table.long()].transpose(1, 2).reshape(seqs, n_kv, per * PAGE)
    j = torch.arange(per * PAGE, device=DEVICE)
    weight = torch.where(torch.isnan(weight), torch.full_like(weight, float("-inf")), weight)
    # rank: kept anyway, then the others by weight, then what is not there; equal ones in their order
    order = torch.sort(weight, dim=-1, descending=True, stable=True).indices
    kind = torch.where(j >= n, 2, torch.where((j < case["first"]) | (j >= n - case["recent"]), 0, 1)).expand_as(weight)
    order = order.gather(-1, torch.sort(kind.gather(-1, order), dim=-1, stable=True).indices)
    most = min(keep, per * PAGE)
    chosen = torch.sort(torch.where(torch.arange(most, device=DEVICE) < n, order[..., :most], per * PAGE), dim=-1).values
    there = chosen < per * PAGE
    state["kept"].fill_(-1)
    state["kept"][..., :most] = torch.where(there, chosen, -1).to(torch.int32)
    # destination blocks: places 0 .. keep - 1, padded to whole blocks
    place = torch.zeros((seqs, n_kv, state["new_table"].shape[1] * PAGE), dtype=torch.long, device=DEVICE)
    live = torch.zeros_like(place, dtype=torch.bool)
    place[..., :most] = torch.where(there, chosen, 0)
    live[..., :most] = there
    page = state["new_table"].long().view(seqs, -1, 1, 1, 1)
    heads = torch.arange(n_kv, device=DEVICE).view(-1, 1, 1)
    for i, name in enumerate(("k", "v")):
        codes, scale = c[name], c[name + "_scale"]
        s = _gathered(scale.repeat_interleave(block, dim=-1), table, place) * live
        new = s.view(seqs, n_kv, -1, block).amax(-1)
        moved = _gathered(codes, table, place).float()
        ratio = s / torch.where(new > 0, new, torch.ones_like(new)).repeat_interleave(block, dim=-1)
        moved = (moved * ratio[..., None]).round() * live[..., None]
        full = new.repeat_interleave(block, dim=-1)[..., None]
        state["values"][i][:, :most] = (moved * full).transpose(1, 2)[:, :most]
        split = moved.view(seqs, n_kv, -1, PAGE, codes.shape[-1]).transpose(1, 2).to(torch.int8)
        written = (new > 0).view(seqs, n_kv, -1, PAGE // block).transpose(1, 2)
        at = state["new_table"].long()
        scale[at] = torch.where(written, new.view(seqs, n_kv, -1, PAGE // block).transpose(1, 2), scale[at])
        rows = live.view(seqs, n_kv, -1, PAGE).transpose(1, 2)[..., None]
        codes[at] = torch.where(rows, split, codes[at])
    rows = live.view(seqs, n_kv, -1, PAGE).transpose(1, 2)
    at = state["new_table"].long()
    moved = _gathered(c["weight"], table, place).view(seqs, n_kv, -1, PAGE).transpose(1, 2)
    c["weight"][at] = torch.where(rows, moved, c["weight"][at])
    return {"kept": state["kept"], "k": state["values"][0], "v": state["values"][1], "k_scale": c["k_scale"],
            "v_scale": c["v_scale"], "weight": c["weight"]}


def _plain_linear(state):
    x, w = state["x"].float(), state["w"].float()
    scale = torch.clamp(x.abs().amax(-1, keepdim=True) / 127.0, min=LEAST_SCALE)
    y = (x / scale).round() @ w.t() * scale * state["w_scale"]
    if state["case"]["add"]:
        state["out"].add_(y)
    else:
        state["out"].copy_(y)
    return state["out"]


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict, "linear": _plain_linear}[state["case"]["op"]](state)


# ---- work ---------------------------------------------------------------------------------------------------------
def _visible(case, held, new):
    """(keys that some row of the sequence sees, (row, key) pairs)"""
    window = case["window"] or (1 << 40)
    first = max(0, held - window + 1)
    keys = held + new - first
    whole = sum(min(held + i + 1, window) for i in range(new))
    return keys, whole


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "linear":
        rows, n, k = case["rows"], case["n"], case["k"]
        out = rows * n * (8 if case["add"] else size)
        return {"bytes": n * k + 4 * n + rows * k * size + out, "flops": 2.0 * rows * n * k}
    held, new = _lengths(case)
    n_q, n_kv, dim, block = case["n_q"], case["n_kv"], case["dim"], case["block"]
    token = n_kv * (2 * dim + 8 / block)                          # codes and scales of keys and values
    if case["op"] == "append":
        rows = sum(new)
        return {"bytes": rows * (2 * (n_q + 2 * n_kv) * dim * size + 4 * dim + token + 4 * n_kv), "flops": 6.0 * rows * (n_q + n_kv) * dim}
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in held)
        # weights read; kept codes read, written and read back as values; the list
        return {"bytes": sum(held) * n_kv * 4 + kept * (3 * token + n_kv * (2 * dim * size + 4 + 8)), "flops": 2.0 * kept * n_kv * 2 * dim}
    rows, keys, pairs = sum(new), 0, 0
    for h, n in zip(held, new):
        a, b = _visible(case, h, n)
        keys, pairs = keys + a, pairs + b
    moved = keys * token + 2 * rows * n_q * dim * size + rows * n_q * 4
    if case["weigh"]:
        moved += keys * n_kv * 8
    return {"bytes": moved, "flops": 4.0 * pairs * n_q * dim}


# ---- the operators' definitions in 64 bits --------------------------------------------------------------------------
def _exact_values(c, name, pages, block):
    """float64 [n_kv, tokens, dim] of one sequence's pages"""
    codes, scale = c[name][pages].double(), c[name + "_scale"][pages].double()
    kv = codes.shape[1]
    full = codes.unflatten(2, (-1, block)) * scale[..., None, None]
    return full.flatten(2, 3).permute(1, 0, 2, 3).reshape(kv, -1, codes.shape[-1])


def _exact_attend(state):
    case, c, step = state["case"], state["cache"], state["step"]
    held, new = _lengths(case)
    n_q, n_kv, dim = case["n_q"], case["n_kv"], case["dim"]
    q = state["q"].double().view(-1, n_kv, n_q // n_kv, dim)
    weight, out, lses, row = c["weight"].double(), [], [], 0
    for b, (h, n) in enumerate(zip(held, new)):
        pages = c["table"][b, : -(-(h + n) // PAGE)].long()
        k, v = (_exact_values(c, name, pages, case["block"])[:, : h + n] for name in ("k", "v"))
        added = torch.zeros((n_kv, h + n), dtype=torch.float64, device=DEVICE)
        for lo in range(0, n, 128):
            hi = min(n, lo + 128)
            at = torch.arange(h + lo, h + hi, device=DEVICE)[:, None]
            j = torch.arange(h + n, device=DEVICE)
            hidden = (j > at) | ((j <= at - case["window"]) if case["window"] else False)
            s = torch.matmul(q[row + lo:row + hi].permute(1, 2, 0, 3), k.transpose(1, 2)[:, None]) / math.sqrt(dim)
            s = s.masked_fill(hidden, -math.inf)
            lse = torch.logsumexp(s, dim=-1)
            p = torch.exp(s - lse[..., None])
            out.append(torch.matmul(p, v[:, None]).permute(2, 0, 1, 3).reshape(hi - lo, -1))
            lses.append(lse.permute(2, 0, 1).reshape(hi - lo, -1))
            first = max(lo, n - case["weigh"]) - lo
            if first < hi - lo:
                added += p[:, :, first:].sum((1, 2))
        padded = torch.zeros((n_kv, len(pages) * PAGE), dtype=torch.float64, device=DEVICE)
        padded[:, : h + n] = added
        weight[pages] += padded.view(n_kv, -1, PAGE).transpose(0, 1)
        row += n
    got = {"out": torch.cat(out), "lse": torch.cat(lses)}
    return dict(got, weight=weight) if case["weigh"] else got


def _exact_append(state):
    case, c, step = state["case"], state["cache"], state["step"]
    held, new = _lengths(case)
    n_q, n_kv, dim, block = case["n_q"], case["n_kv"], case["dim"], case["block"]
    x = state["qkv"].double().view(-1, n_q + 2 * n_kv, dim)
    angles = (state["cos"].double()[step["place"].long()], state["sin"].double()[step["place"].long()])
    turn = torch.complex(*angles)[:, None]
    z = torch.complex(x[:, : n_q + n_kv, : dim // 2], x[:, : n_q + n_kv, dim // 2:]) * turn
    x = torch.cat([torch.cat([z.real, z.imag], -1), x[:, n_q + n_kv:]], 1)
    k_scale, v_scale, weight, row = c["k_scale"].double(), c["v_scale"].double(), c["weight"].double(), 0
    for b, (h, n) in enumerate(zip(held, new)):
        t = h
        while t < h + n:
            end = min(h + n, (t // block + 1) * block)
            page, at, rows = int(c["table"][b, t // PAGE]), t % PAGE // block, slice(row + t - h, row + end - h)
            for scale, heads in ((k_scale, slice(n_q, n_q + n_kv)), (v_scale, slice(n_q + n_kv, None))):
                now = x[rows, heads].abs().amax((0, 2)) / 127
                if t % block:
                    now = torch.maximum(now, scale[page, :, at])
                scale[page, :, at] = now
                x[rows, heads] = torch.round(x[rows, heads] / now[:, None]) * now[:, None]
            weight[page, :, t % PAGE:t % PAGE + end - t] = 0
            t = end
        row += n
    return {"rows": x.reshape(x.shape[0], -1), "k_scale": k_scale, "v_scale": v_scale, "weight": weight}


def _exact_evict(state):
    case, c = state["case"], state["cache"]
    keep, block = case["keep"], case["block"]
    values = [v.double() for v in state["values"]]
    scales = {name: c[name].double() for name in ("k_scale", "v_scale")}
    weight = c["weight"].double()
    for b, n in enumerate(state["lengths"].tolist()):
        pages = c["table"][b].long()
        target = state["new_table"][b].long()
        for head in range(case["n_kv"]):
            w = c["weight"][pages, head].double().flatten()[:n].cpu()
            if n <= keep:
                places = list(range(n))
            else:
                low, high = case["first"], n - case["recent"]
                middle = sorted(range(low, high), key=w.tolist().__getitem__, reverse=True)[: keep - case["first"] - case["recent"]]
                places = sorted(list(range(low)) + middle + list(range(high, n)))
            at = torch.tensor(places, device=DEVICE)
            to = torch.arange(len(places), device=DEVICE)
            weight[target[to // PAGE], head, to % PAGE] = w.to(DEVICE)[at]
            for i, name in enumerate(("k", "v")):
                scale = c[name + "_scale"][pages[at // PAGE], head, at % PAGE // block].double()
                codes = c[name][pages[at // PAGE], head, at % PAGE].double()
                for lo in range(0, len(places), block):
                    now = scale[lo:lo + block].max()
                    scales[name + "_scale"][target[lo // PAGE], head, lo % PAGE // block] = now
                    values[i][b, lo:min(lo + block, len(places)), head] = torch.round(codes[lo:lo + block] * (scale[lo:lo + block] / now)[:, None]) * now
    return {"kept": None, "k": values[0], "v": values[1], "weight": weight, **scales}


def _exact_linear(state):
    x, w = state["x"].double(), state["w"].double()
    scale = x.abs().amax(-1) / 127
    y = torch.matmul(torch.round(x / scale[:, None]), w.t()) * torch.outer(scale, state["w_scale"].double())
    return y + state["out"].double() if state["case"]["add"] else y


def exact(case, seed):
    if case["op"] == "append" and sum(_lengths(case)[1]) > 6000:
        return None
    if case["op"] == "evict" and case["seqs"] * case["n_kv"] * case["keep"] > 40000:
        return None
    state = prepare(case, seed)
    with torch.no_grad():
        return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict, "linear": _exact_linear}[case["op"]](state)
