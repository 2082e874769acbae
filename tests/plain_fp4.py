"""The 4-bit operators once more in float64 (torch, on whatever device the inputs are on): what the kernels are compared with."""
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
MOST = float(torch.finfo(torch.float32).max)


def finite(x):
    return torch.nan_to_num(x.double(), nan=0.0, posinf=MOST, neginf=-MOST).clamp(-MOST, MOST)


def exponents(x):
    """The blocks' scale bytes of float64 rows [n, k]."""
    top = x.unflatten(-1, (-1, 32)).abs().amax(-1)
    _, e = torch.frexp(top)                                     # top = m 2^e, m in [0.5, 1)
    return torch.where(top > 0, e - 1 - 2 + 127, torch.zeros_like(e)).clamp(min=0)


def codes_of(x, bytes_):
    """The nearest codes (0-7, the sign apart) of |x| under these scales, between two the even one."""
    y = x.unflatten(-1, (-1, 32)).abs() * torch.exp2(127.0 - bytes_.double())[..., None]
    d = (y[..., None] - GRID.to(x.device)).abs()
    near = d.amin(-1, keepdim=True)
    ties = d == near
    even = torch.arange(8, device=x.device) % 2 == 0
    first = torch.where(ties & even, 0, torch.where(ties, 1, 2))
    return first.argmin(-1)


def rounded(x, bytes_=None):
    """The values of rows [n, k] in 4 bits, float64."""
    x = finite(x)
    bytes_ = exponents(x) if bytes_ is None else bytes_
    v = GRID.to(x.device)[codes_of(x, bytes_)] * torch.exp2(bytes_.double() - 127.0)[..., None]
    return torch.copysign(v.flatten(-2), x)


def values(matrix):
    """float64 values of an Fp4Matrix, rows in the order its codes have."""
    c = torch.stack([matrix.codes & 15, matrix.codes >> 4], dim=-1).flatten(-2).long()
    v = torch.copysign(GRID.to(c.device)[c & 7], torch.where(c > 7, -1.0, 1.0).double())
    s = torch.exp2(matrix.plain_scales().double() - 127.0)
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def sum_slack(x, w):
    """How far float32 sums of x w^T may be off: a block's products and their sum are exact (multiples of 0.25 up to 1,152, times two powers
    of two), which leaves k / 32 additions and the joining of at most 16 parts, each off by 2^-23 of the magnitudes at most."""
    return (x.shape[-1] / 32 + 16) * 2.0 ** -23 * (x.abs() @ w.abs().transpose(-1, -2))


def gate(g, u, kind="silu", limit=0.0):
    if kind == "silu":
        return g * torch.sigmoid(g) * u
    if kind == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh((2 / torch.pi) ** 0.5 * (g + 0.044715 * g ** 3))) * u
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(1.702 * g) * (u + 1)


def activate(u, kind):
    if kind == "relu_squared":
        return u.clamp(min=0) ** 2
    if kind == "gelu_tanh":
        return gate(u, torch.ones_like(u), "gelu_tanh")
    return u * torch.sigmoid(u)


def inner(x, first, gated, act, row_scale=None):
    """(inner rows before they go into 4 bits, how far they may be off) of rows x and a first matrix's values, gate rows first."""
    s, t = x @ first.t(), sum_slack(x, first)
    if gated:
        (g, u), (tg, tu) = s.chunk(2, -1), t.chunk(2, -1)
        kind, limit = act if act else ("silu", 0.0)
        z = gate(g, u, kind, limit)
        # |d gate / dg| <= 1.8 |u'| for the three, with u' = u or u + 1; |d / du| <= max(|g|, 1); the fast exponential is good to (2 + 1.2 |x|) ulp
        # of an argument 1.8 |g| at most (gelu's cubic: |g| < 8 where it is not flat), the quotient to two
        du = u.abs() + 1
        slack = 1.8 * du * tg + g.abs().clamp(min=1) * tu + z.abs() * (8 + 20 * g.abs().clamp(max=30)) * 2.0 ** -23
    else:
        z = activate(s, act)
        slack = (2 * s.abs() + 1.2) * t + z.abs() * 2.0 ** -19
    if row_scale is not None:
        z, slack = z * row_scale[:, None].double(), slack * row_scale[:, None].double().abs()
    return z, slack + z.abs() * 2.0 ** -22


def between(z, slack):
    """(values in 4 bits of z, how far what is within ``slack`` of z may be from them)."""
    low, high = exponents((z.abs() - slack).clamp(min=0)), exponents(z.abs() + slack)
    q = rounded(z)
    off = torch.maximum((rounded(z + slack, exponents(z)) - q).abs(), (rounded(z - slack, exponents(z)) - q).abs())
    unsure = (low != high).repeat_interleave(32, dim=-1)                  # the block's scale is not sure: a whole step of the larger one
    step = (2.0 * torch.exp2(high.double() - 127.0)).repeat_interleave(32, dim=-1)
    return q, torch.where(unsure, step, off)


def route(logits, correction, scores, groups, keep, by, top, renormalize, scale):
    """(experts, weights) of every token, python lists, from float64 logits [tokens, experts] on the host."""
    import math
    out_e, out_w = [], []
    for row in logits.double().tolist():
        z = [-math.inf if v != v else min(max(v, -MOST), MOST) if v != -math.inf else v for v in row]
        if scores == "softmax":
            m = max(z)
            e = [math.exp(v - m) if v > -math.inf else 0.0 for v in z]
            total = math.fsum(e)
            s = [v / total if total > 0 else 0.0 for v in e]
        else:
            s = [0.0 if v == -math.inf else 1 / (1 + math.exp(-v)) if v > -700 else 0.0 for v in z]
        c = [a + b for a, b in zip(s, correction.double().tolist())] if correction is not None else s
        c = [-math.inf if v != v else v for v in c]
        per = len(c) // groups
        best = [sum(sorted(c[g * per:(g + 1) * per], reverse=True)[: 1 if by == "max" else 2]) for g in range(groups)]
        if correction is None:                   # s grows with z, also where 64 bits no longer show it (exp(-1e30), sigmoid(40) and (41))
            c = z
            if by == "max" or per == 1:
                best = [max(c[g * per:(g + 1) * per]) for g in range(groups)]
        kept = sorted(range(groups), key=lambda g: (-best[g], g))[:keep]
        chosen = sorted((e for g in kept for e in range(g * per, (g + 1) * per)), key=lambda e: (-c[e], e))[:top]
        f = scale / (math.fsum(s[e] for e in chosen) + 1e-20) if renormalize else scale
        out_e.append(chosen)
        out_w.append([s[e] * f for e in chosen])
    return out_e, out_w
