"""The 8-bit operators once more, token by token in float64: what the kernels are compared with.

``Cache`` mirrors one cache entry on the host.  Codes follow from float32 quantities by correctly rounded float32 operations
(division, product), as the operators define them, so they can be compared bit by bit; sums are float64."""
import numpy as np

PAGE = 64
LEAST = np.float32(2.0 ** -100)
MOST = np.float32(2.0 ** 127)


def finite(x):
    x = np.where(np.isnan(x), np.float32(0), x.astype(np.float32))
    return np.clip(x, -MOST, MOST)


def quantize(x, least=np.float32(0)):
    """(codes, scale) of the numbers of ``x`` together, under a scale of at least ``least``"""
    x = finite(x)
    scale = max(np.float32(least), np.float32(np.abs(x).max(initial=0)) * (np.float32(1) / np.float32(127)), LEAST)
    return np.clip(np.rint(x / scale), -127, 127).astype(np.int8), np.float32(scale)


class Cache:
    def __init__(self, pages, n_kv, dim, block):
        self.block, self.n_kv, self.dim = block, n_kv, dim
        self.codes = [np.zeros((pages, n_kv, PAGE, dim), np.int8) for _ in range(2)]
        self.scale = [np.zeros((pages, n_kv, PAGE // block), np.float32) for _ in range(2)]
        self.weight = np.zeros((pages, n_kv, PAGE), np.float32)

    def values(self, which, pages, n):
        """float64 [n, n_kv, dim] of the first n tokens in ``pages``"""
        full = np.repeat(self.scale[which][pages].astype(np.float64), self.block, axis=2)[..., None]
        x = (self.codes[which][pages] * full).transpose(0, 2, 1, 3).reshape(-1, self.n_kv, self.dim)
        return x[:n]

    def append(self, k, v, pages, place):
        """The tokens of one sequence at places ``place`` ..; k, v float32 [tokens, n_kv, dim]; returns their values in float32"""
        back = [np.zeros_like(k), np.zeros_like(v)]
        t = 0
        while t < len(k):
            at = place + t
            end = min(len(k), t + self.block - at % self.block)
            page, blk = pages[at // PAGE], at % PAGE // self.block
            first = at % PAGE // self.block * self.block
            for which, x in ((0, k), (1, v)):
                for h in range(self.n_kv):
                    old = self.scale[which][page, h, blk] if at % self.block else np.float32(0)
                    codes, now = quantize(x[t:end, h], old)
                    if at % self.block and now > old:
                        c = self.codes[which][page, h, first:at % PAGE]
                        c[:] = np.rint(c.astype(np.float32) * (old / now)).astype(np.int8)
                    self.codes[which][page, h, at % PAGE:at % PAGE + end - t] = codes
                    self.scale[which][page, h, blk] = now
                    back[which][t:end, h] = codes.astype(np.float32) * now
            self.weight[page, :, at % PAGE:at % PAGE + end - t] = 0
            t = end
        return back

    def attend(self, q, pages, start, scale, window=None, weigh_last=0):
        """q float64 [rows, n_q, dim] of one sequence; (out, lse, weight added [n_kv, tokens], the largest sum of |q_d k_d| of a score)"""
        rows, n_q, _ = q.shape
        n, group = start + rows, n_q // self.n_kv
        k, v = self.values(0, pages, n), self.values(1, pages, n)
        out, lse, added, terms = np.zeros(q.shape), np.zeros((rows, n_q)), np.zeros((self.n_kv, n)), 0.0
        for i in range(rows):
            lo = max(0, start + i - window + 1) if window else 0
            for h in range(n_q):
                s = k[lo:start + i + 1, h // group] @ q[i, h] * scale
                top = s.max()
                terms = max(terms, (np.abs(k[lo:start + i + 1, h // group]) @ np.abs(q[i, h])).max() * scale)
                p = np.exp(s - top)
                out[i, h] = p @ v[lo:start + i + 1, h // group] / p.sum()
                lse[i, h] = top + np.log(p.sum())
                if i >= rows - weigh_last:
                    added[h // group, lo:start + i + 1] += p / p.sum()
        return out, lse, added, terms

    def evict(self, pages, n, target, keep, first, recent):
        """Moves what stays of one sequence to the pages ``target``; the places [n_kv, keep], -1 behind them"""
        kept = np.full((self.n_kv, keep), -1, np.int64)
        scale, codes = [s.copy() for s in self.scale], [c.copy() for c in self.codes]
        weight = self.weight.copy()
        for h in range(self.n_kv):
            w = self.weight[pages, h].reshape(-1)[:n].astype(np.float64)
            w = np.where(np.isnan(w), -np.inf, w)
            if n <= keep:
                stay = list(range(n))
            else:
                middle = sorted(range(first, n - recent), key=lambda j: (-w[j], j))[:keep - first - recent]
                stay = sorted(list(range(first)) + middle + list(range(n - recent, n)))
            kept[h, :len(stay)] = stay
            for i0 in range(0, len(stay), self.block):
                run = stay[i0:i0 + self.block]
                for which in range(2):
                    s = np.array([scale[which][pages[j // PAGE], h, j % PAGE // self.block] for j in run])
                    now = s.max()
                    self.scale[which][target[i0 // PAGE], h, i0 % PAGE // self.block] = now
                    for i, j in enumerate(run):
                        c = codes[which][pages[j // PAGE], h, j % PAGE].astype(np.float32)
                        self.codes[which][target[i0 // PAGE], h, i0 % PAGE + i] = np.rint(c * (s[i] / now)).astype(np.int8)
                for i, j in enumerate(run):
                    self.weight[target[i0 // PAGE], h, i0 % PAGE + i] = weight[pages[j // PAGE], h, j % PAGE]
        return kept


def rotate(x, cos, sin):
    """float32 rotation of pairs (i, i + half) of x [..., dim] by tables [..., rot / 2], one rounding an operation"""
    half = cos.shape[-1]
    lo, hi = x[..., :half], x[..., half:2 * half]
    return np.concatenate([lo * cos - hi * sin, lo * sin + hi * cos, x[..., 2 * half:]], axis=-1)
