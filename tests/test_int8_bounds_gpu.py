"""Attention over the 8-bit cache at the borders of what it is given: places behind the page table's end, page ids that name no page,
starts near 2^31.  One definition holds for every kernel: a key is seen if its place is within the row's reach and the table and its
page id is one of the pool's; a row that sees none is zeros, with minus infinity for its sum."""
import numpy as np
import pytest
import torch

import plain_int8 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
MOST = 2 ** 31 - 1
GUARD = 4096


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cache(rng, table, n_pages, n_kv, dim, block):
    """Random codes and scales in the pages that the table names; every other page's scales and weights are NaN."""
    cache = plain.Cache(n_pages, n_kv, dim, block)
    named = np.unique(table[(table >= 0) & (table < n_pages)])
    for which in range(2):
        cache.codes[which][:] = np.clip(np.rint(rng.normal(size=cache.codes[which].shape) * 36), -127, 127)
        cache.scale[which][:] = np.nan
        cache.scale[which][named] = 0.02 * np.exp(0.5 * rng.normal(size=cache.scale[which][named].shape))
    cache.weight[:] = np.nan
    cache.weight[named] = np.exp(rng.normal(size=cache.weight[named].shape))
    return cache


def _attend(cache, pages, start, window, weigh, q, scale):
    """(out, lse, weight added [n_kv, places of the table], the largest sum of |q_d k_d| of a score) of one sequence; q float64"""
    rows, n_q, _ = q.shape
    group, n_pages = n_q // cache.n_kv, len(cache.codes[0])
    there = np.repeat((pages >= 0) & (pages < n_pages), plain.PAGE)
    place = np.flatnonzero(there)
    k, v = (cache.values(which, pages[(pages >= 0) & (pages < n_pages)], None) for which in range(2))
    out, lse, added, terms = np.zeros(q.shape), np.full((rows, n_q), -np.inf), np.zeros((cache.n_kv, len(there))), 0.0
    for i in range(rows):
        seen = place <= start + i
        if window:
            seen &= place > start + i - window
        if not seen.any():
            continue
        for h in range(n_q):
            ks = k[seen, h // group]
            s = ks @ q[i, h] * scale
            terms = max(terms, (np.abs(ks) @ np.abs(q[i, h])).max() * scale)
            p = np.exp(s - s.max())
            out[i, h] = p @ v[seen, h // group] / p.sum()
            lse[i, h] = s.max() + np.log(p.sum())
            if i >= rows - weigh:
                added[h // group, place[seen]] += p / p.sum()
    return out, lse, added, terms


def _check(rng, monkeypatch, table, starts, counts, n_q, n_kv, dim, block, kind, window=None, weigh=0, bad=()):
    """``bad``: (row, head) of queries that hold a NaN: their results are NaN, and the weights of what they account for."""
    from supersonic_b200.cache import Int8Pages
    from supersonic_b200.csrc import int8_ops, ops
    dtype, rows, n_pages = TYPES[kind], sum(counts), int(table[(table >= 0) & (table < MOST)].max()) - 1
    cache = _cache(rng, table, n_pages, n_kv, dim, block)
    pages = Int8Pages(*[torch.from_numpy(x).to(DEV) for x in (*cache.codes, *cache.scale, cache.weight.copy())])
    q = torch.from_numpy(rng.normal(size=(rows, n_q, dim)) * 2).to(dtype)
    given = q.clone()
    for row, head in bad:
        given[row, head, dim // 3] = float("nan")
    qt = given.to(DEV).reshape(rows, -1)
    out, lse = torch.full_like(qt, 7.0), torch.full((rows, n_q), 7.0, device=DEV)
    guards, empty = [], torch.empty

    def guarded(shape, *a, **kw):                                     # scratch, with a region behind it that nothing may touch
        if not isinstance(shape, int) or kw.get("dtype") is not torch.float32:
            return empty(shape, *a, **kw)
        whole = torch.full((shape + GUARD,), 12345.0, **kw)
        guards.append(whole[shape:])
        return whole[:shape]
    monkeypatch.setattr(torch, "empty", guarded)
    cu = np.concatenate([[0], np.cumsum(counts)])
    scale = dim ** -0.5
    int8_ops.attention(qt, pages, torch.from_numpy(table).to(DEV), _ints(cu), _ints(starts), _ints(list(range(len(counts)))), max(counts),
                       out, n_q, scale, window=window, lse=lse, weigh_last=weigh)
    monkeypatch.undo()
    ops.check_device_errors()
    assert all((g == 12345.0).all() for g in guards)
    out, lse = out.float().cpu().numpy().reshape(rows, n_q, dim), lse.cpu().numpy()
    weight, want_weight, terms = pages.weight.cpu().numpy(), cache.weight.astype(np.float64), 0.0
    most_added, lost = np.zeros_like(want_weight), np.zeros(weight.shape, bool)
    for b, (start, n) in enumerate(zip(starts, counts)):
        own = slice(cu[b], cu[b + 1])
        spoilt = np.zeros((n, n_q), bool)
        for row, head in bad:
            if cu[b] <= row < cu[b + 1]:
                spoilt[row - cu[b], head] = True
                if row >= cu[b + 1] - weigh:
                    for j in range(max(0, start + row - cu[b] - window + 1 if window else 0), start + row - cu[b] + 1):
                        if 0 <= table[b, j // 64] < n_pages:
                            lost[table[b, j // 64], head // (n_q // n_kv), j % 64] = True
        o, l, added, most = _attend(cache, table[b], start, window, weigh, q[own].double().numpy(), scale)
        terms = max(terms, most)
        # bounds as in test_int8_gpu.py: the rows' type's rounding, probabilities of 11 bits, float32 sums
        top = max([np.abs(cache.values(1, [p], 64)).max() for p in table[b] if 0 <= p < n_pages], default=0.0)
        bound = (2.0 ** -9 + 2.0 ** -10 if kind == "bf16" else 4e-6) * top + (2.0 ** -9 * np.abs(o) if kind == "bf16" else 0)
        seen_nan = spoilt & ~np.isneginf(l)
        assert np.isnan(out[own][seen_nan]).all() and np.isnan(lse[own][seen_nan]).all()
        o, l = np.where(seen_nan[..., None], 0, o), np.where(seen_nan, 0, l)
        out[own], lse[own] = np.where(seen_nan[..., None], 0, out[own]), np.where(seen_nan, 0, lse[own])
        assert (np.abs(out[own] - o) <= bound).all(), b
        none = np.isneginf(l)
        assert np.array_equal(np.isneginf(lse[own]), none) and (out[own][none] == 0).all()
        assert (np.abs(lse[own][~none] - l[~none]) <= 4e-6 * np.maximum(1.0, np.abs(l[~none]))).all()
        for p, page in enumerate(table[b]):
            if 0 <= page < n_pages:
                want_weight[page] += added[:, 64 * p:64 * p + 64]
                most_added[page] += added[:, 64 * p:64 * p + 64]
    assert np.isnan(weight[lost]).all()
    weight, want_weight = np.where(lost, 0, weight), np.where(lost, 0, want_weight)
    ok = np.abs(weight - want_weight) <= (1e-5 + 2.0 ** -21 * terms) * (most_added + 1e-3) + 2.0 ** -22 * np.abs(cache.weight)
    assert (ok | (np.isnan(weight) & np.isnan(want_weight))).all()


# head sizes and groups of the kernel of rows (one, two and four tiles of columns), the prompt kernel, and the plain one
HEADS = [(64, 8, 2), (128, 4, 1), (128, 16, 1), (64, 40, 1), (32, 4, 2)]


def _table(rng, n, width):
    """Pages of ``n`` sequences, in no order; two ids stay outside the pool (see ``_check``: it ends two below the largest)."""
    ids = rng.permutation(n * width)
    return (ids + 3).astype(np.int32).reshape(n, width)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,n_q,n_kv", HEADS)
@pytest.mark.parametrize("window", [None, 50, 1000])
def test_single_tokens_whose_start_lies_behind_the_table(monkeypatch, kind, dim, n_q, n_kv, window):
    rng = np.random.default_rng(dim + n_q)
    starts = [3, 127, 128, 190, 5000, MOST, 64, MOST - 1]
    _check(rng, monkeypatch, _table(rng, len(starts), 2), starts, [1] * len(starts), n_q, n_kv, dim, 16, kind, window, weigh=1)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,n_q,n_kv", HEADS)
@pytest.mark.parametrize("window", [None, 50, 1000])
def test_prompts_whose_start_lies_behind_the_table(monkeypatch, kind, dim, n_q, n_kv, window):
    rng = np.random.default_rng(dim * n_q)
    starts, counts = [0, 100, 150, 192, 4000, MOST - 200, 60], [70, 140, 33, 2, 40, 130, 0]
    _check(rng, monkeypatch, _table(rng, len(starts), 3), starts, counts, n_q, n_kv, dim, 32, kind, window, weigh=20)


def _with_holes(table):
    table[0, 1], table[1, 0], table[2, :], table[3, -1] = -1, MOST, -(2 ** 31), table[table < MOST].max() + 2
    return table


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,n_q,n_kv", HEADS)
def test_single_tokens_over_page_ids_that_name_no_page(monkeypatch, kind, dim, n_q, n_kv):
    rng = np.random.default_rng(dim + n_q)
    for window in (None, 40):
        _check(rng, monkeypatch, _with_holes(_table(rng, 4, 4)), [200, 255, 130, 250], [1] * 4, n_q, n_kv, dim, 16, kind, window, weigh=1)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,n_q,n_kv", HEADS)
def test_prompts_over_page_ids_that_name_no_page(monkeypatch, kind, dim, n_q, n_kv):
    rng = np.random.default_rng(dim + n_q)
    for window in (None, 40):
        _check(rng, monkeypatch, _with_holes(_table(rng, 4, 4)), [0, 100, 3, 200], [200, 140, 130, 56], n_q, n_kv, dim, 64, kind, window, weigh=9)


@pytest.mark.parametrize("kind", ["bf16"])
def test_parts_of_keys_over_page_ids_that_name_no_page(monkeypatch, kind):
    """Few rows behind many keys: parts of them, some of which see nothing."""
    rng = np.random.default_rng(9)
    table = _table(rng, 2, 40)
    table[0, 3:25], table[1, 8:], = -1, MOST
    for window in (None, 700):
        _check(rng, monkeypatch, table.copy(), [2400, 2450], [70, 100], 4, 1, 64, 16, kind, window, weigh=2)


# ---- batches of several launches, odd groups, scales --------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_more_single_tokens_than_a_launch_takes(monkeypatch, kind):
    rng, n = np.random.default_rng(3), 1100
    _check(rng, monkeypatch, _table(rng, n, 2), [(31 * i) % 128 for i in range(n)], [1] * n, 2, 1, 64, 16, kind, weigh=1)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_more_prompts_than_a_launch_takes(monkeypatch, kind):
    rng, n = np.random.default_rng(4), 530
    counts = [33 + i % 5 for i in range(n)]
    _check(rng, monkeypatch, _table(rng, n, 2), [(17 * i) % 90 for i in range(n)], counts, 2, 1, 64, 16, kind, weigh=2)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,n_q,n_kv", [(64, 3, 1), (128, 5, 1), (64, 14, 2)])
@pytest.mark.parametrize("window", [1, 70, 200])
def test_odd_groups_in_a_window(monkeypatch, kind, dim, n_q, n_kv, window):
    rng = np.random.default_rng(n_q)
    _check(rng, monkeypatch, _table(rng, 3, 7), [0, 150, 300], [260, 130, 40], n_q, n_kv, dim, 32, kind, window, weigh=5)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("counts", [[1, 1, 1], [150, 1, 30]])
def test_value_scales_very_far_apart(kind, dim, counts):
    """Scales of values up to 2^90 of each other."""
    from test_int8_gpu import _check_attention
    _check_attention(np.random.default_rng(8), [300, 129, 40], counts, 8, 2, dim, 16, kind, weigh=1, v_spread=45)


# ---- queries that are no numbers --------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,n_q,n_kv", HEADS)
@pytest.mark.parametrize("starts,counts,weigh", [([3, 127, 150, 60], [1] * 4, 1), ([0, 100, 3], [70, 92, 1], 20), ([1500, 40], [70, 60], 3)])
def test_a_query_that_is_no_number_spoils_what_it_sees_and_nothing_else(monkeypatch, kind, dim, n_q, n_kv, starts, counts, weigh):
    rng = np.random.default_rng(dim + n_q)
    table = _table(rng, len(starts), -(-max(s + n for s, n in zip(starts, counts)) // 64))
    cu = np.concatenate([[0], np.cumsum(counts)])
    bad = [(cu[1] - 1, 0), (0, n_q - 1), (cu[2] - 1, n_q // 2)]        # sequences' last rows, and a first one that may not account
    _check(rng, monkeypatch, table, starts, counts, n_q, n_kv, dim, 16, kind, 90, weigh, bad)


# ---- host threads -------------------------------------------------------------------------------------------------
def test_the_scratch_of_a_batch_does_not_depend_on_who_asks_beside_it():
    """Threads that ask for batches of other sizes all the time are told what one that asks alone is told."""
    import threading
    from supersonic_b200.csrc import int8_ops
    ask = int8_ops._fn("ssb_int8_attention_scratch")
    sizes = [8, 200, 1000, 60, 700, 1]
    args = lambda n: (1, n, n, 1, 64, 32, 8, 128, 0, 0, 0.125)                               # noqa: E731
    want, wrong = {n: ask(*args(n)) for n in sizes}, []
    assert len(set(want.values())) > 1

    def go(first):
        for i in range(600):
            n = sizes[(first + i) % len(sizes)]
            if ask(*args(n)) != want[n]:
                wrong.append(n)
    threads = [threading.Thread(target=go, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, len(wrong)


def test_two_host_threads_with_batches_of_different_sizes():
    import threading
    from supersonic_b200.cache import Int8Pages
    from supersonic_b200.csrc import int8_ops, ops

    def batch(n, seed):
        gen = torch.Generator(device=DEV).manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=gen, device=DEV)                          # noqa: E731
        pages = Int8Pages(*[(rand(2 * n, 2, 64, 128) * 36).clamp(-127, 127).to(torch.int8) for _ in range(2)],
                          *[rand(2 * n, 2, 4).abs() + 0.01 for _ in range(2)])
        table = torch.arange(2 * n, dtype=torch.int32, device=DEV).reshape(n, 2)
        ints = (_ints(list(range(n + 1))), _ints([(37 * i) % 128 for i in range(n)]), _ints(list(range(n))))
        q = rand(n, 8 * 128)
        torch.cuda.synchronize()

        def run():
            out = torch.empty_like(q)
            int8_ops.attention(q, pages, table, *ints, 1, out, 8, 0.125)
            return out
        return run
    runs = [batch(8, 1), batch(200, 2)]
    want, wrong = [r() for r in runs], []
    torch.cuda.synchronize()

    def go(which):
        with torch.cuda.stream(torch.cuda.Stream()):
            outs = [runs[which]() for _ in range(100)]
            torch.cuda.current_stream().synchronize()
            wrong.extend(which for o in outs if not torch.equal(o, want[which]))
    threads = [threading.Thread(target=go, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    ops.check_device_errors()
    assert not wrong


@pytest.mark.parametrize("rows,start", [(1, 500), (300, 4000)])
def test_a_scratch_that_is_too_small_is_refused(monkeypatch, rows, start):
    from supersonic_b200.cache import Int8Pages
    from supersonic_b200.csrc import int8_ops, ops
    pages = Int8Pages.allocate(80, 1, 64, 16, device=DEV)
    q = torch.zeros((rows, 64), dtype=torch.bfloat16, device=DEV)
    table = torch.arange(80, dtype=torch.int32, device=DEV).reshape(1, 80)
    args = (q, pages, table, _ints([0, rows]), _ints([start]), _ints([0]), rows, torch.zeros_like(q), 1, 0.125)
    size = int8_ops._scratch_size
    int8_ops.attention(*args)
    monkeypatch.setattr(int8_ops, "_scratch_size", lambda *a: size(*a) - 1)
    with pytest.raises(ops.KernelError):
        int8_ops.attention(*args)


# ---- products -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,k", [(8_400_000, 4), (67_200_000, 8)])
def test_rows_beyond_32_bits_of_threads_are_quantised(rows, k):
    """More rows than a launch's threads can be counted in 32 bits, with 256 and with 32 threads a row."""
    from supersonic_b200.csrc import int8_ops
    gen = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.empty((rows, k), dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    codes, scale = torch.full((rows, k), 99, dtype=torch.int8, device=DEV), torch.zeros(rows, device=DEV)
    int8_ops.quantize_rows(x, codes, scale)
    for part in (slice(0, 2000), slice(rows // 2 - 1000, rows // 2 + 1000), slice(rows - 2000, rows)):
        xs = x[part].float().cpu().numpy()
        for i in range(0, 2000, 97):
            want, s = plain.quantize(xs[i])
            assert np.array_equal(codes[part][i].cpu().numpy(), want) and scale[part][i].item() == s
    assert (scale > 0).all()


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_the_largest_sums_of_weights_of_minus_128(rows):
    """Products of 127 x -128 throughout, at the largest k that is taken: a sum of -(2^31 - 131,072)."""
    from supersonic_b200.csrc import int8_ops, ops
    k = int8_ops.MOST_K
    assert 127 * 128 * k < 2 ** 31 <= 127 * 128 * (k + 16)
    x = torch.ones((rows, k), device=DEV)
    x[:, 1::2] = -1
    w = torch.full((8, k), -128, dtype=torch.int8, device=DEV)
    w[:, 1::2] = 127                                              # whose sum is k / 2 times 127 x 255
    w[5, 0::2], w[5, 1::2] = 127, -128
    w[3] = -128
    out, same = torch.zeros((rows, 8), device=DEV), torch.zeros((rows, 8), device=DEV)
    int8_ops.linear(x, w, torch.ones(8, device=DEV), out)
    by = np.float32(1) / np.float32(127)
    assert (out[:, 0] == float(-np.float32(127 * 255 * (k // 2)) * by)).all() and (out[:, 5] == -out[:, 0]).all() and (out[:, 3] == 0).all()
    int8_ops.linear(x.abs(), w, torch.ones(8, device=DEV), same)
    assert (same[:, 3] == float(-np.float32(127 * 128 * k) * by)).all()
    wide = torch.zeros((8, k + 16), dtype=torch.int8, device=DEV)
    with pytest.raises(ops.KernelError):
        int8_ops.linear(torch.ones((rows, k + 16), device=DEV), wide, torch.ones(8, device=DEV), out)


# ---- eviction -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim,block", [(64, 16), (128, 64), (16, 32)])
def test_evict_over_page_ids_that_name_no_page(dim, block):
    """Tokens without a page are the last to be chosen; those that stay all the same are zeros, and spoil nobody's scale."""
    from supersonic_b200.cache import Int8Pages
    from supersonic_b200.csrc import int8_ops
    rng, n_kv, n, keep, first, recent = np.random.default_rng(dim), 2, 700, 500, 10, 70
    table = np.arange(11, dtype=np.int32)[None, ::-1].copy()
    table[0, [0, 3, 7, 10]] = -1, MOST, 30, -5                            # the first tokens, the last ones, and some between
    target = np.arange(11, 19, dtype=np.int32)[None]
    cache = plain.Cache(20, n_kv, dim, block)
    for which in range(2):
        cache.codes[which][:] = np.clip(np.rint(rng.normal(size=cache.codes[which].shape) * 36), -127, 127)
        cache.scale[which][:] = 0.02 * np.exp(0.5 * rng.normal(size=cache.scale[which].shape))
    cache.weight[:] = rng.normal(size=cache.weight.shape)
    cache.weight[table[0, 5], :, ::2] = -np.inf
    pages = Int8Pages(*[torch.from_numpy(t).to(DEV) for t in (*cache.codes, *cache.scale, cache.weight.copy())])
    kept = torch.zeros((1, n_kv, keep), dtype=torch.int32, device=DEV)
    int8_ops.evict(pages, torch.from_numpy(table).to(DEV), _ints([0]), _ints([n]), torch.from_numpy(target).to(DEV), keep, first, recent, kept)
    out = [torch.full((1, keep, n_kv, dim), 9.0, device=DEV) for _ in range(2)]
    int8_ops.read(pages, torch.from_numpy(target).to(DEV), _ints([0]), _ints([keep]), *out)
    there = np.repeat((table[0] >= 0) & (table[0] < 20), 64)[:n]
    for h in range(n_kv):
        w = [cache.weight[table[0, j // 64], h, j % 64] if there[j] else 0.0 for j in range(n)]
        middle = sorted(range(first, n - recent), key=lambda j: (not there[j], -w[j], j))[:keep - first - recent]
        stay = sorted([*range(first), *middle, *range(n - recent, n)])
        assert kept[0, h].tolist() == stay
        for i0 in range(0, keep, block):
            run = stay[i0:i0 + block]
            for which in range(2):
                s = np.array([cache.scale[which][table[0, j // 64], h, j % 64 // block] if there[j] else 0 for j in run], np.float32)
                for i, j in enumerate(run):
                    c = cache.codes[which][table[0, j // 64], h, j % 64].astype(np.float32) if there[j] else np.zeros(dim, np.float32)
                    want = np.rint(c * (s[i] / s.max())) * s.max() if s.max() > 0 else c
                    assert np.array_equal(out[which][0, i0 + i, h].cpu().numpy(), want), (h, i0 + i)
        moved = pages.weight[torch.from_numpy(target[0]).long().to(DEV), h].reshape(-1)[:keep].cpu().numpy()
        assert np.array_equal(moved, [w[j] for j in stay])
