"""The 8-bit cache, its attention, its eviction and the 8-bit products against ``plain_int8`` in 64 bits."""
import numpy as np
import pytest
import torch

import plain_int8 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _pages_of(cache, weights=True):
    from supersonic_b200.cache import Int8Pages
    return Int8Pages(*[torch.from_numpy(x.copy()).to(DEV) for x in (cache.codes[0], cache.codes[1], cache.scale[0], cache.scale[1])],
                     torch.from_numpy(cache.weight.copy()).to(DEV) if weights else None)


def _random_cache(rng, lengths, n_kv, dim, block, spare=0, poison=False):
    """A cache with every sequence's tokens in random pages; with ``poison`` the scales and weights that no sequence has a token
    under are NaN."""
    counts = [-(-n // 64) for n in lengths]
    total = sum(counts) + spare * len(lengths) + 2
    order = list(rng.permutation(total))
    cache = plain.Cache(total, n_kv, dim, block)
    per = max(1, max(counts))
    table = np.zeros((len(lengths), per), np.int32)
    owned = np.zeros((total, 64), bool)
    for b, n in enumerate(lengths):
        for p in range(counts[b]):
            table[b, p] = order.pop()
            owned[table[b, p], : min(64, n - 64 * p)] = True
    for which in range(2):
        cache.codes[which][:] = np.clip(np.rint(rng.normal(size=cache.codes[which].shape) * 36), -127, 127)
        cache.scale[which][:] = 0.02 * np.exp(0.6 * rng.normal(size=cache.scale[which].shape))
    cache.weight[:] = np.exp(2 * rng.normal(size=cache.weight.shape))
    if poison:
        live = owned.reshape(total, 64 // block, block).any(-1)
        for which in range(2):
            cache.scale[which][~np.broadcast_to(live[:, None], cache.scale[which].shape)] = np.nan
        cache.weight[~np.broadcast_to(owned[:, None], cache.weight.shape)] = np.nan
    targets = np.array([[order.pop() for _ in range(spare)] for _ in lengths], np.int32)
    return cache, table, targets


def _attend(cache, table, q, starts, counts, slots, n_q, dtype, window=None, weigh=0, scale=None, lse=True):
    """The operator on host data: (out, lse, weight) back on the host."""
    from supersonic_b200.csrc import int8_ops
    pages = _pages_of(cache)
    rows = sum(counts)
    qt = torch.from_numpy(q.astype(np.float32)).to(DEV).to(dtype).reshape(rows, -1)
    out = torch.full_like(qt, float("nan"))
    l = torch.full((rows, n_q), float("nan"), device=DEV) if lse else None
    cu = np.concatenate([[0], np.cumsum(counts)])
    int8_ops.attention(qt, pages, torch.from_numpy(table).to(DEV), _ints(cu), _ints(starts), _ints(slots), max(counts), out, n_q,
                       scale, window=window, lse=l, weigh_last=weigh)
    torch.cuda.synchronize()
    from supersonic_b200.csrc import ops
    ops.check_device_errors()
    return out.float().cpu().numpy().reshape(rows, n_q, -1), None if l is None else l.cpu().numpy(), pages.weight.cpu().numpy()


def _check_attention(rng, starts, counts, n_q, n_kv, dim, block, kind, window=None, weigh=0, slots=None, spread=2.0, v_spread=None):
    dtype = TYPES[kind]
    B = len(starts)
    lengths = [s + n for s, n in zip(starts, counts)]
    cache, table, _ = _random_cache(rng, lengths, n_kv, dim, block, poison=True)
    if v_spread:                                                 # value scales that differ by many powers of two
        cache.scale[1] *= np.exp2(rng.integers(-v_spread, v_spread + 1, cache.scale[1].shape)).astype(np.float32)
    q = rng.normal(size=(sum(counts), n_q, dim)) * spread
    q = torch.from_numpy(q).to(dtype).double().numpy()
    slots = list(range(B)) if slots is None else slots
    scale = dim ** -0.5
    out, lse, weight = _attend(cache, table, q, starts, counts, slots, n_q, dtype, window, weigh, scale)
    want_weight = cache.weight.astype(np.float64)
    row, terms = 0, 0.0
    for b in range(B):
        rows = slice(row, row + counts[b])
        row += counts[b]
        if counts[b] == 0:
            continue
        if slots[b] < 0:
            assert (out[rows] == 0).all() and np.isneginf(lse[rows]).all()
            continue
        pages = table[b, : -(-lengths[b] // 64)]
        o, l, added, most = cache.attend(q[rows], pages, starts[b], scale, window, weigh)
        # a result is a mean of values.  float32: scores are sums of head_dim products good to 2^-22 and come through exponentials
        # good to 2^-21; bfloat16: one rounding to 8 bits, and probabilities of 11 bits
        top = np.abs(cache.values(1, pages, lengths[b])).max()
        bound = (2.0 ** -9 + 2.0 ** -10 if kind == "bf16" else 4e-6) * top + (2.0 ** -9 * np.abs(o) if kind == "bf16" else 0)
        assert (np.abs(out[rows] - o) <= bound).all(), np.abs(out[rows] - o).max() / top
        assert np.abs(lse[rows] - l).max() <= 4e-6 * max(1.0, np.abs(l).max())
        terms = max(terms, most)
        for j in range(lengths[b]):
            want_weight[pages[j // 64], :, j % 64] += added[:, j]
    if weigh:
        # a probability is off by its score's error, which a float32 sum of products has in proportion to their magnitudes
        ok = np.abs(weight - want_weight) <= (1e-5 + 2.0 ** -21 * terms) * (want_weight - cache.weight + 1e-3) + 2.0 ** -22 * np.abs(cache.weight)
        assert (ok | (np.isnan(weight) & np.isnan(want_weight))).all()
    else:
        assert np.array_equal(weight, cache.weight, equal_nan=True)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,n_q,n_kv", [(64, 8, 2), (128, 32, 8), (128, 3, 1), (64, 9, 1), (128, 16, 1), (64, 4, 4), (256, 4, 2), (16, 6, 3),
                                          (32, 40, 2)])
@pytest.mark.parametrize("block", [16, 64])
def test_attention_single_tokens(kind, dim, n_q, n_kv, block):
    rng = np.random.default_rng(dim + n_q)
    starts = [0, 1, 15, 16, 62, 63, 64, 127, 128, 700]
    _check_attention(rng, starts, [1] * len(starts), n_q, n_kv, dim, block, kind, weigh=1)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 17, 64, 200])
def test_attention_single_tokens_in_a_window(kind, window):
    rng = np.random.default_rng(window)
    starts = [0, 15, 16, 17, 63, 64, 65, 199, 200, 500]
    _check_attention(rng, starts, [1] * len(starts), 8, 2, 128, 32, kind, window=window, weigh=1)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_attention_of_one_long_sequence_beside_short_ones(kind):
    rng = np.random.default_rng(5)
    _check_attention(rng, [6000, 3, 0, 64], [1, 1, 1, 1], 8, 2, 64, 16, kind, weigh=1)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,n_q,n_kv,block", [(128, 4, 1, 16), (64, 6, 2, 32), (128, 3, 3, 64), (64, 9, 1, 16), (256, 2, 1, 16), (32, 4, 2, 32)])
def test_attention_prompts(kind, dim, n_q, n_kv, block):
    rng = np.random.default_rng(dim * n_q)
    _check_attention(rng, [0, 0, 5, 64, 130, 0], [1, 65, 0, 64, 131, 257], n_q, n_kv, dim, block, kind, weigh=20)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("window", [1, 50, 128])
def test_attention_prompts_in_a_window(kind, window):
    rng = np.random.default_rng(window)
    _check_attention(rng, [0, 100, 63], [200, 130, 1], 4, 2, 64, 16, kind, window=window, weigh=3)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [130, 40, 0, 7]])
def test_attention_rows_without_a_sequence(kind, counts):
    _check_attention(np.random.default_rng(2), [70, 10, 3, 200], counts, 8, 2, 128, 16, kind, weigh=1, slots=[0, -1, 2, -1])


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("counts", [[1, 1, 1], [150, 1, 30]])
def test_attention_scales_and_scores_far_apart(kind, counts):
    """Value scales from 2^-12 to 2^12 of each other, scores that spread by tens."""
    _check_attention(np.random.default_rng(8), [300, 129, 40], counts, 8, 2, 64, 16, kind, weigh=1, spread=30.0, v_spread=12)


def test_attention_is_the_same_in_every_run_and_on_another_stream():
    rng = np.random.default_rng(3)
    cache, table, _ = _random_cache(rng, [3000, 70, 900], 2, 128, 16)
    q = rng.normal(size=(3, 8, 128))
    first = _attend(cache, table, q, [2999, 69, 899], [1, 1, 1], [0, 1, 2], 8, torch.bfloat16, weigh=1, scale=0.1)
    stream = torch.cuda.Stream()
    for s in (torch.cuda.current_stream(), stream):
        with torch.cuda.stream(s):
            again = _attend(cache, table, q, [2999, 69, 899], [1, 1, 1], [0, 1, 2], 8, torch.bfloat16, weigh=1, scale=0.1)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


def test_attention_reads_rows_of_a_wider_matrix():
    from supersonic_b200.csrc import int8_ops
    rng = np.random.default_rng(4)
    cache, table, _ = _random_cache(rng, [100, 300], 2, 64, 16)
    pages, wide = _pages_of(cache), torch.randn((2, 8 * 64 + 256), device=DEV)
    got = torch.zeros((2, 8 * 64 + 64), device=DEV)
    args = (torch.from_numpy(table).to(DEV), _ints([0, 1, 2]), _ints([99, 299]), _ints([0, 1]), 1)
    int8_ops.attention(wide, pages, *args, got, 8, 0.125)
    want = torch.zeros((2, 8 * 64), device=DEV)
    int8_ops.attention(wide[:, : 8 * 64].contiguous(), pages, *args, want, 8, 0.125)
    assert torch.equal(got[:, : 8 * 64], want) and (got[:, 8 * 64:] == 0).all()


# ---- append -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("dim,n_q,n_kv,block,rot", [(128, 4, 2, 16, 128), (64, 3, 1, 32, 64), (64, 2, 2, 64, 32), (256, 2, 1, 64, 256),
                                                    (16, 1, 1, 16, 0), (32, 0, 3, 16, 32), (128, 8, 1, 64, 128)])
def test_append(kind, dim, n_q, n_kv, block, rot):
    """Steps of several sequences one after another: whole blocks, pieces of blocks, single tokens, a scale that grows, zeros."""
    from supersonic_b200.csrc import int8_ops
    rng = np.random.default_rng(dim + block)
    dtype = TYPES[kind]
    cache, table, _ = _random_cache(rng, [200, 300, 64], n_kv, dim, block)
    pages, host = _pages_of(cache), cache
    angle = np.arange(400)[:, None] / 50.0 * np.exp(-np.arange(max(rot // 2, 1)) / 7.0)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    tables = [torch.from_numpy(t).to(DEV) for t in (cos, sin)] if rot else [None, None]
    held = [0, 3, 0]
    for step, counts in enumerate([[70, 17, 1], [1, 1, 1], [1, 0, 13], [block, 2 * block + 1, 0], [1, 1, 1], [2, 90, 40]]):
        T = sum(counts)
        x = rng.normal(size=(T, n_q + 2 * n_kv, dim)) * np.exp(rng.normal(size=(T, 1, 1)))
        if step == 2:
            x[0] = 0
        xt = torch.from_numpy(x).to(DEV).to(dtype).reshape(T, -1)
        x = xt.float().cpu().numpy().reshape(x.shape)
        place = np.concatenate([np.arange(h, h + n) for h, n in zip(held, counts)]).astype(np.int32)
        slot = np.concatenate([np.full(n, b) for b, n in enumerate(counts)]).astype(np.int32)
        pos = place + 5                                            # positions and places differ once tokens were evicted
        out = xt if step == 3 else torch.zeros_like(xt)            # in place, too
        int8_ops.append(xt, *tables, _ints(pos), _ints(place), _ints(slot), torch.from_numpy(table).to(DEV), pages, out, n_q)
        turned = x.copy()
        if rot:
            turned[:, : n_q + n_kv] = plain.rotate(x[:, : n_q + n_kv], cos[pos][:, None], sin[pos][:, None])
        want, row = turned.copy(), 0
        for b, n in enumerate(counts):
            rows = slice(row, row + n)
            row += n
            back = host.append(turned[rows, n_q:n_q + n_kv], turned[rows, n_q + n_kv:], table[b], held[b])
            want[rows, n_q:n_q + n_kv], want[rows, n_q + n_kv:] = back
            held[b] += n
        rounded = torch.from_numpy(want).to(dtype).float().numpy()
        assert np.array_equal(out.float().cpu().numpy().reshape(want.shape), rounded)
        for got, ref in zip(pages, (*host.codes, *host.scale, host.weight)):
            assert np.array_equal(got.cpu().numpy(), ref)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("counts", [[250, 3, 200, 67], [1] * 300, [2100, 33, 1, 500]])
def test_append_of_many_tokens(kind, block, counts):
    """Steps of hundreds and thousands of tokens behind tokens that are there, then one more step of one token each."""
    from supersonic_b200.csrc import int8_ops
    rng = np.random.default_rng(len(counts) + block)
    dtype, n_q, n_kv, dim, rot = TYPES[kind], 3, 2, 64, 64
    held = [5 + 3 * b % 40 for b in range(len(counts))]
    cache, table, _ = _random_cache(rng, [h + n + 1 for h, n in zip(held, counts)], n_kv, dim, block)
    cos, sin = (f(np.arange(2300)[:, None] / 50.0 * np.exp(-np.arange(rot // 2) / 7.0)).astype(np.float32) for f in (np.cos, np.sin))
    tables = [torch.from_numpy(t).to(DEV) for t in (cos, sin)]
    for n_new in (counts, [1] * len(counts)):
        pages, T = _pages_of(cache), sum(n_new)
        x = rng.normal(size=(T, n_q + 2 * n_kv, dim)) * np.exp(rng.normal(size=(T, 1, 1)))
        xt = torch.from_numpy(x).to(DEV).to(dtype).reshape(T, -1)
        x = xt.float().cpu().numpy().reshape(x.shape)
        place = np.concatenate([np.arange(h, h + n) for h, n in zip(held, n_new)]).astype(np.int32)
        slot = np.concatenate([np.full(n, b) for b, n in enumerate(n_new)]).astype(np.int32)
        out = torch.zeros_like(xt)
        int8_ops.append(xt, *tables, _ints(place), _ints(place), _ints(slot), torch.from_numpy(table).to(DEV), pages, out, n_q)
        turned = x.copy()
        turned[:, : n_q + n_kv] = plain.rotate(x[:, : n_q + n_kv], cos[place][:, None], sin[place][:, None])
        want, row = turned.copy(), 0
        for b, n in enumerate(n_new):
            rows = slice(row, row + n)
            row += n
            back = cache.append(turned[rows, n_q:n_q + n_kv], turned[rows, n_q + n_kv:], table[b], held[b])
            want[rows, n_q:n_q + n_kv], want[rows, n_q + n_kv:] = back
            held[b] += n
        rounded = torch.from_numpy(want).to(dtype).float().numpy()
        assert np.array_equal(out.float().cpu().numpy().reshape(want.shape), rounded)
        for got, ref in zip(pages, (*cache.codes, *cache.scale, cache.weight)):
            assert np.array_equal(got.cpu().numpy(), ref)


def test_append_of_numbers_that_have_no_code():
    from supersonic_b200.csrc import int8_ops
    from supersonic_b200.cache import Int8Pages
    pages = Int8Pages.allocate(1, 1, 16, 16, device=DEV)
    x = torch.zeros((2, 48), device=DEV)
    x[0, 16], x[0, 17], x[0, 18], x[1, 32], x[1, 33] = float("nan"), 2.0, -1.0, float("-inf"), 5.0
    out = torch.empty_like(x)
    int8_ops.append(x, None, None, _ints([0, 1]), _ints([0, 1]), _ints([0, 0]), _ints([[0]]), pages, out, 1)
    k, v = pages.k[0, 0].cpu().numpy(), pages.v[0, 0].cpu().numpy()
    assert list(k[0, :3]) == [0, 127, -64] and pages.k_scale[0, 0, 0].item() == float(np.float32(2) * (np.float32(1) / np.float32(127)))
    assert list(v[1, :2]) == [-127, 0] and np.isfinite(pages.v_scale.cpu().numpy()).all()
    assert torch.isfinite(out).all()


def test_append_passes_over_rows_without_a_place():
    from supersonic_b200.csrc import int8_ops
    from supersonic_b200.cache import Int8Pages
    pages = Int8Pages.allocate(3, 2, 64, 16, weights=True, device=DEV)
    before = [t.clone() for t in pages]
    x = torch.randn((4, (2 + 4) * 64), device=DEV)
    out = torch.full_like(x, 7.0)
    int8_ops.append(x, None, None, _ints([0] * 4), _ints([0, 64, -1, 3]), _ints([-1, 0, 0, 9]), _ints([[1]]), pages, out, 2)
    assert all(torch.equal(a, b) for a, b in zip(before, pages)) and (out == 7.0).all()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_read(kind):
    from supersonic_b200.csrc import int8_ops
    rng = np.random.default_rng(1)
    cache, table, _ = _random_cache(rng, [130, 64, 1], 3, 64, 32)
    out = [torch.full((4, 100, 3, 64), 9.0, device=DEV, dtype=TYPES[kind]) for _ in range(2)]
    slots, lengths = [0, 2, -1, 1], [130, 1, 50, 0]
    int8_ops.read(_pages_of(cache), torch.from_numpy(table).to(DEV), _ints(slots), _ints(lengths), *out)
    for which in range(2):
        got = out[which].float().cpu().numpy()
        for b, (s, n) in enumerate(zip(slots, lengths)):
            n = 0 if s < 0 else min(n, 100)
            want = cache.values(which, table[s], n).astype(np.float32)
            assert np.array_equal(got[b, :n], torch.from_numpy(want).to(TYPES[kind]).float().numpy())
            assert (got[b, n:] == 9.0).all()


# ---- eviction ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim,n_kv,block", [(64, 2, 16), (128, 1, 64), (16, 3, 32)])
@pytest.mark.parametrize("keep,first,recent", [(1, 0, 0), (1, 0, 1), (64, 4, 16), (100, 0, 100), (65, 65, 0), (200, 3, 50), (5000, 4, 100)])
def test_evict(dim, n_kv, block, keep, first, recent):
    from supersonic_b200.csrc import int8_ops
    rng = np.random.default_rng(keep + dim)
    lengths = [0, 1, 64, 199, 201, 900, 2100]
    cache, table, targets = _random_cache(rng, lengths, n_kv, dim, block, spare=-(-keep // 64), poison=True)
    cache.weight[table[5, 3]] = np.round(cache.weight[table[5, 3]])       # ties
    cache.weight[table[6, :8]] = 0.25
    cache.weight[table[6, 9, None], :, ::3] = np.nan
    cache.weight[table[6, 10, None], :, ::2] = -np.inf
    cache.weight[table[6, 11, None], :, 1::2] = -0.0
    cache.weight[table[6, 12, None], :, 1::5] = np.inf
    pages = _pages_of(cache)
    slots = [0, 1, 2, 3, 4, 5, 6]
    kept = torch.full((len(slots) + 1, n_kv, keep), 77, dtype=torch.int32, device=DEV)
    more = np.concatenate([targets, targets[:1]])                         # the last row has no slot
    int8_ops.evict(pages, torch.from_numpy(table).to(DEV), _ints(slots + [-1]), _ints(lengths + [50]),
                   torch.from_numpy(more).to(DEV), keep, first, recent, kept)
    kept = kept.cpu().numpy()
    for b, n in enumerate(lengths):
        assert np.array_equal(kept[b], cache.evict(table[b], n, targets[b], keep, first, recent)), b
    assert (kept[-1] == -1).all()
    for got, ref in zip(pages, (*cache.codes, *cache.scale, cache.weight)):
        assert np.array_equal(got.cpu().numpy(), ref, equal_nan=True)


@pytest.mark.parametrize("n,keep", [(40000, 3000), (100001, 70)])
def test_evict_long_sequences(n, keep):
    """Weights with many ties, by sorting."""
    from supersonic_b200.csrc import int8_ops
    rng = np.random.default_rng(n)
    cache, table, targets = _random_cache(rng, [n], 2, 16, 64, spare=-(-keep // 64))
    cache.weight[:] = np.round(np.exp(cache.weight.clip(0, 5)) * 4) / 4
    pages = _pages_of(cache)
    kept = torch.zeros((1, 2, keep), dtype=torch.int32, device=DEV)
    int8_ops.evict(pages, torch.from_numpy(table).to(DEV), _ints([0]), _ints([n]), torch.from_numpy(targets).to(DEV), keep, 4, 20, kept)
    for h in range(2):
        w = cache.weight[table[0], h].reshape(-1)[:n]
        middle = 4 + np.argsort(-w[4:n - 20], kind="stable")[:keep - 24]
        want = np.sort(np.concatenate([np.arange(4), middle, np.arange(n - 20, n)]))
        assert np.array_equal(kept[0, h].cpu().numpy(), want)


@pytest.mark.parametrize("n,keep", [(5000, 300), (140001, 6000)])
def test_evict_with_weights_off_16_bytes(n, keep):
    """Weights that begin anywhere, in sequences of which a block holds more places than it keeps ranks, too."""
    from supersonic_b200.cache import Int8Pages
    from supersonic_b200.csrc import int8_ops
    rng = np.random.default_rng(n)
    cache, table, targets = _random_cache(rng, [n], 1, 16, 64, spare=-(-keep // 64))
    pages = _pages_of(cache)
    off = torch.zeros(pages.weight.numel() + 1, dtype=torch.float32, device=DEV)
    weight = off[1:].view(pages.weight.shape)
    weight.copy_(pages.weight)
    kept = torch.zeros((1, 1, keep), dtype=torch.int32, device=DEV)
    int8_ops.evict(Int8Pages(*pages[:4], weight), torch.from_numpy(table).to(DEV), _ints([0]), _ints([n]), torch.from_numpy(targets).to(DEV),
                   keep, 0, 33, kept)
    w = cache.weight[table[0], 0].reshape(-1)[:n - 33]
    want = np.sort(np.concatenate([np.argsort(-w, kind="stable")[:keep - 33], np.arange(n - 33, n)]))
    got = kept[0, 0].cpu().numpy()
    assert np.array_equal(got, want)
    moved = weight.cpu().numpy()[targets[0, :-(-keep // 64)], 0].reshape(-1)[:keep]
    assert np.array_equal(moved, cache.weight[table[0], 0].reshape(-1)[got])


# ---- products ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("rows,n,k", [(1, 8, 16), (3, 64, 48), (8, 136, 4096), (17, 72, 512), (65, 200, 1040), (130, 128, 128), (257, 520, 272),
                                      (300, 264, 2048), (1030, 776, 144)])
def test_linear(kind, rows, n, k):
    from supersonic_b200.csrc import int8_ops
    rng = np.random.default_rng(rows * n)
    dtype = TYPES[kind]
    x = torch.from_numpy(rng.normal(size=(rows, k)) * np.exp(rng.normal(size=(rows, 1)) * 3)).to(DEV).to(dtype)
    if rows > 2:
        x[1] = 0
        x[2, 0], x[2, 1] = float("nan"), float("inf")
    w = rng.integers(-127, 128, size=(n, k)).astype(np.int8)
    sw = np.exp(rng.normal(size=n)).astype(np.float32)
    wt, swt = torch.from_numpy(w).to(DEV), torch.from_numpy(sw).to(DEV)
    codes, scales = torch.zeros((rows, k), dtype=torch.int8, device=DEV), torch.zeros(rows, device=DEV)
    int8_ops.quantize_rows(x, codes, scales)
    xs = x.float().cpu().numpy()
    want_codes = np.zeros((rows, k), np.int8)
    want_scale = np.zeros(rows, np.float32)
    for i in range(rows):
        want_codes[i], want_scale[i] = plain.quantize(xs[i])
    assert np.array_equal(codes.cpu().numpy(), want_codes) and np.array_equal(scales.cpu().numpy(), want_scale)
    scaled = (want_codes.astype(np.int64) @ w.T.astype(np.int64)).astype(np.float64) * want_scale[:, None].astype(np.float64)
    exact = scaled * sw
    out = torch.full((rows, n), float("nan"), device=DEV, dtype=dtype)
    int8_ops.linear(x, wt, swt, out)
    # an exact integer rounded to float32, and two products; bfloat16 has 8 bits: a rounding is up to 2^-8 of its number.  The row
    # with an infinity may leave float32 before the channel's scale
    bound = (4 * 2.0 ** -24 + (2.0 ** -8 if kind == "bf16" else 0)) * np.abs(exact)
    fine = np.maximum(np.abs(exact), np.abs(scaled)) < 3e38
    got = out.float().cpu().numpy()
    assert (np.abs(got - exact)[fine] <= bound[fine]).all()
    base = torch.from_numpy(rng.normal(size=(rows, n)).astype(np.float32)).to(DEV)
    added = base.clone()
    int8_ops.linear(x, wt, swt, added, accumulate=True)
    total = exact + base.cpu().numpy().astype(np.float64)
    err = np.abs(added.cpu().numpy() - total)
    assert (err[fine] <= (5 * 2.0 ** -24 * np.abs(exact) + 2.0 ** -23 * np.abs(total))[fine]).all()


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_linear_of_the_largest_sums(rows):
    """Every product 127 x 127: the sum needs 31 bits."""
    from supersonic_b200.csrc import int8_ops
    k = int8_ops.MOST_K
    x = torch.ones((rows, k), device=DEV)
    w = torch.full((8, k), -127, dtype=torch.int8, device=DEV)
    w[3] = 127
    out = torch.zeros((rows, 8), device=DEV)
    int8_ops.linear(x, w, torch.ones(8, device=DEV), out)
    want = np.float32(127 * 127 * k) * (np.float32(1) / np.float32(127))
    assert (out[:, 3] == float(want)).all() and (out[:, 0] == -float(want)).all()


@pytest.mark.parametrize("n,k", [(1024, 4096), (4096, 1152), (28672, 1024), (2056, 8208), (16384, 2048), (520, 14336)])
@pytest.mark.parametrize("rows", [1, 9, 31, 50, 72, 128, 200, 320, 700])
def test_linear_has_the_formulas_bits_however_it_is_cut(rows, n, k):
    """Whole tiles, equal parts of tiles, shares that end anywhere and pairs: exact sums, then the formula's two float32 products."""
    from supersonic_b200.csrc import int8_ops
    gen = torch.Generator(device=DEV).manual_seed(rows + n)
    x = torch.randn((rows, k), generator=gen, device=DEV).to(torch.bfloat16)
    w = torch.randint(-127, 128, (n, k), generator=gen, device=DEV, dtype=torch.int8)
    sw = torch.rand((n,), generator=gen, device=DEV) + 0.01
    codes, scales = torch.zeros((rows, k), dtype=torch.int8, device=DEV), torch.zeros(rows, device=DEV)
    int8_ops.quantize_rows(x, codes, scales)
    sums = torch.cat([codes.double() @ part.double().T for part in w.split(4096)], dim=1)      # whole numbers below 2^53: exact
    want = sums.float() * scales[:, None] * sw
    base = torch.randn((rows, n), generator=gen, device=DEV)
    out, added = torch.full((rows, n), float("nan"), device=DEV), base.clone()
    int8_ops.linear(x, w, sw, out)
    int8_ops.linear(x, w, sw, added, accumulate=True)
    assert torch.equal(out, want) and torch.equal(added, want + base)


def test_linear_reads_and_writes_parts_of_wider_matrices():
    from supersonic_b200.csrc import int8_ops
    x = torch.randn((70, 512), device=DEV).bfloat16()
    w = torch.randint(-127, 128, (144, 512), dtype=torch.int8, device=DEV)
    sw = torch.rand(144, device=DEV)
    out, want = torch.zeros((70, 256), device=DEV, dtype=torch.bfloat16), torch.zeros((70, 144), device=DEV, dtype=torch.bfloat16)
    int8_ops.linear(x[:, 128:384], w[:, :256], sw, out[:, 8:152])
    int8_ops.linear(x[:, 128:384].contiguous(), w[:, :256].contiguous(), sw, want)
    assert torch.equal(out[:, 8:152], want) and (out[:, :8] == 0).all() and (out[:, 152:] == 0).all()


def test_linear_is_the_same_in_every_run_and_batch():
    """Integer sums have no order: a row's result does not depend on what is beside it, nor on the kernel that took it."""
    from supersonic_b200.csrc import int8_ops
    x = torch.randn((700, 1024), device=DEV).bfloat16()
    w = torch.randint(-127, 128, (384, 1024), dtype=torch.int8, device=DEV)
    sw = torch.rand(384, device=DEV)
    whole = torch.zeros((700, 384), device=DEV)
    int8_ops.linear(x, w, sw, whole)
    for rows in (1, 2, 9, 33, 64, 65, 129, 300):
        part = torch.zeros((rows, 384), device=DEV)
        int8_ops.linear(x[:rows], w, sw, part)
        assert torch.equal(part, whole[:rows]), rows


@pytest.mark.parametrize("rows", [2, 100, 2000])
def test_linear_on_a_side_stream_and_no_wait_runs_out(rows):
    from supersonic_b200.csrc import int8_ops, ops
    x, w = torch.randn((rows, 640), device=DEV), torch.randint(-127, 128, (2064, 640), dtype=torch.int8, device=DEV)
    sw = torch.rand(2064, device=DEV)
    want, got = torch.zeros((rows, 2064), device=DEV), torch.zeros((rows, 2064), device=DEV)
    int8_ops.linear(x, w, sw, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            int8_ops.linear(x, w, sw, got)
    side.synchronize()
    ops.check_device_errors()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dim,n_q,n_kv,window", [(128, 4, 1, None), (64, 6, 2, None), (128, 3, 3, 700), (64, 4, 1, 1500)])
def test_attention_of_few_new_tokens_behind_many(dim, n_q, n_kv, window):
    """Few tiles of rows and many keys: the keys are cut into parts, as many as each sequence has room for."""
    rng = np.random.default_rng(dim + n_q)
    _check_attention(rng, [2100, 3, 900, 5000], [70, 130, 64, 1], n_q, n_kv, dim, 16, "bf16", window=window, weigh=2)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_attention_of_a_few_tokens_a_sequence(kind):
    """Between one token and a tile of them: rows of several tokens and heads share a block's columns."""
    rng = np.random.default_rng(11)
    for n_q, n_kv, dim in ((4, 1, 64), (6, 2, 128), (8, 8, 64), (16, 1, 128)):
        _check_attention(rng, [300, 61, 0, 1000], [3, 7, 16, 33], n_q, n_kv, dim, 32, kind, weigh=5)


def test_numbers_that_do_not_fit_their_type_are_refused():
    from supersonic_b200.cache import Int8Pages
    from supersonic_b200.csrc import int8_ops, ops
    pages = Int8Pages.allocate(1, 1, 64, 16, device=DEV)
    q = torch.zeros((1, 64), dtype=torch.bfloat16, device=DEV)
    for window in (2 ** 40, -1):
        with pytest.raises(ops.KernelError):
            int8_ops.attention(q, pages, _ints([[0]]), _ints([0, 1]), _ints([0]), _ints([0]), 1, torch.zeros_like(q), 1, 0.125, window=window)
