"""More of the 4-bit operators on the device: whose memory launches work in, forms that few sizes take, and extremes."""
import pytest
import torch

import plain_fp4 as pf
from test_fp4_gpu import DEV, TYPES, check, check_experts, check_inner, check_route, choices, gen, randn, rows4, weight

pytestmark = pytest.mark.gpu


def written_over():
    """Small and larger tensors, so that whatever was given back to the allocator is written over."""
    return [torch.full((n,), i % 251, dtype=torch.uint8, device=DEV) for n in (2048, 1 << 16) for i in range(128)]


def unchanged(held):
    return all(bool((t == i % 128 % 251).all()) for i, t in enumerate(held))


# ---- whose memory ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("numbers", [True, False])
@pytest.mark.parametrize("rows", [3, 40, 64, 200, 300])
def test_a_captured_product_of_rows_made_before(rows, numbers):
    """Inner rows from rows of either kind; the product that reads them is captured and replayed, whatever is allocated since."""
    from supersonic_b200.csrc import fp4_ops
    g = gen(rows)
    (first, _), (down, dv) = weight(g, 2 * 4096, 1024, gated=True, spread=0.01), weight(g, 512, 4096)
    x = randn(g, rows, 1024, dtype=torch.bfloat16)
    x = x if numbers else rows4(x)
    z, out, graph = fp4_ops.gate_up(x, first), torch.empty((rows, 512), device=DEV), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        fp4_ops.linear(z, down, out)
    held = written_over()
    zv = pf.values(z)
    for _ in range(4):
        out.fill_(float("nan"))
        graph.replay()
        check(out, zv @ dv.t(), pf.sum_slack(zv, dv))
    assert unchanged(held)


@pytest.mark.parametrize("numbers", [True, False])
@pytest.mark.parametrize("rows", [16, 40, 300])
def test_inner_rows_read_on_another_stream(rows, numbers):
    """The second product on another stream, while the first one goes on allocating and writing."""
    from supersonic_b200.csrc import fp4_ops
    g = gen(rows + 1)
    (first, _), (down, _) = weight(g, 2 * 2048, 1024, gated=True, spread=0.01), weight(g, 1024, 2048)
    x = randn(g, rows, 1024, dtype=torch.bfloat16)
    x = x if numbers else rows4(x)
    want, out = torch.empty((rows, 1024), device=DEV), torch.empty((rows, 1024), device=DEV)
    fp4_ops.linear(fp4_ops.gate_up(x, first), down, want)
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    busy = torch.zeros((1 << 24,), device=DEV)
    for _ in range(6):
        z = fp4_ops.gate_up(x, first)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            for _ in range(4):
                busy.add_(1.0)                                    # the product waits behind these
            fp4_ops.linear(z, down, out.fill_(float("nan")))
        held = written_over()
        main.wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and unchanged(held)
        del z


# ---- weights that were just written ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows, n, k", [(1, 2048, 2048), (12, 1024, 4096), (40, 2048, 1024), (300, 1024, 512), (4, 19000, 256)])
@pytest.mark.parametrize("numbers", [True, False])
def test_products_behind_writes_of_every_kind(rows, n, k, numbers):
    """Codes copied by torch, a matrix made of parts on the spot, a view of one that was quantised: the next launch is the product."""
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.weights import Fp4Matrix
    g = gen(rows + n)
    x = randn(g, rows, k)
    sources = [rows4(torch.randn((n, k), generator=g, device=DEV) * 2.0 ** i) for i in range(3)]
    xv, x = pf.rounded(x.double()), x if numbers else rows4(x)
    wants = [(xv @ pf.values(m).t(), pf.sum_slack(xv, pf.values(m))) for m in sources]
    plain = [(m.codes.clone(), m.plain_scales()) for m in sources]
    m, out, some = Fp4Matrix.empty(n, k), torch.empty((rows, n), device=DEV), n // 16 * 8
    torch.cuda.synchronize()
    for _ in range(3):
        for source, parts, (want, slack) in zip(sources, plain, wants):
            m.scales.copy_(source.scales)
            m.codes.copy_(source.codes)
            fp4_ops.linear(x, m, out)
            check(out, want, slack)
            fp4_ops.linear(x, Fp4Matrix.from_parts(*parts), out.zero_())
            check(out, want, slack)
            fp4_ops.linear(x, m.first_rows(some), out[:, :some].zero_())
            check(out, want, slack)


@pytest.mark.parametrize("rows", [2, 12, 40, 300])
def test_products_behind_replays_that_write(rows):
    """A graph that quantises a matrix, products of it in the graph, in another and outside of both."""
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.weights import Fp4Matrix
    g = gen(rows + 40)
    x, source, m = randn(g, rows, 1024), torch.empty((512, 1024), device=DEV), Fp4Matrix.empty(512, 1024).settle()
    outs, xv = [torch.empty((rows, 512), device=DEV) for _ in range(3)], pf.rounded(x.double())
    fp4_ops.linear(x, m, outs[0])
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        fp4_ops.quantize(source, m)
        fp4_ops.linear(x, m, outs[0])
    with torch.cuda.graph(second):
        fp4_ops.linear(x, m, outs[1])
    assert not m.reads_ahead(torch.cuda.current_stream().cuda_stream)
    for turn in range(10):
        source.normal_(generator=g)
        torch.cuda.synchronize()
        first.replay()
        if turn % 2:
            second.replay()
        fp4_ops.linear(x, m, outs[2])
        second.replay()
        wv = pf.rounded(source.double())
        for out in outs:
            check(out, xv @ wv.t(), pf.sum_slack(xv, wv))


# ---- scales at the ends of their range ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("numbers", [True, False])
@pytest.mark.parametrize("rows, n, k", [(1, 136, 512), (8, 136, 512), (12, 136, 512), (12, 136, 4096), (30, 264, 512), (40, 264, 512), (100, 136, 512),
                                        (300, 264, 512), (3, 19000, 512), (24, 19000, 512)])
def test_products_of_scales_at_the_ends(rows, n, k, numbers):
    """Weight scales from 2^-126 to 2^125 against rows of the opposite ones, so that a product of codes with one of its scales alone would leave
    float32 (1,152 2^125) while the whole is of ordinary size; beside them blocks whose products are too small for it."""
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.weights import Fp4Matrix
    g = gen(rows + k)

    def ints(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device=DEV)
    blocks = k // 32
    ends = torch.tensor([1, 250, 60, 190, 2, 252, 127, 5, 240, 10], device=DEV)[torch.arange(blocks, device=DEV) % 10]
    other = (254 - ends).clamp(2, 252)
    other[6] = ends[6] = 1                                        # 2^-252 times codes
    jitter = lambda t, c: (t + ints(-3, 4, c, blocks)).clamp(0, 252).to(torch.uint8)
    wm = Fp4Matrix.from_parts(ints(0, 256, n, k // 2).to(torch.uint8), jitter(ends, n))
    xm = Fp4Matrix.from_parts(ints(0, 256, rows, k // 2).to(torch.uint8), jitter(other, rows))
    if numbers:
        x = torch.empty((rows, k), device=DEV)
        fp4_ops.values(xm, x)
        xv = pf.rounded(x.double())                               # (a block whose largest code is below 4 gets a smaller scale)
    else:
        x, xv = xm, pf.values(xm)
    wv = pf.values(wm)
    out = torch.empty((rows, n), device=DEV)
    fp4_ops.linear(x, wm, out)
    check(out, xv @ wv.t(), pf.sum_slack(xv, wv))


# ---- experts: many tiles, cut wherever a block's share ends ----------------------------------------------------------------------
@pytest.mark.parametrize("tokens, k, inter, experts, top", [(85, 1024, 480, 64, 6), (700, 512, 288, 256, 3), (600, 288, 96, 40, 1), (150, 4096, 4096, 4, 1)])
def test_experts_in_cut_tiles_have_the_same_bits_in_every_run(tokens, k, inter, experts, top):
    """More tiles than blocks, popular experts with several of them, more pairs than one block sorts for itself."""
    from supersonic_b200.csrc import fp4_ops
    g = gen(tokens)
    x = randn(g, tokens, k, dtype=torch.bfloat16)
    (first, fv), (down, dv) = weight(g, experts, 2 * inter, k, gated=True, spread=0.02), weight(g, experts, k, inter)
    e, w = choices(g, tokens, experts, top)
    out = check_experts(x, e, w, first, fv, down, dv, None, torch.float32)
    again = torch.empty_like(out)
    for _ in range(20):
        fp4_ops.experts(x, e, w, first, down, again)
        assert torch.equal(again, out)
    # the tokens in another order are other tiles
    order = torch.randperm(tokens, generator=g, device=DEV)
    check_experts(x[order], e[order].contiguous(), w[order].contiguous(), first, fv, down, dv, None, torch.float32)


# ---- the scored router ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n, top, groups, keep, by", [(32, 12, 1, 1, "max"), (64, 40, 1, 1, "max"), (64, 16, 8, 4, "two"), (256, 20, 1, 1, "max"),
                                                      (256, 31, 8, 5, "two"), (300, 64, 3, 2, "max"), (600, 33, 4, 3, "two")])
def test_route_of_corrections_that_are_infinite_or_no_numbers(n, top, groups, keep, by, scores):
    """A choice score that is NaN counts as minus infinity: as one of that size, and the lower index first."""
    g = gen(n + top)
    inf, nan = float("inf"), float("nan")
    logits = torch.randn((9, n), generator=g, device=DEV)
    for share in (0.3, 0.8, 0.97, 1.0):
        correction = torch.randn((n,), generator=g, device=DEV) * 0.1
        pick = torch.rand((n,), generator=g, device=DEV)
        correction[pick < share] = -inf
        correction[pick < share / 2] = nan
        check_route(logits, n, top, correction, scores, groups, keep, by)
        if by == "max":                                           # (of both infinities there is no sum: below)
            correction[pick < share / 8] = inf
            check_route(logits, n, top, correction, scores, groups, keep, by)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_of_a_group_whose_two_best_have_no_sum(scores):
    """Groups of (inf, -inf), (1, 1) and (2, -inf), two of which are kept: the first's sum counts as minus infinity, as the last's is."""
    from supersonic_b200.csrc import ops
    inf = float("inf")
    correction = torch.tensor([inf, -inf, 1.0, 1.0, 2.0, -inf], device=DEV)
    e, w = torch.empty((3, 3), dtype=torch.int32, device=DEV), torch.empty((3, 3), device=DEV)
    ops.route_scored(torch.zeros((3, 6), device=DEV), 6, e, w, scores, correction, 3, 2, "two")
    assert e.tolist() == [[0, 2, 3]] * 3 and bool(((w - 1 / 3).abs() < 1e-6).all())


# ---- a step's rows against more tiles of channels than there are SMs --------------------------------------------------------------
def drawn(g, *shape, gated=False):
    """(Fp4Matrix of random codes, its float64 values with the gate rows first)"""
    from supersonic_b200.weights import Fp4Matrix
    codes = torch.randint(0, 256, shape[:-1] + (shape[-1] // 2,), generator=g, device=DEV).to(torch.uint8)
    scales = torch.randint(115, 121, shape[:-1] + (shape[-1] // 32,), generator=g, device=DEV).to(torch.uint8)
    return Fp4Matrix.from_parts(codes, scales, gated=gated), pf.values(Fp4Matrix.from_parts(codes, scales))


@pytest.mark.parametrize("numbers", [True, False])
@pytest.mark.parametrize("rows", [1, 8, 16, 17, 32])
@pytest.mark.parametrize("n, k", [(19000, 1056), (28672, 4096), (40000, 288)])
def test_wide_products_of_a_steps_rows(n, k, rows, numbers):
    from supersonic_b200.csrc import fp4_ops
    g = gen(n + rows)
    x, (w, wv) = randn(g, rows, k, dtype=torch.bfloat16), drawn(g, n, k)
    xv, x = pf.rounded(x.double()), x if numbers else rows4(x)
    want, slack = xv @ wv.t(), pf.sum_slack(xv, wv)
    for dtype in TYPES.values():
        out = torch.full((rows, n), float("nan"), dtype=dtype, device=DEV)
        fp4_ops.linear(x, w, out)
        check(out, want, slack)
    was = torch.randn((rows, n), generator=g, device=DEV)
    out = was.clone()
    fp4_ops.linear(x, w, out, accumulate=True)
    check(out, want + was.double(), slack)
    fp4_ops.linear(x, w, was, accumulate=True)
    assert torch.equal(out, was)


@pytest.mark.parametrize("numbers", [True, False])
@pytest.mark.parametrize("rows", [1, 8, 16, 17, 32])
@pytest.mark.parametrize("inter, k", [(9504, 1056), (14336, 4096), (20000, 288)])
def test_wide_units_of_a_steps_rows(inter, k, rows, numbers):
    from supersonic_b200.csrc import fp4_ops
    g = gen(inter + rows)
    x, (first, fv), (down, dv) = randn(g, rows, k, dtype=torch.bfloat16), drawn(g, 2 * inter, k, gated=True), drawn(g, 64, inter)
    xv, x = pf.rounded(x.double()), x if numbers else rows4(x)
    z = fp4_ops.gate_up(x, first)
    check_inner(z, *pf.inner(xv, fv, True, None))
    out = torch.empty((rows, 64), device=DEV)
    fp4_ops.linear(z, down, out)
    check(out, pf.values(z) @ dv.t(), pf.sum_slack(pf.values(z), dv))
    wide, wv = drawn(g, 2 * inter, k)
    z = fp4_ops.activated(x, wide, "relu_squared", scale=0.5)
    want, slack = pf.inner(xv, wv, False, "relu_squared")
    check_inner(z, want * 0.5, slack * 0.5)


# ---- inner rows' scales behind the last channel ------------------------------------------------------------------------------------
@pytest.fixture
def poisoned(monkeypatch):
    """Memory that the operators take is full of ones: scales that are no numbers."""
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: empty(*a, **kw).fill_(-1) if kw.get("dtype") is torch.int8 else empty(*a, **kw))


@pytest.mark.parametrize("numbers", [True, False])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("rows, k, inter", [(1, 512, 96), (8, 512, 1056), (12, 2048, 96), (30, 1024, 1056), (40, 512, 96), (40, 512, 1056), (120, 256, 2016),
                                            (300, 512, 96), (300, 512, 1056), (700, 256, 288), (9, 1056, 19008), (20, 1056, 19008)])
def test_inner_rows_end_in_scales_of_zero(poisoned, rows, k, inter, gated, numbers):
    """Up to a whole k-block, as the product that reads them multiplies what lies there by zeros."""
    from supersonic_b200.csrc import fp4_ops
    g = gen(rows + inter)
    x = randn(g, rows, k, dtype=torch.bfloat16)
    x = x if numbers else rows4(x)
    z = fp4_ops.gate_up(x, drawn(g, 2 * inter, k, gated=True)[0]) if gated else fp4_ops.activated(x, drawn(g, inter, k)[0], "silu")
    runs, blocks = -(-rows // 128), -(-inter // 256) * 8
    scales = z.scales.view(runs, blocks // 8, 2, 32, 4, 4).permute(0, 4, 3, 1, 2, 5).reshape(runs * 128, blocks)
    assert torch.equal(scales[:rows, : inter // 32], z.plain_scales())
    assert inter % 256 and bool((scales[:rows, inter // 32:] == 0).all())
    down, dv = drawn(g, 72, inter)
    out = torch.empty((rows, 72), device=DEV)
    fp4_ops.linear(z, down, out)
    check(out, pf.values(z) @ dv.t(), pf.sum_slack(pf.values(z), dv))


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("tokens, k, inter, experts, top", [(1, 288, 96, 8, 2), (20, 288, 96, 8, 3), (150, 288, 96, 40, 2), (90, 4128, 4128, 4, 1),
                                                            (400, 288, 160, 4, 2)])
def test_experts_in_memory_that_holds_anything(poisoned, tokens, k, inter, experts, top, gated):
    g = gen(tokens + 5)
    x = randn(g, tokens, k, dtype=torch.bfloat16)
    (first, fv), (down, dv) = drawn(g, experts, (2 if gated else 1) * inter, k, gated=gated), drawn(g, experts, k, inter)
    e, w = choices(g, tokens, experts, top)
    check_experts(x, e, w, first, fv, down, dv, None if gated else "silu", torch.float32)


# ---- a model's matrices -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "D", "E"])
def test_a_models_matrices_are_its_weights_in_4_bits(model_folders, name, dtype):
    """Every projection and unit of a loaded model, read back, against the folder's tensors rounded by the formula."""
    import supersonic_b200
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.weights import Fp4Matrix, WeightStore
    folder = model_folders[name][0]
    model = supersonic_b200.load(folder, dtype=dtype, context_size=64, weight_format="mxfp4").model
    store = WeightStore.from_dir(folder)

    def read(m):
        out = torch.empty(m.shape, device=DEV)
        fp4_ops.values(m, out)
        return out.double()

    def stored(part, *roles):
        kind = torch.float32 if dtype == "float32" else torch.bfloat16
        return pf.rounded(torch.cat([store.get(part.weights[r], torch.device(DEV)).to(kind) for r in roles]).double())
    seen = 0
    for block, spec in zip(model.blocks, model.spec.blocks):
        mixer, ff = block.mixer, block.feed_forward
        if isinstance(getattr(mixer, "w_qkv", None), Fp4Matrix):
            assert torch.equal(read(mixer.w_qkv), stored(spec.mixer, "q", "k", "v")) and torch.equal(read(mixer.w_o), stored(spec.mixer, "o"))
            assert torch.equal(read(mixer.w_q), stored(spec.mixer, "q"))
            seen += 1
        if isinstance(getattr(ff, "w_gate_up", None), Fp4Matrix):
            assert torch.equal(read(ff.w_gate_up), stored(spec.feed_forward, "gate", "up")) and torch.equal(read(ff.w_down), stored(spec.feed_forward, "down"))
            seen += 1
    assert seen > 0


def test_a_model_without_such_matrices_is_refused_with_a_line(model_folders, capsys):
    """Sizes that are no multiples of 32: an error that the command prints."""
    import supersonic_b200
    from supersonic_b200.cli import main
    from supersonic_b200.config import ConfigError
    folder = model_folders["C"][0]
    with pytest.raises(ConfigError, match="mxfp4"):
        supersonic_b200.load(folder, context_size=64, weight_format="mxfp4")
    assert main(["--model-dir", folder, "--prompt-ids", "5,17,3", "--max-new-tokens", "2", "--weight-format", "mxfp4"]) == 1
    assert "mxfp4" in capsys.readouterr().err
