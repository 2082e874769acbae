"""The 4-bit operators and the scored router on the device, against float64."""
import random

import pytest
import torch

import plain_fp4 as pf

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    x = torch.randn(shape, generator=g, device=DEV)
    x[..., ::37] *= 9.0                                            # some channels are much larger
    return x.to(dtype)


def weight(g, *shape, gated=False, spread=0.05):
    """(Fp4Matrix, its float64 values with the gate rows first)"""
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.weights import Fp4Matrix
    w = torch.randn(shape, generator=g, device=DEV) * spread * torch.exp2(torch.randint(-3, 4, shape[:-1] + (1,), generator=g, device=DEV))
    m = Fp4Matrix.empty(*shape, gated=gated)
    fp4_ops.quantize(w, m)
    return m, pf.rounded(w)


def rows4(x):
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.weights import Fp4Matrix
    m = Fp4Matrix.empty(*x.shape)
    fp4_ops.quantize(x, m)
    return m


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(out, want, slack):
    """|out - want| <= slack, and the rounding to out's type on top."""
    from supersonic_b200.csrc import ops
    ops.check_device_errors()
    bound = slack + (want.abs() + slack) * half_step(out.dtype) + 1e-37
    off = (out.double() - want).abs()
    assert bool((off <= bound).all()), f"{int((off > bound).sum())} of {off.numel()} are off, by {float((off / bound).max())} bounds"


# ---- rows into 4 bits and back ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (64, 2048), (129, 288), (1000, 4096), (5, 40, 64), (1, 8192)])
def test_quantize_has_the_formulas_codes(kind, shape):
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.weights import Fp4Matrix
    x = randn(gen(1), *shape, dtype=TYPES[kind])
    m, out = Fp4Matrix.empty(*shape), torch.full(shape, 7.0, dtype=TYPES[kind], device=DEV)
    fp4_ops.quantize(x, m)
    fp4_ops.values(m, out)
    want = pf.rounded(x.double())
    assert torch.equal(m.plain_scales(), pf.exponents(x.double()).to(torch.uint8))
    assert torch.equal(pf.values(m), want) and torch.equal(out.double(), want)


@pytest.mark.parametrize("shape", [(64, 64), (128, 512), (3, 192, 96)])
def test_quantize_lays_gated_rows(shape):
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.weights import Fp4Matrix
    x = randn(gen(2), *shape)
    m, out = Fp4Matrix.empty(*shape, gated=True), torch.empty(shape, device=DEV)
    fp4_ops.quantize(x, m)
    fp4_ops.values(m, out)
    assert torch.equal(out.double(), pf.rounded(x.double()))
    plain = rows4(x.flatten(0, -2).contiguous())
    again = Fp4Matrix.from_parts(plain.codes.view(shape[:-1] + (-1,)), plain.plain_scales().view(shape[:-1] + (-1,)), gated=True)
    assert torch.equal(again.codes, m.codes) and torch.equal(again.scales, m.scales)


def test_quantize_of_borders_and_of_numbers_that_have_no_code():
    inf, nan = float("inf"), float("nan")
    rows = [[0.0] * 32, [2.0 ** -126] + [2.0 ** -140] * 31, [2.0 ** 127 * 1.99] + [-2.0 ** 120] * 31, [1.0, nan, -nan] + [0.5] * 29,
            [inf, 1.0, -inf] + [2.0 ** 125] * 29, [nan] * 32, [7.999, 6.999, 5.0, 2.5, -3.5, -0.25, 0.75, 1.75] + [4.0] * 24,
            [2.0 ** -149] * 32, [3.0 - 2.0 ** -22] * 32, [-8.0] + [7.5] * 31]
    x = torch.tensor(rows, device=DEV)
    m = rows4(x)
    want = pf.finite(x)
    assert torch.equal(m.plain_scales(), pf.exponents(want).to(torch.uint8)) and torch.equal(pf.values(m), pf.rounded(want))


def test_quantize_reads_and_values_writes_parts_of_wider_matrices():
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.weights import Fp4Matrix
    wide = randn(gen(3), 70, 160, dtype=torch.bfloat16)
    m, out = Fp4Matrix.empty(70, 96), torch.full((70, 160), 5.0, device=DEV)
    fp4_ops.quantize(wide[:, 32:128], m)
    fp4_ops.values(m, out[:, 16:112])
    assert torch.equal(out[:, 16:112].double(), pf.rounded(wide[:, 32:128].double()))
    assert bool((out[:, :16] == 5).all()) and bool((out[:, 112:] == 5).all())


# ---- products ---------------------------------------------------------------------------------------------------------
LINEAR = [(1, 8, 32), (1, 2048, 2048), (2, 136, 288), (8, 1000, 4096), (9, 64, 96), (16, 2040, 2080), (4, 8192, 1024),       # few rows
          (16, 4096, 8192), (3, 16384, 512), (17, 264, 544), (32, 1024, 4096), (33, 2048, 2048), (64, 4096, 1024), (65, 128, 256),
          (100, 1536, 4096), (128, 640, 2016), (129, 4096, 256), (200, 2048, 4096), (300, 264, 288), (257, 256, 32), (1000, 1032, 800),
          (2048, 2048, 512), (70000, 64, 32), (300, 8, 64), (90, 8, 1024), (2, 64, 65536), (1, 40, 32768), (16, 24, 2048), (65, 40, 4096)]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows, n, k", LINEAR)
def test_linear(kind, rows, n, k):
    from supersonic_b200.csrc import fp4_ops
    g = gen(rows * 7 + n + k)
    x = randn(g, rows, k, dtype=TYPES[kind])
    w, wv = weight(g, n, k)
    xv = pf.rounded(x.double())
    want, slack = xv @ wv.t(), pf.sum_slack(xv, wv)
    out = torch.full((rows, n), float("nan"), dtype=TYPES[kind], device=DEV)
    fp4_ops.linear(x, w, out)
    check(out, want, slack)
    was = torch.randn((rows, n), generator=g, device=DEV)
    out = was.clone()
    fp4_ops.linear(x, w, out, accumulate=True)
    check(out, want + was.double(), slack)
    # the same bits from rows that are in 4 bits already, twice
    m = rows4(x)
    for _ in range(2):
        again = torch.full((rows, n), float("nan"), device=DEV)
        fp4_ops.linear(m, w, again)
        both = torch.empty((rows, n), device=DEV)
        fp4_ops.linear(x, w, both)
        assert torch.equal(again, both)


@pytest.mark.parametrize("rows", [1, 12, 40, 300])
def test_linear_of_scales_far_apart(rows):
    """Blocks from 2^-100 to 2^90 beside one another, zeros, and the largest and smallest scales."""
    from supersonic_b200.csrc import fp4_ops
    g = gen(5)
    x = torch.randn((rows, 512), generator=g, device=DEV) * torch.exp2(torch.randint(-100, 40, (rows, 16), generator=g, device=DEV)).repeat_interleave(32, 1)
    x[0, :64] = 0
    w = torch.randn((136, 512), generator=g, device=DEV) * torch.exp2(torch.randint(-20, 50, (136, 16), generator=g, device=DEV)).repeat_interleave(32, 1)
    wm = rows4(w)
    xv, wv = pf.rounded(x.double()), pf.rounded(w.double())
    out = torch.empty((rows, 136), device=DEV)
    fp4_ops.linear(x, wm, out)
    check(out, xv @ wv.t(), pf.sum_slack(xv, wv))


@pytest.mark.parametrize("rows", [2, 20, 260])
def test_linear_of_wild_rows_leaves_the_others(rows):
    from supersonic_b200.csrc import fp4_ops
    g = gen(6)
    x = randn(g, rows, 1024)
    x[1, 5], x[1, 600] = float("nan"), float("inf")
    w, wv = weight(g, 256, 1024)
    out = torch.empty((rows, 256), device=DEV)
    fp4_ops.linear(x, w, out)
    xv = pf.rounded(x.double())
    keep = [r for r in range(rows) if r != 1]
    check(out[keep], (xv @ wv.t())[keep], pf.sum_slack(xv, wv)[keep])


@pytest.mark.parametrize("rows", [3, 24, 400])
def test_linear_reads_and_writes_parts_of_wider_matrices(rows):
    from supersonic_b200.csrc import fp4_ops
    g = gen(7)
    wide = randn(g, rows, 640, dtype=torch.bfloat16)
    w, wv = weight(g, 136, 512)
    out = torch.full((rows, 256), 3.0, dtype=torch.bfloat16, device=DEV)
    fp4_ops.linear(wide[:, 64:576], w, out[:, 64:200])
    xv = pf.rounded(wide[:, 64:576].double())
    check(out[:, 64:200], xv @ wv.t(), pf.sum_slack(xv, wv))
    assert bool((out[:, :64] == 3).all()) and bool((out[:, 200:] == 3).all())


@pytest.mark.parametrize("rows", [4, 20, 50, 100])
@pytest.mark.parametrize("numbers", [True, False])
def test_linear_of_no_rows_and_a_weight_just_made(rows, numbers):
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.weights import Fp4Matrix
    g = gen(8)
    x, w = randn(g, rows, 2048), torch.randn((2048, 2048), generator=g, device=DEV)
    fp4_ops.linear(x[:0], rows4(w), torch.empty((0, 2048), device=DEV))
    xv = pf.rounded(x.double())
    x = x if numbers else rows4(x)
    m, out = Fp4Matrix.empty(2048, 2048), torch.empty((rows, 2048), device=DEV)
    for turn in range(20):                                        # the product is launched behind the kernel that writes its weights
        fresh = w * 2.0 ** turn
        fp4_ops.quantize(fresh, m)
        fp4_ops.linear(x, m, out)
        wv = pf.rounded(fresh.double())
        check(out, xv @ wv.t(), pf.sum_slack(xv, wv))


@pytest.mark.parametrize("rows, n, k", [(1, 2048, 2048), (16, 2048, 8192), (70, 1024, 4096), (512, 512, 1024)])
def test_linear_is_the_same_in_every_run_on_another_stream_and_captured(rows, n, k):
    from supersonic_b200.csrc import fp4_ops
    g = gen(9)
    x, (w, _) = randn(g, rows, k, dtype=torch.bfloat16), weight(g, n, k)
    first = torch.empty((rows, n), device=DEV)
    fp4_ops.linear(x, w, first)
    out = torch.empty_like(first)
    for _ in range(3):
        fp4_ops.linear(x, w, out)
        assert torch.equal(out, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fp4_ops.linear(x, w, out.zero_())
    side.synchronize()
    assert torch.equal(out, first)
    # two captured calls replayed at the same time on two streams, over rows that change
    graphs = []
    for _ in range(2):
        xs, outs, graph = x.clone(), torch.empty_like(first), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            fp4_ops.linear(xs, w, outs)
        graphs.append((graph, xs, outs, torch.cuda.Stream()))
    for turn in range(3):
        for i, (graph, xs, outs, stream) in enumerate(graphs):
            xs.copy_(x * 2.0 ** (turn + i))
        torch.cuda.synchronize()
        for graph, xs, outs, stream in graphs:
            with torch.cuda.stream(stream):
                for _ in range(4):
                    graph.replay()
        torch.cuda.synchronize()
        for i, (graph, xs, outs, stream) in enumerate(graphs):
            assert torch.equal(outs, first * 2.0 ** (turn + i))


# ---- inner rows -------------------------------------------------------------------------------------------------------
def check_inner(z, want, slack):
    """4-bit rows z of numbers that are within ``slack`` of want: every value is the nearest under its block's scale of some such number."""
    from supersonic_b200.csrc import ops
    ops.check_device_errors()
    bytes_, got = z.plain_scales(), pf.values(z)
    low = pf.exponents((want.abs() - slack).clamp(min=0)).to(torch.uint8)
    high = pf.exponents(want.abs() + slack).to(torch.uint8)
    assert bool(((bytes_ >= low) & (bytes_ <= high)).all())
    near = (pf.rounded(want, bytes_) - want).abs()
    # under a scale the numbers above 6 become 6: what is nearest to want is nearest to what is near it, up to twice the slack
    assert bool(((got - want).abs() <= near + 2 * slack + 1e-37).all())
    k = want.shape[-1]
    assert bool((z.scales.view(-1, -(-k // 256), 2, 32, 4, 4)[:, :, :, :, :, :] >= 0).all())


UNIT = [(1, 64, 32), (1, 2048, 2080), (5, 96, 64), (8, 512, 4096), (16, 2048, 8192), (13, 1024, 96), (24, 512, 1056), (40, 1024, 288),
        (70, 512, 2048), (130, 256, 544), (300, 1024, 320), (700, 512, 1056), (1500, 256, 2048)]


@pytest.mark.parametrize("act", [None, ("clamped_swish", 7.0), ("gelu_tanh", 0.0)])
@pytest.mark.parametrize("rows, k, inter", UNIT)
def test_gated_unit(rows, k, inter, act):
    from supersonic_b200.csrc import fp4_ops
    g = gen(rows + k + inter)
    x = randn(g, rows, k, dtype=torch.bfloat16)
    first, fv = weight(g, 2 * inter, k, gated=True, spread=0.01)
    down, dv = weight(g, 64, inter)
    scale = torch.rand((rows,), generator=g, device=DEV) if act else None
    xv = pf.rounded(x.double())
    z = fp4_ops.gate_up(x, first, act, row_scale=scale)
    check_inner(z, *pf.inner(xv, fv, True, act, scale))
    out = torch.empty((rows, 64), device=DEV)
    fp4_ops.linear(z, down, out)
    zv = pf.values(z)
    check(out, zv @ dv.t(), pf.sum_slack(zv, dv))
    fp4_ops.linear(z, down, out.zero_(), accumulate=True)                        # its counters are gone: it takes its own
    check(out, zv @ dv.t(), pf.sum_slack(zv, dv))
    again = fp4_ops.gate_up(rows4(x), first, act, row_scale=scale)
    assert torch.equal(again.codes, z.codes) and torch.equal(again.plain_scales(), z.plain_scales())


@pytest.mark.parametrize("act", ["relu_squared", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows, k, inter", UNIT)
def test_dense_unit(rows, k, inter, act):
    from supersonic_b200.csrc import fp4_ops
    g = gen(rows + k + inter + 1)
    x = randn(g, rows, k)
    up, uv = weight(g, inter, k, spread=0.02)
    down, dv = weight(g, 72, inter)
    z = fp4_ops.activated(x, up, act, scale=0.5)
    want, slack = pf.inner(pf.rounded(x.double()), uv, False, act)
    check_inner(z, want * 0.5, slack * 0.5)
    out = torch.empty((rows, 72), dtype=torch.bfloat16, device=DEV)
    fp4_ops.linear(z, down, out)
    zv = pf.values(z)
    check(out, zv @ dv.t(), pf.sum_slack(zv, dv))


def test_units_one_after_another_on_two_streams():
    """Inner rows made on one stream and read on another, beside a unit of its own there."""
    from supersonic_b200.csrc import fp4_ops
    g = gen(11)
    (first, _), (down, dv) = weight(g, 2 * 2048, 1024, gated=True, spread=0.01), weight(g, 1024, 2048)
    xs = [randn(g, 16, 1024, dtype=torch.bfloat16) for _ in range(2)]
    want = []
    for x in xs:
        out = torch.empty((16, 1024), device=DEV)
        fp4_ops.linear(fp4_ops.gate_up(x, first), down, out)
        want.append(out)
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    outs = [torch.empty((16, 1024), device=DEV) for _ in range(3)]
    for _ in range(10):
        z = fp4_ops.gate_up(xs[0], first)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            fp4_ops.linear(z, down, outs[0])
            fp4_ops.linear(fp4_ops.gate_up(xs[1], first), down, outs[1])
        fp4_ops.linear(z, down, outs[2])
        main.wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(outs[2], want[0])


@pytest.mark.parametrize("rows", [8, 20, 300])
def test_units_captured_and_replayed_at_the_same_time(rows):
    from supersonic_b200.csrc import fp4_ops
    g = gen(12)
    (first, _), (down, _) = weight(g, 2 * 1536, 2048, gated=True, spread=0.01), weight(g, 2048, 1536)
    x = randn(g, rows, 2048, dtype=torch.bfloat16)

    def unit(x, out):
        fp4_ops.linear(fp4_ops.gate_up(x, first), down, out, accumulate=True)
    graphs = []
    for _ in range(2):
        xs, out, graph = x.clone(), torch.zeros((rows, 2048), device=DEV), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            unit(xs, out)
            unit(xs, out)
        graphs.append((graph, xs, out, torch.cuda.Stream()))
    for turn in range(3):
        wants = []
        for graph, xs, out, stream in graphs:
            xs.copy_(randn(g, rows, 2048, dtype=torch.bfloat16))
            out.zero_()
            want = torch.zeros_like(out)
            for _ in range(6):
                unit(xs, want)
            wants.append(want)
        torch.cuda.synchronize()
        for graph, xs, out, stream in graphs:
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for (_, _, out, _), want in zip(graphs, wants))


@pytest.mark.parametrize("rows", [3, 20, 200])
def test_inner_rows_made_before_a_capture(rows):
    """The captured product keeps the counters and the scratch that came with the rows; eager ones beside it have their own."""
    from supersonic_b200.csrc import fp4_ops
    g = gen(13)
    (first, _), (down, _) = weight(g, 2 * 4096, 1024, gated=True, spread=0.01), weight(g, 512, 4096)
    x = randn(g, rows, 1024, dtype=torch.bfloat16)
    want = torch.empty((rows, 512), device=DEV)
    fp4_ops.linear(fp4_ops.gate_up(x, first), down, want)
    z, out, graph = fp4_ops.gate_up(x, first), torch.empty((rows, 512), device=DEV), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        fp4_ops.linear(z, down, out)
    held = [torch.full((1 << 16,), i, dtype=torch.uint8, device=DEV) for i in range(64)]       # whatever was given back is written over
    other = torch.empty_like(out)
    for _ in range(4):
        out.zero_()
        graph.replay()
        fp4_ops.linear(z, down, other)
        assert torch.equal(out, want) and torch.equal(other, want)
    assert all(bool((t == i).all()) for i, t in enumerate(held))


# ---- experts ----------------------------------------------------------------------------------------------------------
EXPERTS = [(1, 64, 32, 4, 2), (1, 2048, 1408, 64, 6), (3, 512, 96, 8, 3), (16, 256, 320, 64, 6), (37, 288, 64, 16, 7), (40, 128, 96, 3, 2),
           (100, 512, 288, 16, 4), (64, 256, 128, 256, 8), (300, 256, 160, 8, 2), (700, 320, 96, 16, 4), (900, 256, 544, 4, 1), (33, 96, 64, 1, 1),
           (300, 256, 160, 40, 2), (40, 4096, 4096, 4, 1), (130, 4096, 4128, 8, 2), (70, 32, 32, 4096, 5), (40, 64, 32, 301, 11)]


def choices(g, tokens, experts, top, lopsided=True):
    score = torch.randn((tokens, experts), generator=g, device=DEV) + (torch.randn((experts,), generator=g, device=DEV) if lopsided else 0)
    best = torch.topk(score, top, dim=-1)
    return best.indices.to(torch.int32), torch.softmax(best.values, dim=-1).contiguous()


def check_experts(x, e, w, first, fv, down, dv, act, dtype, was=None):
    from supersonic_b200.csrc import fp4_ops
    tokens, k = x.shape
    gated = first.gated
    xv = pf.rounded(x.double())
    want = torch.zeros((tokens, k), dtype=torch.float64, device=DEV) if was is None else was.double()
    slack = torch.zeros_like(want)
    for j in range(e.shape[1]):
        for i in range(first.shape[0]):
            at = torch.nonzero(e[:, j] == i).flatten()
            if at.numel() == 0:
                continue
            q, off = pf.between(*pf.inner(xv[at], fv[i], gated, act))
            y, wj = q @ dv[i].t(), w[at, j].double()[:, None]
            want[at] += wj * y
            # what the inner rows may be off, the sums, and the weighted sum's roundings
            slack[at] += wj.abs() * (off @ dv[i].abs().t() + pf.sum_slack(q.abs() + off, dv[i]) + (y.abs() + 1e-30) * (e.shape[1] + 2) * 2.0 ** -23)
    out = torch.full((tokens, k), float("nan"), dtype=dtype, device=DEV) if was is None else was.clone()
    fp4_ops.experts(x, e, w, first, down, out, act, accumulate=was is not None)
    check(out, want, slack + (was.double().abs() * 2.0 ** -23 if was is not None else 0))
    return out


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("tokens, k, inter, experts, top", EXPERTS)
def test_experts(tokens, k, inter, experts, top, kind):
    g = gen(tokens + k + inter + experts)
    x = randn(g, tokens, k, dtype=TYPES[kind])
    (first, fv), (down, dv) = weight(g, experts, 2 * inter, k, gated=True, spread=0.02), weight(g, experts, k, inter)
    e, w = choices(g, tokens, experts, top)
    out = check_experts(x, e, w, first, fv, down, dv, None, TYPES[kind])
    from supersonic_b200.csrc import fp4_ops
    again = torch.empty_like(out)
    for _ in range(2):
        fp4_ops.experts(x, e, w, first, down, again)
        assert torch.equal(again, out)
    was = torch.randn((tokens, k), generator=g, device=DEV)
    check_experts(x, e, w, first, fv, down, dv, None, torch.float32, was)


@pytest.mark.parametrize("tokens", [2, 30, 500])
def test_experts_without_gate(tokens):
    g = gen(20)
    x = randn(g, tokens, 128, dtype=torch.bfloat16)
    (first, fv), (down, dv) = weight(g, 12, 96, 128), weight(g, 12, 128, 96)
    e, w = choices(g, tokens, 12, 3)
    check_experts(x, e, w, first, fv, down, dv, "relu_squared", torch.bfloat16)


@pytest.mark.parametrize("tokens", [1, 9, 80, 600])
def test_experts_that_are_none_or_chosen_twice(tokens):
    g = gen(21)
    x = randn(g, tokens, 96, dtype=torch.bfloat16)
    (first, fv), (down, dv) = weight(g, 5, 128, 96, gated=True, spread=0.02), weight(g, 5, 96, 64)
    e, w = choices(g, tokens, 5, 3)
    e[::2, 1] = e[::2, 0]                                          # twice
    e[::3, 2] = torch.tensor([-1, 5, 2 ** 30, -2 ** 31], device=DEV, dtype=torch.int32)[torch.arange(e[::3].shape[0], device=DEV) % 4]
    check_experts(x, e, w, first, fv, down, dv, None, torch.float32)
    e[:] = -1                                                      # a step that no expert has a part in
    out = torch.full((tokens, 96), float("nan"), device=DEV)
    from supersonic_b200.csrc import fp4_ops
    fp4_ops.experts(x, e, w, first, down, out)
    assert bool((out == 0).all())


@pytest.mark.parametrize("tokens", [4, 200])
def test_experts_all_tokens_to_one_and_parts_of_wider_rows(tokens):
    g = gen(22)
    wide = randn(g, tokens, 256, dtype=torch.bfloat16)
    (first, fv), (down, dv) = weight(g, 64, 64, 128, gated=True, spread=0.02), weight(g, 64, 128, 32)
    e = torch.full((tokens, 1), 63, dtype=torch.int32, device=DEV)
    check_experts(wide[:, 64:192], e, torch.ones((tokens, 1), device=DEV), first, fv, down, dv, None, torch.bfloat16)


def test_experts_captured_with_choices_that_change():
    from supersonic_b200.csrc import fp4_ops
    g = gen(23)
    (first, _), (down, _) = weight(g, 16, 192, 256, gated=True, spread=0.02), weight(g, 16, 256, 96)
    for tokens in (4, 150):
        x, (e, w) = randn(g, tokens, 256, dtype=torch.bfloat16), choices(g, tokens, 16, 4)
        out, graph = torch.empty((tokens, 256), device=DEV), torch.cuda.CUDAGraph()
        fp4_ops.experts(x, e, w, first, down, out)
        with torch.cuda.graph(graph):
            fp4_ops.experts(x, e, w, first, down, out)
        for _ in range(3):
            ne, nw = choices(g, tokens, 16, 4)
            e.copy_(ne)
            w.copy_(nw)
            x.copy_(randn(g, tokens, 256, dtype=torch.bfloat16))
            graph.replay()
            want = torch.empty_like(out)
            fp4_ops.experts(x, ne, nw, first, down, want)
            assert torch.equal(out, want)


# ---- the scored router ------------------------------------------------------------------------------------------------
def check_route(logits, n, top, correction=None, scores="softmax", groups=1, keep=None, by="two", renormalize=True, scale=1.0):
    from supersonic_b200.csrc import ops
    T = logits.shape[0]
    e, w = torch.full((T, top), -7, dtype=torch.int32, device=DEV), torch.full((T, top), float("nan"), device=DEV)
    ops.route_scored(logits, n, e, w, scores, correction, groups, keep, by, renormalize, scale)
    we, ww = pf.route(logits[:, :n].cpu(), None if correction is None else correction.cpu(), scores, groups, groups if keep is None else keep, by, top,
                      renormalize, scale)
    assert e.tolist() == we
    ww = torch.tensor(ww, dtype=torch.float64)
    # the exponential (2 ulp), z - max rounded (|z - max| 2^-24 in the exponent), the sum of up to 2,048 in parts, quotients
    # a logit that is NaN counts as -inf, here as there: a bound of NaN would refuse every weight of its row
    z = logits[:, :n].double().cpu().nan_to_num(nan=-60.0).clamp(-60, 60)
    spread = (z.amax(-1) - z.amin(-1)).clamp(max=120)[:, None]
    assert bool(((w.double().cpu() - ww).abs() <= ww.abs() * (40 + 2 * spread) * 2.0 ** -24 + 1e-36).all())


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n, top, groups, keep, by", [(1, 1, 1, 1, "max"), (8, 2, 1, 1, "max"), (64, 6, 1, 1, "two"), (60, 5, 6, 3, "two"), (256, 8, 8, 4, "two"),
                                                      (256, 8, 8, 4, "max"), (160, 6, 32, 3, "max"), (257, 8, 1, 1, "max"), (512, 10, 16, 5, "two"),
                                                      (2048, 16, 4, 2, "two"), (33, 33, 3, 3, "two"), (40, 40, 1, 1, "max"), (32, 4, 32, 4, "two")])
def test_route(scores, n, top, groups, keep, by):
    g = gen(n + top)
    for T, corrected, renormalize in ((1, True, True), (77, False, False), (301, True, False), (64, True, True)):
        logits = torch.randn((T, n), generator=g, device=DEV) * 2
        correction = torch.randn((n,), generator=g, device=DEV) * 0.1 if corrected else None
        check_route(logits, n, top, correction, scores, groups, keep, by, renormalize, 2.5)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_of_close_and_equal_scores(scores):
    """Logits on a coarse grid, so that many are equal, and corrections that make up for the scores' differences but for a few ulp."""
    g = gen(31)
    logits = torch.randint(-3, 4, (200, 64), generator=g, device=DEV).float() / 2
    check_route(logits, 64, 6, None, scores, 8, 3, "two")
    check_route(logits, 64, 6, torch.zeros(64, device=DEV), scores, 8, 3, "max")
    z = torch.linspace(-2, 2, 64, device=DEV)
    s = torch.softmax(z.double(), 0) if scores == "softmax" else torch.sigmoid(z.double())
    correction = (s.max() - s).float()                              # every choice score is nearly the same
    check_route(z.repeat(50, 1).contiguous(), 64, 8, correction, scores, 8, 4, "two")


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("n, groups, keep", [(24, 1, 1), (24, 8, 3), (128, 1, 1), (512, 16, 5)])
def test_route_of_zeros_of_both_signs(n, groups, keep, scores):
    g = gen(34)
    logits = torch.randint(-2, 2, (40, n), generator=g, device=DEV).float() * 0.5
    logits[torch.rand((40, n), generator=g, device=DEV) < 0.4] = -0.0
    for by in ("max", "two"):
        check_route(logits, n, 5, None, scores, groups, keep, by)
        check_route(logits, n, 5, torch.full((n,), -0.0, device=DEV), scores, groups, keep, by)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_of_rows_that_are_masked_or_wild(scores):
    g = gen(32)
    inf, nan = float("inf"), float("nan")
    logits = torch.randn((12, 32), generator=g, device=DEV)
    logits[0] = -inf
    logits[1] = nan
    logits[2, ::2] = -inf
    logits[3, 5] = nan
    logits[4] = torch.finfo(torch.float32).min
    logits[5, 3] = torch.finfo(torch.float32).max
    logits[6, 1:] = -inf
    logits[7, 20] = inf
    logits[8] = 30.0
    correction = torch.randn((32,), generator=g, device=DEV) * 0.1
    for c in (None, correction):
        check_route(logits, 32, 4, c, scores, 4, 2, "two")
        check_route(logits, 32, 4, c, scores)
    correction[7] = nan
    check_route(logits, 32, 32, correction, scores)


def test_route_reads_wider_rows_and_is_captured():
    from supersonic_b200.csrc import ops
    g = gen(33)
    wide = torch.randn((50, 72), generator=g, device=DEV)
    check_route(wide, 64, 6)
    check_route(wide[:, 4:68], 60, 6, scores="sigmoid")
    e, w, graph = torch.zeros((50, 6), dtype=torch.int32, device=DEV), torch.zeros((50, 6), device=DEV), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.route_scored(wide, 64, e, w)
    wide.copy_(torch.randn((50, 72), generator=g, device=DEV))
    graph.replay()
    assert e.tolist() == pf.route(wide[:, :64].cpu(), None, "softmax", 1, 1, "two", 6, True, 1.0)[0]
    ops.route_scored(wide[:0], 64, e[:0], w[:0])


# ---- parts and models -------------------------------------------------------------------------------------------------
def test_a_router_chooses_and_experts_run_in_one_captured_step():
    """A router's logits, its choice, the experts and the combination, as a layer runs them."""
    from supersonic_b200.csrc import fp4_ops, ops
    g = gen(41)
    (first, fv), (down, dv) = weight(g, 32, 128, 256, gated=True, spread=0.02), weight(g, 32, 256, 64)
    x, router = randn(g, 20, 256, dtype=torch.bfloat16), torch.randn((32, 256), generator=g, device=DEV) * 0.05
    correction = torch.randn((32,), generator=g, device=DEV) * 0.1
    e, w = torch.zeros((20, 4), dtype=torch.int32, device=DEV), torch.zeros((20, 4), device=DEV)
    residual = torch.zeros((20, 256), device=DEV)

    def layer():
        logits = x.float() @ router.t()
        ops.route_scored(logits, 32, e, w, "sigmoid", correction, 4, 2, "two")
        fp4_ops.experts(x, e, w, first, down, residual, accumulate=True)
        return logits
    layer()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = layer()
    x.copy_(randn(g, 20, 256, dtype=torch.bfloat16))
    residual.normal_(generator=g)
    was = residual.clone()
    graph.replay()
    we, ww = pf.route(logits.cpu(), correction.cpu(), "sigmoid", 4, 2, "two", 4, True, 1.0)
    assert e.tolist() == we
    got = residual.clone()
    assert torch.equal(check_experts(x, e, w, first, fv, down, dv, None, torch.float32, was), got)


def build(dtype, tensors):
    from supersonic_b200.csrc.kernel_sets import kernel_set_for
    from supersonic_b200.parts import BuildContext, WeightAccess

    class Store:
        def get(self, name, device):
            return tensors[name].to(device)
    return BuildContext(torch.device(DEV), dtype, kernel_set_for(dtype), WeightAccess(Store(), DEV), 512)


class Ctx:
    def __init__(self, kernels):
        self.kernels = kernels


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("act", [None, {"kind": "gelu_tanh"}])
def test_the_gated_part_in_4_bits(kind, act):
    from supersonic_b200.csrc import fp4_ops
    from supersonic_b200.parts.feed_forward import SwiGLU
    g, dtype = gen(42), TYPES[kind]
    t = {n: (torch.randn(s, generator=g, device=DEV) * 0.05).to(dtype) for n, s in (("gate", (96, 64)), ("up", (96, 64)), ("down", (64, 96)))}
    b = build(dtype, t)
    part = SwiGLU({"hidden_size": 64, "intermediate_size": 96, "activation": act}, {n: n for n in t}, b)
    assert part.to_fp4()
    x, residual = randn(g, 7, 64, dtype=dtype), torch.randn((7, 64), generator=g, device=DEV)
    want = residual.clone()
    first, down = weight_of(torch.cat([t["gate"], t["up"]]), True), weight_of(t["down"])
    fp4_ops.linear(fp4_ops.gate_up(x, first, ("gelu_tanh", 0.0) if act else None), down, want, accumulate=True)
    part.forward(Ctx(b.kernels), x, residual)
    assert torch.equal(residual, want)


def weight_of(w, gated=False):
    from supersonic_b200.parts.fp4 import fp4_of
    return fp4_of(w, gated)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("gated", [True, False])
def test_the_experts_part_in_4_bits_with_a_scored_router(kind, gated):
    from supersonic_b200.csrc import fp4_ops, ops
    from supersonic_b200.parts.experts import Experts
    g, dtype = gen(43), TYPES[kind]
    E, H, I = 6, 64, 32
    t = {}
    for e in range(E):
        t.update({f"gate.{e}": torch.randn((I, H), generator=g, device=DEV) * 0.1, f"up.{e}": torch.randn((I, H), generator=g, device=DEV) * 0.1,
                  f"down.{e}": torch.randn((H, I), generator=g, device=DEV) * 0.1})
    t.update({"weight": torch.randn((E, H), generator=g, device=DEV) * 0.1, "shared.gate": torch.randn((96, H), generator=g, device=DEV) * 0.1,
              "shared.up": torch.randn((96, H), generator=g, device=DEV) * 0.1, "shared.down": torch.randn((H, 96), generator=g, device=DEV) * 0.1})
    t = {n: v.to(dtype) for n, v in t.items()}
    t["correction"] = torch.randn((E,), generator=g, device=DEV) * 0.1
    b = build(dtype, t)
    router = {"kind": "scored", "scores": "sigmoid", "groups": 2, "keep": 1, "group_score": "max", "scale": 2.0}
    params = {"hidden_size": H, "n_experts": E, "top": 2, "expert_size": I, "gated": gated, "router": router,
              "shared": {"intermediate_size": 96} if gated else None, "activation": None if gated else "relu_squared"}
    part = Experts(params, {n: n for n in t}, b)
    assert part.to_fp4() and part.in_fp4 and not part.sums_choices
    x, residual = randn(g, 9, H, dtype=dtype), torch.randn((9, H), generator=g, device=DEV)
    want = residual.clone()
    part.forward(Ctx(b.kernels), x, residual)
    logits = torch.empty((9, 8), device=DEV)
    b.kernels.linear(x, part.router.weight, logits)
    e, w = torch.empty((9, 2), dtype=torch.int32, device=DEV), torch.empty((9, 2), device=DEV)
    ops.route_scored(logits, E, e, w, "sigmoid", t["correction"], 2, 1, "max", True, 2.0)
    names = ("gate", "up") if gated else ("up",)
    first = weight_of(torch.stack([torch.cat([t[f"{n}.{i}"] for n in names]) for i in range(E)]), gated)
    down = weight_of(torch.stack([t[f"down.{i}"] for i in range(E)]))
    fp4_ops.experts(x, e, w, first, down, want, None if gated else "relu_squared", accumulate=True)
    if gated:
        fp4_ops.linear(fp4_ops.gate_up(x, weight_of(torch.cat([t["shared.gate"], t["shared.up"]]), True)), weight_of(t["shared.down"]), want, accumulate=True)
    assert torch.equal(residual, want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "D", "E"])
def test_a_model_in_4_bits_generates_what_it_scores(model_folders, name, dtype):
    """Greedy tokens of captured decode steps against the model's own logits over whole sequences (prompt steps), and its memory."""
    import supersonic_b200
    from supersonic_b200.engine.batch import StepEntry
    d, pc, _ = model_folders[name]
    g = random.Random(5)
    prompts = [[g.randrange(pc["vocab_size"]) for _ in range(n)] for n in (3, 17, 40)]
    eng = supersonic_b200.load(d, dtype=dtype, context_size=128, batch_size=3, weight_format="mxfp4")
    whole = supersonic_b200.load(d, dtype=dtype, context_size=128, batch_size=3)
    assert eng.model.weight_bytes() < whole.model.weight_bytes()
    got = eng.generate(prompts, max_new_tokens=6, ignore_eos=True, batch_size=3)
    assert got == eng.generate(prompts, max_new_tokens=6, ignore_eos=True, batch_size=3)
    assert eng.generate(prompts[1:2], max_new_tokens=6, ignore_eos=True)[0][:1] == got[1][:1]
    scores = eng.score([p + t for p, t in zip(prompts, got)])
    assert all(s.total_nll > 0 and s.scored_tokens == len(p) + 5 for s, p in zip(scores, prompts))
    slot = eng.model.open_sequence()
    logits = eng.model.step([StepEntry(slot, prompts[2], [len(prompts[2]) - 1])])
    eng.model.close_sequence(slot)
    assert int(logits[0].argmax()) == got[2][0]
    with pytest.raises(ValueError):
        eng.int8_session(max_tokens=1024)


def test_experts_on_two_streams_and_of_other_types():
    from supersonic_b200.csrc import fp4_ops
    g = gen(24)
    (first, fv), (down, dv) = weight(g, 16, 192, 256, gated=True, spread=0.02), weight(g, 16, 256, 96)
    runs = []
    for tokens in (6, 200):
        x, (e, w) = randn(g, tokens, 256), choices(g, tokens, 16, 4)
        check_experts(x, e, w, first, fv, down, dv, None, torch.bfloat16)
        want = torch.empty((tokens, 256), device=DEV)
        fp4_ops.experts(x, e, w, first, down, want)
        runs.append((x, e, w, want, torch.empty_like(want), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for x, e, w, want, out, stream in runs:
            with torch.cuda.stream(stream):
                fp4_ops.experts(x, e, w, first, down, out)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, _, _, want, out, _ in runs)


def test_the_command_runs_a_model_in_4_bits(capsys):
    from supersonic_b200.cli import main
    args = ["--preset", "tiny-a", "--random-seed", "2", "--prompt-ids", "5,17,3", "--max-new-tokens", "4"]
    assert main(args + ["--weight-format", "mxfp4"]) == 0
    assert "generated_tokens=4" in "".join(capsys.readouterr())


def test_designs_with_experts_load_in_4_bits():
    """The experts of the other designs, through their own routers."""
    import supersonic_b200
    for preset in ("sotavik-small", "kilisun-small", "ruzunex-small", "ropulix-small"):
        eng = supersonic_b200.load(preset=preset, random_seed=1, context_size=64, batch_size=2, weight_format="mxfp4")
        assert any(getattr(getattr(b, "feed_forward", None), "in_fp4", False) for b in eng.model.blocks), preset
        out = eng.generate([[5, 17, 3], [7, 2, 9, 4, 1]], max_new_tokens=4, ignore_eos=True, batch_size=2)
        assert [len(t) for t in out] == [4, 4]
        eng.model.check_errors()
