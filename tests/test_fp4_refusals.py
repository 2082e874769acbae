"""Matrices in 4 bits on the host, and what the 4-bit operators and the scored router refuse before anything is launched: no GPU."""
import pytest
import torch

import plain_fp4 as pf
from supersonic_b200.csrc import fp4_ops, ops
from supersonic_b200.csrc.ops import KernelError
from supersonic_b200.weights import Fp4Matrix


class OnDevice(torch.Tensor):
    """A host tensor that says it lives on device 0: only the checks are run on it."""

    @staticmethod
    def of(t):
        return t.as_subclass(OnDevice)

    @property
    def is_cuda(self):
        return True

    def get_device(self):
        return 0


@pytest.fixture(autouse=True)
def current_device(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)


def z(*shape, dtype=torch.float32):
    return OnDevice.of(torch.zeros(shape, dtype=dtype))


def matrix(*shape, gated=False):
    m = Fp4Matrix.empty(*shape, device="cpu", gated=gated)
    m.index = 0
    return m


def random_parts(*shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, shape[:-1] + (shape[-1] // 2,), generator=g, dtype=torch.uint8)
    return codes, torch.randint(100, 140, shape[:-1] + (shape[-1] // 32,), generator=g, dtype=torch.uint8)


@pytest.mark.parametrize("shape", [(1, 32), (128, 256), (129, 288), (300, 1024), (3, 40, 64), (2, 200, 544)])
def test_scales_keep_their_places(shape):
    codes, scales = random_parts(*shape)
    m = Fp4Matrix.from_parts(codes, scales)
    assert m.shape == shape and torch.equal(m.plain_scales(), scales) and torch.equal(m.codes, codes)
    # a row's block by the layout's own words: runs of 128 rows x 8 blocks, halves of 4 blocks, 16 bytes a lane
    n, blocks = shape[-2], shape[-1] // 32
    flat, runs = scales.reshape(-1, n, blocks), m.scales.view(-1, -(-n // 128), -(-blocks // 8), 1024)
    for r, b in ((0, 0), (n - 1, blocks - 1), (n // 2, blocks // 2)):
        at = (b // 4 % 2) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4
        assert runs[-1, r // 128, b // 8, at] == flat[-1, r, b]


def test_rows_behind_the_last_and_blocks_behind_k_are_zeros():
    m = Fp4Matrix.from_parts(*random_parts(100, 96))
    assert int((m.scales != 0).sum()) == 100 * 3


@pytest.mark.parametrize("shape", [(64, 32), (128, 64), (2, 192, 96)])
def test_gated_rows_lie_in_sixteens(shape):
    codes, scales = random_parts(*shape)
    m = Fp4Matrix.from_parts(codes, scales, gated=True)
    n = shape[-2]
    for r in range(n // 2):
        at = r // 16 * 32 + r % 16
        assert torch.equal(m.codes[..., at, :], codes[..., r, :]) and torch.equal(m.codes[..., at + 16, :], codes[..., n // 2 + r, :])
    assert torch.equal(m.plain_scales()[..., 16, :], scales[..., n // 2, :])


def test_first_rows_share_memory():
    m = Fp4Matrix.from_parts(*random_parts(300, 64))
    f = m.first_rows(200)
    assert f.shape == (200, 64) and f.codes_at == m.codes_at and torch.equal(f.plain_scales(), m.plain_scales()[:200])
    for bad in (0, 301):
        with pytest.raises(ValueError):
            m.first_rows(bad)
    with pytest.raises(ValueError):
        Fp4Matrix.empty(64, 32, device="cpu", gated=True).first_rows(32)


def test_values_of_every_code():
    codes = torch.arange(16, dtype=torch.uint8).repeat(2).view(1, 32)
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    for byte in (0, 1, 127, 254):
        got = pf.values(Fp4Matrix.from_parts(packed, torch.full((1, 1), byte, dtype=torch.uint8)))[0, :16]
        want = [0, .5, 1, 1.5, 2, 3, 4, 6, -0.0, -.5, -1, -1.5, -2, -3, -4, -6]
        assert got.tolist() == [w * 2.0 ** (byte - 127) for w in want]


@pytest.mark.parametrize("make", [
    lambda: Fp4Matrix.empty(0, 32, device="cpu"), lambda: Fp4Matrix.empty(4, 33, device="cpu"), lambda: Fp4Matrix.empty(4, device="cpu"),
    lambda: Fp4Matrix.empty(2, 2, 2, 32, device="cpu"), lambda: Fp4Matrix.empty(32, 32, device="cpu", gated=True),
    lambda: Fp4Matrix.from_parts(torch.zeros((4, 16), dtype=torch.int8), torch.zeros((4, 1), dtype=torch.uint8)),
    lambda: Fp4Matrix.from_parts(torch.zeros((4, 16), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8)),
    lambda: Fp4Matrix.from_parts(torch.zeros((4, 12), dtype=torch.uint8), torch.zeros((4, 1), dtype=torch.uint8)),
    lambda: Fp4Matrix.from_parts(torch.zeros((4, 16), dtype=torch.uint8), torch.full((4, 1), 255, dtype=torch.uint8)),
    lambda: Fp4Matrix.from_parts(torch.zeros((48, 16), dtype=torch.uint8), torch.zeros((48, 1), dtype=torch.uint8), gated=True),
    lambda: Fp4Matrix(torch.zeros((4, 16), dtype=torch.uint8), torch.zeros((2, 1024), dtype=torch.uint8), (4, 32)),
    lambda: Fp4Matrix(torch.zeros((4, 32), dtype=torch.uint8)[:, :16], torch.zeros((1, 1024), dtype=torch.uint8), (4, 32)),
])
def test_no_such_matrix(make):
    with pytest.raises(ValueError):
        make()


@pytest.mark.parametrize("x, m", [
    (z(4, 64), matrix(4, 32)), (z(4, 32, dtype=torch.float16), matrix(4, 32)), (z(4, 33)[:, 1:], matrix(4, 32)),
    (torch.zeros((4, 32)), matrix(4, 32)), (z(2, 4, 32), matrix(4, 32)), (z(3, 4, 32).transpose(0, 1), matrix(4, 3, 32)),
])
def test_quantize_and_values_refuse(x, m):
    with pytest.raises(KernelError):
        fp4_ops.quantize(x, m)
    with pytest.raises(KernelError):
        fp4_ops.values(m, x)


@pytest.mark.parametrize("kw", [
    {"x": z(3, 32)}, {"x": z(64)}, {"x": z(3, 64, dtype=torch.float16)}, {"x": torch.zeros((3, 64))}, {"x": z(64, 3).t()}, {"x": z(3, 65)[:, 1:]},
    {"x": matrix(3, 32)}, {"x": matrix(2, 3, 64)}, {"w": matrix(12, 64)}, {"w": matrix(2, 16, 64)}, {"w": z(16, 64)},
    {"w": matrix(64, 64, gated=True), "out": z(3, 64)}, {"out": z(3, 24)}, {"out": z(4, 16)}, {"out": z(3, 16, dtype=torch.float64)},
    {"out": z(3, 16, dtype=torch.bfloat16), "add": True}, {"out": torch.zeros((3, 16))}, {"w": Fp4Matrix.empty(16, 64, device="cpu")},
])
def test_linear_refuses(kw):
    with pytest.raises(KernelError):
        fp4_ops.linear(kw.get("x", z(3, 64)), kw.get("w", matrix(16, 64)), kw.get("out", z(3, 16)), accumulate=kw.get("add", False))


def test_inner_rows_are_no_weights_and_results_no_rows():
    size, both = Fp4Matrix.rows_layout(64, 64)
    rows = Fp4Matrix.over_rows(torch.zeros(both, dtype=torch.int8), 64, 64, size)
    rows.index = 0
    for weight in (rows, rows.first_rows(32)):
        weight.index = 0
        with pytest.raises(KernelError, match="not weights"):
            fp4_ops.linear(z(4, 64), weight, z(4, weight.shape[0]))
    x = z(4, 64)
    with pytest.raises(KernelError, match="must not be x"):
        fp4_ops.linear(x, matrix(64, 64), x)


@pytest.mark.parametrize("call", [
    lambda: fp4_ops.gate_up(z(3, 64), matrix(64, 64)), lambda: fp4_ops.gate_up(z(3, 64), matrix(64, 64, gated=True), ("tanh", 0.0)),
    lambda: fp4_ops.gate_up(z(0, 64), matrix(64, 64, gated=True)), lambda: fp4_ops.gate_up(z(3, 32), matrix(64, 64, gated=True)),
    lambda: fp4_ops.gate_up(z(3, 64), matrix(64, 64, gated=True), row_scale=z(2)),
    lambda: fp4_ops.gate_up(z(3, 64), matrix(64, 64, gated=True), row_scale=z(3, dtype=torch.bfloat16)),
    lambda: fp4_ops.activated(z(3, 64), matrix(64, 64, gated=True), "silu"), lambda: fp4_ops.activated(z(3, 64), matrix(64, 64), "tanh"),
    lambda: fp4_ops.activated(z(3, 64), matrix(40, 64), "silu"),
])
def test_inner_rows_refuse(call):
    with pytest.raises(KernelError):
        call()


def experts(x=None, e=None, w=None, first=None, down=None, out=None, act=None, add=False):
    fp4_ops.experts(z(3, 64) if x is None else x, z(3, 2, dtype=torch.int32) if e is None else e, z(3, 2) if w is None else w,
                    matrix(4, 64, 64, gated=True) if first is None else first, matrix(4, 64, 32) if down is None else down,
                    z(3, 64) if out is None else out, act, add)


@pytest.mark.parametrize("kw", [
    {"x": z(3, 32)}, {"e": z(3, 2)}, {"e": z(3, dtype=torch.int32)}, {"e": z(3, 0, dtype=torch.int32), "w": z(3, 0)}, {"w": z(3, 3)},
    {"w": z(3, 2, dtype=torch.bfloat16)}, {"w": z(2, 3).t()}, {"first": matrix(64, 64, gated=True)}, {"first": matrix(4, 64, 64)},
    {"first": matrix(5, 64, 64, gated=True)}, {"down": matrix(4, 64, 64)}, {"down": matrix(4, 32, 64)}, {"out": z(3, 32)}, {"out": z(2, 64)},
    {"act": ("tanh", 0.0)}, {"first": matrix(4, 32, 64), "act": None}, {"first": matrix(4, 32, 64), "act": "tanh"},
    {"out": z(3, 64, dtype=torch.bfloat16), "add": True}, {"e": torch.zeros((3, 2), dtype=torch.int32)},
])
def test_experts_refuse(kw):
    with pytest.raises(KernelError):
        experts(**kw)


def route(logits=None, n=8, e=None, w=None, **kw):
    ops.route_scored(z(3, 8) if logits is None else logits, n, z(3, 2, dtype=torch.int32) if e is None else e, z(3, 2) if w is None else w, **kw)


@pytest.mark.parametrize("kw", [
    {"logits": z(3, 7)}, {"logits": z(3, 8, dtype=torch.bfloat16)}, {"logits": z(2, 8)}, {"logits": z(8, 3).t()}, {"logits": torch.zeros((3, 8))},
    {"e": z(3, 2)}, {"e": z(3, 2, dtype=torch.int64)}, {"w": z(3, 3)}, {"scores": "tanh"}, {"group_score": "three"}, {"groups": 3}, {"groups": 0},
    {"groups": 4, "keep": 5}, {"groups": 8, "keep": 1}, {"groups": 2, "keep": 0}, {"correction": z(7)}, {"correction": z(8, dtype=torch.float64)},
    {"correction": torch.zeros(8)}, {"n": 0}, {"logits": z(3, 4096), "n": 4096}, {"logits": z(3, 64), "n": 64, "groups": 64},
    {"e": z(3, 9, dtype=torch.int32), "w": z(3, 9)}, {"e": z(3, 0, dtype=torch.int32), "w": z(3, 0)},
])
def test_route_refuses(kw):
    with pytest.raises(KernelError):
        route(**kw)


def test_plain_rounding_is_the_nearest_number():
    """The reference itself, on every border between two numbers: the even code, and 6 for what is above it."""
    x = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9] + [0.0] * 23 + [4.0]], dtype=torch.float64)
    assert pf.rounded(x)[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]
    assert pf.rounded(-x)[0, :8].tolist() == [-0.0, -1.0, -1.0, -2.0, -2.0, -4.0, -4.0, -6.0]


def test_a_model_refuses_formats_it_does_not_know():
    from supersonic_b200.config import preset_config, spec_from_config
    from supersonic_b200.engine.model import Model
    spec = spec_from_config(preset_config("tiny-a"))
    with pytest.raises(ValueError, match="weight_format"):
        Model(spec, None, weight_format="int3")
    with pytest.raises(ValueError, match="deterministic"):
        Model(spec, None, weight_format="mxfp4", deterministic=True)


def test_memory_is_estimated_in_the_format():
    from supersonic_b200.config import preset_config
    from supersonic_b200.engine import preflight
    from supersonic_b200.weights import RandomWeightStore
    cfg = preset_config("llama3.1-8b")
    store = RandomWeightStore(cfg, 2)
    spec = cfg.build_spec()
    whole, four = (preflight.weight_bytes(spec, store, torch.bfloat16, f) for f in (None, "mxfp4"))
    layer = 2 * 4096 * 4096 + 2 * 1024 * 4096 + 3 * 14336 * 4096
    assert whole - four == 32 * layer * 2 - 32 * layer * 17 // 32 - 2 * layer


def test_the_command_line_names_the_format():
    from supersonic_b200.cli import build_parser
    assert build_parser().parse_args(["--weight-format", "mxfp4"]).weight_format == "mxfp4"
    assert build_parser().parse_args([]).weight_format is None
    with pytest.raises(SystemExit):
        build_parser().parse_args(["--weight-format", "int3"])
