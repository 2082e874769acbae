"""More of what the 4-bit operators and the scored router refuse before anything is launched: no GPU."""
import pytest
import torch

from supersonic_b200.csrc import fp4_ops, ops
from supersonic_b200.csrc.ops import KernelError
from supersonic_b200.weights import Fp4Matrix
from test_fp4_refusals import OnDevice, current_device, matrix, z  # noqa: F401


def route(logits, e, w):
    ops.route_scored(logits, 8, e, w)


@pytest.mark.parametrize("logits, e, w", [
    (z(8), z(3, 2, dtype=torch.int32), z(3, 2)), (z(), z(3, 2, dtype=torch.int32), z(3, 2)), (z(3, 8), z(dtype=torch.int32), z()),
    (z(3, 8), z(3, dtype=torch.int32), z(3)), (z(2, 3, 8), z(3, 2, dtype=torch.int32), z(3, 2)), (z(3, 8), z(1, 3, 2, dtype=torch.int32), z(1, 3, 2)),
])
def test_route_refuses_tensors_of_other_dimensions(logits, e, w):
    with pytest.raises(KernelError):
        route(logits, e, w)


@pytest.fixture
def launched(monkeypatch):
    """Whether a call came as far as its launch."""
    made = []
    monkeypatch.setattr(fp4_ops, "_fn", lambda name: lambda *args: made.append(name) or 0)
    monkeypatch.setattr(fp4_ops, "_scratch_size", lambda name, *sizes: 0)
    monkeypatch.setattr(fp4_ops, "_error_word", lambda m: 0)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    monkeypatch.setattr(fp4_ops, "_stream", lambda *indices: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return made


def f32(flat, offset, rows, step, width):
    return OnDevice.of(flat.as_strided((rows, width), (step, 1), offset))


@pytest.mark.parametrize("rows, xs, outs, over", [
    (4, (0, 128, 64), (64, 128, 64), False),                     # two halves of the same rows
    (4, (64, 128, 64), (0, 128, 64), False), (4, (64, 128, 64), (128, 128, 64), False),
    (4, (0, 128, 64), (60, 128, 64), True), (4, (0, 128, 64), (68, 128, 64), True), (4, (64, 128, 64), (188, 128, 64), True),
    (4, (0, 64, 64), (0, 64, 64), True), (4, (0, 64, 64), (4, 64, 64), True), (4, (0, 64, 64), (64, 64, 64), True),
    (4, (0, 64, 64), (252, 64, 64), True), (4, (0, 64, 64), (256, 64, 64), False), (4, (256, 64, 64), (0, 64, 64), False),
    (1, (0, 64, 64), (64, 64, 64), False), (1, (0, 64, 64), (60, 64, 64), True), (1, (64, 64, 64), (4, 64, 64), True),
    (4, (0, 64, 64), (128, 128, 64), True), (4, (0, 64, 64), (0, 64, 8), True), (4, (0, 96, 64), (64, 96, 32), False),
])
def test_linear_refuses_results_over_its_rows(launched, rows, xs, outs, over):
    flat = torch.zeros(2048)
    x, out = f32(flat, xs[0], rows, *xs[1:]), f32(flat, outs[0], rows, *outs[1:])
    shared = {flat.data_ptr() + 4 * (at + r * step + c) for at, step, width in (xs,) for r in range(rows) for c in range(width)} \
        & {flat.data_ptr() + 4 * (at + r * step + c) for at, step, width in (outs,) for r in range(rows) for c in range(width)}
    assert bool(shared) == over
    if over:
        with pytest.raises(KernelError, match="must not be x"):
            fp4_ops.linear(x, matrix(outs[2], 64), out)
        assert not launched
    else:
        fp4_ops.linear(x, matrix(outs[2], 64), out)
        assert launched == ["ssb_fp4_linear"]


def test_linear_refuses_results_over_rows_in_4_bits(launched):
    held = torch.zeros(4096, dtype=torch.uint8)
    m = Fp4Matrix(held[1024:1152].view(4, 32), torch.zeros((1, 1024), dtype=torch.uint8), (4, 64))
    m.index = 0
    for at in (1024, 1136, 2048, 1024 - 16 * 4, 0):
        out = OnDevice.of(held[at:at + 4 * 8 * 4].view(torch.float32).view(4, 8))
        if at in (2048, 0):
            fp4_ops.linear(m, matrix(8, 64), out)
        else:
            with pytest.raises(KernelError, match="must not be x"):
                fp4_ops.linear(m, matrix(8, 64), out)
