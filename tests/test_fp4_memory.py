"""Whose memory the launches of the 4-bit products work in, with the library's functions taken down instead of called: no GPU."""
import pytest
import torch

from supersonic_b200.csrc import fp4_ops
from supersonic_b200.weights import Fp4Matrix

COUNTERS = 4 * 256                                                # bytes that a product counts in


def matrix(*shape, gated=False):
    m = Fp4Matrix.empty(*shape, device="cpu", gated=gated)
    m.index = 0
    return m


@pytest.fixture
def launches(monkeypatch):
    """What was launched, as [(name, arguments)]; every product needs 4,096 bytes of scratch and counters."""
    made = []

    def fn(name):
        return lambda *args: made.append((name, args)) or 0
    monkeypatch.setattr(fp4_ops, "_fn", fn)
    monkeypatch.setattr(fp4_ops, "_stream", lambda *indices: 0)
    monkeypatch.setattr(fp4_ops, "_error_word", lambda m: 0)
    monkeypatch.setattr(fp4_ops, "_scratch_size", lambda name, *sizes: 2 * 4096 + 1)
    return made


def inside(at, size, tensor):
    return tensor.data_ptr() <= at and at + size <= tensor.data_ptr() + tensor.numel() * tensor.element_size()


@pytest.mark.parametrize("numbers", [True, False])
@pytest.mark.parametrize("gated", [True, False])
def test_what_a_units_second_product_counts_in_is_there_as_long_as_the_rows(launches, numbers, gated):
    x = torch.zeros((40, 64)) if numbers else matrix(40, 64)
    z = fp4_ops.gate_up(x, matrix(128, 64, gated=True)) if gated else fp4_ops.activated(x, matrix(64, 64), "silu")
    *_, scratch, counters, _, _ = launches[-1][1]
    assert inside(counters, 2 * COUNTERS, z._buffer) and inside(scratch, 4096, z._buffer) and counters + 2 * COUNTERS <= scratch
    if not numbers:
        assert not bool(z._buffer[counters - z._buffer.data_ptr():][: 2 * COUNTERS].any())
    fp4_ops.linear(z, matrix(64, 64), torch.zeros((40, 64)))
    *_, scratch2, counters2, _, _ = launches[-1][1]
    assert counters2 == counters + COUNTERS and scratch2 == scratch and z._counters is None
    # rows that are read again: nothing of the first product's is taken twice
    fp4_ops.linear(z, matrix(64, 64), torch.zeros((40, 64)))
    *_, scratch3, counters3, _, _ = launches[-1][1]
    assert not inside(scratch3, 1, z._buffer) and not inside(counters3, 1, z._buffer)


def test_scratch_without_room_is_the_second_products_own(launches, monkeypatch):
    z = fp4_ops.gate_up(matrix(40, 64), matrix(128, 64, gated=True))
    monkeypatch.setattr(fp4_ops, "_scratch_size", lambda name, *sizes: 2 * 8192 + 1)
    fp4_ops.linear(z, matrix(64, 64), torch.zeros((40, 64)))
    *_, scratch, counters, _, _ = launches[-1][1]
    assert inside(counters, COUNTERS, z._buffer) and not inside(scratch, 1, z._buffer)
