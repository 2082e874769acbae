"""Whose memory the launches of the 4-bit products work in, with the library's functions taken down instead of called: no GPU."""
import pytest
import torch

from supersonic_b200.csrc import fp4_ops
from supersonic_b200.weights import Fp4Matrix

COUNTERS = 4 * 256                                                # bytes that a product counts in


def matrix(*shape, gated=False):
    return Fp4Matrix.empty(*shape, device="cpu", gated=gated)


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
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
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


# ---- weights that were just written: a product may read them ahead of its turn only behind another one on its stream ----------
AHEAD = -5                                                        # where a product's arguments say that it may


def product(launches, w, x=None):
    fp4_ops.linear(torch.zeros((3, 64)) if x is None else x, w, torch.zeros((3, w.shape[0])))
    return launches[-1][1][AHEAD]


@pytest.mark.parametrize("write", [
    lambda m: fp4_ops.quantize(torch.zeros((64, 64)), m), lambda m: m.codes.fill_(3), lambda m: m.scales[0].fill_(120),
    lambda m: m.codes[3:5].copy_(torch.ones((2, 32), dtype=torch.uint8)), lambda m: m.first_rows(16).codes.zero_(),
    lambda m: fp4_ops.quantize(torch.zeros((16, 64)), m.first_rows(16)), lambda m: m.written(),
])
def test_the_first_product_behind_a_write_waits_for_it(launches, write):
    m = matrix(64, 64)
    assert [product(launches, m) for _ in range(3)] == [0, 1, 1]
    write(m)
    assert [product(launches, m) for _ in range(3)] == [0, 1, 1]
    m.settle()
    assert product(launches, m) == 1
    write(m)
    assert [product(launches, m) for _ in range(2)] == [0, 1]


def test_every_stream_has_a_first_product(launches, monkeypatch):
    m, at = matrix(64, 64), 0
    monkeypatch.setattr(fp4_ops, "_stream", lambda *indices: at)
    seen = []
    for at in (7, 7, 9, 7, 9):
        seen.append(product(launches, m))
    assert seen == [0, 1, 0, 1, 1]


def test_a_captured_product_orders_nothing_outside_its_graph(launches, monkeypatch):
    m, capturing = matrix(64, 64), True
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    assert [product(launches, m) for _ in range(2)] == [0, 1]
    capturing = False
    assert [product(launches, m) for _ in range(2)] == [0, 1]
    capturing = True
    assert product(launches, m) == 1                              # written before the capture


def test_tensors_of_inference_mode_are_read_ahead_when_settled(launches):
    with torch.inference_mode():
        m = matrix(64, 64)
        assert [product(launches, m) for _ in range(2)] == [0, 0]
        m.settle()
        assert product(launches, m) == 1
        fp4_ops.quantize(torch.zeros((64, 64)), m)
        assert [product(launches, m) for _ in range(2)] == [0, 0]
    assert [product(launches, m) for _ in range(2)] == [0, 0]


def test_units_look_at_both_matrices_and_views_are_matrices_too(launches):
    first, down = matrix(128, 64, gated=True), matrix(64, 64).settle()
    z = fp4_ops.gate_up(torch.zeros((3, 64)), first)
    assert launches[-1][1][AHEAD] == 0
    assert product(launches, down, z) == 1
    fp4_ops.gate_up(torch.zeros((3, 64)), first)
    assert launches[-1][1][AHEAD] == 1
    view = down.first_rows(16)
    assert product(launches, view) == 1
    down.written()
    assert [product(launches, view) for _ in range(2)] == [0, 1]
    assert product(launches, down) == 0


def test_the_parts_matrices_are_settled(launches):
    from supersonic_b200.parts.fp4 import fp4_of
    w = fp4_of(torch.zeros((64, 64)))
    assert w.reads_ahead(0) and w.reads_ahead(5) and not matrix(64, 64).reads_ahead(0)


# ---- what Python declares of the library's functions is what the sources say ---------------------------------------------------
def declared(name):
    """The kinds of a C entry's arguments, from its definition."""
    import os
    import re
    folder = os.path.dirname(fp4_ops.__file__)
    for f in sorted(os.listdir(folder)):
        if f.startswith("fp4_") and f.endswith(".cu"):
            with open(os.path.join(folder, f), encoding="utf-8") as fh:
                got = re.search(r"SSB_API (?:int|long long) " + name + r"\(([^)]*)\) \{", fh.read())
            if got:
                kinds = [" ".join(a.split()[:-1]) + "*" * (a.split()[-1][0] == "*") for a in got.group(1).split(",")]
                return ["P" if "*" in k or k == "cudaStream_t" else {"int": "i", "long long": "q", "float": "f"}[k] for k in kinds]
    raise AssertionError(f"no definition of {name}")


@pytest.mark.parametrize("name", sorted(fp4_ops._SIGNATURES))
def test_signatures(name):
    assert [fp4_ops._FORMATS[t] for t in fp4_ops._SIGNATURES[name]] == declared(name)


# ---- what is set once is set on every device ------------------------------------------------------------------------------------
def test_settings_are_each_devices_own(tmp_path):
    """csrc/per_device.h against a runtime of three devices, and one whose device has no place."""
    import os
    import subprocess
    from supersonic_b200.csrc import build
    (tmp_path / "cuda_runtime.h").write_text("""
enum cudaError_t { cudaSuccess = 0, cudaErrorNoDevice = 100 };
extern int device;
inline cudaError_t cudaGetDevice(int* d) { if (device == -2) return cudaErrorNoDevice; *d = device; return cudaSuccess; }
""")
    (tmp_path / "check.cpp").write_text("""
#include "per_device.h"
int device = 0;
template <int K> int settings() { static SsbPerDevice<int> set; int* here = set.here(); return here ? ++*here : -1; }
int main() {
    int wrong = 0;
    for (device = 0; device < 3; ++device) wrong += settings<0>() != 1;
    for (device = 0; device < 3; ++device) wrong += settings<0>() != 2;
    wrong += (device = 1, settings<1>()) != 1;
    wrong += (device = 64, settings<0>()) != -1;
    wrong += (device = -2, settings<0>()) != -1;
    return wrong;
}
""")
    header = os.path.join(os.path.dirname(build.__file__))
    subprocess.run([build.find_cxx(), "-std=c++17", "-I", str(tmp_path), "-I", header, str(tmp_path / "check.cpp"), "-o", str(tmp_path / "check")], check=True)
    assert subprocess.run([str(tmp_path / "check")]).returncode == 0


@pytest.mark.parametrize("source", ["fp4_few.cu", "fp4_linear.cu", "fp4_rows.cu", "fp4_step.cu"])
def test_launches_keep_nothing_for_the_whole_process(source):
    import os
    import re
    with open(os.path.join(os.path.dirname(fp4_ops.__file__), source), encoding="utf-8") as fh:
        assert not re.findall(r"^\s+static (?!SsbPerDevice|const)[a-z_ ]+\w+( = [^;]*)?;", fh.read(), flags=re.M)


def test_a_steps_rows_can_be_settled_as_any_matrix(launches):
    z = fp4_ops.gate_up(torch.zeros((40, 64)), matrix(128, 64, gated=True))
    assert z.settle() is z and z.codes.shape == (40, 32)
    z.written()


def test_a_captured_write_comes_again_with_every_replay(launches, monkeypatch):
    capturing = False
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    m = matrix(64, 64)
    m.index = 0
    view = m.first_rows(16)
    assert [product(launches, m) for _ in range(2)] == [0, 1]
    capturing = True
    m.written()
    assert [product(launches, m) for _ in range(2)] == [0, 1]     # in the graph
    capturing = False
    assert [product(launches, w) for w in (m, m, view, m.first_rows(8))] == [0, 0, 0, 0]
    m.settle()
    assert product(launches, m) == 0
    capturing = True
    assert product(launches, m) == 1
