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


def weight_bytes_of(config, weight_format):
    from supersonic_b200.config import config_from_dict
    from supersonic_b200.engine import preflight
    from supersonic_b200.weights import RandomWeightStore
    cfg = config_from_dict(config)
    return preflight.weight_bytes(cfg.build_spec(), RandomWeightStore(cfg, 1), torch.bfloat16, weight_format)


@pytest.mark.parametrize("hidden, inter, heads, head_dim, attention, unit", [
    (96, 256, 3, 32, True, True), (96, 200, 3, 32, True, False), (72, 256, 3, 32, False, False), (96, 256, 3, 16, False, True),
    (72, 200, 3, 16, False, False), (64, 72, 5, 16, False, False),
])
def test_memory_of_matrices_that_have_no_4_bit_form(hidden, inter, heads, head_dim, attention, unit):
    import tiny_configs
    config = dict(tiny_configs.B, hidden_size=hidden, intermediate_size=inter, num_attention_heads=heads, num_key_value_heads=1, head_dim=head_dim)
    held = (2 * heads + 2) * head_dim * hidden * attention + 3 * inter * hidden * unit
    layers = config["num_hidden_layers"]
    assert weight_bytes_of(config, "mxfp4") == weight_bytes_of(config, None) - 2 * layers * held + layers * held * 17 // 32 + 2 * held


@pytest.mark.parametrize("hidden, inter, shared, n", [(64, 96, None, 4), (64, 96, 32, 4), (64, 96, 40, 4), (64, 40, 32, 4), (72, 96, 32, 4), (64, 32, None, 4097)])
def test_what_a_part_says_of_its_sizes_is_what_it_does(monkeypatch, hidden, inter, shared, n):
    """``fp4_roles`` from the parameters, ``to_fp4`` from the matrices."""
    from supersonic_b200.parts import attention, experts, feed_forward

    def of(w, gated=False):
        return Fp4Matrix.empty(*w.shape, device="cpu", gated=gated)

    class Kernels:
        @staticmethod
        def pack_gate_up(gate, up):
            return torch.cat([gate, up]), "halves"

    class Weights:
        def __init__(self, shapes):
            self.shapes = shapes

        def as_dtype(self, name, dtype):
            return torch.zeros(1, dtype=dtype).expand(self.shapes[name.split(".")[0] if name not in self.shapes else name])
        stored = as_dtype

    class Build:
        device, dtype, kernels = torch.device("cpu"), torch.bfloat16, Kernels

        def __init__(self, shapes):
            self.weights = Weights(shapes)
    for module in (attention, experts, feed_forward):
        monkeypatch.setattr(module, "fp4_of", of)
    unit = {"gate": (inter, hidden), "up": (inter, hidden), "down": (hidden, inter)}
    params = {"hidden_size": hidden, "intermediate_size": inter}
    part = feed_forward.SwiGLU(params, {r: r for r in unit}, Build(unit))
    assert part.to_fp4() == bool(part.fp4_roles(params)) == isinstance(part.w_down, Fp4Matrix)
    part = feed_forward.DenseFeedForward(params, {r: r for r in unit}, Build(unit))
    assert part.to_fp4() == bool(part.fp4_roles(params)) == isinstance(part.w_down, Fp4Matrix)
    params = {"hidden_size": hidden, "num_heads": 1, "num_kv_heads": 1, "head_dim": 16 * (inter // 16), "scale": 1.0}
    sizes = {r: (params["head_dim"], hidden) for r in "qkv"}
    sizes["o"] = (hidden, params["head_dim"])
    part = attention.Attention(params, {r: r for r in sizes}, Build(sizes))
    assert part.to_fp4() == bool(part.fp4_roles(params)) == isinstance(part.w_o, Fp4Matrix)
    params = {"hidden_size": hidden, "n_experts": n, "top": 1, "expert_size": inter, "router": {"kind": "none here"},
              "shared": {"intermediate_size": shared} if shared else None}
    sizes = dict(unit, **{f"shared.{r}": tuple(shared or 1 if s == inter else s for s in shape) for r, shape in unit.items()})
    monkeypatch.setitem(experts.ROUTERS, "none here", lambda *a: None)
    names = {f"{r}.{e}": f"{r}.{e}" for r in unit for e in range(n)}
    names.update({f"shared.{r}": f"shared.{r}" for r in unit})
    part = experts.Experts(params, names, Build(sizes))
    roles = part.fp4_roles(params)
    assert part.to_fp4() == bool(roles) == part.in_fp4
    assert bool(shared) is False or isinstance(part.shared.w_down, Fp4Matrix) == ("shared.gate" in roles)
