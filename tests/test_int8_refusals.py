"""What the 8-bit operators refuse, before anything is launched: these need no GPU."""
import pytest
import torch

from supersonic_b200.cache import CacheError, Int8Pages
from supersonic_b200.csrc import int8_ops
from supersonic_b200.csrc.ops import KernelError


class OnDevice(torch.Tensor):
    """A host tensor that says it lives on a device: only the checks are run on it."""

    @staticmethod
    def of(t):
        return t.as_subclass(OnDevice)

    @property
    def is_cuda(self):
        return True


def z(*shape, dtype=torch.float32):
    return OnDevice.of(torch.zeros(shape, dtype=dtype))


def i32(*shape):
    return z(*shape, dtype=torch.int32)


def pages(n=4, n_kv=2, dim=64, per=4, weight=True):
    return Int8Pages(z(n, n_kv, 64, dim, dtype=torch.int8), z(n, n_kv, 64, dim, dtype=torch.int8), z(n, n_kv, per), z(n, n_kv, per),
                     z(n, n_kv, 64) if weight else None)


def attend(p=None, table=None, q=None, out=None, n_q=4, cu=None, lse=None, weigh=0, start=None):
    int8_ops.attention(z(3, 256) if q is None else q, pages() if p is None else p, i32(2, 5) if table is None else table,
                       i32(3) if cu is None else cu, i32(2) if start is None else start, i32(2), 2, z(3, 256) if out is None else out,
                       n_q, 0.125, lse=lse, weigh_last=weigh)


@pytest.mark.parametrize("kw", [
    {"p": Int8Pages(torch.zeros((4, 2, 64, 64), dtype=torch.int8), *pages()[1:])},               # not on a device
    {"p": pages()._replace(k=z(4, 2, 64, 64))}, {"p": pages()._replace(v=z(4, 2, 64, 32, dtype=torch.int8))},
    {"p": pages(per=3)}, {"p": pages()._replace(v_scale=z(4, 2, 2))}, {"p": pages()._replace(k_scale=z(4, 2, 4, dtype=torch.float64))},
    {"p": pages()._replace(weight=z(4, 2, 32))}, {"p": pages(dim=48)},
    {"table": i32(10)}, {"table": z(2, 5)}, {"q": z(3, 128)}, {"q": z(3, 256, dtype=torch.float16)}, {"q": z(256, 3).t()},
    {"out": z(2, 256)}, {"out": z(3, 256, dtype=torch.bfloat16)}, {"n_q": 3}, {"n_q": 0}, {"cu": i32(2)}, {"cu": z(3)},
    {"lse": z(3, 3)}, {"lse": z(3, 4, dtype=torch.bfloat16)}, {"p": pages(weight=False), "weigh": 1}, {"weigh": -1},
    {"start": i32(4)[::2]}, {"q": z(3, 257)[:, 1:]},
])
def test_attention_refuses(kw):
    with pytest.raises(KernelError):
        attend(**kw)


@pytest.mark.parametrize("kw", [
    {"qkv": z(3, 511)}, {"qkv": z(3, 512, dtype=torch.int32)}, {"out": z(3, 512, dtype=torch.bfloat16)}, {"out": z(2, 512)},
    {"cos": z(9, 33)}, {"cos": z(9, 40), "sin": z(9, 40)}, {"cos": z(9, 4), "sin": z(9, 4)}, {"sin": z(9, 16)}, {"sin": None},
    {"pos": i32(2)}, {"slot": z(3)}, {"n_q": -1}, {"qkv": torch.zeros((3, 512))},
])
def test_append_refuses(kw):
    a = dict(qkv=z(3, 512), cos=z(9, 32), sin=z(9, 32), pos=i32(3), place=i32(3), slot=i32(3), page_table=i32(2, 5), pages=pages(),
             out=z(3, 512), n_q=4)
    a.update(kw)
    with pytest.raises(KernelError):
        int8_ops.append(**a)


@pytest.mark.parametrize("kw", [
    {"pages": pages(weight=False)}, {"keep": 0}, {"first": -1}, {"recent": -1}, {"first": 60, "recent": 41}, {"new_table": i32(2, 1)},
    {"new_table": i32(3, 2)}, {"new_table": z(2, 2)}, {"kept": i32(2, 2, 99)}, {"kept": z(2, 2, 100)}, {"lengths": i32(3)},
])
def test_evict_refuses(kw):
    a = dict(pages=pages(), page_table=i32(2, 5), seq_slot=i32(2), lengths=i32(2), new_table=i32(2, 2), keep=100, first=4, recent=10,
             kept=i32(2, 2, 100))
    a.update(kw)
    with pytest.raises(KernelError):
        int8_ops.evict(**a)


@pytest.mark.parametrize("kw", [{"k_out": z(2, 10, 2, 32)}, {"v_out": z(2, 9, 2, 64)}, {"v_out": z(2, 10, 2, 64, dtype=torch.bfloat16)},
                                {"lengths": i32(1)}])
def test_read_refuses(kw):
    a = dict(pages=pages(), page_table=i32(2, 5), seq_slot=i32(2), lengths=i32(2), k_out=z(2, 10, 2, 64), v_out=z(2, 10, 2, 64))
    a.update(kw)
    with pytest.raises(KernelError):
        int8_ops.read(**a)


@pytest.mark.parametrize("kw", [
    {"x": z(3, 40)}, {"x": z(3, 32, dtype=torch.int32)}, {"weight": z(16, 32)}, {"weight": z(16, 48, dtype=torch.int8)},
    {"weight": z(12, 32, dtype=torch.int8)}, {"weight": z(16, 33, dtype=torch.int8)[:, 1:]}, {"weight_scale": z(15)},
    {"weight_scale": z(16, dtype=torch.float64)}, {"out": z(3, 8)}, {"out": z(2, 16)},
    {"out": z(3, 16, dtype=torch.bfloat16), "accumulate": True}, {"x": z(3, 0), "weight": z(16, 0, dtype=torch.int8)},
    {"x": z(1, 133152), "weight": z(16, 133152, dtype=torch.int8), "out": z(1, 16)},
])
def test_linear_refuses(kw):
    a = dict(x=z(3, 32), weight=z(16, 32, dtype=torch.int8), weight_scale=z(16), out=z(3, 16))
    a.update(kw)
    with pytest.raises(KernelError):
        int8_ops.linear(**a)


@pytest.mark.parametrize("kw", [{"x": z(3)}, {"codes": z(3, 31, dtype=torch.int8)}, {"codes": z(3, 32)}, {"scale": z(4)}, {"x": z(32, 3).t()}])
def test_quantize_rows_refuses(kw):
    a = dict(x=z(3, 32), codes=z(3, 32, dtype=torch.int8), scale=z(3))
    a.update(kw)
    with pytest.raises(KernelError):
        int8_ops.quantize_rows(**a)


def test_pages_refuse_sizes_they_cannot_have():
    for kw in ({"block": 8}, {"head_dim": 48}, {"n_pages": 0}, {"n_kv_heads": 0}):
        with pytest.raises(CacheError):
            Int8Pages.allocate(**{**dict(n_pages=2, n_kv_heads=1, head_dim=64, device="cpu"), **kw})
    p = Int8Pages.allocate(2, 3, 64, block=32, weights=True, device="cpu")
    assert p.block == 32 and p.bytes_held() == 2 * (2 * 3 * 64 * 64) + 2 * (2 * 3 * 2 * 4) + 2 * 3 * 64 * 4


@pytest.mark.parametrize("kw", [{"x": z(32)}, {"x": z(2, 3, 32)}, {"weight": z(16, dtype=torch.int8)}, {"weight": z(2, 16, 32, dtype=torch.int8)},
                                {"weight": OnDevice.of(torch.tensor(1, dtype=torch.int8))}])
def test_linear_refuses_what_is_no_matrix(kw):
    a = dict(x=z(3, 32), weight=z(16, 32, dtype=torch.int8), weight_scale=z(16), out=z(3, 16))
    a.update(kw)
    with pytest.raises(KernelError):
        int8_ops.linear(**a)
