"""Python faces of the kernels in microscaled 4-bit floats: rows into 4 bits and back, matrix products of 4-bit rows and weights, and
feed-forwards whose inner rows never leave 4 bits.

Like :mod:`.ops`, every function checks what its kernel assumes, raises :class:`KernelError`, and launches on the current stream;
nothing synchronises.  Weights, and rows that several products read, are :class:`~supersonic_b200.weights.Fp4Matrix`.

A number's block is 32 neighbours along its row.  With m the block's largest magnitude (NaN counts as zero, an infinity as the largest
finite number), its scale is 2^(floor(log2 m) - 2) (2^-127 at least, and where m is 0), and a number becomes the one of 0, 0.5, 1, 1.5,
2, 3, 4, 6 (times the scale, with its sign) that is nearest, between two the one with the even code; what is above 6 becomes 6.
Products of codes and their scales are exact, and are summed in float32.

The modelled project's 4-bit lanes multiply int4 weights by activations of the model's type
(crates/runner/src/llama31_engine.rs:289-430).
"""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p
from struct import Struct, error as StructError
from typing import Optional, Union

import torch

from ..weights.fp4 import FP4_BLOCK, Fp4Matrix
from . import ops
from .build import load_library
from .int8_ops import _SIZES
from .ops import KernelError, _CODES, _check, _raw_stream

_P, _I, _F, _L = c_void_p, c_int, c_float, c_longlong
_SIGNATURES = {
    "ssb_fp4_quantize": [_P, _L, _I, _P, _P, _I, _I, _I, _I, _P, _I, _I, _P],
    "ssb_fp4_values": [_P, _P, _P, _L, _I, _I, _I, _I, _I, _P],
    "ssb_fp4_linear": [_P, _L, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P, _P],
    "ssb_fp4_inner": [_P, _L, _I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _F, _P, _I, _P, _P, _P, _P],
    "ssb_fp4_experts": [_P, _L, _I, _P, _P, _P, _P, _P, _P, _P, _L, _I, _I, _I, _I, _I, _I, _I, _I, _F, _I, _P, _P, _P],
    "ssb_fp4_product_scratch": [_I] * 5,
    "ssb_fp4_experts_scratch": [_I] * 5,
}
_FORMATS = {_P: "P", _I: "i", _F: "f", _L: "q"}
_functions = {}
_scratch_sizes = {}
_COUNTERS = 256                # words a product counts in


def _fn(name: str):
    """The library's function; arguments of a launch go as one run of bytes (packed_call.cuh)."""
    f = _functions.get(name)
    if f is None:
        types = _SIGNATURES[name]
        if name.endswith("_scratch"):
            f = getattr(load_library("fp4"), name)
            f.restype, f.argtypes = c_longlong, types
        else:
            call, pack = getattr(load_library("fp4"), name + "_packed"), Struct("@" + "".join(_FORMATS[t] for t in types)).pack
            call.restype = c_int

            def f(*args):
                try:
                    packed = pack(*args)
                except (StructError, OverflowError) as e:
                    raise KernelError(f"{name}: {e}") from None
                return call(packed)
        _functions[name] = f
    return f


def _scratch_size(name: str, *sizes) -> int:
    """What the library says a launch of these sizes needs."""
    n = _scratch_sizes.get((name, sizes))
    if n is None:
        if len(_scratch_sizes) > 4096:
            _scratch_sizes.clear()
        n = _scratch_sizes[name, sizes] = _fn(name)(*sizes)
    return n


def _stream(*indices) -> int:
    """The current stream's handle; raises unless these device indices (-1: no CUDA device) are the current device's."""
    current = torch.cuda.current_device()
    for i in indices:
        if i != current:
            raise KernelError(f"tensors must be on the current CUDA device {current}, are on {sorted(set(indices))}")
    return _raw_stream(current) if _raw_stream is not None else ops._stream().value or 0


_error_words = {}


def _error_word(m: Fp4Matrix) -> int:
    """The address of the device's error word (:func:`.ops.tc_error_word`), for a launch with bounded waits, which counts as unread."""
    ops.note_bounded_wait_launches(1)
    at = _error_words.get(m.index)
    if at is None:
        at = _error_words[m.index] = ops.tc_error_word(m.device).data_ptr()
    return at


def _rows(t: torch.Tensor, name: str, rows: int, width: int):
    """(address, row stride) of a matrix [rows, width] whose rows start on 16 bytes; its device is checked where it is launched."""
    size, shape = _SIZES.get(t.dtype), t.shape
    if size is None or len(shape) != 2 or shape[0] != rows or shape[1] != width:
        raise KernelError(f"{name} must be [{rows}, {width}] of float32 or bfloat16, is {t.dtype} {tuple(shape)}")
    at, (ld, step) = t.data_ptr(), t.stride()
    if rows == 1:
        ld = width + -width % 8
    if (step != 1 and width > 1) or (at | ld * size) % 16 or ld < width:
        raise KernelError(f"{name}: rows of contiguous elements that start on 16 bytes")
    return at, ld


def _matrix_rows(t: torch.Tensor, name: str, m: Fp4Matrix):
    """(address, row stride, rows, type code) of a tensor of a 4-bit matrix's shape, all its rows equally far apart."""
    shape = t.shape
    if shape != m.shape or t.dtype not in _CODES or t.get_device() != m.index:
        raise KernelError(f"{name} must be float32 or bfloat16 {m.shape} on the matrix's device, is {t.dtype} {tuple(shape)} on {t.device}")
    if len(shape) == 3:
        if not t.is_contiguous():
            raise KernelError(f"{name}: matrices of several experts are contiguous")
        t = t.view(-1, shape[2])
        shape = t.shape
    at, ld = _rows(t, name, shape[0], shape[1])
    return at, ld, shape[0], _CODES[t.dtype]


def quantize(x: torch.Tensor, matrix: Fp4Matrix) -> None:
    """``matrix`` gets the numbers of ``x`` (float32 or bfloat16, of its shape; of a gated matrix the gate rows, then the up rows)."""
    at, ld, rows, code = _matrix_rows(x, "x", matrix)
    n, k = matrix.shape[-2:]
    matrix.written()
    _check(_fn("ssb_fp4_quantize")(at, ld, code, matrix.codes_at, matrix.scales_at, rows, k, n,
                                   n // 2 if matrix.gated else 0, 0, 0, 0, _stream(matrix.index)), "fp4_quantize")


def values(matrix: Fp4Matrix, out: torch.Tensor) -> None:
    """``out`` (float32 or bfloat16, of its shape) gets the numbers that ``matrix`` stands for, which both types hold exactly (from
    2^-128; what is 2^128 or more, of scales that only parts can bring, is an infinity); of a gated matrix the gate rows, then the up rows."""
    at, ld, rows, code = _matrix_rows(out, "out", matrix)
    n, k = matrix.shape[-2:]
    _check(_fn("ssb_fp4_values")(matrix.codes_at, matrix.scales_at, at, ld, code, rows, k, n,
                                 n // 2 if matrix.gated else 0, _stream(matrix.index)), "fp4_values")


Rows = Union[torch.Tensor, Fp4Matrix]
_MODE_STORE, _MODE_GATED, _MODE_ACT = 0, 1, 2


def _operands(what: str, x: Rows, weight: Fp4Matrix):
    """(rows, x's address, row stride, type code, scales' address and device) of rows that a dense weight takes."""
    if not isinstance(weight, Fp4Matrix) or len(weight.shape) != 2:
        raise KernelError(f"{what}: weight must be a 4-bit matrix [n, k], is {weight if isinstance(weight, Fp4Matrix) else type(weight)}")
    n, k = weight.shape
    if n % 8:
        raise KernelError(f"{what}: n {n} must be a multiple of 8")
    if weight._buffer is not None:             # a product reads its weights ahead of the launch before it
        raise KernelError(f"{what}: a unit's inner rows are rows, not weights")
    if isinstance(x, Fp4Matrix):
        if len(x.shape) != 2 or x.shape[1] != k or x.gated:
            raise KernelError(f"{what}: rows of {k} numbers, not {x}")
        return x.shape[0], x.codes_at, 0, -1, x.scales_at, x.index
    shape = x.shape
    if len(shape) != 2 or shape[1] != k:
        raise KernelError(f"{what}: rows of {k} numbers, not {tuple(shape)}")
    at, ld = _rows(x, "x", shape[0], k)
    return shape[0], at, ld, _CODES[x.dtype], 0, x.get_device()


def _workspace(x: Rows, needs: int, device, words: int, ahead: int = 0):
    """(a buffer or None, the address of scratch behind its first ``ahead`` bytes, the address of ``words`` counters) of a product that
    ``needs`` so much (ssb_fp4_product_scratch).  Counters are zeroed by the launch that quantises rows; a product of rows in 4 bits takes
    those that came with them, and the scratch of the launch that made them where it has room, which nobody takes twice and which lie in the
    rows' own buffer, there as long as the rows are; or it has its own zeroed."""
    size, counts = needs >> 1, needs & 1
    if not counts:
        if size + ahead == 0:
            return None, 0, 0
        buffer = torch.empty(ahead + size, dtype=torch.int8, device=device)
        return buffer, buffer.data_ptr() + ahead, 0
    own = isinstance(x, Fp4Matrix)
    if own:
        left, x._counters = x._counters, None
        if left is not None and ahead == 0 and words <= _COUNTERS:
            counters, scratch, room = left
            if size <= room:
                return None, scratch, counters
            buffer = torch.empty(size, dtype=torch.int8, device=device)
            return buffer, buffer.data_ptr(), counters
    buffer = torch.empty(ahead + 4 * words + size, dtype=torch.int8, device=device)
    if own:
        buffer[ahead:ahead + 4 * words].zero_()
    at = buffer.data_ptr() + ahead
    return buffer, at + 4 * words, at


def _over(at: int, step: int, width: int, at2: int, step2: int, width2: int, rows: int) -> bool:
    """Whether two matrices of so many rows, ``width`` bytes every ``step``, have memory in common."""
    if at2 >= at + (rows - 1) * step + width or at >= at2 + (rows - 1) * step2 + width2:
        return False
    if rows == 1 or step != step2:
        return True
    off = (at2 - at) % step                     # parts of the same wider rows
    return off < width or off + width2 > step


def linear(x: Rows, weight: Fp4Matrix, out: torch.Tensor, accumulate: bool = False) -> None:
    """``out`` [rows, n] (+)= x W^T with ``x`` [rows, k] (float32 or bfloat16, quantised as it comes, or a 4-bit matrix) and ``weight``
    [n, k].  ``accumulate`` adds to a float32 ``out``.  n: a multiple of 8."""
    rows, x_at, ldx, code, xs_at, index = _operands("linear", x, weight)
    if weight.gated:
        raise KernelError("linear: a gated unit's first matrix goes through gate_up")
    n, k = weight.shape
    o_at, ldo = _rows(out, "out", rows, n)
    if accumulate and out.dtype is not torch.float32:
        raise KernelError("linear: results are added in float32 only")
    step, width = (ldx * x.element_size(), k * x.element_size()) if code >= 0 else (k // 2, k // 2)
    size = out.element_size()
    if rows and _over(x_at, step, width, o_at, ldo * size, n * size, rows):
        raise KernelError("linear: out must not be x, or lie over it")
    stream = _stream(index, weight.index, out.get_device())
    if rows == 0:
        return
    device = weight.device
    needs = _scratch_size("ssb_fp4_product_scratch", rows, n, k, code >= 0, _MODE_STORE)
    held, scratch, counters = _workspace(x, needs, device, _COUNTERS)
    _check(_fn("ssb_fp4_linear")(x_at, ldx, code, xs_at, weight.codes_at, weight.scales_at, o_at, ldo, _CODES[out.dtype], rows, n, k,
                                 1 if accumulate else 0, 1 if weight.reads_ahead(stream) else 0, scratch, counters, _error_word(weight),
                                 stream), "fp4_linear")


def _inner(what: str, x: Rows, weight: Fp4Matrix, kind: int, limit: float, row_scale: Optional[torch.Tensor]) -> Fp4Matrix:
    rows, x_at, ldx, code, xs_at, index = _operands(what, x, weight)
    n, k = weight.shape
    gated = weight.gated
    inter = n // 2 if gated else n
    if inter % FP4_BLOCK:
        raise KernelError(f"{what}: {inter} inner channels must be a multiple of {FP4_BLOCK}")
    if rows == 0:
        raise KernelError(f"{what}: no rows")
    device = weight.device
    if row_scale is not None and (row_scale.dtype != torch.float32 or row_scale.shape != (rows,) or not row_scale.is_contiguous()
                                  or row_scale.get_device() != weight.index):
        raise KernelError(f"{what}: row_scale must be {rows} contiguous float32 values beside the weight")
    stream = _stream(index, weight.index)
    needs = _scratch_size("ssb_fp4_product_scratch", rows, n, k, code >= 0, _MODE_GATED if gated else _MODE_ACT)
    size, ahead = Fp4Matrix.rows_layout(rows, inter)
    buffer, scratch, counters = _workspace(x, needs, device, 2 * _COUNTERS, ahead)
    z = Fp4Matrix.over_rows(buffer, rows, inter, size)
    _check(_fn("ssb_fp4_inner")(x_at, ldx, code, xs_at, weight.codes_at, weight.scales_at, z.codes_at, z.scales_at, rows, n, k,
                                1 if gated else 0, kind, limit, 0 if row_scale is None else row_scale.data_ptr(),
                                1 if weight.reads_ahead(stream) else 0, scratch, counters, _error_word(weight), stream), "fp4_inner")
    if counters:
        z._counters = (counters + 4 * _COUNTERS, scratch, needs >> 1)          # of z's own buffer
    return z


def gate_up(x: Rows, weight: Fp4Matrix, act=None, row_scale: Optional[torch.Tensor] = None) -> Fp4Matrix:
    """The inner rows of a gated unit, f(x Wgate^T, x Wup^T) * row_scale from the float32 sums, in 4 bits [rows, inter].  ``weight``: a
    gated matrix [2 x inter, k].  ``act``: None for silu(g) u, or (kind, limit) as :func:`.ops.gated_activation` takes them;
    ``row_scale``: a float32 factor for each row."""
    if not isinstance(weight, Fp4Matrix) or not weight.gated:
        raise KernelError("gate_up: weight must be a gated 4-bit matrix")
    kind, limit = act if act else ("silu", 0.0)
    if kind not in ops.GATE_KINDS_FF:
        raise KernelError(f"gate_up: {kind!r} is not known (known: {sorted(ops.GATE_KINDS_FF)})")
    return _inner("gate_up", x, weight, ops.GATE_KINDS_FF[kind], float(limit), row_scale)


def activated(x: Rows, weight: Fp4Matrix, act: str, scale: float = 1.0) -> Fp4Matrix:
    """The inner rows of a feed-forward without gate, act(x W^T) * scale from the float32 sums, in 4 bits [rows, inter].  ``act``: one of
    ``ops.ACTIVATIONS``."""
    if act not in ops.ACTIVATIONS:
        raise KernelError(f"activated: {act!r} is not known (known: {sorted(ops.ACTIVATIONS)})")
    if isinstance(weight, Fp4Matrix) and weight.gated:
        raise KernelError("activated: a gated unit's first matrix goes through gate_up")
    return _inner("activated", x, weight, ops.ACTIVATIONS[act], float(scale), None)


MOST_PAIRS = 1 << 24           # (token, choice) pairs of a call


def experts(x: torch.Tensor, expert_of: torch.Tensor, pair_weight: torch.Tensor, first: Fp4Matrix, down: Fp4Matrix, out: torch.Tensor,
            act=None, accumulate: bool = False) -> None:
    """``out`` [tokens, k] (+)= sum over a token's choices j of pair_weight[t, j] * E(x_t), E the unit of expert ``expert_of[t, j]``:
    down(f(gate x, up x)) with a gated ``first`` [experts, 2 x inter, k] (``act`` as :func:`gate_up` takes it), down(act(up x)) with
    ``first`` [experts, inter, k] (``act``: one of ``ops.ACTIVATIONS``); ``down`` [experts, k, inter].  Rows and inner rows go into 4
    bits, an inner row from the float32 sums; choices are summed in float32, in their order.  A choice that names no expert counts
    nothing.  ``expert_of`` int32 and ``pair_weight`` float32 [tokens, top]; ``accumulate`` adds to a float32 ``out``."""
    if not (isinstance(first, Fp4Matrix) and isinstance(down, Fp4Matrix) and len(first.shape) == len(down.shape) == 3):
        raise KernelError("experts: first and down must be 4-bit matrices of several experts")
    E, n, k = first.shape
    inter = n // 2 if first.gated else n
    if down.shape != (E, k, inter) or down.gated or k % FP4_BLOCK or inter % FP4_BLOCK:
        raise KernelError(f"experts: first {first} takes a down of {[E, k, inter]}, not {down}")
    if first.gated:
        kind, limit = act if act else ("silu", 0.0)
        kinds = ops.GATE_KINDS_FF
    else:
        kind, limit, kinds = act, 1.0, ops.ACTIVATIONS
    if kind not in kinds:
        raise KernelError(f"experts: {kind!r} is not known (known: {sorted(kinds)})")
    if x.dim() != 2 or x.shape[1] != k or out.shape != x.shape:
        raise KernelError(f"experts: x and out must be [tokens, {k}], are {tuple(x.shape)} and {tuple(out.shape)}")
    tokens = x.shape[0]
    x_at, ldx = _rows(x, "x", tokens, k)
    o_at, ldo = _rows(out, "out", tokens, k)
    if accumulate and out.dtype != torch.float32:
        raise KernelError("experts: results are added in float32 only")
    device = first.device
    top = expert_of.shape[-1] if expert_of.dim() == 2 else 0
    if top < 1 or expert_of.dtype != torch.int32 or pair_weight.dtype != torch.float32 or expert_of.shape != (tokens, top) \
            or pair_weight.shape != (tokens, top) or not expert_of.is_contiguous() or not pair_weight.is_contiguous():
        raise KernelError(f"experts: expert_of and pair_weight must be contiguous int32 and float32 [{tokens}, top], are {expert_of.dtype} "
                          f"{tuple(expert_of.shape)} and {pair_weight.dtype} {tuple(pair_weight.shape)}")
    if tokens * top > MOST_PAIRS or E > 4096:
        raise KernelError(f"experts: {tokens} tokens of {top} choices among {E} experts are more than {MOST_PAIRS} pairs or 4096 experts")
    stream = _stream(x.get_device(), out.get_device(), expert_of.get_device(), pair_weight.get_device(), first.index, down.index)
    if tokens == 0:
        return
    scratch = torch.empty(_scratch_size("ssb_fp4_experts_scratch", tokens, top, E, k, inter), dtype=torch.int8, device=device)
    _check(_fn("ssb_fp4_experts")(x_at, ldx, _CODES[x.dtype], expert_of.data_ptr(), pair_weight.data_ptr(), first.codes_at,
                                  first.scales_at, down.codes_at, down.scales_at, o_at, ldo, _CODES[out.dtype],
                                  tokens, top, E, k, inter, 1 if first.gated else 0, kinds[kind], float(limit), 1 if accumulate else 0,
                                  scratch.data_ptr(), _error_word(first), stream), "fp4_experts")
