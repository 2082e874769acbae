"""Python faces of the 8-bit serving kernels: a cache of int8 codes and the attention that reads it, eviction from that cache by
the attention weight its tokens gathered, and matrix products in 8-bit integers.

Like :mod:`.ops`, every function checks what its kernel assumes, raises :class:`KernelError`, and launches on the current stream;
nothing synchronises.  A cache entry is an :class:`~supersonic_b200.cache.Int8Pages`, addressed through a page table
``[slots, pages a sequence]`` as the float caches are.

The modelled project's 8-bit lanes: an int8/int4 tiered cache (kernels/certified_kv_bridge_cuda.cu:32-420) and int8 weights
(crates/runner/src/llama31_engine.rs:289-430); both compute in the model's type.
"""
from __future__ import annotations

from ctypes import c_char_p, c_float, c_int, c_longlong, c_void_p
from struct import Struct, error as StructError
from typing import Optional, Tuple

import torch

from ..cache import Int8Pages
from . import ops
from .build import load_library
from .ops import KernelError, _CODES, _check

_P, _I, _F, _L = c_void_p, c_int, c_float, c_longlong
_SIGNATURES = {
    "ssb_int8_append": ("int8_cache", [_P, _I, _I, _P, _I, _P, _P, _I, _I, _P, _P, _P, _I, _P, _I, _I, _P, _P, _P, _P, _P, _I, _I, _I,
                                       _I, _I, _P]),
    "ssb_int8_read": ("int8_cache", [_P, _P, _P, _P, _P, _I, _I, _I, _P, _P, _I, _P, _P, _I, _I, _I, _I, _I, _P]),
    "ssb_int8_evict": ("int8_cache", [_P, _P, _P, _P, _P, _P, _I, _I, _I, _P, _P, _I, _P, _I, _I, _I, _I, _I, _I, _I, _P, _P]),
    "ssb_int8_attention": ("int8_attention", [_P, _I, _I, _P, _I, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _P, _P, _P, _I, _I, _I, _I, _I,
                                              _I, _I, _I, _I, _F, _P, _L, _P, _P]),
    "ssb_int8_attention_scratch": ("int8_attention", [_I] * 10 + [_F]),
    "ssb_int8_quantize_rows": ("int8_linear", [_P, _I, _I, _P, _I, _P, _I, _I, _P]),
    "ssb_int8_linear": ("int8_linear", [_P, _I, _I, _P, _I, _P, _P, _I, _I, _I, _I, _I, _I, _P, _P, _P]),
    "ssb_int8_linear_scratch": ("int8_linear", [_I, _I, _I]),
}
_FORMATS = {_P: "P", _I: "i", _F: "f", _L: "q"}
_functions = {}


def _fn(name: str):
    """The library's function.  Arguments of a launch go as one run of bytes (packed_call.cuh): one conversion instead of up to 31, at a
    third of the cost; a number that its type does not hold is an error."""
    f = _functions.get(name)
    if f is None:
        library, types = _SIGNATURES[name]
        if name.endswith("_scratch"):
            f = getattr(load_library(library), name)
            f.restype, f.argtypes = c_longlong, types
        else:
            call, pack = getattr(load_library(library), name + "_packed"), Struct("@" + "".join(_FORMATS[t] for t in types)).pack
            call.restype, call.argtypes = c_int, [c_char_p]

            def f(*args):
                try:
                    packed = pack(*args)
                except (StructError, OverflowError) as e:
                    raise KernelError(f"{name}: {e}") from None
                return call(packed)
        _functions[name] = f
    return f


_INT32, _INT8, _FLOAT32 = torch.int32, torch.int8, torch.float32
_SIZES = {torch.float32: 4, torch.bfloat16: 2}
_DIMS = (16, 32, 64, 128, 256)


def _ints(t: torch.Tensor, name: str, n: int) -> int:
    """The address of ``n`` int32 values in a row on the device."""
    if t.dtype is not _INT32 or t.shape != (n,) or not t.is_cuda or not t.is_contiguous():
        raise KernelError(f"{name} must be {n} contiguous int32 values on a CUDA device, is {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, rows: int, width: int, dtype=None) -> Tuple[int, int]:
    """(address, row stride) of a matrix of at least ``width`` columns whose rows start on 16 bytes."""
    size, shape = _SIZES.get(t.dtype), t.shape
    if size is None or len(shape) != 2 or shape[0] != rows or shape[1] < width or not t.is_cuda or (dtype is not None and t.dtype is not dtype):
        raise KernelError(f"{name} must be [{rows}, {width}] of {dtype or 'float32 or bfloat16'} on a CUDA device, "
                          f"is {t.dtype} {tuple(shape)}")
    at, (ld, step) = t.data_ptr(), t.stride()
    if rows == 1:
        ld = width + -width % 8
    if (step != 1 and width > 1) or (at | ld * size) % 16 or ld < width:
        raise KernelError(f"{name}: rows of contiguous elements that start on 16 bytes")
    return at, ld


def _pages(pages: Int8Pages, table: torch.Tensor):
    """(pages, kv heads, head size, block) of a cache entry that holds together, the addresses of its five tensors (0: no weight), and
    its table's address, rows and width.  One condition over all of it: this runs in every call of a decode step."""
    k, v, ks, vs, weight = pages
    shape, scales, tab = k.shape, ks.shape, table.shape
    if len(shape) == 4 and len(scales) == 3 and len(tab) == 2:
        n_pages, n_kv, page, dim = shape
        scale_pages, scale_heads, per = scales
        if (page == 64 and dim in _DIMS and v.shape == shape and k.dtype is _INT8 and v.dtype is _INT8
                and k.is_cuda and v.is_cuda and k.is_contiguous() and v.is_contiguous()
                and scale_pages == n_pages and scale_heads == n_kv and per in (1, 2, 4) and vs.shape == scales
                and ks.dtype is _FLOAT32 and vs.dtype is _FLOAT32 and ks.is_cuda and vs.is_cuda and ks.is_contiguous() and vs.is_contiguous()
                and (weight is None or (weight.shape == (n_pages, n_kv, 64) and weight.dtype is _FLOAT32 and weight.is_cuda
                                        and weight.is_contiguous()))
                and table.dtype is _INT32 and table.is_cuda and table.is_contiguous()):
            k_at, v_at = k.data_ptr(), v.data_ptr()
            if (k_at | v_at) % 16 == 0:
                at = (k_at, v_at, ks.data_ptr(), vs.data_ptr(), 0 if weight is None else weight.data_ptr())
                return n_pages, n_kv, dim, 64 // per, at, table.data_ptr(), tab[0], tab[1]
    raise KernelError(
        "pages: k and v must be int8 [pages, kv heads, 64, 16 32 64 128 or 256], their scales float32 [pages, kv heads, 4 2 or 1], weight "
        "float32 [pages, kv heads, 64] or None, the page table int32 [rows, pages a sequence], all contiguous on a CUDA device; are "
        f"{k.dtype} {tuple(shape)}, {v.dtype} {tuple(v.shape)}, {ks.dtype} {tuple(scales)}, {vs.dtype} {tuple(vs.shape)}, "
        f"{None if weight is None else (weight.dtype, tuple(weight.shape))} and {table.dtype} {tuple(tab)}")


def _stream() -> int:
    """The current stream's handle."""
    return ops._stream().value or 0


_error_words = {}
_scratch_sizes = {}


def _error_word(device: torch.device) -> int:
    """The address of the device's error word (:func:`.ops.tc_error_word`), for a launch with bounded waits, which counts as unread."""
    ops.note_bounded_wait_launches(1)
    at = _error_words.get(device)
    if at is None:
        at = _error_words[device] = ops.tc_error_word(device).data_ptr()
    return at


def _scratch_size(name: str, *sizes) -> int:
    """What the library says a launch of these sizes needs."""
    n = _scratch_sizes.get((name, sizes))
    if n is None:
        if len(_scratch_sizes) > 4096:
            _scratch_sizes.clear()
        n = _scratch_sizes[name, sizes] = _fn(name)(*sizes)
    return n


def append(qkv: torch.Tensor, cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], pos: torch.Tensor, place: torch.Tensor,
           slot: torch.Tensor, page_table: torch.Tensor, pages: Int8Pages, out: torch.Tensor, n_q: int) -> None:
    """The queries, keys and values of a step: ``qkv`` [T, (n_q + 2 kv heads) x head size] holds a token's query heads, key heads
    and value heads.  Queries and keys are rotated by ``pos`` (tables ``cos``, ``sin`` [positions, rotated / 2], pairs
    (i, i + rotated / 2); None: not at all), keys and values go into ``pages`` as codes at ``place``, the token's place in the
    sequence's cache (the same as ``pos`` until tokens are evicted).  ``out`` (may be ``qkv``): queries rotated, keys and values as
    the cache now holds them.  The weight of a new token is zero.

    A block's scale is max(its scale so far, max |x| * (1/127) over its new tokens, 2^-100); when it grows, the block's earlier codes
    are rounded again under it.  NaN counts as zero and an infinity as 2^127.  The tokens of a sequence come in
    consecutive rows, in order; rows with a negative slot, or a place outside the table, are passed over."""
    n_pages, n_kv, dim, block, at, table, slots, per_seq = _pages(pages, page_table)
    T, width = qkv.shape[0], (n_q + 2 * n_kv) * dim
    if n_q < 0:
        raise KernelError(f"append: {n_q} query heads")
    q_at, ldq = _rows(qkv, "qkv", T, width)
    o_at, ldo = _rows(out, "out", T, width, qkv.dtype)
    rot = positions = cos_at = sin_at = 0
    if cos is not None:
        positions, rot = cos.shape[0], 2 * cos.shape[-1]
        if sin is None or cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32 \
                or not cos.is_cuda or not sin.is_cuda or not cos.is_contiguous() or not sin.is_contiguous() \
                or rot % 16 or rot > dim or (cos.data_ptr() | sin.data_ptr()) % 16:
            raise KernelError(f"append: cos and sin must be contiguous float32 [positions, a multiple of 8 up to {dim // 2}]")
        cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
    _check(_fn("ssb_int8_append")(
        q_at, ldq, _CODES[qkv.dtype], o_at, ldo, cos_at, sin_at, positions, rot, _ints(pos, "pos", T), _ints(place, "place", T),
        _ints(slot, "slot", T), T, table, slots, per_seq, *at, n_pages, n_q, n_kv, dim, block, _stream()), "int8_append")


def read(pages: Int8Pages, page_table: torch.Tensor, seq_slot: torch.Tensor, lengths: torch.Tensor, k_out: torch.Tensor,
         v_out: torch.Tensor) -> None:
    """The values a cache stands for: ``k_out``, ``v_out`` [sequences, most, kv heads, head size] (float32 or bfloat16) get the
    first ``lengths`` (and at most ``most``) tokens of every sequence; what is behind them stays."""
    n_pages, n_kv, dim, block, at, table, slots, per_seq = _pages(pages, page_table)
    shape = k_out.shape
    if len(shape) != 4 or shape[2] != n_kv or shape[3] != dim or v_out.shape != shape or k_out.dtype not in _CODES \
            or v_out.dtype is not k_out.dtype or not k_out.is_cuda or not v_out.is_cuda or not k_out.is_contiguous() \
            or not v_out.is_contiguous() or (k_out.data_ptr() | v_out.data_ptr()) % 16:
        raise KernelError(f"read: k_out and v_out must be contiguous [sequences, most, {n_kv}, {dim}] of float32 or bfloat16, are "
                          f"{k_out.dtype} {tuple(shape)} and {v_out.dtype} {tuple(v_out.shape)}")
    B, most = shape[0], shape[1]
    _check(_fn("ssb_int8_read")(
        *at[:4], table, slots, per_seq, n_pages, _ints(seq_slot, "seq_slot", B), _ints(lengths, "lengths", B), B,
        k_out.data_ptr(), v_out.data_ptr(), _CODES[k_out.dtype], most, n_kv, dim, block, _stream()), "int8_read")


def evict(pages: Int8Pages, page_table: torch.Tensor, seq_slot: torch.Tensor, lengths: torch.Tensor, new_table: torch.Tensor,
          keep: int, first: int, recent: int, kept: torch.Tensor) -> None:
    """Cut sequences of ``lengths`` tokens down to ``keep`` each, for every kv head by itself: the first ``first`` and the last
    ``recent`` tokens stay, and of the others those with the largest ``pages.weight`` (equal ones: the lower place; NaN ranks
    lowest).  Sequences of up to ``keep`` tokens stay whole.

    What stays is moved, in its order, to the pages named by ``new_table`` [sequences, pages], which no sequence may hold: codes
    under the largest scale of their new block, weights as they are.  ``kept`` (int32 [sequences, kv heads, keep]) gets the places
    that stayed, -1 behind the last.  Afterwards a sequence has min(length, keep) tokens, in ``new_table``'s row; its old pages
    can be given back.  Keys stay rotated by the positions they had.  A place whose page id names no page is the last to be
    chosen, and zeros where it stays."""
    n_pages, n_kv, dim, block, at, table, slots, per_seq = _pages(pages, page_table)
    B = seq_slot.shape[0]
    if pages.weight is None:
        raise KernelError("evict: the pages keep no weights (Int8Pages.weight)")
    if not (keep > 0 and first >= 0 and recent >= 0 and first + recent <= keep):
        raise KernelError(f"evict: first {first} and recent {recent} must fit into keep {keep}")
    if new_table.dtype != torch.int32 or new_table.dim() != 2 or not new_table.is_cuda or not new_table.is_contiguous() \
            or new_table.shape[0] != B or new_table.shape[1] * 64 < keep:
        raise KernelError(f"evict: new_table must be contiguous int32 [{B}, at least {(keep + 63) // 64}], is {tuple(new_table.shape)}")
    if kept.dtype != torch.int32 or kept.shape != (B, n_kv, keep) or not kept.is_cuda or not kept.is_contiguous():
        raise KernelError(f"evict: kept must be contiguous int32 [{B}, {n_kv}, {keep}], is {kept.dtype} {tuple(kept.shape)}")
    _check(_fn("ssb_int8_evict")(
        *at, table, slots, per_seq, n_pages, _ints(seq_slot, "seq_slot", B),
        _ints(lengths, "lengths", B), B, new_table.data_ptr(), new_table.shape[1], n_kv, dim, block, keep, first, recent,
        kept.data_ptr(), _stream()), "int8_evict")


def attention(q: torch.Tensor, pages: Int8Pages, page_table: torch.Tensor, cu_new: torch.Tensor, seq_start: torch.Tensor,
              seq_slot: torch.Tensor, max_new: int, out: torch.Tensor, n_q: int, scale: float, window: Optional[int] = None,
              lse: Optional[torch.Tensor] = None, weigh_last: int = 0) -> None:
    """Causal attention of packed sequences over an 8-bit cache that holds the step's keys already.  ``q`` and ``out`` [rows,
    n_q x head size]; sequence b brings rows ``cu_new[b]`` to ``cu_new[b + 1]`` (at most ``max_new``; none is allowed), held
    ``seq_start[b]`` tokens before them, and its row i sees the keys at places start + i - ``window`` + 1 (None or 0: 0) to start + i.
    ``lse`` (float32 [rows, n_q]) gets the logarithm of a row's sum of exponentials.  ``weigh_last``: that many last rows of every
    sequence add their probabilities, summed over the query heads of a kv head, to ``pages.weight``.  Rows of a sequence with a
    negative slot are zeros, and their ``lse`` minus infinity.  A place behind the table's end, or under a page id that names no page,
    holds a key that no row sees.  The values' scales that a row sees have to be within 2^90 of one another."""
    n_pages, n_kv, dim, block, at, table, slots, width = _pages(pages, page_table)
    rows, B = q.shape[0], seq_slot.shape[0]
    if n_q <= 0 or n_q % n_kv:
        raise KernelError(f"attention: {n_q} query heads do not split over {n_kv} kv heads")
    q_at, ldq = _rows(q, "q", rows, n_q * dim)
    o_at, ldo = _rows(out, "out", rows, n_q * dim, q.dtype)
    if weigh_last < 0 or (weigh_last and pages.weight is None):
        raise KernelError("attention: weigh_last needs pages that keep weights (Int8Pages.weight)")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (rows, n_q) or not lse.is_cuda or not lse.is_contiguous()):
        raise KernelError(f"attention: lse must be contiguous float32 [{rows}, {n_q}], is {lse.dtype} {tuple(lse.shape)}")
    if weigh_last and lse is None:
        lse = torch.empty((rows, n_q), dtype=_FLOAT32, device=q.device)
    if rows == 0 or B == 0:
        return
    if max_new <= 0 or (window or 0) < 0:
        raise KernelError(f"attention: max_new {max_new} new tokens, window {window}")
    code, device = _CODES[q.dtype], q.device
    size = _scratch_size("ssb_int8_attention_scratch", code, B, rows, max_new, width, n_q, n_kv, dim, window or 0, weigh_last, scale)
    scratch = torch.empty(size, dtype=_FLOAT32, device=device)
    _check(_fn("ssb_int8_attention")(
        q_at, ldq, code, o_at, ldo, 0 if lse is None else lse.data_ptr(), *at, table, slots, width, n_pages,
        _ints(cu_new, "cu_new", B + 1), _ints(seq_start, "seq_start", B), _ints(seq_slot, "seq_slot", B), B, rows, max_new, n_q, n_kv,
        dim, block, window or 0, weigh_last, scale, scratch.data_ptr(), size, _error_word(device), _stream()), "int8_attention")


# ---- matrix products ------------------------------------------------------------------------------------------------
MOST_K = 132096        # 127 * 128 * k stays below 2^31: rows' codes go to 127, weights may be -128


def quantize_rows(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor) -> None:
    """``codes`` (int8) and ``scale`` (float32, one a row) of the rows of ``x`` (float32 or bfloat16): scale = max |x| * (1/127)
    (float32, at least 2^-100), codes = rint(x / scale).  NaN counts as zero and an infinity as 2^127.  Also what turns a weight
    matrix [outputs, inputs] into 8 bits for :func:`linear`."""
    if x.dim() != 2 or x.dtype not in _CODES or not x.is_cuda or (x.shape[1] > 1 and x.stride(1) != 1):
        raise KernelError("quantize_rows: x must be a float32 or bfloat16 matrix of contiguous rows on a CUDA device")
    rows, k = x.shape
    if codes.dtype != torch.int8 or codes.shape != x.shape or not codes.is_cuda or (k > 1 and codes.stride(1) != 1):
        raise KernelError(f"quantize_rows: codes must be int8 {tuple(x.shape)}, are {codes.dtype} {tuple(codes.shape)}")
    if scale.dtype != torch.float32 or scale.shape != (rows,) or not scale.is_cuda or not scale.is_contiguous():
        raise KernelError(f"quantize_rows: scale must be {rows} contiguous float32 values")
    if rows == 0:
        return
    _check(_fn("ssb_int8_quantize_rows")(x.data_ptr(), x.stride(0), _CODES[x.dtype], codes.data_ptr(), codes.stride(0),
                                         scale.data_ptr(), rows, k, _stream()), "int8_quantize_rows")


def linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, out: torch.Tensor, accumulate: bool = False) -> None:
    """``out`` [rows, n] (+)= x W^T with ``x`` (float32 or bfloat16 [rows, k]) quantised row by row as it comes and ``weight`` int8
    [n, k] with ``weight_scale`` (float32 [n]): the sum of products of codes is an exact integer, times the row's scale, times the
    channel's.  ``accumulate`` adds to a float32 ``out``.  k: a multiple of 16 up to 132,096; n: a multiple of 8."""
    if x.dim() != 2 or weight.dim() != 2:
        raise KernelError(f"linear: x and weight must be matrices, are {tuple(x.shape)} and {tuple(weight.shape)}")
    rows, k = x.shape
    n = weight.shape[0]
    if weight.dtype is not _INT8 or weight.shape[1] != k or not weight.is_cuda or weight.stride(1) != 1 \
            or (weight.data_ptr() | weight.stride(0)) % 16:
        raise KernelError(f"linear: weight must be int8 [n, {k}] with rows on 16 bytes, is {weight.dtype} {tuple(weight.shape)}")
    if k % 16 or not 0 < k <= MOST_K or n % 8:
        raise KernelError(f"linear: k {k} must be a multiple of 16 up to {MOST_K}, n {n} a multiple of 8")
    if weight_scale.dtype != torch.float32 or weight_scale.shape != (n,) or not weight_scale.is_cuda or not weight_scale.is_contiguous():
        raise KernelError(f"linear: weight_scale must be {n} contiguous float32 values")
    x_at, ldx = _rows(x, "x", rows, k)
    o_at, ldo = _rows(out, "out", rows, n)
    if accumulate and out.dtype != torch.float32:
        raise KernelError("linear: results are added in float32 only")
    if rows == 0 or n == 0:
        return
    device = x.device
    scratch = torch.empty(_scratch_size("ssb_int8_linear_scratch", rows, n, k), dtype=_INT8, device=device)
    _check(_fn("ssb_int8_linear")(x_at, ldx, _CODES[x.dtype], weight.data_ptr(), weight.stride(0), weight_scale.data_ptr(), o_at, ldo,
                                  _CODES[out.dtype], rows, n, k, 1 if accumulate else 0, scratch.data_ptr(), _error_word(device),
                                  _stream()), "int8_linear")
