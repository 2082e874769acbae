"""What turns a part's matrices into 4-bit ones (``weight_format="mxfp4"``).

A part that can has ``to_fp4()`` (its matrices become :class:`Fp4Matrix`, or it answers False and stays as it is) and
``fp4_roles(params)``, the roles of the tensors that these matrices are made of, none where it would answer False (a role ending in "."
stands for all that begin with it)."""
from __future__ import annotations

from ..weights.fp4 import FP4_BLOCK, Fp4Matrix


def fp4_fits(weight) -> bool:
    """Whether a product can take a matrix of this shape in 4 bits."""
    n, k = weight.shape[-2:]
    return n % 8 == 0 and k % FP4_BLOCK == 0 and n > 0 and k > 0


def fp4_sizes(*sizes: int) -> bool:
    """Whether matrices between rows of these sizes have that form: each is one's n and another's k."""
    return all(s > 0 and s % FP4_BLOCK == 0 for s in sizes)


def fp4_of(weight, gated: bool = False) -> Fp4Matrix:
    """``weight`` ([n, k] or [experts, n, k]) in 4 bits; ``gated``: gate rows, then up rows."""
    from ..csrc import fp4_ops
    out = Fp4Matrix.empty(*weight.shape, device=weight.device, gated=gated)
    fp4_ops.quantize(weight, out)
    return out.settle()
