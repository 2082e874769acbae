"""One cache entry in 8 bits: codes, their scales, and the attention weight that cached tokens have gathered.

The layout is that of :class:`KvGroup`'s entries, so the page tables of a :class:`SequenceCache` serve both: ``k`` and ``v`` are
int8 codes ``[pages, kv_heads, 64, head_dim]``; ``k_scale`` and ``v_scale`` float32 ``[pages, kv_heads, 64 / block]`` with one scale
for every ``block`` (16, 32 or 64) consecutive tokens of a head; a value is code times scale.  ``weight`` (float32
``[pages, kv_heads, 64]``, or None where nobody asks) is what ``int8_ops.attention`` adds to and ``int8_ops.evict`` goes by.

The reference's 8-bit cache keeps its codes in its bridge's own blocks (kernels/certified_kv_bridge_cuda.cu:32-420).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .allocators import CacheError
from .sequence_cache import PAGE_TOKENS


class Int8Pages(NamedTuple):
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    weight: Optional[torch.Tensor] = None

    @classmethod
    def allocate(cls, n_pages: int, n_kv_heads: int, head_dim: int, block: int = 16, weights: bool = False,
                 device="cuda") -> "Int8Pages":
        """Zeroed storage of ``n_pages`` pages."""
        if block not in (16, 32, 64) or head_dim not in (16, 32, 64, 128, 256) or n_pages <= 0 or n_kv_heads <= 0:
            raise CacheError(f"no 8-bit pages of {n_pages} x {n_kv_heads} heads of {head_dim} in blocks of {block}: heads of 16, 32, "
                             "64, 128 or 256 in blocks of 16, 32 or 64 tokens")
        shape = (n_pages, n_kv_heads, PAGE_TOKENS, head_dim)
        scales = (n_pages, n_kv_heads, PAGE_TOKENS // block)
        return cls(torch.zeros(shape, dtype=torch.int8, device=device), torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(scales, dtype=torch.float32, device=device), torch.zeros(scales, dtype=torch.float32, device=device),
                   torch.zeros(shape[:3], dtype=torch.float32, device=device) if weights else None)

    @property
    def block(self) -> int:
        """Tokens a scale."""
        return PAGE_TOKENS // self.k_scale.shape[2]

    def bytes_held(self) -> int:
        return sum(t.numel() * t.element_size() for t in self if t is not None)
