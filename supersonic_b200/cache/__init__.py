"""Slots, paged keys and values, and fixed-size per-sequence state."""
from .allocators import CacheError, CacheFull, FreeList
from .int8_pages import Int8Pages
from .sequence_cache import (PAGE_SHIFT, PAGE_TOKENS, KvGroup, KvNeed, SequenceCache,
                             StateNeed, flatten_needs, pages_for)

__all__ = ["CacheError", "CacheFull", "FreeList", "Int8Pages", "PAGE_SHIFT", "PAGE_TOKENS", "KvGroup",
           "KvNeed", "SequenceCache", "StateNeed", "flatten_needs", "pages_for"]
