"""16-bit paged KV cache: PagedKV (pages, their tables and the attention over them) and packed_attention (causal attention of
prompts that lie one behind the other)."""

from .packed import packed_attention
from .pool import PagedKV

__all__ = ["PagedKV", "packed_attention"]
