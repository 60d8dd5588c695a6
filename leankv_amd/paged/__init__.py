"""16-bit paged KV cache: PagedKV (pages, their tables and the attention over them), packed_attention (causal attention of
prompts that lie one behind the other) and PagedCache (a cache for HF models built from them)."""

from .cache import PagedCache
from .packed import packed_attention
from .pool import PagedKV

__all__ = ["PagedCache", "PagedKV", "packed_attention"]
