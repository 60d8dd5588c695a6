"""8-bit block-scaled KV cache: KV8Store (one layer's keys and values, with the attention that reads them) and
BlockInt8Cache (a cache for HF models built from it)."""

from .cache import BlockInt8Cache
from .store import BLOCK, KV8Store

__all__ = ["BLOCK", "BlockInt8Cache", "KV8Store"]
