"""The part of HF's cache interface that the KV caches here share: transformers calls these on past_key_values (its Cache
contract, as the reference's cache implements it, leankv/turboquant/cache.py:193-291).  A cache provides num_layers,
_device, _seq_lengths (tokens per layer), _seen_tokens and _get_full_cache(layer)."""

from __future__ import annotations

import torch


class HFCache:
    is_compileable = False
    layer_type = None

    def get_seq_length(self, layer_idx: int = 0) -> int:
        return self._seq_lengths[layer_idx] if layer_idx < len(self._seq_lengths) else 0

    def get_mask_sizes(self, query_length, layer_idx: int = 0):
        q = query_length if isinstance(query_length, int) else int(query_length.shape[0])
        return self.get_seq_length(layer_idx) + q, 0

    def get_query_offset(self, layer_idx: int = 0) -> int:
        """Position of the first query of the next forward (transformers' Cache contract: the cached length)."""
        return self.get_seq_length(layer_idx)

    def get_max_cache_shape(self, *args, **kwargs):
        return None

    def get_max_length(self):
        return None

    def has_previous_state(self, layer_idx=None):
        if layer_idx is not None:
            return layer_idx < len(self._seq_lengths) and self._seq_lengths[layer_idx] > 0
        return any(s > 0 for s in self._seq_lengths)

    @property
    def seen_tokens(self):
        return self._seen_tokens

    @property
    def key_cache(self):
        return [torch.empty(0, device=self._device)] * len([s for s in self._seq_lengths if s > 0])

    @property
    def value_cache(self):
        return self.key_cache

    @property
    def is_initialized(self):
        return any(s > 0 for s in self._seq_lengths)

    @property
    def is_sliding(self):
        return [False] * self.num_layers

    @property
    def max_cache_len(self):
        return max(self._seq_lengths) if self._seq_lengths else 0

    def __len__(self) -> int:
        return len([s for s in self._seq_lengths if s > 0])

    def __getitem__(self, layer_idx: int):
        if self._seq_lengths[layer_idx] > 0:
            return self._get_full_cache(layer_idx)
        raise IndexError("Layer %d not in cache" % layer_idx)

    def __iter__(self):
        for i in range(self.num_layers):
            if self._seq_lengths[i] > 0:
                yield self._get_full_cache(i)

    def __bool__(self):
        return True

    def to_legacy_cache(self):
        return tuple(self._get_full_cache(i) for i in range(self.num_layers) if self._seq_lengths[i] > 0)
