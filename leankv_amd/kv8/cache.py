"""BlockInt8Cache: an HF past_key_values in 8 bits with one scale for each block of 64 tokens and head.

Next to TurboQuantCache (1 to 4 bits, a rotation and a codebook): twice its 4-bit store, and values within amax / 254 of
the fp16 ones.  By default update() returns the whole K / V as attention sees it, so the cache works under any attention
implementation.  With fused_attention=True (what optimize_model(kv8=True) and leankv_amd.turboquant.attention.use_on(model,
cache) set) it defers attention to the kernels that read the 8-bit store, and the model has to run the "leankv_tq"
attention implementation; a deferred update that none of its calls consumed makes the next update raise.  sparse_blocks=n
lets a single-token step read, of every head's finished blocks, only the n with the highest score (KV8Store.select_blocks)
once there are more.

No gradient flows through the stored tokens: with gradients enabled a forward pass runs, its backward pass raises.
Lengths live on the host here: a step that is to be captured into a HIP graph and replayed at other lengths is built from
KV8Store, whose lengths are device tensors.
"""

from __future__ import annotations

import math

import torch

from ..hf_cache import HFCache
from ..turboquant.cache import set_active
from .store import BLOCK, HEAD_DIM, KV8Store


class BlockInt8Cache(HFCache):
    """KV cache of num_layers layers, 8 bits with block scales (one KV8Store a layer, allocated by its first update)."""

    def __init__(self, head_dim: int = 128, num_layers: int = 32, device=None, dtype: torch.dtype | None = None,
                 max_seq_len: int = 4096, fused_attention: bool = False, sparse_blocks: int | None = None,
                 sink_blocks: int = 1, recent_blocks: int = 1):
        if head_dim != HEAD_DIM:
            raise ValueError("BlockInt8Cache: head_dim=%d is not built (the HIP kernels take head_dim %d)"
                             % (head_dim, HEAD_DIM))
        if num_layers < 1:
            raise ValueError("BlockInt8Cache: num_layers must be at least 1")
        if sink_blocks < 0 or recent_blocks < 0 or (sparse_blocks is not None
                                                    and sparse_blocks < max(1, sink_blocks + recent_blocks)):
            raise ValueError("BlockInt8Cache: sparse_blocks=%s has no room for the first %d and the last %d blocks"
                             % (sparse_blocks, sink_blocks, recent_blocks))
        self.head_dim, self.num_layers = head_dim, num_layers
        self._device = torch.device(device) if device is not None else torch.device("cuda")
        self._asked_dtype = dtype  # of the K / V that update returns and that are read back (None: the keys')
        self._dtype = dtype
        self._init_cap = max(int(max_seq_len), 1)
        self.fused_attention = bool(fused_attention)
        self.sparse_blocks, self.sink_blocks, self.recent_blocks = sparse_blocks, sink_blocks, recent_blocks
        self._seen_tokens = 0
        self._seq_lengths = [0] * num_layers
        self._stores: list = [None] * num_layers
        self._pos_dev: list = [None] * num_layers  # int32 [B]: length before the newest update
        self._len_dev: list = [None] * num_layers  # int32 [B]: length after it
        self._fused_pending = [False] * num_layers    # a one-token update awaits decode_attention
        self._prefill_pending = [False] * num_layers  # a several-token update awaits prefill_attention
        self._pending_len = [0] * num_layers

    # ----------------------------------------------------------- storage
    def _store(self, li: int, B: int, H: int, tokens: int, device) -> KV8Store:
        """Layer li's store with room for `tokens`: allocated once, and grown by doubling."""
        st = self._stores[li]
        if st is None:
            st = KV8Store(B, H, max(self._init_cap, tokens), device=device)
            self._pos_dev[li] = torch.zeros(B, dtype=torch.int32, device=st.device)
            self._len_dev[li] = torch.zeros(B, dtype=torch.int32, device=st.device)
            self._stores[li] = st
        if (st.batch, st.kv_heads) != (B, H):
            raise ValueError("BlockInt8Cache: layer %d holds %d sequences of %d heads, got %d of %d"
                             % (li, st.batch, st.kv_heads, B, H))
        if tokens > st.capacity:
            cap = st.capacity
            while cap < tokens:
                cap *= 2
            self._stores[li] = st = st.grown(cap)
        return st

    # ----------------------------------------------------------- update
    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int, cache_kwargs=None):
        if self._fused_pending[layer_idx] or self._prefill_pending[layer_idx]:
            raise RuntimeError(
                "BlockInt8Cache(fused_attention=True): layer %d's previous update was never attended by the "
                "'leankv_tq' attention implementation, so the model attended to the newest tokens only; call "
                "leankv_amd.turboquant.attention.use_on(model, cache) or build the cache with "
                "fused_attention=False" % layer_idx)
        set_active(self)
        B, H, S, _ = key_states.shape
        p0 = self._seq_lengths[layer_idx]
        T = p0 + S
        st = self._store(layer_idx, B, H, T, key_states.device)
        self._pos_dev[layer_idx].fill_(p0)
        st.update(key_states, value_states, self._pos_dev[layer_idx])
        self._len_dev[layer_idx].fill_(T)
        self._seq_lengths[layer_idx] = T
        if layer_idx == 0:
            self._seen_tokens += S
        if self._dtype is None:
            self._dtype = key_states.dtype
        if self.fused_attention and S:
            (self._fused_pending if S == 1 else self._prefill_pending)[layer_idx] = True
            self._pending_len[layer_idx] = T
            return key_states, value_states
        return self._get_full_cache(layer_idx)

    def _get_full_cache(self, layer_idx: int):
        """K, V [B, H, tokens, 128] of the layer: finished blocks from their codes, the unfinished one as stored."""
        st, n = self._stores[layer_idx], self._seq_lengths[layer_idx]
        k, v = st.read(self._len_dev[layer_idx], n)
        return (k, v) if self._dtype == torch.float16 else (k.to(self._dtype), v.to(self._dtype))

    def take_full_cache(self, layer_idx: int):
        """The whole K / V for a pending update whose attention runs elsewhere (a padding mask, a sliding window)."""
        self._prefill_pending[layer_idx] = False
        self._fused_pending[layer_idx] = False
        return self._get_full_cache(layer_idx)

    # ----------------------------------------------------------- attention over the 8-bit store
    def decode_attention(self, layer_idx: int, query: torch.Tensor, scaling: float | None = None) -> torch.Tensor:
        """Attention of a single query [B, Hq, 1, D] over this layer's cache -> [B, Hq, 1, D]."""
        if not self._fused_pending[layer_idx]:
            raise RuntimeError("BlockInt8Cache.decode_attention: no one-token update pending for layer %d" % layer_idx)
        self._fused_pending[layer_idx] = False
        st, lens = self._stores[layer_idx], self._len_dev[layer_idx]
        q = query.squeeze(2)
        scale = 1.0 / math.sqrt(self.head_dim) if scaling is None else float(scaling)
        # (sized for the store's capacity: the same split of the work at every step, which a short sequence pays for in a
        # store with much more room: 4133 tokens 12 us a layer in one of 8192, 31 in one of 131072)
        if self.sparse_blocks is not None and self._seq_lengths[layer_idx] // BLOCK > self.sparse_blocks:
            out, _ = st.sparse_decode_attention(q, lens, self.sparse_blocks, self.sink_blocks, self.recent_blocks,
                                                scale=scale)
        else:
            out = st.decode_attention(q, lens, scale=scale)
        return out.unsqueeze(2)

    def prefill_attention(self, layer_idx: int, query: torch.Tensor, scaling: float | None = None) -> torch.Tensor:
        """Causal attention of the newest S tokens' queries [B, Hq, S, D] over this layer's cache -> [B, Hq, S, D]."""
        if not self._prefill_pending[layer_idx]:
            raise RuntimeError("BlockInt8Cache.prefill_attention: no several-token update pending for layer %d"
                               % layer_idx)
        self._prefill_pending[layer_idx] = False
        scale = 1.0 / math.sqrt(self.head_dim) if scaling is None else float(scaling)
        return self._stores[layer_idx].prefill_attention(query, self._len_dev[layer_idx],
                                                         max_len=self._pending_len[layer_idx], scale=scale)

    # ----------------------------------------------------------- HF interface (the rest: HFCache)
    def _unsupported(self, what: str):
        raise NotImplementedError("BlockInt8Cache: %s is not built (finished blocks cannot be cut or reordered)" % what)

    def crop(self, max_length: int):
        self._unsupported("crop")

    def batch_repeat_interleave(self, repeats: int):
        self._unsupported("batch_repeat_interleave")

    def batch_select_indices(self, indices: torch.Tensor):
        self._unsupported("batch_select_indices")

    def reorder_cache(self, beam_idx: torch.LongTensor):
        self._unsupported("reorder_cache")

    @property
    def max_batch_size(self):
        return next((s.batch for s in self._stores if s is not None), 0)

    def reset(self):
        n = self.num_layers
        self._stores, self._pos_dev, self._len_dev = [None] * n, [None] * n, [None] * n
        self._seq_lengths = [0] * n
        self._fused_pending, self._prefill_pending = [False] * n, [False] * n
        self._seen_tokens = 0
        self._dtype = self._asked_dtype

    def get_total_cache_bytes(self) -> int:
        """Bytes that the held tokens take: codes and scales and ranges of finished blocks, fp16 of the others."""
        total = 0
        for st, n in zip(self._stores, self._seq_lengths):
            if st is not None:
                per_block = 2 * BLOCK * HEAD_DIM + 8 + 2 * HEAD_DIM
                total += st.batch * st.kv_heads * (n // BLOCK * per_block + n % BLOCK * 4 * HEAD_DIM)
        return total

    def get_fp16_equivalent_bytes(self) -> int:
        return sum(st.batch * st.kv_heads * n * 4 * HEAD_DIM for st, n in zip(self._stores, self._seq_lengths)
                   if st is not None)

    def get_compression_ratio(self) -> float:
        actual = self.get_total_cache_bytes()
        return 0.0 if actual == 0 else self.get_fp16_equivalent_bytes() / actual
