"""PagedCache: an HF past_key_values in 16-bit pages, whose sequences share pages while they are alike.

Next to TurboQuantCache and BlockInt8Cache, which hold fewer bits: the keys and values as the model computed them, so that
results are those of HF's own cache.  Beam search reorders it by forking pages (PagedKV.fork), assisted generation cuts it
(crop).  By default update() returns the whole K / V, so it works under any attention implementation.  With
fused_attention=True (what optimize_model(paged_kv=True) and leankv_amd.turboquant.attention.use_on(model, cache) set) it defers
attention to the kernels that read the pages, and the model has to run the "leankv_tq" attention implementation; a deferred
update that none of its calls consumed makes the next update raise.

No gradient flows through the stored tokens: with gradients enabled a forward pass runs, its backward pass raises.
Lengths live on the host here; a step that is to be captured into a HIP graph is built from PagedKV.
"""

from __future__ import annotations

import math

import torch

from ..hf_cache import HFCache
from ..turboquant.cache import set_active
from .packed import DTYPES, HEAD_DIM, packed_attention
from .pool import PAGE_SIZES, PagedKV


def _packed(t: torch.Tensor) -> torch.Tensor:
    """[B, heads, S, 128] as rows [B * S, heads, 128] (a view for one sequence or one token each)."""
    B, H, S, D = t.shape
    if S == 1:
        return t[:, :, 0]
    return t[0].transpose(0, 1) if B == 1 else t.transpose(1, 2).reshape(B * S, H, D)


class PagedCache(HFCache):
    """KV cache of num_layers layers in pages of page_size tokens (one PagedKV, allocated by the first update and grown by
    doubling past max_seq_len)."""

    def __init__(self, head_dim: int = HEAD_DIM, num_layers: int = 32, device=None, max_seq_len: int = 4096,
                 page_size: int = 64, fused_attention: bool = False):
        if head_dim != HEAD_DIM:
            raise ValueError("PagedCache: head_dim=%d is not built (the HIP kernels take head_dim %d)" % (head_dim, HEAD_DIM))
        if num_layers < 1:
            raise ValueError("PagedCache: num_layers must be at least 1")
        if page_size not in PAGE_SIZES:
            raise ValueError("PagedCache: page_size=%s must be one of %s" % (page_size, PAGE_SIZES))
        self.head_dim, self.num_layers, self.page_size = head_dim, num_layers, page_size
        self._device = torch.device(device) if device is not None else torch.device("cuda")
        self._init_cap = max(int(max_seq_len), 1)
        self.fused_attention = bool(fused_attention)
        self.reset()

    def reset(self):
        n = self.num_layers
        self.kv: PagedKV | None = None
        self._seen_tokens = 0
        self._seq_lengths = [0] * n
        self._fused_pending = [False] * n    # a one-token update awaits decode_attention
        self._prefill_pending = [False] * n  # a several-token update awaits prefill_attention
        self._pending_len = [0] * n
        self._rows: list = [None] * n        # a whole prompt's keys and values, until its attention
        self._cu = None

    # ----------------------------------------------------------- storage
    def _room(self, B: int, H: int, tokens: int, t: torch.Tensor) -> PagedKV:
        """The pages, with room for `tokens` of every sequence (what they share is to spare)."""
        if self.kv is None:
            cap = max(self._init_cap, tokens)
            self.kv = PagedKV(self.num_layers, H, B * -(-cap // self.page_size), B, cap, self.page_size, t.dtype, t.device)
        kv = self.kv
        self._alike(t)
        if tokens > kv.max_len:
            cap = kv.max_len
            while cap < tokens:
                cap *= 2
            self.kv = kv = kv.resized(max(kv.num_pages, B * (cap // self.page_size)), cap)
        return kv

    def _alike(self, t: torch.Tensor):
        kv, (B, H) = self.kv, t.shape[:2]
        if (kv.max_seqs, kv.kv_heads, kv.dtype, kv.device) != (B, H, t.dtype, t.device):
            raise ValueError("PagedCache: holds %d sequences of %d heads in %s on %s, got %d of %d in %s on %s"
                             % (kv.max_seqs, kv.kv_heads, kv.dtype, kv.device, B, H, t.dtype, t.device))

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int, cache_kwargs=None):
        if self._fused_pending[layer_idx] or self._prefill_pending[layer_idx]:
            raise RuntimeError(
                "PagedCache(fused_attention=True): layer %d's previous update was never attended by the "
                "'leankv_tq' attention implementation, so the model attended to the newest tokens only; call "
                "leankv_amd.turboquant.attention.use_on(model, cache) or build the cache with "
                "fused_attention=False" % layer_idx)
        if key_states.dtype not in DTYPES:
            raise ValueError("PagedCache: float16 or bfloat16 keys and values expected, got %s" % key_states.dtype)
        if key_states.dim() != 4 or key_states.shape[3] != HEAD_DIM or value_states.shape != key_states.shape \
                or value_states.dtype != key_states.dtype or value_states.device != key_states.device:
            raise ValueError("PagedCache: keys and values must be [B, heads, tokens, %d] of one type on one device, got %s %s on "
                             "%s and %s %s on %s" % (HEAD_DIM, tuple(key_states.shape), key_states.dtype, key_states.device,
                                                     tuple(value_states.shape), value_states.dtype, value_states.device))
        B, H, S, _ = key_states.shape
        p0 = self._seq_lengths[layer_idx]
        T = p0 + S
        if layer_idx == 0:
            kv = self._room(B, H, T, key_states)
            # (one more token a sequence: extend and store take the rows as they are)
            self._cu = None if S == 1 and p0 else torch.arange(B + 1, dtype=torch.int32, device=kv.device) * S
            kv.extend(self._cu)
        elif self.kv is None or T != self._seq_lengths[0]:
            raise RuntimeError("PagedCache: layer %d would hold %d tokens, layer 0 holds %d (layers are updated in order)"
                               % (layer_idx, T, self._seq_lengths[0]))
        else:
            self._alike(key_states)
        set_active(self)
        kv = self.kv
        try:
            k, v = _packed(key_states), _packed(value_states)
            if S:
                kv.store(layer_idx, k, v, self._cu)
        except Exception:
            if layer_idx == 0:  # the room that was made for them
                kv.truncate(torch.full((B,), p0, dtype=torch.int32, device=kv.device))
            raise
        self._seq_lengths[layer_idx] = T
        if layer_idx == 0:
            self._seen_tokens += S
        if self.fused_attention and S:
            (self._fused_pending if S == 1 and p0 else self._prefill_pending)[layer_idx] = True
            self._pending_len[layer_idx] = T
            self._rows[layer_idx] = (k, v) if not p0 else None
            return key_states, value_states
        return self._get_full_cache(layer_idx)

    def _get_full_cache(self, layer_idx: int):
        """K, V [B, H, tokens, 128] of the layer."""
        return self.kv.read(layer_idx, self._seq_lengths[layer_idx])

    def _take(self, layer_idx: int):
        self._prefill_pending[layer_idx] = self._fused_pending[layer_idx] = False
        rows, self._rows[layer_idx] = self._rows[layer_idx], None
        return rows

    def take_full_cache(self, layer_idx: int):
        """The whole K / V for a pending update whose attention runs elsewhere (a padding mask, a sliding window)."""
        self._take(layer_idx)
        return self._get_full_cache(layer_idx)

    # ----------------------------------------------------------- attention over the pages
    def _scale(self, scaling):
        return 1.0 / math.sqrt(self.head_dim) if scaling is None else float(scaling)

    def decode_attention(self, layer_idx: int, query: torch.Tensor, scaling: float | None = None) -> torch.Tensor:
        """Attention of a single query [B, Hq, 1, D] over this layer's cache -> [B, Hq, 1, D]."""
        if not self._fused_pending[layer_idx]:
            raise RuntimeError("PagedCache.decode_attention: no one-token update pending for layer %d" % layer_idx)
        self._take(layer_idx)
        # (a bound in whole steps of the work, so that most calls find the workspace's size where it was last looked up)
        bound = min(-(-self._pending_len[layer_idx] // 128) * 128, self.kv.max_len)
        return self.kv.decode_attention(layer_idx, query.squeeze(2), max_len=bound, scale=self._scale(scaling)).unsqueeze(2)

    def prefill_attention(self, layer_idx: int, query: torch.Tensor, scaling: float | None = None) -> torch.Tensor:
        """Causal attention of the newest S tokens' queries [B, Hq, S, D] over this layer's cache -> [B, Hq, S, D]."""
        if not self._prefill_pending[layer_idx]:
            raise RuntimeError("PagedCache.prefill_attention: no several-token update pending for layer %d" % layer_idx)
        rows, q = self._take(layer_idx), _packed(query)
        B, H, S, D = query.shape
        if rows is not None:  # a whole prompt: its keys and values as they came
            out = packed_attention(q, *rows, self._cu, max_len=S, scale=self._scale(scaling))
        else:
            out = self.kv.prefill_attention(layer_idx, q, self._cu, max_new=S, max_len=self._pending_len[layer_idx],
                                            scale=self._scale(scaling))
        return out.view(B, S, H, D).transpose(1, 2)

    # ----------------------------------------------------------- HF interface (the rest: HFCache)
    def _idle(self, what: str):
        if any(self._fused_pending) or any(self._prefill_pending):
            raise RuntimeError("PagedCache.%s: an update awaits its attention" % what)

    def crop(self, max_length: int):
        """Keeps the first max_length tokens (0 or negative: drops that many from the end, as HF's caches do).  An integer, or
        a tensor of one (assisted generation gives it; one on the device is waited for)."""
        self._idle("crop")
        n, max_length = self._seq_lengths[0], int(max_length)
        keep = max(0, n + max_length) if max_length <= 0 else min(n, max_length)
        if self.kv is not None and keep < n:
            self.kv.truncate(torch.full((self.kv.max_seqs,), keep, dtype=torch.int32, device=self.kv.device))
        self._seq_lengths = [min(keep, x) for x in self._seq_lengths]
        self._seen_tokens = self._seq_lengths[0]

    def activate_past_recording(self):
        """Called before tokens that may be cut again (assisted generation); pages need no record of them."""

    def reorder_cache(self, beam_idx: torch.LongTensor):
        """Sequence b goes on from sequence beam_idx[b] (beam search): pages are shared, not copied.  (Beams on the device are
        waited for: one out of range would empty its sequence there, while its tokens are counted here.)"""
        self._idle("reorder_cache")
        if self.kv is None:
            return
        if beam_idx.numel() != self.kv.max_seqs:
            raise ValueError("PagedCache.reorder_cache: %d beams of %d sequences" % (beam_idx.numel(), self.kv.max_seqs))
        if beam_idx.dtype not in (torch.int32, torch.int64) or bool(((beam_idx < 0) | (beam_idx >= self.kv.max_seqs)).any()):
            raise ValueError("PagedCache.reorder_cache: beams are sequence numbers 0 .. %d" % (self.kv.max_seqs - 1))
        self.kv.fork(beam_idx.reshape(-1).to(device=self.kv.device, dtype=torch.int32).contiguous())

    def _chosen(self, index: torch.Tensor):
        if self.kv is not None:
            self.kv = self.kv.chosen(index.to(self.kv.device))

    def batch_repeat_interleave(self, repeats: int):
        self._idle("batch_repeat_interleave")
        if self.kv is not None:
            self._chosen(torch.arange(self.kv.max_seqs, device=self.kv.device).repeat_interleave(repeats))

    def batch_select_indices(self, indices: torch.Tensor):
        self._idle("batch_select_indices")
        self._chosen(indices)

    @property
    def max_batch_size(self):
        return 0 if self.kv is None else self.kv.max_seqs

    def get_total_cache_bytes(self) -> int:
        """Bytes of the pages in use (this waits for the device)."""
        if self.kv is None:
            return 0
        return int((self.kv.refs > 0).sum()) * self.kv.pool[:, 0].numel() * 2

    def get_fp16_equivalent_bytes(self) -> int:
        if self.kv is None:
            return 0
        return sum(self.kv.max_seqs * self.kv.kv_heads * n * 4 * HEAD_DIM for n in self._seq_lengths)

    def get_compression_ratio(self) -> float:
        actual = self.get_total_cache_bytes()
        return 0.0 if actual == 0 else self.get_fp16_equivalent_bytes() / actual
