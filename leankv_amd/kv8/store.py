"""One layer's keys and values in 8 bits, and the attention that reads them (lkv_kv8_* in include/leankv_amd.h).

Every finished block of 64 tokens of a kv head is held as one byte a number with one fp32 scale for its keys and one
for its values (amax / 127; no rotation, no codebook); the unfinished last block of a sequence is fp16.  A stored token
costs 256 bytes a kv head instead of 512, and a number is off by at most half a code, amax / 254.  For each finished
block the store also keeps the lowest and the highest key code of every dim, from which the sparse decode attention
finds the blocks worth reading; of the last finished block it keeps the fp16 tokens too, so that a sequence can be taken
back into it (drafted tokens that were not accepted).

The store does not know its sequences' lengths: they live with the caller, as int32 device tensors that every call
takes, so that a decode step can be captured into a HIP graph and replayed with other lengths.  Nothing here
synchronises, and every workspace is allocated for its call on the current stream.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._lib import LeanKVError, check

HEAD_DIM = 128
BLOCK = 64
_DTYPES = {torch.float32: _lib.LKV_DTYPE_F32, torch.float16: _lib.LKV_DTYPE_F16, torch.bfloat16: _lib.LKV_DTYPE_BF16}
_I64x3 = ctypes.c_int64 * 3
_SCALE = 1.0 / math.sqrt(HEAD_DIM)


@functools.lru_cache(maxsize=256)
def _strides3(b: int, h: int, s: int):
    return _I64x3(b, h, s)


@functools.lru_cache(maxsize=256)
def _attn_bytes(batch: int, heads: int, kv_heads: int, S: int, max_len: int, n_index: int) -> int:
    return _lib.load().lkv_kv8_attn_workspace_bytes(batch, heads, kv_heads, S, max_len, n_index)


@functools.lru_cache(maxsize=256)
def _select_bytes(batch: int, kv_heads: int, max_len: int) -> int:
    return _lib.load().lkv_kv8_select_workspace_bytes(batch, kv_heads, max_len)


@functools.lru_cache(maxsize=256)
def _sparse_bytes(batch: int, heads: int, kv_heads: int, max_len: int, blocks: int) -> int:
    return _lib.load().lkv_kv8_sparse_attn_workspace_bytes(batch, heads, kv_heads, max_len, blocks)


def _dtype(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise LeanKVError("%s: float16, bfloat16 or float32 expected, got %s" % (what, t.dtype))
    return code


def _in_place(shape, strides, t: torch.Tensor):
    """The strides of batch, head and token of t [B, H, S, 128] as the kernels take them, None where its rows are not
    dense or not 16-byte aligned.  Strides of single sizes count as 0 (torch leaves them free)."""
    b = strides[0] if shape[0] > 1 else 0
    h = strides[1] if shape[1] > 1 else 0
    s = strides[2] if shape[2] > 1 else 0
    if strides[3] != 1 or (b | h | s) % (16 // t.element_size()) or t.data_ptr() % 16:
        return None
    return _strides3(b, h, s)


@functools.lru_cache(maxsize=256)
def _apart(sizes, strides) -> bool:
    """Whether rows of 128 numbers at these strides lie apart from each other (outputs are written by many workgroups at
    once)."""
    dims = sorted((st, n) for n, st in zip(sizes, strides) if n != 1)
    if not all(n for _, n in dims):
        return True
    end = HEAD_DIM  # numbers from the first to the last of the sizes so far
    for st, n in dims:
        if st < end:
            break
        end += st * (n - 1)
    else:
        return True
    at = torch.zeros(1, dtype=torch.int64, device="cpu")  # rows of one size between those of another: look at every row
    for st, n in dims:
        at = (at.unsqueeze(1) + st * torch.arange(n, device="cpu")).flatten()
    return bool((at.sort().values.diff() >= HEAD_DIM).all())


def _rows(t: torch.Tensor):
    """(t or a copy of it, strides) for t [B, H, S, 128] that is read."""
    strides = _in_place(t.shape, t.stride(), t)
    if strides is None:
        t = t.detach().clone(memory_format=torch.contiguous_format)
        strides = _in_place(t.shape, t.stride(), t)
    return t, strides


def _query_rows(q: torch.Tensor):
    """The same for q [B, H, 128]: one token a sequence."""
    b, h, d = q.stride()
    strides = _in_place((q.shape[0], q.shape[1], 1), (b, h, 0, d), q)
    if strides is None:
        q = q.detach().clone(memory_format=torch.contiguous_format)
        strides = _strides3(q.stride(0), q.stride(1), 0)
    return q, strides


def _follow(what: str, a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether autograd follows a or b.  A forward-mode tangent would be lost at once and is refused."""
    if getattr(forward_ad, "_current_level", -1) >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (a, b)):
        raise LeanKVError("%s: the 8-bit store has no forward-mode derivative" % what)
    return (a.requires_grad or b.requires_grad) and torch.is_grad_enabled()


class _NoBackward(torch.autograd.Function):
    """Ties an output to what autograd follows, so that a backward pass through it raises instead of leaving it out."""

    @staticmethod
    def forward(ctx, out, what, anchor):
        ctx.what = what
        ctx.mark_dirty(out)
        return out

    @staticmethod
    def backward(ctx, grad):
        raise LeanKVError("%s: the 8-bit store has no backward pass" % ctx.what)


class KV8Store:
    """Keys and values of `batch` sequences x `kv_heads` heads of 128 dims, up to `capacity` tokens each (rounded up to
    whole blocks of 64), in 8 bits with a scale for each block and head.

        store = KV8Store(batch, kv_heads, capacity, device="cuda")
        store.update(k, v, pos)                        # S new tokens of every sequence, at positions pos[b] ..
        out = store.prefill_attention(q, lens)         # their queries, causal over everything stored
        out = store.decode_attention(q1, lens)         # one new token's queries
        out, index = store.sparse_decode_attention(q1, lens, blocks=64)
        k, v = store.read(lens, n)                     # the K / V that attention sees, fp16

    pos, lens, n_new and q_lens are int32 device tensors [batch]; lens counts every stored token, the queries' own among
    them, and may not pass the capacity or max_len (a longer sequence counts as one that ends with the last finished block
    below, its queries the last tokens of that).  The work is split for max_len: give it where the capacity is many times
    the lengths.  Inputs are float16, bfloat16 or float32 of any strides; they are rounded to
    float16 first (infinities and larger numbers to +-65504; a NaN key or value is stored as 0).  There is no gradient: a
    backward pass through the outputs of queries, keys or values that autograd follows raises."""

    _followed = False  # autograd followed keys or values that were stored

    def __init__(self, batch: int, kv_heads: int, capacity: int, device="cuda"):
        if batch < 1 or kv_heads < 1 or capacity < 1:
            raise ValueError("KV8Store: batch, kv_heads and capacity must be at least 1, got %d, %d, %d"
                             % (batch, kv_heads, capacity))
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise LeanKVError("leankv_amd kernels run on the GPU only; got device %s" % self.device)
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.batch, self.kv_heads = int(batch), int(kv_heads)
        self.blocks = -(-int(capacity) // BLOCK)
        rows = (self.batch, self.kv_heads)

        def zeros(*shape, dtype):
            return torch.zeros(*rows, *shape, dtype=dtype, device=self.device)

        self.k_codes = zeros(self.blocks, BLOCK, HEAD_DIM, dtype=torch.uint8)
        self.v_codes = zeros(self.blocks, HEAD_DIM, BLOCK, dtype=torch.uint8)
        self.scales = zeros(self.blocks, 2, dtype=torch.float32)
        self.ranges = zeros(self.blocks, 2, HEAD_DIM, dtype=torch.int8)
        # fp16 tokens of the last two blocks, block j's in [:, :, j & 1]
        self.k_tails = zeros(2, BLOCK, HEAD_DIM, dtype=torch.float16)
        self.v_tails = zeros(2, HEAD_DIM, BLOCK, dtype=torch.float16)
        self._struct = _lib.KV8StoreStruct(self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.scales.data_ptr(),
                                           self.ranges.data_ptr(), self.k_tails.data_ptr(), self.v_tails.data_ptr(),
                                           self.batch, self.kv_heads, self.blocks)
        self._ref = ctypes.byref(self._struct)
        self._index = self.device.index
        self._lib = _lib.load()

    @property
    def capacity(self) -> int:
        return self.blocks * BLOCK

    def nbytes(self) -> int:
        """Device bytes of the store."""
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.v_codes, self.scales, self.ranges,
                                                          self.k_tails, self.v_tails))

    def _open(self, tails: torch.Tensor) -> torch.Tensor:
        """Of every sequence and head the tail of its unfinished block, which the update left with scales of -1."""
        block = (self.scales[..., 0] < 0).int().argmax(-1)  # (the lowest such)
        return torch.where((block & 1).bool()[..., None, None], tails[:, :, 1], tails[:, :, 0])

    @property
    def k_tail(self) -> torch.Tensor:
        """fp16 [batch, kv_heads, 64, 128]: a copy of the unfinished blocks' keys, as the newest update left them."""
        return self._open(self.k_tails)

    @property
    def v_tail(self) -> torch.Tensor:
        """fp16 [batch, kv_heads, 128, 64]: the same of their values, in the order of the codes."""
        return self._open(self.v_tails)

    def grown(self, capacity: int) -> "KV8Store":
        """A store of `capacity` tokens that holds what this one does."""
        new = KV8Store(self.batch, self.kv_heads, max(capacity, self.capacity), self.device)
        for name in ("k_codes", "v_codes", "scales", "ranges"):
            getattr(new, name)[:, :, :self.blocks] = getattr(self, name)
        new.k_tails.copy_(self.k_tails)
        new.v_tails.copy_(self.v_tails)
        new._followed = self._followed
        return new

    def __deepcopy__(self, memo):
        """A store of its own with the same contents (a prompt's cache that several continuations start from)."""
        new = memo[id(self)] = self.grown(self.capacity)
        return new

    # ------------------------------------------------------------------------------------------------ checks
    def _call(self, name: str, *args):
        """One C entry on the store's device and that device's current stream."""
        idx = self._index
        if torch._C._cuda_getDevice() == idx:
            rc = getattr(self._lib, name)(self._ref, *args, torch._C._cuda_getCurrentRawStream(idx))
        else:
            with torch.cuda.device(idx):
                rc = getattr(self._lib, name)(self._ref, *args, torch._C._cuda_getCurrentRawStream(idx))
        if rc:
            check(rc, name)

    def _ints(self, t, what: str, name: str):
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or not t.is_cuda \
                or t.get_device() != self._index or t.numel() != self.batch or not t.is_contiguous():
            raise LeanKVError("%s: %s must be a contiguous int32 tensor of %d entries on %s"
                              % (what, name, self.batch, self.device))
        return t.data_ptr()

    def _queries(self, q, dims: int, what: str):
        """Heads of q [batch, heads(, S), 128] and its dtype code."""
        n = q.shape
        if len(n) != dims or n[0] != self.batch or n[-1] != HEAD_DIM or n[1] % self.kv_heads or not n[1] \
                or not q.is_cuda or q.get_device() != self._index:
            raise LeanKVError("%s: q must be [%d, heads, %s%d] on %s with a multiple of %d heads, got %s on %s"
                              % (what, self.batch, "S, " if dims == 4 else "", HEAD_DIM, self.device, self.kv_heads,
                                 tuple(n), q.device))
        return n[1], _dtype(q, what)

    def _bound(self, max_len, what: str) -> int:
        if max_len is None:
            return self.blocks * BLOCK
        if not 0 <= int(max_len) <= self.blocks * BLOCK:
            raise LeanKVError("%s: max_len=%d outside a store of %d tokens" % (what, max_len, self.blocks * BLOCK))
        return int(max_len)

    # Workspaces too are allocated for their call, on the current stream: calls on several streams and captured graphs share
    # none.  (new_empty of a tensor at hand is half a microsecond less a call than empty with a device.)
    def _empty(self, shape, dtype):
        return torch.empty(shape, dtype=dtype, device=self.device)

    def _workspace(self, nbytes: int):
        return self.k_codes.new_empty(nbytes) if nbytes else None

    def _output(self, out: torch.Tensor, what: str, q: torch.Tensor | None = None) -> torch.Tensor:
        """out as the caller gets it: with autograd following q or what is stored, tied to it."""
        follows = q is not None and _follow(what, q, q)
        if not follows and not (self._followed and torch.is_grad_enabled()):
            return out
        return _NoBackward.apply(out, what, q if follows else torch.zeros((), device="cpu", requires_grad=True))

    def _no_grad_out(self, q: torch.Tensor, what: str) -> None:
        if _follow(what, q, q) or (self._followed and torch.is_grad_enabled()):
            raise LeanKVError("%s: out= does not support autograd, which follows q or what is stored" % what)

    # ------------------------------------------------------------------------------------------------ storing
    def update(self, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, n_new: torch.Tensor | None = None) -> None:
        """Store S new tokens of every sequence: k, v [batch, kv_heads, S, 128], sequence b's at positions pos[b] .. (what
        it holds already).  n_new: how many of the S are sequence b's (a padded batch; the rest is not read).  Tokens
        past the capacity are dropped.  One launch; blocks that become whole are quantized.

        A sequence may be taken back (a smaller pos and length from then on): to any multiple of 64, where it begins anew,
        or, no further than where it began, to any length from 64 * (n // 64 - 1) on, n the most tokens that it has held
        since then (so up to 64 drafted tokens may be dropped wherever blocks end).  An older block is not opened again:
        to drop some of its tokens, take the sequence back to its start and store the others anew (read gives them as they
        are held)."""
        what = "KV8Store.update"
        nk, nv = k.shape, v.shape
        for t, n, name in ((k, nk, "k"), (v, nv, "v")):
            if len(n) != 4 or n[0] != self.batch or n[1] != self.kv_heads or n[3] != HEAD_DIM or not t.is_cuda \
                    or t.get_device() != self._index:
                raise LeanKVError("%s: %s must be [%d, %d, S, %d] on %s, got %s on %s"
                                  % (what, name, self.batch, self.kv_heads, HEAD_DIM, self.device, tuple(n), t.device))
        if nk != nv or k.dtype != v.dtype:
            raise LeanKVError("%s: k and v must be alike, got %s %s and %s %s"
                              % (what, k.dtype, tuple(nk), v.dtype, tuple(nv)))
        dtype = _dtype(k, what)
        if _follow(what, k, v):
            self._followed = True
        p = self._ints(pos, what, "pos")
        m = None if n_new is None else self._ints(n_new, what, "n_new")
        (k, ks), (v, vs) = _rows(k), _rows(v)
        self._call("lkv_kv8_update", k.data_ptr(), ks, v.data_ptr(), vs, dtype, nk[2], p, m)

    def read(self, lens: torch.Tensor, n: int, first: int = 0):
        """(K, V) float16 [batch, kv_heads, n - first, 128]: tokens first .. n - 1 of every sequence as attention sees
        them, zeros past its length."""
        what = "KV8Store.read"
        if not 0 <= first <= n <= self.blocks * BLOCK:
            raise LeanKVError("%s: tokens %d .. %d outside a store of %d" % (what, first, n, self.blocks * BLOCK))
        p = self._ints(lens, what, "lens")
        kv = self._empty((2, self.batch, self.kv_heads, n - first, HEAD_DIM), torch.float16)
        if self._followed:
            kv = self._output(kv, what)
        k, v = kv.unbind(0)
        self._call("lkv_kv8_read", p, first, n - first, k.data_ptr(), v.data_ptr())
        return k, v

    # ---------------------------------------------------------------------------------------------- attention
    def decode_attention(self, q: torch.Tensor, lens: torch.Tensor, max_len: int | None = None,
                         scale: float | None = None, out: torch.Tensor | None = None,
                         index: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one query per sequence and head, q [batch, heads, 128], over everything stored (its own token
        among it): [batch, heads, 128] in q's type.  A sequence of length 0 gives zeros.  max_len: the caller's bound on
        lens (default the capacity), which the work is split for.  scale: 1 / sqrt(128) by default.  index: int32
        [batch, kv_heads, n], only these finished blocks of a kv head (as select_blocks gives them; others than finished
        ones are skipped, one listed twice counts twice) and the unfinished one.  out: a buffer like q whose rows are
        dense, 16-byte aligned and apart from each other (q itself may be it)."""
        what = "KV8Store.decode_attention"
        heads, dtype = self._queries(q, 3, what)
        p, L = self._ints(lens, what, "lens"), self._bound(max_len, what)
        n, list_ = 0, None
        if index is not None:
            if not isinstance(index, torch.Tensor) or index.dtype is not torch.int32 or index.dim() != 3 or index.shape[0] != self.batch \
                    or index.shape[1] != self.kv_heads or not index.shape[2] or index.device != self.device \
                    or not index.is_contiguous():
                raise LeanKVError("%s: index must be a contiguous int32 tensor [%d, %d, n] on %s"
                                  % (what, self.batch, self.kv_heads, self.device))
            n, list_ = index.shape[2], index.data_ptr()
        if out is None:
            out = self._output(q.new_empty((self.batch, heads, HEAD_DIM)), what, q)
            os = _strides3(heads * HEAD_DIM, HEAD_DIM, 0)
        else:
            self._no_grad_out(q, what)
            os = None if out.dim() != 3 else _in_place((self.batch, heads, 1), (*out.stride()[:2], 0, out.stride(2)), out)
            if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or os is None:
                raise LeanKVError("%s: out must be like q, %s %s on %s, with dense 16-byte aligned rows"
                                  % (what, q.dtype, tuple(q.shape), q.device))
            if not _apart(tuple(out.shape[:2]), out.stride()[:2]):
                raise LeanKVError("%s: rows of out overlap, strides %s" % (what, out.stride()))
        q, qs = _query_rows(q)
        nbytes = _attn_bytes(self.batch, heads, self.kv_heads, 1, L, n)
        ws = self._workspace(nbytes)
        self._call("lkv_kv8_attn", q.data_ptr(), qs, dtype, heads, 1, p, None, L, list_, n,
                   _SCALE if scale is None else scale, out.data_ptr(), os, None if ws is None else ws.data_ptr(), nbytes)
        return out

    def prefill_attention(self, q: torch.Tensor, lens: torch.Tensor, q_lens: torch.Tensor | None = None,
                          max_len: int | None = None, scale: float | None = None,
                          out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of the S newest tokens' queries q [batch, heads, S, 128] (after their update): query i of a
        sequence with q_lens[b] of them (default S, at most its length) sees tokens 0 .. lens[b] - q_lens[b] + i.  Rows
        from q_lens[b] on are zeros.  Returns [batch, heads, S, 128] in q's type, laid out [batch, S, heads, 128], or out
        (as for decode_attention)."""
        what = "KV8Store.prefill_attention"
        heads, dtype = self._queries(q, 4, what)
        p, L = self._ints(lens, what, "lens"), self._bound(max_len, what)
        m = None if q_lens is None else self._ints(q_lens, what, "q_lens")
        S = q.shape[2]
        if out is None:  # laid out token by token, as an output projection reads it
            out = self._output(q.new_empty((self.batch, S, heads, HEAD_DIM)), what, q).transpose(1, 2)
        else:
            self._no_grad_out(q, what)
            if out.dim() == 4 and not _apart(tuple(out.shape[:3]), out.stride()[:3]):
                raise LeanKVError("%s: rows of out overlap, strides %s" % (what, out.stride()))
        os = _in_place(q.shape, out.stride(), out) if out.dim() == 4 else None
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or os is None:
            raise LeanKVError("%s: out must be like q, %s %s on %s, with dense 16-byte aligned rows"
                              % (what, q.dtype, tuple(q.shape), q.device))
        q, qs = _rows(q)
        nbytes = _attn_bytes(self.batch, heads, self.kv_heads, S, L, 0)
        ws = self._workspace(nbytes)
        self._call("lkv_kv8_attn", q.data_ptr(), qs, dtype, heads, S, p, m, L, None, 0,
                   _SCALE if scale is None else scale, out.data_ptr(), os, None if ws is None else ws.data_ptr(), nbytes)
        return out

    # ------------------------------------------------------------------------------------------------- sparse
    def _choice(self, blocks, sink, recent, what):
        blocks, sink, recent = int(blocks), int(sink), int(recent)
        if blocks < 1 or sink < 0 or recent < 0 or sink + recent > blocks:
            raise LeanKVError("%s: %d blocks with the first %d and the last %d among them" % (what, blocks, sink, recent))
        return blocks, sink, recent

    def select_blocks(self, q: torch.Tensor, lens: torch.Tensor, blocks: int, sink: int = 1, recent: int = 1,
                      max_len: int | None = None) -> torch.Tensor:
        """int32 [batch, kv_heads, blocks]: for one query per sequence, q [batch, heads, 128], the finished blocks with
        the highest upper bound of q.k (over the kv head's queries), ascending, -1 where a sequence has fewer.  The first
        `sink` and the last `recent` finished blocks are always among them; of equal scores the lower index wins."""
        what = "KV8Store.select_blocks"
        heads, dtype = self._queries(q, 3, what)
        p, L = self._ints(lens, what, "lens"), self._bound(max_len, what)
        blocks, sink, recent = self._choice(blocks, sink, recent, what)
        q, qs = _query_rows(q)
        index = self._empty((self.batch, self.kv_heads, blocks), torch.int32)
        nbytes = _select_bytes(self.batch, self.kv_heads, L)
        ws = self._workspace(nbytes)
        self._call("lkv_kv8_select_blocks", q.data_ptr(), qs, dtype, heads, p, L, blocks, sink, recent,
                   index.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
        return index

    def sparse_decode_attention(self, q: torch.Tensor, lens: torch.Tensor, blocks: int, sink: int = 1, recent: int = 1,
                                max_len: int | None = None, scale: float | None = None):
        """decode_attention over the blocks that select_blocks chooses and the unfinished block: (out [batch, heads, 128],
        index)."""
        what = "KV8Store.sparse_decode_attention"
        heads, dtype = self._queries(q, 3, what)
        p, L = self._ints(lens, what, "lens"), self._bound(max_len, what)
        blocks, sink, recent = self._choice(blocks, sink, recent, what)
        q, qs = _query_rows(q)
        index = self._empty((self.batch, self.kv_heads, blocks), torch.int32)
        out = self._output(q.new_empty((self.batch, heads, HEAD_DIM)), what, q)
        nbytes = _sparse_bytes(self.batch, heads, self.kv_heads, L, blocks)
        ws = self._workspace(nbytes)
        self._call("lkv_kv8_sparse_attn", q.data_ptr(), qs, dtype, heads, p, L, blocks, sink, recent,
                   _SCALE if scale is None else scale, index.data_ptr(), out.data_ptr(),
                   _strides3(heads * HEAD_DIM, HEAD_DIM, 0), None if ws is None else ws.data_ptr(), nbytes)
        return out, index
