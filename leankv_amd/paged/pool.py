"""Keys and values of many sequences in 16-bit pages, and the attention that reads them (lkv_pages_* in include/leankv_amd.h).

A pool has pages of page_size tokens in every layer; a sequence is a row of page ids and a length.  Pages are given out as
sequences grow, shared when one is forked (beams, several answers to one prompt), copied when a shared one is written to, and
free again when no sequence names them.  All of that happens on the device, on the current stream and without a
synchronisation, so that a step that grows or forks sequences can be captured into a HIP graph and replayed.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from .. import _lib
from .._lib import LeanKVError
from .packed import DTYPES, HEAD_DIM, MAX_SEQS, SCALE, apart, call, follow, out_rows, rows, strides2, tied

PAGE_SIZES = (16, 32, 64, 128, 256)


@functools.lru_cache(maxsize=256)
def _decode_bytes(seqs: int, heads: int, kv_heads: int, max_len: int) -> int:
    return _lib.load().lkv_pages_decode_attn_workspace_bytes(seqs, heads, kv_heads, max_len)


@functools.lru_cache(maxsize=256)
def _prefill_bytes(rows_: int, seqs: int, heads: int, kv_heads: int, max_new: int, max_len: int) -> int:
    return _lib.load().lkv_pages_prefill_attn_workspace_bytes(rows_, seqs, heads, kv_heads, max_new, max_len)


class PagedKV:
    """A pool of num_pages pages of page_size tokens (16 to 256, a power of two) in each of num_layers layers, kv_heads heads
    of 128 dims, float16 or bfloat16, for up to max_seqs sequences of up to max_len tokens (rounded up to whole pages).

        cache = PagedKV(num_layers, kv_heads, num_pages, max_seqs, max_len)
        cache.extend(cu)                                     # room for packed prompts: sequence s has rows cu[s] .. cu[s + 1]
        for layer in ...:
            cache.store(layer, k, v, cu)                     # [rows, kv_heads, 128]
            out = cache.prefill_attention(layer, q, cu)      # [rows, heads, 128], causal over everything stored
        cache.fork(parent)                                   # sequence s goes on from sequence parent[s]
        cache.extend()                                       # one token for every sequence that holds some
        for layer in ...:
            cache.store(layer, k1, v1)                       # [max_seqs, kv_heads, 128]
            out = cache.decode_attention(layer, q1)          # [max_seqs, heads, 128]
        cache.free(done)
        pages = cache.compact()

    Device tensors that may be read (and, by a program that knows what it does, written):
      pool   [num_layers, num_pages, 2 (K, V), kv_heads, page_size, 128]
      table  int32 [max_seqs, max_len / page_size], the pages of every sequence, -1 behind the last
      lens   int32 [max_seqs], tokens held
      refs   int32 [num_pages], how many entries of table name a page (0: free)
      taken  int32 [max_seqs], what the last extend made room for
    cu is int32 [max_seqs + 1] on the device, ascending: where the rows of every sequence begin.  Calls on one pool must be
    ordered on one stream (or by events).  Keys, values and queries have the pool's type and any strides.  There is no
    gradient: a backward pass through the outputs of queries, keys or values that autograd follows raises."""

    _followed = False  # autograd followed keys or values that were stored

    def __init__(self, num_layers: int, kv_heads: int, num_pages: int, max_seqs: int, max_len: int, page_size: int = 64,
                 dtype: torch.dtype = torch.float16, device="cuda"):
        if num_layers < 1 or kv_heads < 1 or num_pages < 1 or max_len < 1:
            raise ValueError("PagedKV: num_layers, kv_heads, num_pages and max_len must be at least 1, got %d, %d, %d, %d"
                             % (num_layers, kv_heads, num_pages, max_len))
        if not 1 <= max_seqs <= MAX_SEQS:
            raise ValueError("PagedKV: max_seqs=%d must be 1 to %d" % (max_seqs, MAX_SEQS))
        if page_size not in PAGE_SIZES:
            raise ValueError("PagedKV: page_size=%s must be one of %s" % (page_size, PAGE_SIZES))
        if max_seqs * (-(-max_len // page_size) + 1) >= 1 << 31:
            raise ValueError("PagedKV: a table of %d sequences of up to %d tokens is too large" % (max_seqs, max_len))
        if dtype not in DTYPES:
            raise ValueError("PagedKV: dtype=%s must be float16 or bfloat16" % dtype)
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise LeanKVError("leankv_amd kernels run on the GPU only; got device %s" % self.device)
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.num_layers, self.kv_heads, self.num_pages = int(num_layers), int(kv_heads), int(num_pages)
        self.max_seqs, self.page_size, self.dtype = int(max_seqs), int(page_size), dtype
        self.width = -(-int(max_len) // self.page_size)
        self.pool = torch.zeros(self.num_layers, self.num_pages, 2, self.kv_heads, self.page_size, HEAD_DIM, dtype=dtype,
                                device=self.device)
        # one buffer, so that a snapshot is one copy
        sizes = (self.max_seqs * self.width, self.max_seqs, self.num_pages, self.max_seqs)
        self._books = torch.zeros(sum(sizes), dtype=torch.int32, device=self.device)
        table, self.lens, self.refs, self.taken = self._books.split(sizes)
        self.table = table.view(self.max_seqs, self.width).fill_(-1)
        self._struct = _lib.PagesStruct(self.pool.data_ptr(), self.table.data_ptr(), self.lens.data_ptr(),
                                        self.refs.data_ptr(), self.taken.data_ptr(), self.num_layers, self.num_pages,
                                        self.kv_heads, self.page_size, self.max_seqs, self.width, DTYPES[dtype])
        self._ref = ctypes.byref(self._struct)
        self._index = self.device.index
        self._lib = lib = _lib.load()
        self._extend_bytes = lib.lkv_pages_extend_workspace_bytes(self.num_pages, self.max_seqs)
        self._fork_bytes = lib.lkv_pages_fork_workspace_bytes(self.max_seqs, self.width)
        self._compact_bytes = lib.lkv_pages_compact_workspace_bytes(self.num_pages)
        # of the calls that change the tables, which are ordered as the tables are
        self._scratch = self._books.new_empty(max(self._extend_bytes, self._fork_bytes, self._compact_bytes) // 4)
        self._scratch_ptr = self._scratch.data_ptr()

    @property
    def max_len(self) -> int:
        return self.width * self.page_size

    def nbytes(self) -> int:
        """Device bytes of the pool and its tables."""
        return self.pool.numel() * 2 + self._books.numel() * 4

    # ------------------------------------------------------------------------------------------------ checks
    def _ints(self, t, n: int, what: str, name: str):
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or not t.is_cuda or t.get_device() != self._index \
                or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
            raise LeanKVError("%s: %s must be a contiguous int32 tensor [%d] on %s" % (what, name, n, self.device))
        return t.data_ptr()

    def _cu(self, cu, what: str):
        return None if cu is None else self._ints(cu, self.max_seqs + 1, what, "cu")

    def _layer(self, layer: int, what: str) -> int:
        if not 0 <= layer < self.num_layers:
            raise LeanKVError("%s: layer %d of %d" % (what, layer, self.num_layers))
        return layer

    def _row_shape(self, t: torch.Tensor, what: str, name: str):
        if t.dim() != 3 or t.shape[2] != HEAD_DIM or t.dtype != self.dtype or not t.is_cuda or t.get_device() != self._index:
            raise LeanKVError("%s: %s must be [rows, heads, %d] %s on %s, got %s %s on %s"
                              % (what, name, HEAD_DIM, self.dtype, self.device, tuple(t.shape), t.dtype, t.device))

    def _queries(self, q: torch.Tensor, what: str) -> int:
        self._row_shape(q, what, "q")
        heads = q.shape[1]
        if not heads or heads % self.kv_heads:
            raise LeanKVError("%s: %d query heads over %d kv heads" % (what, heads, self.kv_heads))
        return heads

    def _bound(self, max_len, what: str) -> int:
        if max_len is None:
            return self.width * self.page_size
        if not 0 <= int(max_len) <= self.width * self.page_size:
            raise LeanKVError("%s: max_len=%d outside sequences of up to %d tokens" % (what, max_len, self.max_len))
        return int(max_len)

    # Workspaces of attention are allocated for their call, on the current stream: calls on several streams and captured graphs
    # share none.
    def _workspace(self, nbytes: int):
        return self._books.new_empty(nbytes // 4)

    def _output(self, q: torch.Tensor, out, what: str):
        """(out, its strides): a new one, tied to what autograd follows, or the caller's."""
        follows = follow(what, q) or (self._followed and torch.is_grad_enabled())
        if out is None:
            out = q.new_empty(q.shape)
            if follows:
                out = tied(out, what, q, torch.zeros((), device="cpu", requires_grad=True))
            return out, strides2(q.shape[1] * HEAD_DIM, HEAD_DIM)
        if follows:
            raise LeanKVError("%s: out= does not support autograd, which follows q or what is stored" % what)
        return out, out_rows(out, q, what)

    # ------------------------------------------------------------------------------------------------ storing
    def extend(self, cu: torch.Tensor | None = None) -> None:
        """Room for the rows of every sequence (without cu: one token for every sequence that holds some): lens grows, new
        pages are the lowest free ones in the order of the sequences.  A last page that is not full and that others name too
        is replaced by a copy of its tokens, unless all that name it are to grow and this sequence is the first of them,
        which goes on in it.  A sequence that would pass max_len, and one whose pages with those of all sequences before it
        are more than are free, takes nothing, and neither does the first on a page of which another, refused for want of
        pages, holds more tokens (what a sequence holds is never written over): taken says what each took.  Two launches."""
        p = self._cu(cu, "PagedKV.extend")
        call(self._index, self._lib.lkv_pages_extend, self._ref, p, self._scratch_ptr, self._extend_bytes)

    def store(self, layer: int, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor | None = None) -> None:
        """Keys and values [rows, kv_heads, 128] of what the last extend made room for, in one layer: rows cu[s] .. of
        sequence s, as many as it took (without cu: row s is sequence s's).  Other rows are not read."""
        what = "PagedKV.store"
        self._layer(layer, what)
        self._row_shape(k, what, "k")
        self._row_shape(v, what, "v")
        if k.shape != v.shape or k.shape[1] != self.kv_heads or (cu is None and k.shape[0] != self.max_seqs):
            raise LeanKVError("%s: k and v must be [%s, %d, %d], got %s and %s"
                              % (what, "rows" if cu is not None else self.max_seqs, self.kv_heads, HEAD_DIM, tuple(k.shape),
                                 tuple(v.shape)))
        p = self._cu(cu, what)
        if follow(what, k, v):
            self._followed = True
        (k, ks), (v, vs) = rows(k), rows(v)
        call(self._index, self._lib.lkv_pages_store, self._ref, layer, k.data_ptr(), ks, v.data_ptr(), vs, k.shape[0], p)

    def read(self, layer: int, n: int):
        """(K, V) [max_seqs, kv_heads, n, 128]: tokens 0 .. n - 1 of every sequence in one layer, zeros past its length."""
        what = "PagedKV.read"
        self._layer(layer, what)
        if not 0 <= n <= self.max_len:
            raise LeanKVError("%s: n=%d outside sequences of up to %d tokens" % (what, n, self.max_len))
        kv = self.pool.new_empty((2, self.max_seqs, self.kv_heads, n, HEAD_DIM))
        if self._followed and torch.is_grad_enabled():
            kv = tied(kv, what, torch.zeros((), device="cpu", requires_grad=True))
        k, v = kv.unbind(0)
        call(self._index, self._lib.lkv_pages_read, self._ref, layer, n, k.data_ptr(), v.data_ptr())
        return k, v

    # -------------------------------------------------------------------------------------------------- pages
    def fork(self, parent: torch.Tensor | None, lens: torch.Tensor | None = None) -> None:
        """Sequence s becomes the first lens[s] tokens (default: all) of what sequence parent[s] (None: s itself) held before
        the call; a parent outside 0 .. max_seqs - 1 empties it.  Pages are shared, and free when no sequence names them any
        more.  int32 tensors [max_seqs].  Two launches."""
        what = "PagedKV.fork"
        p = None if parent is None else self._ints(parent, self.max_seqs, what, "parent")
        c = None if lens is None else self._ints(lens, self.max_seqs, what, "lens")
        call(self._index, self._lib.lkv_pages_fork, self._ref, p, c, self._scratch_ptr, self._fork_bytes)

    def truncate(self, lens: torch.Tensor) -> None:
        """Every sequence keeps at most its first lens[s] tokens (int32 [max_seqs]; drafted tokens that were not accepted)."""
        self.fork(None, lens)

    def free(self, which) -> None:
        """Empties sequences: their numbers (a list or an integer), or a bool tensor [max_seqs] on the device."""
        if isinstance(which, torch.Tensor):
            if which.dtype is not torch.bool or which.shape != (self.max_seqs,) or which.device != self.device:
                raise LeanKVError("PagedKV.free: a bool tensor [%d] on %s expected, got %s %s on %s"
                                  % (self.max_seqs, self.device, which.dtype, tuple(which.shape), which.device))
            parent = torch.arange(self.max_seqs, dtype=torch.int32, device=self.device).masked_fill_(which, -1)
        else:
            which = [which] if isinstance(which, int) else list(which)
            if not all(isinstance(s, int) and not isinstance(s, bool) and 0 <= s < self.max_seqs for s in which):
                raise LeanKVError("PagedKV.free: sequence numbers 0 .. %d expected, got %s" % (self.max_seqs - 1, which))
            done = set(which)
            parent = torch.tensor([-1 if s in done else s for s in range(self.max_seqs)], dtype=torch.int32,
                                  device=self.device)
        self.fork(parent)

    def compact(self) -> torch.Tensor:
        """The pages in use become the first ones of the pool, in every layer: those behind fill the gaps, in order.  Returns
        their number, int32 [1] on the device.  Two launches."""
        in_use = self._books.new_empty(1)
        call(self._index, self._lib.lkv_pages_compact, self._ref, in_use.data_ptr(), self._scratch_ptr, self._compact_bytes)
        return in_use

    def _like(self, num_pages: int, max_seqs: int, max_len: int) -> "PagedKV":
        """A pool of other sizes whose first pages are this one's."""
        new = PagedKV(self.num_layers, self.kv_heads, num_pages, max_seqs, max_len, self.page_size, self.dtype, self.device)
        n = min(num_pages, self.num_pages)
        new.pool[:, :n] = self.pool[:, :n]
        new._followed = self._followed
        return new

    def resized(self, num_pages: int, max_len: int | None = None) -> "PagedKV":
        """A pool of num_pages pages (and sequences of up to max_len tokens, at least as many as now) that holds what this one
        does.  A smaller one is for the pages that compact has moved to the front; pages in use behind them raise (this looks
        at the device and waits for it)."""
        n = min(int(num_pages), self.num_pages)
        if num_pages < 1 or (n < self.num_pages and bool((self.refs[n:] > 0).any())):
            raise LeanKVError("PagedKV.resized: pages from %d on are in use (compact moves them)" % num_pages)
        new = self._like(int(num_pages), self.max_seqs, max(self.max_len, max_len or 0))
        new.table[:, :self.width] = self.table
        new.lens.copy_(self.lens)
        new.taken.copy_(self.taken)
        new.refs[:n] = self.refs[:n]
        return new

    def chosen(self, index: torch.Tensor) -> "PagedKV":
        """A pool of index.numel() sequences, the i-th of which holds what sequence index[i] of this one does (a batch made
        larger or smaller).  Pages are shared as fork shares them; there are as many pages a sequence as here, and at least
        as many in all."""
        if index.dim() != 1 or not 1 <= index.shape[0] <= MAX_SEQS or index.dtype not in (torch.int32, torch.int64) \
                or index.device != self.device:
            raise LeanKVError("PagedKV.chosen: 1 to %d sequence numbers on %s expected" % (MAX_SEQS, self.device))
        if bool(((index < 0) | (index >= self.max_seqs)).any()):  # (this waits for the device)
            raise LeanKVError("PagedKV.chosen: sequence numbers outside 0 .. %d" % (self.max_seqs - 1))
        n, each = index.shape[0], -(-self.num_pages // self.max_seqs)
        new = self._like(max(self.num_pages, n * each), n, self.max_len)
        new.table.copy_(self.table[index])
        new.lens.copy_(self.lens[index])
        named = new.table[new.table >= 0].long()
        new.refs.index_add_(0, named, torch.ones_like(named, dtype=torch.int32))
        return new

    def __deepcopy__(self, memo):
        """A pool of its own with the same contents."""
        new = memo[id(self)] = self.resized(self.num_pages)
        return new

    def snapshot(self) -> torch.Tensor:
        """The tables as they are (pages are not copied), for rollback."""
        return self._books.clone()

    def rollback(self, snapshot: torch.Tensor) -> None:
        """The tables as a snapshot of this pool has them.  What the pages hold is not taken back: tokens that were added since
        are gone, and those of the snapshot are there as long as, since then, none of its pages was released and taken again or
        moved by compact, no sequence was cut (truncate, fork with lens) and grew over what was cut off, and sequences that
        grew on one last page were as long as each other (extend lets the first of them go on in it)."""
        if not isinstance(snapshot, torch.Tensor) or snapshot.shape != self._books.shape \
                or snapshot.dtype is not torch.int32 or snapshot.device != self.device:
            raise LeanKVError("PagedKV.rollback: a snapshot of this pool expected")
        self._books.copy_(snapshot)

    # ---------------------------------------------------------------------------------------------- attention
    def decode_attention(self, layer: int, q: torch.Tensor, max_len: int | None = None, scale: float | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one query per sequence and head, q [max_seqs, heads, 128], over everything that it holds (its own token
        among it): [max_seqs, heads, 128].  An empty sequence gives zeros.  max_len: the caller's bound on lens (default: the
        longest that the table holds), which the work is split for; a longer sequence counts as its first max_len tokens.
        Neighbouring sequences (as far as 16 query heads of a kv head go) that name the same pages read them once.  scale:
        1 / sqrt(128) by default.  out: a buffer like q, rows dense, 16-byte aligned and apart (q itself may be it; where it
        lies over q in another way, q is copied first)."""
        what = "PagedKV.decode_attention"
        self._layer(layer, what)
        heads = self._queries(q, what)
        if q.shape[0] != self.max_seqs:
            raise LeanKVError("%s: q must have a row for each of %d sequences, got %s" % (what, self.max_seqs, tuple(q.shape)))
        bound = self._bound(max_len, what)
        given = out is not None
        out, os = self._output(q, out, what)
        if given and (q.data_ptr() != out.data_ptr() or q.stride() != out.stride()):
            q = apart(q, out)
        q, qs = rows(q)
        nbytes = _decode_bytes(self.max_seqs, heads, self.kv_heads, bound)
        ws = self._workspace(nbytes) if nbytes else None
        call(self._index, self._lib.lkv_pages_decode_attn, self._ref, layer, q.data_ptr(), qs, heads, bound,
             SCALE if scale is None else scale, out.data_ptr(), os, None if ws is None else ws.data_ptr(), nbytes)
        return out

    def prefill_attention(self, layer: int, q: torch.Tensor, cu: torch.Tensor, max_new: int | None = None,
                          max_len: int | None = None, scale: float | None = None,
                          out: torch.Tensor | None = None) -> torch.Tensor:
        """Causal attention of the newest tokens' queries (after their store), q [rows, heads, 128]: rows cu[s] .. cu[s + 1] - 1
        are those of sequence s (further ones than it holds tokens are zeros), and query i of m sees tokens 0 .. lens[s] - m +
        i.  Returns [rows, heads, 128]; rows of no sequence are zeros, or, in a buffer given as `out` (queries that it is written
        over are copied first), left as they are.
        max_new, max_len: the caller's bounds on the rows of a sequence and on lens, which the work is split for.  (A sequence
        that extend refused, taken[s] = 0, has its rows computed as those of the tokens that it holds.)"""
        what = "PagedKV.prefill_attention"
        self._layer(layer, what)
        heads = self._queries(q, what)
        p = self._ints(cu, self.max_seqs + 1, what, "cu")
        bound = self._bound(max_len, what)
        n = q.shape[0]
        if max_new is not None and max_new < 0:
            raise LeanKVError("%s: max_new=%d" % (what, max_new))
        new = n if max_new is None else min(int(max_new), n)
        fill = out is None
        out, os = self._output(q, out, what)
        q, qs = rows(q if fill else apart(q, out))
        nbytes = _prefill_bytes(n, self.max_seqs, heads, self.kv_heads, new, bound)
        ws = self._workspace(nbytes) if nbytes else None
        call(self._index, self._lib.lkv_pages_prefill_attn, self._ref, layer, q.data_ptr(), qs, n, heads, p, new, bound,
             SCALE if scale is None else scale, out.data_ptr(), os, int(fill), None if ws is None else ws.data_ptr(), nbytes)
        return out
