"""Causal attention of packed sequences (lkv_packed_attn in include/leankv_amd.h), and what the paged cache's calls share."""

from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._lib import LeanKVError, check

HEAD_DIM = 128
DTYPES = {torch.float16: _lib.LKV_DTYPE_F16, torch.bfloat16: _lib.LKV_DTYPE_BF16}
SCALE = 1.0 / math.sqrt(HEAD_DIM)
MAX_SEQS = 2048
_I64x2 = ctypes.c_int64 * 2


@functools.lru_cache(maxsize=256)
def strides2(row: int, head: int):
    return _I64x2(row, head)


def in_place(t: torch.Tensor):
    """The strides of row and head of t [rows, heads, 128] as the kernels take them, None where its rows are not dense or not
    16-byte aligned.  Strides of single sizes count as 0 (torch leaves them free)."""
    if t.is_contiguous() and not t.data_ptr() % 16:
        return strides2(t.shape[1] * HEAD_DIM, HEAD_DIM)
    n, (r, h, d) = t.shape, t.stride()
    if n[0] <= 1:
        r = 0
    if n[1] <= 1:
        h = 0
    if d != 1 or (r | h) % 8 or t.data_ptr() % 16 or r >= 1 << 26 or h >= 1 << 31:
        return None
    return strides2(r, h)


def rows(t: torch.Tensor, apart: bool = False):
    """(t or a copy of it, strides) for t [rows, heads, 128] that is read; with rows apart, if they have to be."""
    st = in_place(t)
    if st is None or (apart and st[0] < HEAD_DIM and t.shape[0] > 1):
        t = t.detach().clone(memory_format=torch.contiguous_format)
        st = in_place(t)
    return t, st


def out_rows(out: torch.Tensor, like: torch.Tensor, what: str):
    """The strides of a buffer that the caller gives for the result: rows apart from each other."""
    st = in_place(out) if out.dim() == 3 else None
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device or st is None:
        raise LeanKVError("%s: out must be like q, %s %s on %s, with dense 16-byte aligned rows"
                          % (what, like.dtype, tuple(like.shape), like.device))
    end = HEAD_DIM  # numbers from the first to the last of the sizes so far
    for step, n in sorted((step, n) for step, n in zip(out.stride()[:2], out.shape[:2]) if n > 1):
        if step < end:
            raise LeanKVError("%s: rows of out overlap, strides %s" % (what, out.stride()))
        end += step * (n - 1)
    return st


def _size(t: torch.Tensor, first: int) -> int:
    """Bytes from the first to the last number of t's dims from `first` on."""
    return 2 * (1 + sum(st * (n - 1) for st, n in zip(t.stride()[first:], t.shape[first:])))


def meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether a and b [rows, heads, 128] may have numbers in common: not if they lie behind each other, or are parts of the
    rows of one buffer that do (q, k and v of a projection)."""
    if not a.numel() or not b.numel():
        return False
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + _size(a, 0) <= pb or pb + _size(b, 0) <= pa:
        return False
    row = 2 * a.stride(0)
    if row and a.stride(0) == b.stride(0):
        off = (pb - pa) % row
        return off < _size(a, 1) or off + _size(b, 1) > row
    return True


def apart(t: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """t, or a copy where out is written over it: the call reads t until it ends (queries too, whose rows are read again where a
    value is no number)."""
    return t.clone(memory_format=torch.contiguous_format) if meet(t, out) else t


def follow(what: str, *tensors: torch.Tensor) -> bool:
    """Whether autograd follows one of them.  A forward-mode tangent would be lost at once and is refused."""
    if getattr(forward_ad, "_current_level", -1) >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise LeanKVError("%s: there is no forward-mode derivative" % what)
    for t in tensors:
        if t.requires_grad:
            return torch.is_grad_enabled()
    return False


class _NoBackward(torch.autograd.Function):
    """Ties an output to what autograd follows, so that a backward pass through it raises instead of leaving it out."""

    @staticmethod
    def forward(ctx, out, what, *anchors):
        ctx.what = what
        ctx.mark_dirty(out)
        return out

    @staticmethod
    def backward(ctx, grad):
        raise LeanKVError("%s: there is no backward pass" % ctx.what)


def tied(out: torch.Tensor, what: str, *anchors: torch.Tensor) -> torch.Tensor:
    return _NoBackward.apply(out, what, *anchors)


def call(index: int, fn, *args) -> None:
    """One C entry (of the loaded library) on a device and that device's current stream."""
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, fn.__name__)


@functools.lru_cache(maxsize=256)
def _bytes(rows_: int, batch: int, heads: int, kv_heads: int, max_len: int) -> int:
    return _lib.load().lkv_packed_attn_workspace_bytes(rows_, batch, heads, kv_heads, max_len)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     max_len: int | None = None, scale: float | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of sequences that lie one behind the other: q [tokens, heads, 128], k and v [tokens, kv_heads, 128]
    (heads a multiple of kv_heads; query head h reads kv head h * kv_heads // heads), float16 or bfloat16.  cu_seqlens: int32
    [n + 1] on the device, ascending; rows cu_seqlens[i] .. cu_seqlens[i + 1] - 1 are sequence i, up to 2048 of them.  Returns
    [tokens, heads, 128] in q's type; rows of no sequence are zeros, or, in a buffer given as `out` (dense 16-byte aligned
    rows apart from each other), left as they are.  Inputs that out is written over are copied first.  max_len: the caller's
    bound on the lengths (default: all tokens), which the work is split for.  scale: 1 / sqrt(128) by default.

    Inputs may have any strides (rows that are not dense or not 16-byte aligned are copied).  A token that a query does not
    see has no part in its row, whatever it holds; a NaN in a query gives a row of NaN.  There is no gradient: a backward pass
    through the result raises."""
    what = "packed_attention"
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.dim() != 3 or t.shape[2] != HEAD_DIM or not t.is_cuda:
            raise LeanKVError("%s: %s must be [tokens, heads, %d] on the GPU, got %s on %s"
                              % (what, name, HEAD_DIM, tuple(t.shape), t.device))
        if t.dtype != q.dtype or t.dtype not in DTYPES or t.device != q.device:
            raise LeanKVError("%s: q, k and v must be of one type, float16 or bfloat16, on one device, got %s %s on %s"
                              % (what, name, t.dtype, t.device))
    n, heads, kv_heads = q.shape[0], q.shape[1], k.shape[1]
    if k.shape != v.shape or k.shape[0] != n or not kv_heads or not heads or heads % kv_heads:
        raise LeanKVError("%s: q %s, k %s and v %s do not belong together"
                          % (what, tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    index = q.get_device()
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dtype is not torch.int32 or cu_seqlens.dim() != 1 \
            or not 2 <= cu_seqlens.shape[0] <= MAX_SEQS + 1 or not cu_seqlens.is_cuda \
            or cu_seqlens.get_device() != index or not cu_seqlens.is_contiguous():
        raise LeanKVError("%s: cu_seqlens must be a contiguous int32 tensor of 2 to %d entries on %s"
                          % (what, MAX_SEQS + 1, q.device))
    if max_len is not None and max_len < 0:
        raise LeanKVError("%s: max_len=%d" % (what, max_len))
    bound = n if max_len is None else min(int(max_len), n)
    follows = follow(what, q, k, v)
    fill = out is None
    if fill:
        out = q.new_empty((n, heads, HEAD_DIM))
        if follows:
            out = tied(out, what, q, k, v)
        os = strides2(heads * HEAD_DIM, HEAD_DIM)
    else:
        if follows:
            raise LeanKVError("%s: out= does not support autograd, which follows q, k or v" % what)
        os = out_rows(out, q, what)
        q, k, v = apart(q, out), apart(k, out), apart(v, out)
    (q, qs), (k, ks), (v, vs) = rows(q), rows(k, apart=True), rows(v, apart=True)
    batch = cu_seqlens.shape[0] - 1
    nbytes = _bytes(n, batch, heads, kv_heads, bound)
    ws = q.new_empty(nbytes // 2) if nbytes else None
    call(index, _lib.load().lkv_packed_attn, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, DTYPES[q.dtype], n, heads,
         kv_heads, cu_seqlens.data_ptr(), batch, bound, SCALE if scale is None else scale, out.data_ptr(), os, int(fill),
         None if ws is None else ws.data_ptr(), nbytes)
    return out
