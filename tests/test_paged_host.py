"""What the 16-bit paged cache's entry points refuse, and what their plans need; no GPU."""

import ctypes

import pytest
import torch

F16 = torch.float16


def _store(**other):
    from leankv_amd import _lib

    args = dict(pool=16, table=16, lens=16, refs=16, taken=16, layers=2, pages=8, kv_heads=2, page_size=64, seqs=4, width=4,
                dtype=_lib.LKV_DTYPE_F16)
    args.update(other)
    return ctypes.byref(_lib.PagesStruct(*args.values()))


def _strides(row=512, head=128):
    return (ctypes.c_int64 * 2)(row, head)


@pytest.mark.parametrize("other,text", [
    (dict(dtype=0), "dtype"), (dict(page_size=48), "page_size"), (dict(page_size=512), "page_size"),
    (dict(page_size=8), "page_size"), (dict(seqs=0), "seqs"), (dict(seqs=4097), "seqs"), (dict(width=0), "width"),
    (dict(width=1 << 26), "width"), (dict(pages=0), "pages"), (dict(layers=0), "layers"), (dict(kv_heads=0), "kv_heads"),
    (dict(pool=None), "null"), (dict(table=None), "null"), (dict(refs=None), "null"), (dict(pool=24), "16-byte"),
    (dict(lens=18), "4-byte"),
])
def test_stores_are_checked(other, text):
    from leankv_amd import _lib

    lib, p = _lib.load(), ctypes.c_void_p(16)
    st = _store(**other)
    s = _strides()
    for rc in (lambda: lib.lkv_pages_extend(st, None, p, 1 << 20, None),
               lambda: lib.lkv_pages_fork(st, None, None, p, 1 << 20, None),
               lambda: lib.lkv_pages_compact(st, p, p, 1 << 20, None),
               lambda: lib.lkv_pages_store(st, 0, p, s, p, s, 4, None, None),
               lambda: lib.lkv_pages_read(st, 0, 16, p, p, None),
               lambda: lib.lkv_pages_decode_attn(st, 0, p, s, 4, 64, 0.1, p, s, p, 1 << 20, None),
               lambda: lib.lkv_pages_prefill_attn(st, 0, p, s, 4, 4, p, 4, 64, 0.1, p, s, 1, p, 1 << 20, None)):
        assert rc() == -1 and text in _lib.last_error(), _lib.last_error()


def test_calls_are_checked():
    from leankv_amd import _lib

    lib, p, st, s = _lib.load(), ctypes.c_void_p(16), _store(), _strides()

    def refused(rc, text):
        assert rc == -1 and text in _lib.last_error(), _lib.last_error()

    need = lib.lkv_pages_extend_workspace_bytes(8, 4)
    assert need == 4 * (8 + 1 + 12)
    refused(lib.lkv_pages_extend(st, None, p, need - 1, None), "workspace")
    refused(lib.lkv_pages_extend(st, None, None, need, None), "workspace")
    refused(lib.lkv_pages_extend(st, 18, p, need, None), "cu")
    refused(lib.lkv_pages_fork(st, None, None, p, lib.lkv_pages_fork_workspace_bytes(4, 4) - 1, None), "workspace")
    refused(lib.lkv_pages_fork(st, 18, None, p, 1 << 20, None), "parent")
    refused(lib.lkv_pages_compact(st, None, p, 1 << 20, None), "in_use")
    refused(lib.lkv_pages_compact(st, p, p, lib.lkv_pages_compact_workspace_bytes(8) - 1, None), "workspace")
    refused(lib.lkv_pages_store(st, 2, p, s, p, s, 4, None, None), "layer")
    refused(lib.lkv_pages_store(st, -1, p, s, p, s, 4, None, None), "layer")
    refused(lib.lkv_pages_store(st, 0, p, s, p, s, 3, None, None), "one row for each")
    refused(lib.lkv_pages_store(st, 0, p, _strides(row=513), p, s, 4, None, None), "rows of k")
    refused(lib.lkv_pages_store(st, 0, p, s, 24, s, 4, None, None), "rows of v")
    refused(lib.lkv_pages_store(st, 0, p, s, None, s, 4, None, None), "null")
    refused(lib.lkv_pages_store(st, 0, p, s, p, s, -1, p, None), "rows")
    assert lib.lkv_pages_store(st, 0, None, None, None, None, 0, p, None) == 0
    refused(lib.lkv_pages_read(st, 0, 257, p, p, None), "n=257")
    refused(lib.lkv_pages_read(st, 0, 16, p, None, None), "16-byte")
    refused(lib.lkv_pages_decode_attn(st, 0, p, s, 3, 64, 0.1, p, s, p, 1 << 20, None), "query heads")
    refused(lib.lkv_pages_decode_attn(st, 0, p, s, 4, 257, 0.1, p, s, p, 1 << 20, None), "max_len")
    refused(lib.lkv_pages_decode_attn(st, 5, p, s, 4, 64, 0.1, p, s, p, 1 << 20, None), "layer")
    refused(lib.lkv_pages_decode_attn(st, 0, p, _strides(row=-512), 4, 64, 0.1, p, s, p, 1 << 20, None), "rows of q")
    wide = _store(width=400, page_size=256)
    need = lib.lkv_pages_decode_attn_workspace_bytes(4, 4, 2, 102400)
    assert need > 0
    refused(lib.lkv_pages_decode_attn(wide, 0, p, s, 4, 102400, 0.1, p, s, p, need - 1, None), "workspace")
    refused(lib.lkv_pages_decode_attn(wide, 0, p, s, 4, 102400, 0.1, p, s, None, need, None), "workspace")
    refused(lib.lkv_pages_prefill_attn(st, 0, p, s, 4, 4, None, 4, 64, 0.1, p, s, 1, p, 1 << 20, None), "cu")
    refused(lib.lkv_pages_prefill_attn(st, 0, p, s, -1, 4, p, 4, 64, 0.1, p, s, 1, p, 1 << 20, None), "rows")
    refused(lib.lkv_pages_prefill_attn(st, 0, p, s, 4, 4, p, 4, 300, 0.1, p, s, 1, p, 1 << 20, None), "max_len")
    refused(lib.lkv_pages_prefill_attn(st, 0, p, s, 1 << 28, 4, p, 4, 64, 0.1, p, s, 1, p, 1 << 20, None), "rows")
    assert lib.lkv_pages_prefill_attn(st, 0, None, None, 0, 4, p, 4, 64, 0.1, None, None, 1, None, 0, None) == 0

    def packed(q=p, qs=s, k=p, ks=s, dtype=1, rows=4, Hq=4, Hkv=2, cu=p, B=1, max_len=4, ws=p, ws_bytes=1 << 20):
        return lib.lkv_packed_attn(q, qs, k, ks, p, s, dtype, rows, Hq, Hkv, cu, B, max_len, 0.1, p, s, 1, ws, ws_bytes, None)

    refused(packed(dtype=0), "dtype")
    refused(packed(Hq=5), "query heads")
    refused(packed(cu=None), "cu")
    refused(packed(B=0), "B=0")
    refused(packed(B=4097), "B=4097")
    refused(packed(max_len=-1), "max_len")
    refused(packed(k=24), "rows of k")
    refused(packed(qs=_strides(head=12)), "rows of q")
    refused(packed(ks=_strides(row=1 << 26)), "2^26")
    refused(packed(rows=1 << 29), "rows")
    need = lib.lkv_packed_attn_workspace_bytes(4096, 1, 2, 2, 4096)
    assert need > 0
    refused(packed(rows=4096, Hq=2, max_len=4096, ws_bytes=need - 1), "workspace")
    assert packed(rows=0) == 0


def test_constructor_refuses():
    from leankv_amd._lib import LeanKVError
    from leankv_amd.paged import PagedKV

    for args, kw in (((0, 1, 1, 1, 1), {}), ((1, 0, 1, 1, 1), {}), ((1, 1, 0, 1, 1), {}), ((1, 1, 1, 0, 1), {}),
                     ((1, 1, 1, 4097, 1), {}), ((1, 1, 1, 1, 0), {}), ((1, 1, 1, 1, 1), dict(page_size=24)),
                     ((1, 1, 1, 1, 1), dict(dtype=torch.float32))):
        with pytest.raises(ValueError, match="PagedKV"):
            PagedKV(*args, **kw)
    with pytest.raises(LeanKVError, match="GPU only"):
        PagedKV(1, 1, 1, 1, 1, device="cpu")


def test_packed_attention_refuses_host_tensors():
    from leankv_amd._lib import LeanKVError
    from leankv_amd.paged import packed_attention

    q = torch.zeros(4, 2, 128, dtype=F16)
    with pytest.raises(LeanKVError, match="on the GPU"):
        packed_attention(q, q, q, torch.zeros(2, dtype=torch.int32))


def test_out_rows():
    from leankv_amd._lib import LeanKVError
    from leankv_amd.paged.packed import in_place, out_rows

    q = torch.zeros(6, 4, 128, dtype=F16)
    assert list(out_rows(torch.zeros(6, 4, 128, dtype=F16), q, "x")) == [512, 128]
    assert list(out_rows(torch.zeros(4, 6, 128, dtype=F16).transpose(0, 1), q, "x")) == [128, 768]
    base = torch.zeros(4096, dtype=F16)
    for bad in (base.as_strided((6, 4, 128), (0, 128, 1)), base.as_strided((6, 4, 128), (128, 128, 1)),
                base.as_strided((6, 4, 128), (512, 64, 1))):
        with pytest.raises(LeanKVError, match="overlap"):
            out_rows(bad, q, "x")
    for bad in (torch.zeros(6, 4, 130, dtype=F16)[..., :128], torch.zeros(6, 4, 128), torch.zeros(6, 4, 64, dtype=F16),
                torch.zeros(6, 128, 4, dtype=F16).transpose(1, 2), torch.zeros(24, 128, dtype=F16)):
        with pytest.raises(LeanKVError, match="out must be"):
            out_rows(bad, q, "x")
    assert in_place(torch.zeros(5, 4, 136, dtype=F16)[..., :128]) is not None
    assert in_place(torch.zeros(5, 4, 132, dtype=F16)[..., :128]) is None


def test_the_model_of_the_tables():
    """The lists that the GPU tests compare with: pages are shared, copied and moved as the entry points say."""
    from paged_ref import Tables

    t = Tables(6, 3, 4, 16)
    t.extend([20, 0, 0])
    t.fork([0, 0, 0])
    t.extend([1, 1, 0])
    assert t.rows == [[0, 2], [0, 3], [0, 1]] and t.copies == [(1, 2, 4), (1, 3, 4)] and t.refs() == [3, 1, 1, 1, 0, 0]
    t.fork([-1, 1, -1])
    assert t.compact() == 2 and t.rows == [[], [0, 1], []] and t.moves == {3: 1}
    t.extend([0, 100, 0])
    assert t.taken == [0, 0, 0] and t.lens == [0, 21, 0]


def test_hf_cache_refuses():
    from leankv_amd.paged import PagedCache

    for kw in (dict(head_dim=64), dict(num_layers=0), dict(page_size=24)):
        with pytest.raises(ValueError, match="PagedCache"):
            PagedCache(**kw)
    cache = PagedCache(num_layers=2, device="cuda")
    assert cache.get_seq_length() == 0 and not len(cache) and cache.max_batch_size == 0 and not cache.is_initialized
    assert cache.get_total_cache_bytes() == 0 and cache.get_compression_ratio() == 0.0
    cache.crop(5)
    cache.reorder_cache(torch.tensor([0]))
    cache.batch_repeat_interleave(2)
    with pytest.raises(IndexError):
        cache[0]


def test_optimize_model_takes_one_cache():
    from leankv_amd.combined import optimize_model

    for kw in (dict(kv8=True), dict(turboquant_bits=3), dict(use_paged_cache=True)):
        with pytest.raises(ValueError, match="paged_kv"):
            optimize_model(None, paged_kv=True, **kw)
