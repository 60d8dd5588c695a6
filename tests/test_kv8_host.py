"""The 8-bit block-scaled KV cache without a GPU: the C entry points' argument checks (a refused call launches nothing),
the store struct against the header, and the refusals of the Python classes."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096  # a 16-byte aligned address that no refused call reads


def _lib():
    from leankv_amd import _lib

    return _lib


def _store(**kw):
    m = _lib()
    f = dict(k_codes=P, v_codes=P, scales=P, ranges=P, k_tail=P, v_tail=P, batch=2, kv_heads=4, blocks=8)
    f.update(kw)
    return m.KV8StoreStruct(*[f[n] for n, _ in m.KV8StoreStruct._fields_])


def _strides(*s):
    return (ctypes.c_int64 * 3)(*s)


OK3 = (4096, 128, 512)


def test_struct_matches_the_header():
    src = open(os.path.join(ROOT, "include", "leankv_amd.h")).read()
    body = re.search(r"typedef struct lkv_kv8_store \{(.*?)\} lkv_kv8_store;", src, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    names = [n.strip().lstrip("*") for line in body.split(";") if line.strip()
             for n in line.strip().split(None, 1)[1].split(",")]
    assert names == [n for n, _ in _lib().KV8StoreStruct._fields_]
    assert ctypes.sizeof(_lib().KV8StoreStruct) == 9 * 8


def _refused(rc, text):
    assert rc == -1 and text in _lib().last_error(), (rc, _lib().last_error())


def test_update_and_read_arguments():
    lib = _lib().load()

    def update(st=None, k=P, ks=OK3, v=P, vs=OK3, dtype=1, S=4, pos=P, store=True):
        st = _store() if st is None else st
        return lib.lkv_kv8_update(ctypes.byref(st) if store else None, k, _strides(*ks), v, _strides(*vs), dtype, S, pos,
                                  None, None)

    _refused(update(store=False), "null store")
    _refused(update(_store(blocks=0)), "out of range")
    _refused(update(_store(kv_heads=0)), "out of range")
    _refused(update(_store(batch=-1)), "out of range")
    _refused(update(_store(batch=70000)), "out of range")
    _refused(update(_store(v_tail=None)), "null pointer")
    _refused(update(_store(ranges=P + 8)), "16-byte aligned")
    _refused(update(dtype=3), "dtype")
    _refused(update(S=-1), "out of range")
    _refused(update(k=None), "null pointer")
    _refused(update(pos=None), "null pointer")
    _refused(update(k=P + 2), "16-byte aligned")
    _refused(update(vs=(4096, 128, 516)), "16-byte aligned")
    assert update(S=0) == 0 and update(_store(batch=0)) == 0  # nothing to do

    def read(first=0, n=4, lens=P, k=P):
        st = _store()
        return lib.lkv_kv8_read(ctypes.byref(st), lens, first, n, k, P, None)

    _refused(read(first=-1), "outside")
    _refused(read(n=513), "outside")
    _refused(read(first=500, n=13), "outside")
    _refused(read(first=2 ** 62, n=2 ** 62), "outside")
    _refused(read(lens=None), "null pointer")
    _refused(read(k=P + 4), "aligned")
    assert read(n=0) == 0


def test_attention_arguments():
    lib = _lib().load()

    def attn(st=None, q=P, qs=OK3, dtype=1, Hq=8, S=1, lens=P, max_len=512, index=None, n=0, out=P, os_=OK3, ws=P,
             nbytes=1 << 30):
        st = _store() if st is None else st
        return lib.lkv_kv8_attn(ctypes.byref(st), q, _strides(*qs), dtype, Hq, S, lens, None, max_len, index, n, 0.1, out,
                                _strides(*os_), ws, nbytes, None)

    _refused(attn(Hq=6), "query heads")
    _refused(attn(Hq=0), "query heads")
    _refused(attn(S=-1), "out of range")
    _refused(attn(max_len=513), "max_len")
    _refused(attn(max_len=-1), "max_len")
    _refused(attn(dtype=-1), "dtype")
    _refused(attn(index=P, n=0), "list")
    _refused(attn(index=None, n=3), "list")
    _refused(attn(index=P, n=3, S=2), "one query")
    _refused(attn(lens=None), "null pointer")
    _refused(attn(q=P + 8), "16-byte aligned")
    _refused(attn(os_=(4096, 130, 512)), "16-byte aligned")
    need = lib.lkv_kv8_attn_workspace_bytes(2, 8, 4, 1, 8192, 0)
    assert need > 0  # several splits for so few heads
    big = _store(blocks=128)
    _refused(attn(big, max_len=8192, nbytes=need - 1), "workspace")
    _refused(attn(big, max_len=8192, ws=None, nbytes=need), "workspace")
    assert lib.lkv_kv8_attn_workspace_bytes(2, 8, 4, 1, 512, 0) == 0  # so little work is one split
    many = lib.lkv_kv8_attn_workspace_bytes(1, 8, 4, 512, 8192, 0)
    assert many > 0 and many % (8 * 512 * 130 * 4) == 0
    assert attn(S=0) == 0 and attn(_store(batch=0)) == 0
    assert lib.lkv_kv8_attn_workspace_bytes(2, 6, 4, 1, 512, 0) == 0
    # many sequences need no split, and no workspace
    assert lib.lkv_kv8_attn_workspace_bytes(512, 32, 8, 1, 8192, 0) == 0
    # the partial sums of every split of every row
    assert need % (2 * 8 * 130 * 4) == 0


def test_selection_arguments():
    lib = _lib().load()

    def select(n=3, sink=1, recent=1, max_len=512, q=P, index=P, nbytes=0, ws=None, st=None):
        st = _store() if st is None else st
        return lib.lkv_kv8_select_blocks(ctypes.byref(st), q, _strides(*OK3), 1, 8, P, max_len, n, sink, recent, index, ws,
                                         nbytes, None)

    _refused(select(n=0), "blocks")
    _refused(select(n=2, sink=2, recent=1), "blocks")
    _refused(select(sink=-1), "blocks")
    _refused(select(n=3, sink=1, recent=2 ** 62), "blocks")
    _refused(select(max_len=1000), "max_len")
    _refused(select(index=None), "null pointer")
    big = _store(blocks=4096)
    need = lib.lkv_kv8_select_workspace_bytes(2, 4, 4096 * 64)
    assert need == 2 * 4 * 4096 * 4 and lib.lkv_kv8_select_workspace_bytes(2, 4, 512) == 0
    _refused(select(st=big, max_len=4096 * 64, nbytes=need - 4, ws=P), "workspace")

    def sparse(out=P, n=3, nbytes=1 << 30):
        st = _store()
        return lib.lkv_kv8_sparse_attn(ctypes.byref(st), P, _strides(*OK3), 1, 8, P, 512, n, 1, 1, 0.1, P, out,
                                       _strides(*OK3), P, nbytes, None)

    _refused(sparse(out=None), "null pointer")
    _refused(sparse(n=1), "blocks")
    need = lib.lkv_kv8_sparse_attn_workspace_bytes(2, 8, 4, 512, 64)
    assert need > 0
    _refused(sparse(n=64, nbytes=need - 1), "workspace")


def test_store_refuses():
    from leankv_amd._lib import LeanKVError
    from leankv_amd.kv8 import KV8Store

    with pytest.raises(LeanKVError, match="GPU only"):
        KV8Store(1, 1, 64, device="cpu")
    for bad in ((0, 1, 64), (1, 0, 64), (1, 1, 0)):
        with pytest.raises(ValueError):
            KV8Store(*bad)


def test_cache_refuses():
    from leankv_amd.kv8 import BlockInt8Cache

    for kw in (dict(head_dim=64), dict(num_layers=0), dict(sparse_blocks=1), dict(sparse_blocks=0, sink_blocks=0,
                                                                                 recent_blocks=0), dict(sink_blocks=-1)):
        with pytest.raises(ValueError):
            BlockInt8Cache(**kw)
    c = BlockInt8Cache(num_layers=2, device="cpu")
    assert len(c) == 0 and c.get_seq_length(0) == 0 and c.max_batch_size == 0 and c.get_compression_ratio() == 0.0
    with pytest.raises(RuntimeError, match="pending"):
        c.decode_attention(0, torch.zeros(1, 1, 1, 128))
    with pytest.raises(RuntimeError, match="pending"):
        c.prefill_attention(0, torch.zeros(1, 1, 2, 128))
    for f in (lambda: c.crop(3), lambda: c.reorder_cache(None), lambda: c.batch_select_indices(None),
              lambda: c.batch_repeat_interleave(2)):
        with pytest.raises(NotImplementedError):
            f()


def test_optimize_model_takes_one_cache():
    from leankv_amd.combined import optimize_model

    for kw in (dict(kv8=True, turboquant_bits=3), dict(kv8=True, use_paged_cache=True), dict(kv8_sparse_blocks=8)):
        with pytest.raises(ValueError, match="kv8"):
            optimize_model(object(), **kw)
