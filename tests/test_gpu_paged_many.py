"""Many sequences in a table that has room for long ones: splits of more pages than are held at a time."""

import pytest
import torch

from paged_ref import D, check, packed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decode_in_splits_of_many_pages(cuda, dtype):
    """2048 sequences of up to 131072 tokens in pages of 16, 7 splits of 1176 pages.  Four are longer than that or nearly, one of
    them forked from another; most are empty."""
    from leankv_amd.paged import PagedKV

    seqs, heads, kv, page = 2048, 32, 2, 16
    lens = {5: 40000, 6: 40000, 900: 18817, 2047: 16385, 17: 3}
    gen = torch.Generator().manual_seed(9)
    rows = {s: tuple(torch.randn(n, kv, D, generator=gen).to(dtype) for _ in range(2)) for s, n in lens.items() if s != 6}
    cache = PagedKV(1, kv, 4800, seqs, 131072, page_size=page, dtype=dtype)
    at = [0]
    for s in range(seqs):
        at.append(at[-1] + (rows[s][0].shape[0] if s in rows else 0))
    cu = torch.tensor(at, dtype=torch.int32, device="cuda")
    cache.extend(cu)
    cache.store(0, *(torch.cat([rows[s][i] for s in sorted(rows)]).cuda() for i in range(2)), cu)
    parent = torch.arange(seqs, dtype=torch.int32, device="cuda")
    parent[6] = 5
    cache.fork(parent)
    rows[6] = rows[5]
    assert cache.lens.cpu().nonzero().flatten().tolist() == sorted(lens)
    q = torch.randn(seqs, heads, D, generator=gen).to(dtype)
    got = cache.decode_attention(0, q.cuda())
    some = sorted(lens)
    want, bound = packed(q[some], None, None, list(range(len(some) + 1)), paged=lambda b: rows[some[b]])
    check(got[some], want, bound)
    assert not got[[s for s in range(0, seqs, 50) if s not in lens]].any()
    # a bound on the lengths: other splits
    check(cache.decode_attention(0, q.cuda(), max_len=40000)[some], want, bound)
    # and as drafted tokens' queries
    news = torch.tensor([0] + [1 if s in lens else 0 for s in range(seqs)], dtype=torch.int32, device="cuda").cumsum(0).int()
    check(cache.prefill_attention(0, q[some].cuda(), news, max_new=1), want, bound)
