"""Results written over inputs: as if the inputs lay elsewhere."""

import pytest
import torch

pytestmark = pytest.mark.gpu
F16 = torch.float16


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _buffer(seed, n, heads):
    return torch.randn(n, heads, 128, generator=torch.Generator().manual_seed(seed)).half().cuda()


@pytest.mark.parametrize("n", [40, 700])
@pytest.mark.parametrize("over", ["k", "v", "later rows", "earlier rows", "other heads"])
def test_packed(cuda, n, over):
    from leankv_amd.paged import packed_attention

    heads, cu = 4, _ints([0, n // 3, n])
    x = _buffer(1, n + 50, 3 * heads)
    q, k, v = (x[20:20 + n, heads * i:heads * (i + 1)] for i in range(3))
    out = dict(k=k, v=v, **{"later rows": x[37:37 + n, :heads], "earlier rows": x[:n, :heads],
                            "other heads": x[20:20 + n, 2:2 + heads]})[over]
    want = packed_attention(q.clone(), k.clone(), v.clone(), cu)
    kept = x.clone()
    assert packed_attention(q, k, v, cu, out=out) is out
    assert torch.equal(out, want)
    out.zero_()
    (kept.as_strided(out.shape, out.stride(), out.storage_offset())).zero_()
    assert torch.equal(x, kept)


def test_pages(cuda):
    from leankv_amd.paged import PagedKV

    seqs = heads = 8
    kv = _buffer(2, seqs * 500, 4)
    cache = PagedKV(1, 2, 100, seqs, 4096, page_size=64, dtype=F16)
    at = _ints([500 * s for s in range(seqs + 1)])
    cache.extend(at)
    cache.store(0, kv[:, :2], kv[:, 2:], at)
    for max_len in (500, None):  # one part, and several
        x = _buffer(3, seqs + 3, heads)
        want = cache.decode_attention(0, x[:seqs].clone(), max_len=max_len)
        for view in (lambda x: x[:seqs].transpose(0, 1), lambda x: x[3:], lambda x: x[:seqs]):
            y = x.clone()
            assert torch.equal(cache.decode_attention(0, y[:seqs], max_len=max_len, out=view(y)), want)
        for new in (1, 20):
            q = _buffer(4, seqs * new + 5, heads)
            cu = _ints([new * s for s in range(seqs + 1)])
            want_new = cache.prefill_attention(0, q[:seqs * new].clone(), cu, max_new=new, max_len=max_len)
            for first in (0, 5):
                y = q.clone()
                got = cache.prefill_attention(0, y[:seqs * new], cu, max_new=new, max_len=max_len,
                                              out=y[first:first + seqs * new])
                assert torch.equal(got, want_new)
