"""Values of the whole range of their type: a row is infinite only where a token that it sees is."""

import pytest
import torch

from paged_ref import D, check, packed

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rows(gen, n, heads, size=1.0):
    return (torch.randn(n, heads, D, generator=gen).clamp(-3, 3) / 3 * size).to(BF16)


# the bound of paged_ref.attention scales with the values.  1e-28: the smallest of the largest weights is 2^-29, a product of
# that and a value 2^-122, and fp32 numbers below 2^-126 are off by at most 2^-150, of a sum by 3000 * 2^-150 / 2^-29 < 2^-109,
# less than a hundredth of the bound's 2^-9 * 2^-93
@pytest.mark.parametrize("size", [3.3e38, 1e36, 1e-28])
@pytest.mark.parametrize("lens", [[1], [5, 40], [150, 3], [700], [3000]], ids=str)
def test_packed(cuda, lens, size):
    from leankv_amd.paged import packed_attention

    gen = torch.Generator().manual_seed(sum(lens))
    at = [sum(lens[:i]) for i in range(len(lens) + 1)]
    q, k, v = _rows(gen, at[-1], 4, 4.0), _rows(gen, at[-1], 1, 4.0), _rows(gen, at[-1], 1, size)
    want, bound = packed(q, k, v, at)
    got = packed_attention(q.cuda(), k.cuda(), v.cuda(), _ints(at))
    assert got.isfinite().all()
    check(got, want, bound)


@pytest.mark.parametrize("size", [3.3e38, 1e36, 1e-28])
@pytest.mark.parametrize("shared", [False, True])
def test_pages(cuda, shared, size):
    """Decode, drafted tokens and chunks, of one part and of several, with shared pages too; rising scores, so that the offsets
    move; all values alike and as large as they get."""
    from leankv_amd.paged import PagedKV

    gen = torch.Generator().manual_seed(5)
    n, heads, seqs = 2600, 4, 3
    cache = PagedKV(1, 1, 200, seqs, 4096, page_size=64, dtype=BF16)
    k, v = _rows(gen, n, 1, 4.0), _rows(gen, n, 1, size)
    k = (k.float() * torch.linspace(0.2, 6, n).view(n, 1, 1)).to(BF16)
    v[n // 2:] = size
    at = [0, n, n, n] if shared else [0, n, n + 40, n + 140]
    rows = torch.cat([k, k[:140]])[:at[-1]], torch.cat([v, v[:140]])[:at[-1]]
    cache.extend(_ints(at))
    cache.store(0, rows[0].cuda(), rows[1].cuda(), _ints(at))
    held = [(rows[0][a:b], rows[1][a:b]) for a, b in zip(at, at[1:])]
    if shared:
        cache.fork(_ints([0, 0, 0]))
        held = [held[0]] * seqs
    for new in ([1, 1, 1], [7, 5, 8], [300, 40, 90]):
        starts = [sum(new[:i]) for i in range(seqs + 1)]
        q = _rows(gen, starts[-1], heads, 4.0)
        want, bound = packed(q, None, None, starts, paged=lambda b: held[b])
        got = cache.prefill_attention(0, q.cuda(), _ints(starts), max_new=max(new))
        assert got.isfinite().all()
        check(got, want, bound, str(new))
        if new == [1, 1, 1]:
            for kw in ({}, dict(max_len=n)):
                got = cache.decode_attention(0, q.cuda(), **kw)
                assert got.isfinite().all()
                check(got, want, bound, str(kw))
