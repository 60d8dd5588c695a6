"""As many rows of queries as there may be, and starts of rows that are not ascending."""

import pytest
import torch

pytestmark = pytest.mark.gpu
F16 = torch.float16


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_rows_past_2_to_27(cuda):
    """Rows that a sequence holds no tokens for are zeros, however many: 34 GB of them, all of one query (stride 0)."""
    from leankv_amd.paged import PagedKV

    n = 2 ** 27 + 1000
    cache = PagedKV(1, 1, 4, 1, 64, page_size=16, dtype=F16)
    cache.extend(_ints([0, 2]))
    kv = torch.randn(2, 2, 128, generator=torch.Generator().manual_seed(1)).half().cuda()
    cache.store(0, kv[:, :1], kv[:, 1:], _ints([0, 2]))
    q = torch.ones(1, 1, 128, dtype=F16, device="cuda")
    want = cache.prefill_attention(0, q.expand(2, 1, 128), _ints([0, 2]))
    out = torch.ones(n, 1, 128, dtype=F16, device="cuda")
    cache.prefill_attention(0, q.expand(n, 1, 128), _ints([0, n]), max_new=4, out=out)
    assert torch.equal(out[:2], want)
    assert not any(bool(part.any()) for part in out[2:].split(2 ** 24))
    del out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("starts", [[0, 40, 20, 60], [0, 60, 0, 60, 0, 60, 0, 60], [0, 60, 30, 31]])
def test_starts_that_fall(cuda, starts):
    """Sequences that would lie over each other are left out, and rows beside them are as they were."""
    from leankv_amd.paged import PagedKV, packed_attention

    B, n, heads, kv = len(starts) - 1, 60, 64, 2
    gen = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(n, h, 128, generator=gen).half().cuda() for h in (heads, kv, kv))
    out = torch.full((n + 8, heads, 128), 7.0, dtype=F16, device="cuda")
    packed_attention(q, k, v, _ints(starts), out=out[4:n + 4])
    assert (out == 7).all()
    cache = PagedKV(1, kv, 4 * B, B, 64, page_size=16, dtype=F16)
    at = _ints([20 * s for s in range(B + 1)])
    rows = torch.randn(20 * B, 2 * kv, 128, generator=gen).half().cuda()
    cache.extend(at)
    cache.store(0, rows[:, :kv], rows[:, kv:], at)
    cache.prefill_attention(0, q, _ints(starts), max_new=40, out=out[4:n + 4])
    assert (out == 7).all()
    # ascending ones that leave rows out at both ends
    good = _ints([3, 23, *[43] * (B - 2), 60][:B + 1])
    want = packed_attention(q, k, v, good)
    assert torch.equal(packed_attention(q, k, v, good, out=out[4:n + 4])[3:43], want[3:43]) and (out[:7] == 7).all()
