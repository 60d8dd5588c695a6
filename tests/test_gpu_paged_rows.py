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
