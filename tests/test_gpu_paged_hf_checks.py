"""PagedCache: what it refuses leaves it as it was."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cache(cuda, layers=2, **kw):
    from leankv_amd.paged import PagedCache

    return PagedCache(num_layers=layers, device=cuda, max_seq_len=64, page_size=16, **kw)


def _kv(seed, B=2, H=2, S=5, dtype=torch.float16):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(B, H, S, 128, generator=gen).to(dtype).cuda() for _ in range(2)]


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_beams_out_of_range(cuda, where):
    cache = _cache(cuda)
    k, v = _kv(1)
    for layer in range(2):
        cache.update(k, v, layer)
    for bad in ([0, 2], [-1, 0], [0, 2 ** 32], [0.0, 1.0], [True, False]):
        with pytest.raises(ValueError, match="sequence numbers"):
            cache.reorder_cache(torch.tensor(bad, device=where))
        assert cache.kv.lens.tolist() == [5, 5] and torch.equal(cache[1][0], k)
    for good in (torch.int32, torch.int64):
        cache.reorder_cache(torch.tensor([1, 0], device=where, dtype=good))
    assert torch.equal(cache[1][0], k)
    cache.reorder_cache(torch.tensor([1, 1], device=where))
    assert torch.equal(cache[0][1], v[[1, 1]])
