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


def test_refused_updates_leave_the_cache_as_it_was(cuda):
    cache = _cache(cuda)
    k, v = _kv(2)
    for bad in (v.bfloat16(), v[:1], v[:, :1], v[:, :, :4], v[..., :64], v.cpu(), v[0]):
        with pytest.raises(ValueError, match="of one type on one device"):
            cache.update(k, bad, 0)
    with pytest.raises(ValueError, match="of one type on one device"):
        cache.update(k[..., :64], v[..., :64], 0)
    assert cache.kv is None and cache.get_seq_length() == 0 and cache.seen_tokens == 0
    for layer in range(2):
        cache.update(k, v, layer)
    for S in (1, 3):
        k1, v1 = _kv(3 + S, S=S)
        with pytest.raises(ValueError, match="of one type on one device"):
            cache.update(k1, v1.bfloat16(), 0)
        with pytest.raises(ValueError, match="holds 2 sequences"):
            cache.update(k1.bfloat16(), v1.bfloat16(), 0)
        n = cache.get_seq_length(0)
        cache.update(k1, v1, 0)
        for bad in ((k1[:1], v1[:1]), (k1[:, :1], v1[:, :1]), (k1.bfloat16(), v1.bfloat16())):
            with pytest.raises(ValueError, match="holds 2 sequences"):
                cache.update(*bad, 1)
        cache.update(k1, v1, 1)
        assert cache.kv.lens.tolist() == [n + S] * 2 and cache.seen_tokens == n + S
        assert torch.equal(cache[0][0][:, :, n:], k1) and torch.equal(cache[1][1][:, :, n:], v1)
        assert torch.equal(cache[1][0][:, :, :5], k)


def test_a_tangent_takes_no_room(cuda):
    from leankv_amd._lib import LeanKVError
    from torch.autograd import forward_ad

    cache = _cache(cuda, layers=1)
    k, v = _kv(7)
    cache.update(k, v, 0)
    with forward_ad.dual_level():
        with pytest.raises(LeanKVError, match="forward-mode"):
            cache.update(forward_ad.make_dual(k, torch.ones_like(k)), v, 0)
    assert cache.kv.lens.tolist() == [5, 5] and cache.get_seq_length() == 5 and cache.seen_tokens == 5
    cache.update(k, v, 0)
    assert torch.equal(cache[0][0], torch.cat([k, k], 2))


def test_decode_is_divided_by_what_is_held(cuda, monkeypatch):
    """A cache with room for long sequences: the bound that decode is given holds the tokens and little more."""
    from leankv_amd.paged import PagedCache, PagedKV

    cache = PagedCache(num_layers=1, device=cuda, max_seq_len=30000, fused_attention=True)
    k, v = _kv(8, S=254)
    q = torch.randn(2, 4, 254, 128, generator=torch.Generator().manual_seed(9)).half().cuda()
    cache.update(k, v, 0)
    cache.prefill_attention(0, q)
    bounds, plain = [], PagedKV.decode_attention

    def decode(self, layer, q, max_len=None, **kw):
        bounds.append(max_len)
        return plain(self, layer, q, max_len=max_len, **kw)

    monkeypatch.setattr(PagedKV, "decode_attention", decode)
    for _ in range(4):
        cache.update(k[:, :, :1], v[:, :, :1], 0)
        got = cache.decode_attention(0, q[:, :, :1])
        want = plain(cache.kv, 0, q[:, :, 0].contiguous(), max_len=cache.get_seq_length()).unsqueeze(2)
        assert torch.equal(got, want)
    assert bounds == [256, 256, 384, 384]
    short = PagedCache(num_layers=1, device=cuda, max_seq_len=20, page_size=16, fused_attention=True)
    short.update(k[:, :, :20], v[:, :, :20], 0)
    short.prefill_attention(0, q[:, :, :20])
    short.update(k[:, :, :1], v[:, :, :1], 0)
    short.decode_attention(0, q[:, :, :1])
    assert bounds[-1] == 32
