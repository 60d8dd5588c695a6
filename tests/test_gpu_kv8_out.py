"""Output buffers of KV8Store's attention: over the queries, any strides that single sizes may have, and no
rows over each other."""
import pytest
import torch
from kv8_ref import D

pytestmark = pytest.mark.gpu


def _store(dev, B, H, n, seed):
    from leankv_amd.kv8 import KV8Store

    g = torch.Generator().manual_seed(seed)
    store = KV8Store(B, H, n, device=dev)
    store.update(*(torch.randn(B, H, n, D, generator=g).half().to(dev) for _ in range(2)),
                 torch.zeros(B, dtype=torch.int32, device=dev))
    return store, torch.full((B,), n, dtype=torch.int32, device=dev)


def test_rows_over_each_other_are_refused(cuda):
    from leankv_amd._lib import LeanKVError

    store, lens = _store(cuda, 2, 1, 100, seed=1)
    q = torch.randn(2, 4, D, generator=torch.Generator().manual_seed(2)).half().to(cuda)
    one = torch.zeros(1, 4, D, dtype=q.dtype, device=cuda)
    for call in (lambda: store.decode_attention(q, lens, out=one.expand(2, 4, D)),
                 lambda: store.prefill_attention(q.unsqueeze(2), lens, out=one.unsqueeze(2).expand(2, 4, 1, D))):
        with pytest.raises(LeanKVError, match="overlap"):
            call()
    assert (one == 0).all()


@pytest.mark.parametrize("S", [1, 3, 8, 70, 300])
@pytest.mark.parametrize("n", [310, 64 * 150 + 3])
def test_over_its_own_queries(cuda, S, n):
    store, lens = _store(cuda, 2, 2, n, seed=3)
    q = torch.randn(2, 10, S, D, generator=torch.Generator().manual_seed(4)).half().to(cuda)
    want = store.prefill_attention(q, lens)
    assert store.prefill_attention(q, lens, out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("B,H,Hq", [(1, 1, 1), (1, 2, 4), (3, 1, 1)])
def test_strides_of_single_sizes_are_free(cuda, B, H, Hq):
    store, lens = _store(cuda, B, H, 100, seed=1)
    q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(2)).half().to(cuda)
    want = store.decode_attention(q, lens)
    strides = (1 if B == 1 else Hq * D, 3 if Hq == 1 else D, 1)
    out = torch.zeros(B * Hq * D, dtype=q.dtype, device=cuda).as_strided((B, Hq, D), strides)
    assert store.decode_attention(q, lens, out=out) is out and torch.equal(out, want)
    out4 = torch.zeros(B * Hq * D, dtype=q.dtype, device=cuda).as_strided((B, Hq, 1, D), (*strides[:2], 5, 1))
    assert torch.equal(store.prefill_attention(q.unsqueeze(2), lens, out=out4).squeeze(2), want)
