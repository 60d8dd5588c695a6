"""Attention over a list of blocks that names every finished one, in order: the dense attention bit for bit, since the same
blocks go to the same waves (a longer or shorter list shares them out otherwise)."""
import pytest
import torch
from kv8_ref import D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("blocks", [1, 9, 40, 300])
def test_every_block_in_order_is_dense(cuda, blocks, dtype):
    from leankv_amd.kv8 import KV8Store

    n = 64 * blocks + 20
    g = torch.Generator().manual_seed(blocks)
    store = KV8Store(2, 2, n, device=cuda)
    store.update(*(torch.randn(2, 2, n, D, generator=g).to(dtype).to(cuda) for _ in range(2)),
                 torch.zeros(2, dtype=torch.int32, device=cuda))
    lens = torch.full((2,), n, dtype=torch.int32, device=cuda)
    q = torch.randn(2, 8, D, generator=g).to(dtype).to(cuda)
    index = torch.arange(blocks, dtype=torch.int32, device=cuda).expand(2, 2, -1).contiguous()
    dense = store.decode_attention(q, lens)
    assert torch.equal(store.decode_attention(q, lens, index=index), dense)
    out, chosen = store.sparse_decode_attention(q, lens, blocks, 0, 0)
    assert torch.equal(chosen, index) and torch.equal(out, dense)
