"""BlockInt8Cache gives back keys and values in the keys' type: also after a reset, with a model of another type."""
import pytest
import torch
from kv8_ref import D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("asked", [None, torch.float32])
def test_type_after_reset(cuda, asked):
    from leankv_amd.kv8 import BlockInt8Cache

    cache = BlockInt8Cache(num_layers=2, device=cuda, dtype=asked, max_seq_len=64)
    x = torch.randn(1, 2, 5, D, generator=torch.Generator().manual_seed(1)).to(cuda)
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        for li in range(2):
            kk, vv = cache.update(x.to(dtype), x.to(dtype), li)
            assert kk.dtype == vv.dtype == (asked or dtype)
        cache.reset()
