"""Drafted tokens dropped again across the end of a block: the store taken back into its last finished block is, bit for bit,
a store that never held the dropped tokens."""
import pytest
import torch
from kv8_ref import BLOCK, D

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _kv(dev, B, H, n, seed, dtype=torch.float16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return tuple((torch.randn(B, H, n, D, generator=g) * scale).to(dtype).to(dev) for _ in range(2))


def _equal(a, b, lens, H, seed):
    """Everything that two stores say of their sequences, and the blocks that are finished."""
    dev, n = a.device, max(lens)
    held = _ints(dev, lens)
    for x, y in zip(a.read(held, n), b.read(held, n)):
        assert torch.equal(x, y)
    g = torch.Generator().manual_seed(seed)
    for S in (1, 5, 40):  # one column tile, two, and the many-row kernel
        q = torch.randn(len(lens), 4 * H, S, D, generator=g).half().to(dev)
        if S == 1:
            assert torch.equal(a.decode_attention(q[:, :, 0], held), b.decode_attention(q[:, :, 0], held))
            for x, y in zip(a.sparse_decode_attention(q[:, :, 0], held, 2), b.sparse_decode_attention(q[:, :, 0], held, 2)):
                assert torch.equal(x, y)
        assert torch.equal(a.prefill_attention(q, held), b.prefill_attention(q, held))
    for name in ("k_codes", "v_codes", "scales", "ranges"):
        x, y = getattr(a, name), getattr(b, name)
        for i, m in enumerate(lens):
            assert torch.equal(x[i, :, :m // BLOCK], y[i, :, :m // BLOCK]), (name, i)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("have,S,keep", [
    ([62], 5, [63]),                                  # five drafts past a boundary, one of them accepted
    ([62, 63, 60, 190], 5, [62, 65, 61, 193]),        # none, over the boundary, inside the block
    ([64, 127, 128, 1], 64, [65, 128, 129, 1]),       # a whole block more
    ([62, 100, 65, 7], 140, [140, 200, 130, 128]),    # the last finished block lies two past the first
    ([10, 64, 63, 0], 200, [150, 200, 192, 131]),
    ([62, 30, 0, 127], 66, [100, 64, 40, 150])])      # older tokens dropped too
def test_taken_back_into_the_last_finished_block(cuda, have, S, keep, dtype):
    from leankv_amd.kv8 import KV8Store

    B, H, more = len(have), 2, 150
    k, v = _kv(cuda, B, H, max(have) + 1, seed=1, dtype=dtype)
    dk, dv = _kv(cuda, B, H, S, seed=2, dtype=dtype, scale=7.0)  # (they would change a block's scale)
    nk, nv = _kv(cuda, B, H, more, seed=3, dtype=dtype)
    a, b = (KV8Store(B, H, 512, device=cuda) for _ in range(2))
    for n, m in zip(have, keep):
        assert m >= BLOCK * ((n + S) // BLOCK - 1)
    a.update(k, v, _ints(cuda, [0] * B), _ints(cuda, have))
    a.update(dk, dv, _ints(cuda, have))
    # b: only the tokens that stay
    b.update(k, v, _ints(cuda, [0] * B), _ints(cuda, [min(n, m) for n, m in zip(have, keep)]))
    b.update(dk, dv, _ints(cuda, [min(n, m) for n, m in zip(have, keep)]),
             _ints(cuda, [max(0, m - n) for n, m in zip(have, keep)]))
    _equal(a, b, keep, H, 4)
    # and goes on from there: by one token, by what finishes the block, past it
    lens, at = list(keep), 0
    for s in (1, 3, 70, more - 74):
        for st in (a, b):
            st.update(nk[:, :, at:at + s], nv[:, :, at:at + s], _ints(cuda, lens))
        lens, at = [m + s for m in lens], at + s
        _equal(a, b, lens, H, 5 + at)


def test_drafts_step_after_step(cuda):
    """Speculative decoding: five drafts a step, 0 to 5 of them accepted, over several blocks; every step's attention is
    that of a store which only ever held the accepted tokens."""
    from leankv_amd.kv8 import KV8Store

    B, H, n = 3, 2, 260
    k, v = _kv(cuda, B, H, n, seed=11)
    wrong = _kv(cuda, B, H, 5, seed=12, scale=30.0)
    a, b = (KV8Store(B, H, 320, device=cuda) for _ in range(2))
    lens, step = [50, 57, 126], 0
    for st in (a, b):
        st.update(k, v, _ints(cuda, [0] * B), _ints(cuda, lens))
    while max(lens) + 5 < n:
        taken = [(step * 5 + 3 * i) % 6 for i in range(B)]
        drafts = [torch.stack([torch.cat([x[i, :, m:m + t], w[i, :, t:]], 1) for i, (m, t) in enumerate(zip(lens, taken))])
                  for x, w in zip((k, v), wrong)]
        a.update(*drafts, _ints(cuda, lens))
        b.update(*drafts, _ints(cuda, lens), _ints(cuda, taken))
        lens, step = [m + t for m, t in zip(lens, taken)], step + 1
        _equal(a, b, lens, H, step)
    assert step > 20


def test_copies_hold_both_blocks(cuda):
    """A copy and a grown store are taken back like the store itself."""
    import copy

    from leankv_amd.kv8 import KV8Store

    k, v = _kv(cuda, 1, 2, 70, seed=21)
    a, b = (KV8Store(1, 2, 128, device=cuda) for _ in range(2))
    a.update(k, v, _ints(cuda, [0]))
    b.update(k[:, :, :50], v[:, :, :50], _ints(cuda, [0]))
    for st in (copy.deepcopy(a), a.grown(400)):
        _equal(st, b, [50], 2, 22)


def test_taken_back_in_a_full_store(cuda):
    """The store's last block finished, tokens past it dropped: the sequence goes back into that block."""
    from leankv_amd.kv8 import KV8Store

    k, v = _kv(cuda, 2, 2, 150, seed=31)
    a, b = (KV8Store(2, 2, 128, device=cuda) for _ in range(2))
    a.update(k[:, :, :120], v[:, :, :120], _ints(cuda, [0, 0]))
    a.update(k[:, :, 120:], v[:, :, 120:], _ints(cuda, [120, 120]))
    b.update(k, v, _ints(cuda, [0, 0]), _ints(cuda, [64, 125]))
    _equal(a, b, [64, 125], 2, 32)
    for st in (a, b):
        st.update(k[:, :, :30], v[:, :, :30], _ints(cuda, [64, 125]))
    _equal(a, b, [94, 128], 2, 33)
