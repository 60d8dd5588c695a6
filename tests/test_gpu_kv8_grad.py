"""Autograd and the 8-bit KV cache: no gradient flows through the store, and a backward pass that would need one says so."""
import pytest
import torch
from kv8_ref import D
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _inputs(dev, follow=(), n=70):
    g = torch.Generator().manual_seed(1)
    x = dict(k=torch.randn(2, 2, n, D, generator=g), v=torch.randn(2, 2, n, D, generator=g),
             q=torch.randn(2, 4, 3, D, generator=g))
    return {name: t.half().to(dev).requires_grad_(name in follow) for name, t in x.items()}


def _outs(store, x, n=70):
    dev = store.device
    store.update(x["k"], x["v"], _ints(dev, [0, 0]))
    lens, q = _ints(dev, [n, n]), x["q"]
    outs = [store.decode_attention(q[:, :, 0], lens), store.prefill_attention(q, lens),
            store.sparse_decode_attention(q[:, :, 0], lens, 2)[0]]
    return outs, list(store.read(lens, n))


@pytest.mark.parametrize("follow", ["q", "k", "v", "qkv"])
def test_a_backward_pass_raises(cuda, follow):
    from leankv_amd._lib import LeanKVError
    from leankv_amd.kv8 import KV8Store

    plain = _outs(KV8Store(2, 2, 128, device=cuda), _inputs(cuda))
    assert not any(t.requires_grad for part in plain for t in part)
    store = KV8Store(2, 2, 128, device=cuda)
    got = _outs(store, _inputs(cuda, follow))
    for part, want in zip(got, plain):
        assert all(torch.equal(a.detach(), b) for a, b in zip(part, want))  # the numbers are the same
    for t in got[0] + (got[1] if follow != "q" else []):
        with pytest.raises(LeanKVError, match="backward"):
            t.float().sum().backward()
    if follow == "q":
        assert not any(t.requires_grad for t in got[1])  # (what is stored has nothing to do with it)
    else:  # a copy knows what was stored into it
        with pytest.raises(LeanKVError, match="backward"):
            store.grown(512).read(_ints(cuda, [70, 70]), 70)[0].float().sum().backward()


def test_without_grad_mode_nothing_changes(cuda):
    from leankv_amd.kv8 import KV8Store

    with torch.no_grad():
        store = KV8Store(2, 2, 128, device=cuda)
        got = _outs(store, _inputs(cuda, "qkv"))
        assert not any(t.requires_grad for part in got for t in part)
    q, lens = _inputs(cuda)["q"][:, :, 0], _ints(cuda, [70, 70])
    assert not store.decode_attention(q, lens).requires_grad  # stored without grad mode: nothing was to be followed
    out = torch.empty_like(q)
    assert store.decode_attention(q, lens, out=out) is out


def test_out_and_tangents_are_refused(cuda):
    from leankv_amd._lib import LeanKVError
    from leankv_amd.kv8 import KV8Store

    store, x = KV8Store(2, 2, 128, device=cuda), _inputs(cuda)
    _outs(store, x)
    lens, q = _ints(cuda, [70, 70]), x["q"]
    for call in (lambda: store.decode_attention(q[:, :, 0].clone().requires_grad_(), lens, out=torch.empty_like(q[:, :, 0])),
                 lambda: store.prefill_attention(q.clone().requires_grad_(), lens, out=torch.empty_like(q))):
        with pytest.raises(LeanKVError, match="out="):
            call()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        dk = forward_ad.make_dual(x["k"], torch.ones_like(x["k"]))
        for call in (lambda: store.prefill_attention(dual, lens), lambda: store.decode_attention(dual[:, :, 0], lens),
                     lambda: store.sparse_decode_attention(dual[:, :, 0], lens, 2),
                     lambda: store.update(dk, x["v"], _ints(cuda, [0, 0])), lambda: store.update(x["k"], dk, _ints(cuda, [0, 0]))):
            with pytest.raises(LeanKVError, match="forward-mode"):
                call()
        assert store.prefill_attention(q, lens).shape == q.shape  # (no tangent, no refusal)


@pytest.mark.parametrize("fused", [True, False])
def test_a_model_trained_through_the_cache_raises(cuda, fused):
    """A forward pass with gradients enabled runs as before; its backward pass does not leave out attention's part."""
    from leankv_amd._lib import LeanKVError
    from leankv_amd.engine import random_mistral
    from leankv_amd.kv8 import BlockInt8Cache
    from leankv_amd.turboquant.attention import use_on

    model = random_mistral(device=cuda, seed=3, vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                           num_attention_heads=4, num_key_value_heads=2, head_dim=128, max_position_embeddings=2048)
    model.requires_grad_(True)
    cache = BlockInt8Cache(num_layers=2, device=cuda, max_seq_len=128)
    if fused:
        use_on(model, cache)
    ids = torch.randint(0, 512, (1, 70), generator=torch.Generator().manual_seed(4)).to(cuda)
    out = model(ids, past_key_values=cache, use_cache=True).logits
    if fused:  # (SDPA chooses among its kernels by whether there is a gradient)
        with torch.no_grad():
            cache.reset()
            assert torch.equal(model(ids, past_key_values=cache, use_cache=True).logits, out)
    with pytest.raises(LeanKVError, match="backward"):
        out.float().sum().backward()
