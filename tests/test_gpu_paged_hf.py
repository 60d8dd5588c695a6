"""PagedCache as HF past_key_values: generate, beam search, cut and chosen batches, growth.  It holds the keys and values as the
model computed them, so under HF's own attention results are those of HF's cache to the bit; with the kernels that read the
pages logits are compared at the bound of the other HF tests."""
import copy

import pytest
import torch
from oracle import teal as ot

pytestmark = pytest.mark.gpu

TINY = dict(vocab_size=512, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4,
            num_key_value_heads=2, head_dim=128, max_position_embeddings=2048)
RTOL = 2e-2


def _model(cuda, seed):
    from leankv_amd.engine import random_mistral

    m = random_mistral(device=cuda, seed=seed, **TINY)
    m.generation_config.eos_token_id = None
    return m


def _ids(n, seed, B=1):
    return torch.randint(0, TINY["vocab_size"], (B, n), generator=torch.Generator().manual_seed(seed))


def _scores(model, ids, cache, mask=None, steps=20, reorder=None):
    """Teacher-forced: the prompt in two chunks, then one token at a time."""
    n0 = ids.shape[1] - steps
    out, dev = [], model.device
    with torch.no_grad():
        for a, b in [(0, n0 // 2), (n0 // 2, n0)] + [(i, i + 1) for i in range(n0, ids.shape[1])]:
            kw = {} if mask is None else dict(attention_mask=mask[:, :b].to(dev))
            out.append(model(ids[:, a:b].to(dev), past_key_values=cache, use_cache=True, **kw).logits[:, -1].float().cpu())
            if reorder is not None and a >= n0:
                cache.reorder_cache(reorder[a % len(reorder)].to(dev))
    return out


def _close(a, b):
    return max(ot.rel_err(x.numpy(), y.numpy()) for x, y in zip(a, b))


@pytest.mark.parametrize("B,n,page", [(1, 150, 64), (3, 90, 16), (2, 300, 32)])
def test_fused_steps_match_hf(cuda, B, n, page):
    from leankv_amd.combined import optimize_model
    from leankv_amd.paged import PagedCache
    from transformers import DynamicCache

    ids = _ids(n, 3, B)
    want = _scores(_model(cuda, 21), ids, DynamicCache())
    model, cache = optimize_model(_model(cuda, 21), paged_kv=True, page_size=page, max_seq_len=64)
    assert isinstance(cache, PagedCache) and model.config._attn_implementation == "leankv_tq"
    assert _close(_scores(model, ids, cache), want) < RTOL
    assert cache.get_seq_length(0) == n and len(cache) == 2 and cache.kv.max_len >= n
    assert cache.get_compression_ratio() > 0.5
    # the same tokens again after a cut, and in a cache of its own
    cache.crop(n - 20)
    other = copy.deepcopy(cache)
    for c in (cache, other):
        with torch.no_grad():
            got = [model(ids[:, i:i + 1].to(cuda), past_key_values=c, use_cache=True).logits[:, -1].float().cpu()
                   for i in range(n - 20, n)]
        assert _close(got, want[2:]) < RTOL and c.get_seq_length(1) == n


@pytest.mark.parametrize("fused", [False, True])
def test_reordered_batches(cuda, fused):
    """Beams that go on from each other at every step."""
    from leankv_amd.paged import PagedCache
    from leankv_amd.turboquant.attention import use_on
    from transformers import DynamicCache

    B, n = 4, 75
    ids = _ids(n, 8, B)
    orders = [torch.tensor(o) for o in ([0, 0, 0, 0], [1, 0, 3, 2], [2, 2, 1, 0], [0, 1, 2, 3], [3, 3, 3, 1])]
    want = _scores(_model(cuda, 4), ids, DynamicCache(), reorder=orders)
    model = _model(cuda, 4)
    cache = PagedCache(num_layers=2, device=cuda, max_seq_len=32, page_size=16)
    if fused:
        use_on(model, cache)
    got = _scores(model, ids, cache, reorder=orders)
    assert _close(got, want) < RTOL
    if not fused:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_beam_search(cuda):
    """generate with beams: HF's attention over the cache's K / V finds the beams of HF's own cache, the pages' kernels score
    theirs as HF scores the same sequences."""
    from leankv_amd.combined import optimize_model
    from leankv_amd.paged import PagedCache
    from transformers import DynamicCache

    ids = _ids(40, 9, 2).to(cuda)

    def go(model, cache):
        with torch.no_grad():
            return model.generate(ids, attention_mask=torch.ones_like(ids), max_new_tokens=25, past_key_values=cache,
                                  num_beams=3, num_return_sequences=2, do_sample=False, pad_token_id=0,
                                  output_scores=True, return_dict_in_generate=True, length_penalty=0.0)

    want = go(_model(cuda, 6), DynamicCache())
    plain = go(_model(cuda, 6), PagedCache(num_layers=2, device=cuda, max_seq_len=32, page_size=16))
    assert torch.equal(plain.sequences, want.sequences) and torch.equal(plain.sequences_scores, want.sequences_scores)
    model, cache = optimize_model(_model(cuda, 6), paged_kv=True, max_seq_len=128)
    got = go(model, cache)
    assert got.sequences.shape == want.sequences.shape and cache.get_seq_length(0) == 64
    # 24 steps' log probabilities, each within the logits' bound of the largest logit
    with torch.no_grad():
        logits = _model(cuda, 6)(got.sequences).logits.float()
    logp = logits.log_softmax(-1)[:, 39:-1].gather(-1, got.sequences[:, 40:].unsqueeze(-1)).squeeze(-1).sum(-1)
    bound = 25 * 2 * RTOL * float(logits.abs().max())
    assert float((logp - got.sequences_scores).abs().max()) < bound
    # beams of a prompt share its pages: 6 sequences of 64 tokens in pages of 16 are 24 pages apart
    assert int((cache.kv.refs > 0).sum()) < 24


def test_assisted_generation(cuda):
    """Tokens looked up in the prompt are checked several at a time, and those not taken cut off again."""
    from leankv_amd.combined import optimize_model
    from leankv_amd.paged import PagedCache
    from transformers import DynamicCache

    ids = _ids(12, 21).repeat(1, 4).to(cuda)

    def go(model, cache):
        with torch.no_grad():
            return model.generate(ids, attention_mask=torch.ones_like(ids), max_new_tokens=40, past_key_values=cache,
                                  prompt_lookup_num_tokens=5, do_sample=False, pad_token_id=0)

    want = go(_model(cuda, 8), DynamicCache())
    assert torch.equal(go(_model(cuda, 8), PagedCache(num_layers=2, device=cuda, max_seq_len=32, page_size=16)), want)
    model, cache = optimize_model(_model(cuda, 8), paged_kv=True, max_seq_len=64)
    got = go(model, cache)
    assert got.shape == want.shape and cache.get_seq_length(0) < got.shape[1]
    # a step's choice is the largest logit within the bound of its row's logits, twice (its own and the largest one's)
    with torch.no_grad():
        logits = _model(cuda, 8)(got).logits.float()[:, 47:-1]
    lost = logits.amax(-1) - logits.gather(-1, got[:, 48:].unsqueeze(-1)).squeeze(-1)
    assert float(lost.max()) < 2 * RTOL * float(logits.abs().max())


def test_padding_and_generate(cuda):
    from leankv_amd.combined import optimize_model
    from transformers import DynamicCache

    ids, mask = _ids(60, 4, 2), torch.ones(2, 60, dtype=torch.long)
    mask[0, :17] = 0
    want = _scores(_model(cuda, 5), ids, DynamicCache(), mask=mask)
    model, cache = optimize_model(_model(cuda, 5), paged_kv=True, max_seq_len=64)
    assert _close(_scores(model, ids, cache, mask=mask), want) < RTOL
    cache.reset()
    x = ids[1:].to(cuda)
    with torch.no_grad():
        a = model.generate(x, attention_mask=torch.ones_like(x), max_new_tokens=70, past_key_values=cache, do_sample=False,
                           pad_token_id=0)
        n = cache.get_seq_length(1)
        cache.reset()
        b = model.generate(x, attention_mask=torch.ones_like(x), max_new_tokens=70, past_key_values=cache, do_sample=False,
                           pad_token_id=0)
    assert torch.equal(a, b) and n == 129


def test_chosen_batches_and_bf16(cuda):
    from leankv_amd.paged import PagedCache

    gen = torch.Generator().manual_seed(2)
    cache = PagedCache(num_layers=2, device=cuda, max_seq_len=32, page_size=16)
    k = [torch.randn(2, 2, 21, 128, generator=gen).bfloat16().cuda() for _ in range(4)]
    for layer in range(2):
        cache.update(k[2 * layer], k[2 * layer + 1], layer)
    cache.batch_repeat_interleave(2)
    assert cache.max_batch_size == 4 and int((cache.kv.refs > 0).sum()) == 4
    more = torch.randn(4, 2, 1, 128, generator=gen).bfloat16().cuda()
    for layer in range(2):
        a, b = cache.update(more, -more, layer)
        want = torch.cat([k[2 * layer].repeat_interleave(2, 0), more], 2)
        assert torch.equal(a, want) and torch.equal(b, torch.cat([k[2 * layer + 1].repeat_interleave(2, 0), -more], 2))
    cache.batch_select_indices(torch.tensor([3, 0, 3], device=cuda))
    assert torch.equal(cache[1][0], want[[3, 0, 3]]) and cache.max_batch_size == 3
    grown = copy.deepcopy(cache)  # fewer sequences than before, past the length that there was room for
    grown.batch_select_indices(torch.tensor([0], device=cuda))
    tail = torch.randn(1, 2, 50, 128, generator=gen).bfloat16().cuda()
    for layer in range(2):
        a, _ = grown.update(tail, tail, layer)
    assert torch.equal(a, torch.cat([want[3:], tail], 2)) and grown.kv.max_len >= 72
    cache.crop(-3)
    assert cache.get_seq_length(0) == 19 and torch.equal(cache[1][0], want[[3, 0, 3], :, :19])
    cache.crop(0)  # (HF's caches drop as many tokens as a number below 1 says)
    assert cache.get_seq_length(1) == 19
    cache.crop(torch.tensor(-19))
    assert cache.get_seq_length(1) == 0 and not (cache.kv.refs > 0).any()
    a, _ = cache.update(more[:3], more[:3], 0)
    assert torch.equal(a, more[:3])


def test_refusals(cuda):
    from leankv_amd.paged import PagedCache

    cache = PagedCache(num_layers=2, device=cuda, max_seq_len=64, fused_attention=True)
    x = torch.zeros(1, 2, 3, 128, dtype=torch.float16, device=cuda)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        cache.update(x.float(), x.float(), 0)
    with pytest.raises(RuntimeError, match="in order"):
        cache.update(x, x, 1)
    cache.update(x, x, 0)
    with pytest.raises(RuntimeError, match="never attended"):
        cache.update(x, x, 0)
    with pytest.raises(RuntimeError, match="awaits"):
        cache.reorder_cache(torch.zeros(1, dtype=torch.long))
    with pytest.raises(RuntimeError, match="no one-token update"):
        cache.decode_attention(0, x[:, :, :1])
    cache.prefill_attention(0, x)
    with pytest.raises(ValueError, match="holds 1 sequences"):
        cache.update(x.expand(2, -1, -1, -1), x.expand(2, -1, -1, -1), 0)
    with pytest.raises(ValueError, match="beams"):
        cache.reorder_cache(torch.zeros(2, dtype=torch.long))
    from leankv_amd._lib import LeanKVError

    cache = PagedCache(num_layers=1, device=cuda, max_seq_len=64)
    cache.update(x, x, 0)
    for bad in (torch.tensor([0, 1]), torch.tensor([-1])):
        with pytest.raises(LeanKVError, match="outside"):
            cache.batch_select_indices(bad)
