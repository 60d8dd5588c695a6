"""BlockInt8Cache as HF past_key_values: optimize_model(kv8=True) and generate, a step's attention against the store's in
64 bits, growth, batches, padding, sparse steps.  The models are small random ones; what generate scores is compared with
the same model over the K / V that the cache reads back, under plain SDPA, at the bound of the other HF tests."""
import pytest
import torch
from kv8_ref import BLOCK, SCALE, D, Ref, choose, query, stored
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


def _scores(model, ids, cache, mask=None):
    """Teacher-forced: the prompt's last logits, then one token at a time."""
    n0 = ids.shape[1] - 20
    out, dev = [], model.device
    with torch.no_grad():
        for a, b in [(0, n0)] + [(i, i + 1) for i in range(n0, ids.shape[1])]:
            kw = {} if mask is None else dict(attention_mask=mask[:, :b].to(dev))
            out.append(model(ids[:, a:b].to(dev), past_key_values=cache, use_cache=True, **kw).logits[:, -1].float().cpu())
    return out


def _close(a, b):
    return max(ot.rel_err(x.numpy(), y.numpy()) for x, y in zip(a, b))


@pytest.mark.parametrize("B,n", [(1, 150), (3, 90), (1, 64 + 20)])
def test_fused_steps_match_sdpa_over_the_read_back_cache(cuda, B, n):
    from leankv_amd.combined import optimize_model
    from leankv_amd.kv8 import BlockInt8Cache

    ids = _ids(n, 3, B)
    plain = _scores(_model(cuda, 21), ids, BlockInt8Cache(num_layers=2, device=cuda, max_seq_len=256))
    model, cache = optimize_model(_model(cuda, 21), kv8=True, max_seq_len=256)
    assert isinstance(cache, BlockInt8Cache) and model.config._attn_implementation == "leankv_tq"
    assert _close(_scores(model, ids, cache), plain) < RTOL
    assert cache.get_seq_length(0) == n and len(cache) == 2
    # and both against no quantization at all: 8 bits with block scales are near fp16
    from transformers import DynamicCache

    assert _close(_scores(_model(cuda, 21), ids, DynamicCache()), plain) < RTOL


def test_generate_and_growth(cuda):
    """generate on the fused cache, the store growing while it runs, twice over (reset)."""
    from leankv_amd.combined import optimize_model
    from leankv_amd.kv8 import BlockInt8Cache

    model, cache = optimize_model(_model(cuda, 5), kv8=True, max_seq_len=64)
    ids = _ids(60, 4).to(cuda)

    def go(c):
        with torch.no_grad():
            return model.generate(ids, attention_mask=torch.ones_like(ids), max_new_tokens=90, past_key_values=c,
                                  do_sample=False, pad_token_id=0, output_scores=True, return_dict_in_generate=True)

    first = go(cache)
    assert cache._stores[0].capacity == 256 and cache.get_seq_length(1) == 149
    roomy = BlockInt8Cache(num_layers=2, device=cuda, max_seq_len=256, fused_attention=True)
    again = go(roomy)
    assert torch.equal(first.sequences, again.sequences)
    for li in range(2):
        for a, b in zip(cache[li], roomy[li]):
            assert torch.equal(a, b)
    cache.reset()
    assert torch.equal(go(cache).sequences, first.sequences)
    assert 1.5 < cache.get_compression_ratio() < 2.0


def test_padded_batch_takes_the_masked_path(cuda):
    """Left padding: HF's mask applies, through SDPA over the read-back cache, as without leankv_tq."""
    from leankv_amd.combined import optimize_model
    from leankv_amd.kv8 import BlockInt8Cache

    ids, mask = _ids(90, 8, 2), torch.ones(2, 90, dtype=torch.long)
    mask[1, :30] = 0
    plain = _scores(_model(cuda, 21), ids, BlockInt8Cache(num_layers=2, device=cuda), mask)
    model, cache = optimize_model(_model(cuda, 21), kv8=True)
    got = _scores(model, ids, cache, mask)
    assert _close(got, plain) < RTOL


def test_copies_of_a_prompt_go_their_own_ways(cuda):
    """A prompt's cache copied for two continuations: each as from a prompt of its own."""
    import copy

    from leankv_amd.combined import optimize_model
    from leankv_amd.kv8 import BlockInt8Cache

    model, cache = optimize_model(_model(cuda, 3), kv8=True, max_seq_len=128)
    prompt, tails = _ids(100, 1).to(cuda), [_ids(40, s).to(cuda) for s in (2, 3)]
    with torch.no_grad():
        model(prompt, past_key_values=cache, use_cache=True)
        for tail in tails:
            mine = copy.deepcopy(cache)
            got = model(tail, past_key_values=mine, use_cache=True).logits
            fresh = BlockInt8Cache(num_layers=mine.num_layers, max_seq_len=128, device=cuda, fused_attention=True)
            model(prompt, past_key_values=fresh, use_cache=True)
            assert torch.equal(got, model(tail, past_key_values=fresh, use_cache=True).logits)
            assert mine.get_seq_length() == 140 and cache.get_seq_length() == 100


def test_unattended_update_raises(cuda):
    from leankv_amd.kv8 import BlockInt8Cache

    cache = BlockInt8Cache(num_layers=1, device=cuda, fused_attention=True)
    k = torch.randn(1, 2, 3, D, device=cuda, dtype=torch.float16)
    cache.update(k, k, 0)
    with pytest.raises(RuntimeError, match="never attended"):
        cache.update(k, k, 0)
    assert [t.shape for t in cache.take_full_cache(0)] == [(1, 2, 3, D)] * 2
    with pytest.raises(ValueError, match="holds"):
        cache.update(k[:, :1], k[:, :1], 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sparse", [None, 3])
def test_a_prompt_a_chunk_and_steps(cuda, dtype, sparse):
    """What a model's layer does with the cache, run together: a prompt, a chunk, one-token steps (sparse ones once there
    are more blocks than it reads), each attention against 64 bits, and the tokens read back at the end."""
    from leankv_amd.kv8 import BlockInt8Cache
    from leankv_amd.turboquant.attention import leankv_tq_attention

    B, H, Hq = 2, 2, 8
    lengths = [130, 61] + [1] * 70
    n = sum(lengths)
    g = torch.Generator().manual_seed(17)
    k = (torch.randn(B, n, H, D, generator=g) * 1.3).to(dtype).to(cuda).transpose(1, 2)
    v = torch.randn(B, n, H, D, generator=g).to(dtype).to(cuda).transpose(1, 2)
    q = (torch.randn(B, n, Hq, D, generator=g) * 1.5).to(dtype).to(cuda).transpose(1, 2)
    cache = BlockInt8Cache(num_layers=1, device=cuda, max_seq_len=100, fused_attention=True, sparse_blocks=sparse)
    module = torch.nn.Module()
    module.layer_idx, module.is_causal = 0, True
    ks, vs = stored(k.cpu()), stored(v.cpu())
    at = 0
    for S in lengths:
        kk, vv = cache.update(k[:, :, at:at + S], v[:, :, at:at + S], 0)
        out, _ = leankv_tq_attention(module, q[:, :, at:at + S], kk, vv, None, scaling=SCALE)
        assert out.shape == (B, S, Hq, D) and out.dtype == dtype and out.is_contiguous()
        at += S
        rows = range(S) if S == 1 else (0, 1, S // 2, S - 1)
        if S == 1 and at % 7 and at % BLOCK > 1:
            continue
        for b in range(B):
            refs = [Ref(ks[b, h, :at], vs[b, h, :at]) for h in range(H)]
            for h in range(Hq):
                r = refs[h * H // Hq]
                for i in rows:
                    qi = query(q[b, :, at - S + i].cpu())
                    seen, pick = at - S + i + 1, None
                    if S == 1 and sparse is not None and r.nb > sparse:
                        G = Hq // H
                        chosen = choose(r, qi[h // G * G:(h // G + 1) * G], sparse, 1, 1)
                        pick = [BLOCK * j + e for j in chosen for e in range(BLOCK)] + list(range(r.nb * BLOCK, at))
                        seen = len(pick)
                    want, bound = r.attend(qi[h], seen, SCALE, torch.finfo(dtype).eps, pick)
                    err = (out[b, i, h].cpu().double() - want).abs()
                    assert (err <= bound).all(), (at, b, h, i, (err / bound).max())
    kk, vv = cache[0]
    assert kk.dtype == dtype and kk.shape == (B, H, n, D)
    r = Ref(ks[1, 1], vs[1, 1])
    val = r.vals["k"]  # rounded to fp32, fp16 and (bf16) once more
    eps = torch.finfo(dtype).eps / 2 + 2.0 ** -11 + 2.0 ** -24
    assert ((kk[1, 1].cpu().double() - val).abs() <= eps * val.abs() * (1 + eps) + 2.0 ** -24).all()
