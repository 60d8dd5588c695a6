"""The 8-bit block-scaled KV cache: what update stores (bit for bit), reading it back, and its attention against the
same in 64 bits, with the bounds that its documented roundings give (kv8_ref.Ref.attend)."""
import pytest
import torch
from kv8_ref import BLOCK, SCALE, STEP, D, Ref, choose, factor, query, stored, v_tokens

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _store(*a, **k):
    from leankv_amd.kv8 import KV8Store

    return KV8Store(*a, **k)


def _ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _kv(dev, B, H, n, seed, dtype=F16, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    spread = torch.exp(0.5 * torch.randn(H, 1, D, generator=g)) * scale
    k = torch.randn(B, H, n, D, generator=g) * spread + 0.3 * torch.randn(H, 1, D, generator=g)
    v = torch.randn(B, H, n, D, generator=g) * scale
    return k.to(dtype).to(dev), v.to(dtype).to(dev)


def _refs(k, v, lens):
    k, v = stored(k.cpu()), stored(v.cpu())
    return [[Ref(k[b, h, :n], v[b, h, :n]) for h in range(k.shape[1])] for b, n in enumerate(lens)]


def _check_store(store, refs, k, v, lens):
    """Codes, scales, ranges and tails of every sequence, bit for bit."""
    vt = torch.tensor(v_tokens())
    kc, vc, sc, rg = (t.cpu() for t in (store.k_codes, store.v_codes, store.scales, store.ranges))
    kt, vtail = store.k_tail.cpu(), store.v_tail.cpu()
    k, v = stored(k.cpu()), stored(v.cpu())
    for b, n in enumerate(lens):
        for h in range(store.kv_heads):
            r, nb, rest = refs[b][h], n // BLOCK, n % BLOCK
            assert torch.equal(kc[b, h, :nb].long() - 128, r.codes["k"])
            assert torch.equal(vc[b, h, :nb].long() - 128, r.codes["v"].transpose(1, 2)[:, :, vt])
            assert torch.equal(sc[b, h, :nb], torch.stack([r.scales["k"], r.scales["v"]], 1))
            if nb:
                assert torch.equal(rg[b, h, :nb].long(), torch.stack([r.codes["k"].amin(1), r.codes["k"].amax(1)], 1))
            assert torch.equal(kt[b, h, :rest], k[b, h, n - rest:n])
            pos = torch.argsort(vt)[:rest]
            assert torch.equal(vtail[b, h][:, pos], v[b, h, n - rest:n].t())


def _check_read(store, refs, lens_dev, lens, n, first=0):
    for got, name in zip(store.read(lens_dev, n, first), "kv"):
        got = got.cpu()
        for b, m in enumerate(lens):
            for h in range(store.kv_heads):
                r = refs[b][h]
                nb = r.nb * BLOCK
                full = (r.codes[name].float() * r.scales[name][:, None, None]).half().reshape(-1, D)
                want = torch.cat([full, r.vals[name][nb:].half(), torch.zeros(max(0, n - m), D, dtype=F16)])[first:n]
                assert torch.equal(got[b, h], want), (name, b, h)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("B,H,lens", [(1, 1, [1]), (2, 3, [64, 63]), (1, 2, [65]), (3, 1, [0, 128, 191]),
                                      (2, 2, [300, 1000])])
def test_update_and_read(cuda, B, H, lens, dtype):
    S = max(lens)
    k, v = _kv(cuda, B, H, S, seed=S + B, dtype=dtype)
    store = _store(B, H, S, device=cuda)
    store.update(k, v, _ints(cuda, [0] * B), _ints(cuda, lens))
    refs, ln = _refs(k, v, lens), _ints(cuda, lens)
    _check_store(store, refs, k, v, lens)
    _check_read(store, refs, ln, lens, S)
    _check_read(store, refs, ln, lens, S, first=S // 2)
    _check_read(store, refs, ln, lens, store.capacity)


@pytest.mark.parametrize("steps", [[1] * 70, [60, 3, 1, 1, 64, 63, 130], [127, 129, 1, 62, 65], [63, 1, 64, 200]])
def test_update_in_steps_equals_one(cuda, steps):
    """Every sequence at its own position: the store after any sequence of updates holds what one update would."""
    B, H, n = 3, 2, sum(steps)
    k, v = _kv(cuda, B, H, n + 40, seed=n)
    store = _store(B, H, n + 40, device=cuda)
    start = [0, 17, 40]
    store.update(k[:, :, :40], v[:, :, :40], _ints(cuda, [0] * B), _ints(cuda, start))
    pos = list(start)
    for s in steps:
        kk = torch.stack([k[b, :, p:p + s] for b, p in enumerate(pos)])
        vv = torch.stack([v[b, :, p:p + s] for b, p in enumerate(pos)])
        store.update(kk, vv, _ints(cuda, pos))
        pos = [p + s for p in pos]
    refs = _refs(k, v, pos)
    _check_store(store, refs, k, v, pos)
    _check_read(store, refs, _ints(cuda, pos), pos, max(pos))


def test_update_strides_and_alignment(cuda):
    """Projection-layout views, rows that are not 16-byte aligned, single sizes with odd strides."""
    B, H, S = 2, 3, 130
    base_k, base_v = _kv(cuda, B, H, S, seed=5)
    want = _refs(base_k, base_v, [S] * B)
    for make in (lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda t: torch.cat([torch.zeros(1, dtype=t.dtype, device=t.device), t.reshape(-1)])[1:].view_as(t),
                 lambda t: torch.cat([t, t], -1)[..., :D], lambda t: torch.cat([t, t[..., :3]], -1)[..., :D],
                 lambda t: t.flip(2).flip(2), lambda t: t.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)):
        k, v = make(base_k), make(base_v)
        assert torch.equal(k, base_k)
        store = _store(B, H, S, device=cuda)
        store.update(k, v, _ints(cuda, [0] * B))
        _check_store(store, want, base_k, base_v, [S] * B)


def test_update_special_values(cuda):
    """Zero blocks, NaN, infinities, numbers past fp16, subnormals and a lone large number."""
    B, H, S = 1, 2, 64 * 5 + 9
    k, v = _kv(cuda, B, H, S, seed=9, dtype=F32)
    for t in (k, v):
        t[:, :, :64] = 0
        t[:, :, 64] = float("nan")
        t[:, :, 70, 3], t[:, :, 71, 4] = float("inf"), -float("inf")
        t[:, :, 128:192] *= 2.0 ** -22
        t[:, :, 200, 7] = 70000.0
        t[:, :, 325, 5] = float("nan")
        t[:, :, 326, 6] = -float("inf")
    store = _store(B, H, S, device=cuda)
    store.update(k, v, _ints(cuda, [0]))
    refs = _refs(k, v, [S])
    _check_store(store, refs, k, v, [S])
    q = torch.randn(1, 4, D, generator=torch.Generator().manual_seed(1)).half().to(cuda)
    assert torch.isfinite(store.decode_attention(q, _ints(cuda, [S]))).all()


def test_update_stays_inside(cuda):
    """Tokens past the capacity are dropped, a position outside the store stores nothing, n_new is cut at S; other
    sequences and bytes stay as they were."""
    B, H = 4, 2
    store = _store(B, H, 128, device=cuda)
    k, v = _kv(cuda, B, H, 100, seed=2)
    store.update(k, v, _ints(cuda, [0, 0, 0, 0]), _ints(cuda, [100, 100, 0, 60]))
    before = [t.clone() for t in (store.k_codes, store.v_codes, store.scales, store.ranges, store.k_tail, store.v_tail)]
    k2, v2 = _kv(cuda, B, H, 70, seed=3)
    store.update(k2, v2, _ints(cuda, [100, -1, 128, 60]), _ints(cuda, [70, 70, 70, -5]))
    full_k, full_v = torch.cat([k, k2[:, :, :28]], 2), torch.cat([v, v2[:, :, :28]], 2)
    lens = [128, 100, 0, 60]
    _check_store(store, _refs(full_k, full_v, lens), full_k, full_v, lens)
    for t, old in zip((store.k_codes, store.v_codes, store.scales, store.ranges, store.k_tail, store.v_tail), before):
        assert torch.equal(t[1:], old[1:])
    store.update(k2, v2, _ints(cuda, [128, 100, 0, 60]), _ints(cuda, [0, 0, 1000, 0]))
    k3, v3 = torch.cat([k2, k2], 2)[2:3], torch.cat([v2, v2], 2)[2:3]
    r = _refs(k3, v3, [70])
    assert torch.equal(store.k_codes[2, :, :1].cpu().long() - 128, torch.stack([x.codes["k"] for x in r[0]]))


def _check_attn(out, refs, q, lens, q_lens, scale=SCALE, tokens=None):
    """out, q [B, Hq, S, D]."""
    B, Hq, S, _ = q.shape
    got, q16 = out.cpu().double(), query(q.cpu())
    H = len(refs[0])
    worst = 0.0
    for b in range(B):
        for h in range(Hq):
            r = refs[b][h * H // Hq]
            for i in range(S):
                m = q_lens[b] if q_lens is not None else S
                if i >= m or lens[b] - m + i < 0:
                    assert (got[b, h, i] == 0).all(), (b, h, i)
                    continue
                pick = None if tokens is None else tokens[b][h * H // Hq]
                seen = lens[b] - m + i + 1 if pick is None else len(pick)
                want, bound = r.attend(q16[b, h, i], seen, scale, torch.finfo(out.dtype).eps, pick)
                ratio = ((got[b, h, i] - want).abs() / bound.clamp(min=1e-30)).max().item()
                assert ratio <= 1.0, (b, h, i, ratio)
                worst = max(worst, ratio)
    return worst


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("Hq,H,lens", [(1, 1, [1]), (4, 4, [63, 64, 65]), (8, 2, [0, 129, 640]), (16, 1, [257]),
                                       (17, 1, [100, 700]), (24, 8, [320]), (71, 1, [150]), (32, 8, [1999]),
                                       (12, 4, [64, 1, 0, 500, 64, 127])])
def test_decode_attention(cuda, Hq, H, lens, dtype):
    B, n = len(lens), max(lens)
    k, v = _kv(cuda, B, H, n, seed=n + Hq, dtype=dtype)
    store = _store(B, H, n, device=cuda)
    store.update(k, v, _ints(cuda, [0] * B), _ints(cuda, lens))
    q = (torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(3)) * 1.5).to(dtype).to(cuda)
    out = store.decode_attention(q, _ints(cuda, lens))
    assert out.shape == q.shape and out.dtype == dtype
    _check_attn(out.unsqueeze(2), _refs(k, v, lens), q.unsqueeze(2), lens, None)


def test_decode_attention_long_and_bounds(cuda):
    """A long sequence by many splits and by few (other bounds on its length), a scale of its own, an out buffer."""
    n = 64 * 500 + 13
    k, v = _kv(cuda, 1, 2, n, seed=4)
    store = _store(1, 2, 200000, device=cuda)
    store.update(k, v, _ints(cuda, [0]))
    refs, lens = _refs(k, v, [n]), _ints(cuda, [n])
    q = torch.randn(1, 8, D, generator=torch.Generator().manual_seed(5)).half().to(cuda)
    for bound in (None, n, 40000):
        _check_attn(store.decode_attention(q, lens, max_len=bound).unsqueeze(2), refs, q.unsqueeze(2), [n], None)
    out = torch.full_like(q, 7.0)
    assert store.decode_attention(q, lens, scale=0.3, out=out) is out
    _check_attn(out.unsqueeze(2), refs, q.unsqueeze(2), [n], None, scale=0.3)


def test_length_past_the_bound(cuda):
    """Of a sequence longer than max_len (or than the store) the finished blocks below the bound count; a negative length
    is none."""
    n = 64 * 7 + 9
    k, v = _kv(cuda, 3, 1, n, seed=4)
    store = _store(3, 1, n, device=cuda)
    store.update(k, v, _ints(cuda, [0] * 3), _ints(cuda, [n, 130, 0]))
    q = torch.randn(3, 2, D, generator=torch.Generator().manual_seed(5)).half().to(cuda)
    out = store.decode_attention(q, _ints(cuda, [n, 130, -3]), max_len=200)
    _check_attn(out.unsqueeze(2), _refs(k, v, [192, 130, 0]), q.unsqueeze(2), [192, 130, 0], None)
    out = store.prefill_attention(q.unsqueeze(2).expand(-1, -1, 80, -1), _ints(cuda, [n, 130, -3]), max_len=200)
    _check_attn(out, _refs(k, v, [192, 130, 0]), q.unsqueeze(2).expand(-1, -1, 80, -1), [192, 130, 0], [80, 80, 0])
    far = _ints(cuda, [2 ** 31 - 1, 130, -(2 ** 31)])
    out = store.decode_attention(q, far)
    _check_attn(out[1:].unsqueeze(2), _refs(k, v, [0, 130, 0])[1:], q[1:].unsqueeze(2), [130, 0], None)
    assert torch.isfinite(out).all() and (store.select_blocks(q, far, 9)[0, 0].cpu() == torch.tensor([*range(8), -1])).all()


def test_decode_attention_value_scales_apart(cuda):
    """Value blocks of very different scale (zero ones too) beside weights that favour the small ones."""
    n = 64 * 12 + 30
    k, v = _kv(cuda, 1, 1, n, seed=8, dtype=F32)
    q = torch.randn(1, 4, D, generator=torch.Generator().manual_seed(6)).half().to(cuda)
    for j, s in enumerate((1.0, 0.0, 2.0 ** -20, 1000.0, 2.0 ** -10, 60000.0 / 6, 1.0, 0.0, 2.0 ** -23, 1.0, 30.0, 1e-3)):
        v[:, :, 64 * j:64 * j + 64] *= s
        if s < 1e-2:
            k[:, :, 64 * j:64 * j + 64] += q[0, 0].float() * 0.8
    store = _store(1, 1, n, device=cuda)
    store.update(k, v, _ints(cuda, [0]))
    out = store.decode_attention(q.float(), _ints(cuda, [n]))
    _check_attn(out.unsqueeze(2), _refs(k, v, [n]), q.unsqueeze(2), [n], None)


def test_attention_nan_query_stays_in_its_row(cuda):
    k, v = _kv(cuda, 1, 1, 200, seed=8)
    store = _store(1, 1, 200, device=cuda)
    store.update(k, v, _ints(cuda, [0]))
    q = torch.randn(1, 3, D, generator=torch.Generator().manual_seed(6)).half().to(cuda)
    want = store.decode_attention(q, _ints(cuda, [200]))
    bad = q.clone()
    bad[0, 1, 5] = float("nan")
    out = store.decode_attention(bad, _ints(cuda, [200]))
    assert torch.isnan(out[0, 1]).all() and torch.equal(out[0, ::2], want[0, ::2])


def test_attention_nan_query_through_partial_sums(cuda):
    """The same where a row's sums come from several workgroups, for few rows and for many."""
    n = 64 * 90 + 3
    k, v = _kv(cuda, 1, 1, n, seed=8)
    store = _store(1, 1, n, device=cuda)
    store.update(k, v, _ints(cuda, [0]))
    lens = _ints(cuda, [n])
    for S in (1, 3, 130):
        q = torch.randn(1, 2, S, D, generator=torch.Generator().manual_seed(6)).half().to(cuda)
        want = store.prefill_attention(q, lens)
        bad = q.clone()
        bad[0, 1, S // 2, 5] = float("nan")
        out = store.prefill_attention(bad, lens)
        assert torch.isnan(out[0, 1, S // 2]).all()
        out[0, 1, S // 2] = want[0, 1, S // 2]
        assert torch.equal(out, want) and torch.isfinite(out).all()


@pytest.mark.parametrize("B,H,Hq,S,n", [(2, 8, 8, 4400, 4500), (1, 3, 3, 22100, 22100), (1, 8, 24, 3000, 3001)])
def test_prefill_more_pieces_than_workgroups(cuda, B, H, Hq, S, n):
    """Workgroups that take several pieces, one after the other: rows from everywhere."""
    k, v = _kv(cuda, B, H, n, seed=S)
    store = _store(B, H, n, device=cuda)
    store.update(k, v, _ints(cuda, [0] * B))
    q = torch.randn(B, S, Hq, D, generator=torch.Generator().manual_seed(3)).half().to(cuda).transpose(1, 2)
    out = store.prefill_attention(q, _ints(cuda, [n] * B)).cpu()
    assert torch.isfinite(out).all()
    g = torch.Generator().manual_seed(S)
    k, v = stored(k.cpu()), stored(v.cpu())
    refs = {}
    for _ in range(60):
        b, h, i = (int(torch.randint(0, m, (1,), generator=g)) for m in (B, Hq, S))
        if (b, h * H // Hq) not in refs:
            refs[b, h * H // Hq] = Ref(k[b, h * H // Hq], v[b, h * H // Hq])
        want, bound = refs[b, h * H // Hq].attend(query(q[b, h, i].cpu()), n - S + i + 1, SCALE, torch.finfo(F16).eps)
        assert ((out[b, h, i].double() - want).abs() <= bound).all(), (b, h, i)


@pytest.mark.parametrize("S", [3, 200])
def test_out_buffers_of_other_layouts(cuda, S):
    """Outputs written into views: by token, with rows apart, beside other data that stays."""
    k, v = _kv(cuda, 2, 2, 300, seed=2)
    store = _store(2, 2, 300, device=cuda)
    store.update(k, v, _ints(cuda, [0, 0]))
    lens = _ints(cuda, [300, 300])
    q = torch.randn(2, 4, S, D, generator=torch.Generator().manual_seed(3)).half().to(cuda)
    want = store.prefill_attention(q, lens)
    for make in (lambda: torch.full((2, 4, S, D), 9.0, dtype=F16, device=cuda),
                 lambda: torch.full((2, 4, S, 2 * D), 9.0, dtype=F16, device=cuda)[..., 8:8 + D],
                 lambda: torch.full((S, 2, 4, D), 9.0, dtype=F16, device=cuda).permute(1, 2, 0, 3),
                 lambda: torch.full((2, 7, S + 1, D), 9.0, dtype=F16, device=cuda)[:, 2:6, 1:]):
        out = make()
        assert store.prefill_attention(q, lens, out=out) is out and torch.equal(out, want)
        base = out._base
        if base is not None and base.numel() > out.numel():
            assert (base == 9.0).sum() >= base.numel() - out.numel()
    one = torch.full((2, 4, 3 * D), 9.0, dtype=F16, device=cuda)[..., D:2 * D]
    store.decode_attention(q[:, :, 0], lens, out=one)
    assert torch.equal(one, store.decode_attention(q[:, :, 0], lens)) and (one._base[..., :D] == 9.0).all()
    inplace = q[:, :, 0].clone()  # over its own queries
    assert torch.equal(store.decode_attention(inplace, lens, out=inplace), one)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("Hq,H,S,lens,q_lens", [
    (2, 1, 5, [70], None), (8, 2, 3, [3, 200, 64], None), (4, 4, 64, [64], None), (8, 8, 65, [65, 130], [65, 20]),
    (8, 2, 33, [40, 300], [1, 33]), (6, 2, 130, [130, 500, 131], [130, 77, 0]), (3, 1, 200, [263, 200], None),
    (16, 1, 24, [24, 640], [10, 24]), (20, 4, 16, [16, 17, 333], None), (7, 1, 300, [300], None),
    (32, 8, 96, [700], None)])
def test_prefill_attention(cuda, Hq, H, S, lens, q_lens, dtype):
    B, n = len(lens), max(lens)
    k, v = _kv(cuda, B, H, n, seed=n + S, dtype=dtype)
    store = _store(B, H, n, device=cuda)
    store.update(k, v, _ints(cuda, [0] * B), _ints(cuda, lens))
    q = (torch.randn(B, S, Hq, D, generator=torch.Generator().manual_seed(3)) * 1.5).to(dtype).to(cuda).transpose(1, 2)
    out = store.prefill_attention(q, _ints(cuda, lens), None if q_lens is None else _ints(cuda, q_lens))
    assert out.shape == q.shape and out.dtype == dtype
    _check_attn(out, _refs(k, v, lens), q, lens, q_lens)


def test_prefill_more_queries_than_tokens(cuda):
    """q_lens beyond the length: the queries before the first token do not exist, the others are the newest."""
    k, v = _kv(cuda, 2, 1, 10, seed=1)
    store = _store(2, 1, 64, device=cuda)
    store.update(k, v, _ints(cuda, [0, 0]), _ints(cuda, [4, 0]))
    q = torch.randn(2, 2, 9, D, generator=torch.Generator().manual_seed(3)).half().to(cuda)
    out = store.prefill_attention(q, _ints(cuda, [4, 0]))
    # the sequence has 4 tokens, so 4 of the 9 rows are its queries
    _check_attn(out, _refs(k, v, [4, 0]), q, [4, 0], [4, 0])


@pytest.mark.parametrize("Hq,H,lens,blocks,sink,recent", [
    (4, 1, [64 * 30 + 5], 4, 1, 1), (8, 2, [64 * 40, 64 * 3 + 1, 63, 0], 6, 1, 1), (32, 8, [64 * 50 + 63], 8, 0, 0),
    (17, 1, [64 * 20], 5, 2, 3), (3, 3, [64 * 33 + 1, 64], 2, 1, 1), (2, 1, [64 * 300 + 2], 40, 1, 2)])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_sparse(cuda, Hq, H, lens, blocks, sink, recent, dtype):
    B, n = len(lens), max(lens)
    k, v = _kv(cuda, B, H, n, seed=n + Hq, dtype=dtype)
    store = _store(B, H, n, device=cuda)
    store.update(k, v, _ints(cuda, [0] * B), _ints(cuda, lens))
    q = (torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(3)) * 1.5).to(dtype).to(cuda)
    out, index = store.sparse_decode_attention(q, _ints(cuda, lens), blocks, sink, recent)
    refs, q16 = _refs(k, v, lens), query(q.cpu())
    G = Hq // H
    tokens = []
    for b in range(B):
        tokens.append([])
        for h in range(H):
            pick = choose(refs[b][h], q16[b, h * G:(h + 1) * G], blocks, sink, recent)
            assert index[b, h].tolist() == pick + [-1] * (blocks - len(pick)), (b, h)
            tail = list(range(lens[b] // BLOCK * BLOCK, lens[b]))
            tokens[b].append([BLOCK * j + i for j in pick for i in range(BLOCK)] + tail)
    _check_attn(out.unsqueeze(2), refs, q.unsqueeze(2), lens, None, tokens=tokens)


@pytest.mark.parametrize("Hq,H", [(71, 1), (130, 2), (400, 1)])
def test_block_list_with_many_heads(cuda, Hq, H):
    """More query heads than the few-row kernel has columns, over a list of blocks: still only those blocks."""
    n, blocks = 64 * 20 + 3, 4
    k, v = _kv(cuda, 2, H, n, seed=Hq)
    lens = [n, 64 * 9]
    store = _store(2, H, n, device=cuda)
    store.update(k, v, _ints(cuda, [0, 0]), _ints(cuda, lens))
    q = torch.randn(2, Hq, D, generator=torch.Generator().manual_seed(4)).half().to(cuda)
    out, index = store.sparse_decode_attention(q, _ints(cuda, lens), blocks)
    refs, q16 = _refs(k, v, lens), query(q.cpu())
    picks = [[choose(refs[b][h], q16[b, h * Hq // H:(h + 1) * Hq // H], blocks, 1, 1) for h in range(H)]
             for b in range(2)]
    assert index.tolist() == picks
    tokens = [[[64 * j + i for j in p for i in range(64)] + list(range(lens[b] // 64 * 64, lens[b])) for p in picks[b]]
              for b in range(2)]
    _check_attn(out.unsqueeze(2), refs, q.unsqueeze(2), lens, None, tokens=tokens)
    assert torch.equal(store.decode_attention(q, _ints(cuda, lens), index=index), out)


def test_sequence_taken_back(cuda):
    """Tokens dropped again: within the unfinished block, to a multiple of 64, and inside a finished block through read."""
    n = 64 * 5 + 30
    k, v = _kv(cuda, 3, 2, n, seed=21)
    k2, v2 = _kv(cuda, 3, 2, 200, seed=22)
    store = _store(3, 2, n + 300, device=cuda)
    store.update(k, v, _ints(cuda, [0, 0, 0]))
    back = [64 * 5 + 7, 64 * 5, 64 * 2]
    store.update(k2, v2, _ints(cuda, back))
    fk = torch.cat([torch.cat([k[b:b + 1, :, :m], k2[b:b + 1], k[b:b + 1, :, :back[0] - m]], 2) for b, m in enumerate(back)])
    fv = torch.cat([torch.cat([v[b:b + 1, :, :m], v2[b:b + 1], v[b:b + 1, :, :back[0] - m]], 2) for b, m in enumerate(back)])
    lens = [m + 200 for m in back]
    _check_store(store, _refs(fk, fv, lens), fk, fv, lens)
    # 10 tokens of every sequence's third block stay
    kr, vr = store.read(_ints(cuda, lens), 64 * 2 + 10, 64 * 2)
    store.update(kr, vr, _ints(cuda, [64 * 2] * 3))
    gk, gv = store.read(_ints(cuda, [64 * 2 + 10] * 3), 64 * 2 + 10, 64 * 2)
    assert torch.equal(gk, kr) and torch.equal(gv, vr)
    q = torch.randn(3, 4, D, generator=torch.Generator().manual_seed(4)).half().to(cuda)
    fk, fv = (torch.cat([f[:, :, :64 * 2], r], 2) for f, r in ((fk, kr), (fv, vr)))
    out = store.decode_attention(q, _ints(cuda, [64 * 2 + 10] * 3))
    _check_attn(out.unsqueeze(2), _refs(fk, fv, [64 * 2 + 10] * 3), q.unsqueeze(2), [64 * 2 + 10] * 3, None)


def test_sparse_ties_take_the_lower_index(cuda):
    """Equal blocks: the lowest of them."""
    B, H, nb = 1, 2, 700
    k, v = _kv(cuda, B, H, 64, seed=1)
    k, v = k.repeat(1, 1, nb, 1), v.repeat(1, 1, nb, 1)
    store = _store(B, H, 64 * nb, device=cuda)
    store.update(k, v, _ints(cuda, [0]))
    q = torch.randn(1, 4, D, generator=torch.Generator().manual_seed(2)).half().to(cuda)
    index = store.select_blocks(q, _ints(cuda, [64 * nb]), 300, 0, 0)
    assert (index.cpu() == torch.arange(300)).all()
    index = store.select_blocks(q, _ints(cuda, [64 * nb]), 300, 2, 5)
    assert (index.cpu() == torch.cat([torch.arange(295), torch.arange(695, 700)])).all()
    index = store.select_blocks(torch.zeros_like(q), _ints(cuda, [64 * nb]), 300, 0, 1)  # every score 0
    assert (index.cpu() == torch.cat([torch.arange(299), torch.arange(699, 700)])).all()


@pytest.mark.parametrize("nb,n", [(1024, 9), (1025, 40), (1600, 700), (2047, 3), (2048, 500), (2049, 500), (9001, 500)])
@pytest.mark.parametrize("tied", [False, True])
def test_sparse_many_blocks(cuda, nb, n, tied):
    """More blocks than one round's, than the selection keeps in registers and in LDS, against a stable sort of the same
    scores."""
    store = _store(1, 1, 64 * nb, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    k = torch.randn(1, 1, 64 * nb, D, generator=g, device=cuda).half()
    if tied:
        k = k[:, :, :64 * 13].repeat(1, 1, nb // 13 + 1, 1)[:, :, :64 * nb].contiguous()
    store.update(k, k, _ints(cuda, [0]))
    q = torch.randn(1, 2, D, generator=g, device=cuda).half()
    index = store.select_blocks(q, _ints(cuda, [64 * nb]), n, 1, 1)
    lo, hi = store.ranges[0, 0, :, 0].double(), store.ranges[0, 0, :, 1].double()
    best = None
    for row in q[0].float():
        a = row.abs().max()
        q8 = torch.round(row * factor(a)).double()
        sc = torch.maximum(q8 * lo, q8 * hi).sum(1).float() * (a * STEP.to(cuda))
        best = sc if best is None else torch.maximum(best, sc)
    score = best * store.scales[0, 0, :, 0]
    score[0] = score[-1] = float("inf")
    want = torch.sort(score, descending=True, stable=True).indices[:n].sort().values
    assert torch.equal(index[0, 0].long(), want)


def test_all_blocks_equal_dense(cuda):
    """A list of every block gives the dense attention's numbers (the same work in the same order)."""
    lens = [64 * 9 + 20, 64 * 4]
    k, v = _kv(cuda, 2, 2, max(lens), seed=3)
    store = _store(2, 2, max(lens), device=cuda)
    store.update(k, v, _ints(cuda, [0, 0]), _ints(cuda, lens))
    q = torch.randn(2, 8, D, generator=torch.Generator().manual_seed(2)).half().to(cuda)
    out, index = store.sparse_decode_attention(q, _ints(cuda, lens), 10)
    assert index[0, 0].tolist() == list(range(9)) + [-1] and index[1, 0].tolist() == list(range(4)) + [-1] * 6
    dense = store.decode_attention(q, _ints(cuda, lens))
    assert (out.float() - dense.float()).abs().max() <= 2.0 ** -9 * dense.float().abs().max()


def test_given_blocks(cuda):
    """Attention over a list of blocks of the caller's: any order, entries that are no finished block skipped."""
    n = 64 * 20 + 11
    k, v = _kv(cuda, 2, 2, n, seed=12)
    lens = [n, 64 * 6]
    store = _store(2, 2, n, device=cuda)
    store.update(k, v, _ints(cuda, [0, 0]), _ints(cuda, lens))
    q = torch.randn(2, 6, D, generator=torch.Generator().manual_seed(2)).half().to(cuda)
    lists = [[[3, -1, 19, 0, 20, 7], [5, 4, 3, 2, 1, 1 << 30]], [[-1] * 6, [5, 6, -7, 0, 19, 2]]]
    index = torch.tensor(lists, dtype=torch.int32, device=cuda)
    out = store.decode_attention(q, _ints(cuda, lens), index=index)
    tokens = [[[64 * j + i for j in lists[b][h] if 0 <= j < lens[b] // 64 for i in range(64)]
               + list(range(lens[b] // 64 * 64, lens[b])) for h in range(2)] for b in range(2)]
    _check_attn(out.unsqueeze(2), _refs(k, v, lens), q.unsqueeze(2), lens, None, tokens=tokens)


@pytest.mark.parametrize("bound", [None, 64 * 1000])
@pytest.mark.parametrize("nb", [2, 3, 5, 63, 64, 65, 127, 128, 129, 130, 255, 256, 257, 300, 511, 513])
def test_select_counts(cuda, nb, bound):
    """Every way to choose, around the numbers of blocks where it changes; blocks that repeat, so that scores tie."""
    B, H = 2, 2
    store = _store(B, H, 64 * 1000, device=cuda)
    k, _ = _kv(cuda, B, H, 64 * 7, seed=nb)
    order = torch.randint(0, 7, (nb,), generator=torch.Generator().manual_seed(nb)).tolist()
    k = torch.cat([k[:, :, 64 * j:64 * j + 64] for j in order], 2)
    lens = [64 * nb, 64 * (nb - 1) + 63]
    store.update(k, k, _ints(cuda, [0] * B), _ints(cuda, lens))
    q = torch.randn(B, 4, D, generator=torch.Generator().manual_seed(2)).half().to(cuda)
    refs = _refs(k, k, lens)
    for blocks, sink, recent in ((1, 0, 0), (2, 1, 1), (nb // 2 + 1, 2 if nb > 4 else 0, 0), (nb, 0, 1), (max(nb - 1, 1), 0, 0)):
        index = store.select_blocks(q, _ints(cuda, lens), blocks, sink, recent, max_len=bound)
        for b in range(B):
            for h in range(H):
                want = choose(refs[b][h], query(q[b, 2 * h:2 * h + 2].cpu()), blocks, sink, recent)
                assert index[b, h].tolist() == want + [-1] * (blocks - len(want)), (blocks, b, h)


@pytest.mark.parametrize("sink,recent,blocks", [(3, 4, 7), (0, 0, 1), (5, 0, 5), (0, 6, 6), (2, 2, 60)])
def test_select_forced_blocks(cuda, sink, recent, blocks):
    """No place left for the others, no forced block, as many places as blocks."""
    nb = 60
    k, v = _kv(cuda, 1, 1, 64 * nb, seed=5)
    store = _store(1, 1, 64 * nb, device=cuda)
    store.update(k, v, _ints(cuda, [0]))
    q = torch.randn(1, 3, D, generator=torch.Generator().manual_seed(2)).half().to(cuda)
    index = store.select_blocks(q, _ints(cuda, [64 * nb]), blocks, sink, recent)
    want = choose(_refs(k, v, [64 * nb])[0][0], query(q[0].cpu()), blocks, sink, recent)
    assert index[0, 0].tolist() == want


def test_other_stream_and_graph(cuda):
    """A decode step (update, both attentions) captured once and replayed at other lengths, with eager work between, each
    replay against the eager result; the same on a second stream."""
    B, H, Hq, n = 2, 2, 8, 300
    k, v = _kv(cuda, B, H, n, seed=11)
    eager, graphed = _store(B, H, 512, device=cuda), _store(B, H, 512, device=cuda)
    lens = [100, 61]
    for s in (eager, graphed):
        s.update(k[:, :, :100], v[:, :, :100], _ints(cuda, [0, 0]), _ints(cuda, lens))
    pos, after = _ints(cuda, lens), _ints(cuda, lens) + 1
    kn, vn = k[:, :, :1].contiguous(), v[:, :, :1].contiguous()
    q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(2)).half().to(cuda)

    def step(s, p, a):
        s.update(kn, vn, p)
        return (s.decode_attention(q, a), *s.sparse_decode_attention(q, a, 3),
                s.prefill_attention(q.unsqueeze(2).expand(-1, -1, 40, -1), a))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            outs = step(graphed, pos, after)
    torch.cuda.current_stream().wait_stream(side)
    for i in range(70):
        kn.copy_(k[:, :, 100 + i:101 + i])
        vn.copy_(v[:, :, 100 + i:101 + i])
        graph.replay()
        want = step(eager, pos, after)
        for a, b in zip(outs, want):
            assert torch.equal(a, b), i
        if i % 10 == 0:
            torch.cuda.synchronize()
        pos.add_(1)
        after.add_(1)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = eager.decode_attention(q, after)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, eager.decode_attention(q, after))


def test_two_graphs_and_threads_at_once(cuda):
    """Calls in flight together (two graphs on two streams, two threads on two more) share no workspace."""
    import threading

    n = 64 * 200 + 9
    k, v = _kv(cuda, 1, 2, n, seed=31)
    store = _store(1, 2, n, device=cuda)
    store.update(k, v, _ints(cuda, [0]))
    lens = _ints(cuda, [n])
    qs = [torch.randn(1, 8, D, generator=torch.Generator().manual_seed(i)).half().to(cuda) for i in range(4)]

    def step(q):
        return (store.decode_attention(q, lens), *store.sparse_decode_attention(q, lens, 40),
                store.prefill_attention(q.unsqueeze(2).expand(-1, -1, 70, -1), lens))

    want = [step(q) for q in qs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(4)], [], []
    for q, s in zip(qs[:2], streams):
        g = torch.cuda.CUDAGraph()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
            outs.append(step(q))
        graphs.append(g)
    torch.cuda.synchronize()
    got = {}

    def work(i):
        with torch.cuda.stream(streams[i]):
            got[i] = [step(qs[i]) for _ in range(30)]

    threads = [threading.Thread(target=work, args=(i,)) for i in (2, 3)]
    for t in threads:
        t.start()
    for _ in range(30):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
    for i in (2, 3):
        assert len(got[i]) == 30 and all(torch.equal(a, b) for r in got[i] for a, b in zip(r, want[i]))


def test_deepcopy_is_a_store_of_its_own(cuda):
    import copy

    k, v = _kv(cuda, 2, 2, 200, seed=7)
    store = _store(2, 2, 300, device=cuda)
    store.update(k[:, :, :100], v[:, :, :100], _ints(cuda, [0, 0]))
    other = copy.deepcopy(store)
    store.update(k[:, :, 100:], v[:, :, 100:], _ints(cuda, [100, 100]))
    other.update(k[:, :, :70], v[:, :, :70], _ints(cuda, [100, 100]))
    _check_store(store, _refs(k, v, [200, 200]), k, v, [200, 200])
    ok, ov = torch.cat([k[:, :, :100], k[:, :, :70]], 2), torch.cat([v[:, :, :100], v[:, :, :70]], 2)
    _check_store(other, _refs(ok, ov, [170, 170]), ok, ov, [170, 170])


def test_offsets_past_32_bits(cuda):
    """A store whose codes pass 2^32 bytes: tokens at its end."""
    B, H, cap = 5, 8, 64 * 16400  # 5 x 8 x 16400 blocks x 8192 bytes: 5.4e9
    store = _store(B, H, cap, device=cuda)
    k, v = _kv(cuda, B, H, 100, seed=7)
    pos = cap - 100 - 28
    store.scales[:, :, :pos // BLOCK] = 0  # (older tokens: zeros)
    store.k_codes.fill_(128)
    store.v_codes.fill_(128)
    store.update(k, v, _ints(cuda, [pos] * B))
    lens = _ints(cuda, [pos + 100] * B)
    kk, vv = store.read(lens, pos + 100, pos)
    first = -pos % BLOCK
    assert torch.equal(kk[-1, -1, -36:], k[-1, -1, -36:]) and torch.equal(vv[-1, -1, -36:], v[-1, -1, -36:])
    r = Ref(k[-1, -1, first:].cpu(), v[-1, -1, first:].cpu())
    assert torch.equal(store.k_codes[-1, -1, -2].cpu().long() - 128, r.codes["k"][0])
    q = torch.randn(B, H, D, generator=torch.Generator().manual_seed(2)).half().to(cuda) * 30
    out = store.decode_attention(q, lens)
    # the zero keys have score 0 and value 0: the same attention over the last blocks plus that many zero tokens
    got = out[-1, -1].double().cpu()
    kd, vd = (t[-1, -1].double().cpu() for t in (kk, vv))
    s = (kd @ query(q[-1, -1].cpu()).double()) * SCALE
    m = max(s.max().item(), 0.0)
    den = torch.exp(s - m).sum() + pos * torch.exp(torch.tensor(-m, dtype=torch.float64))
    want = (torch.exp(s - m) @ vd) / den
    assert (got - want).abs().max() <= 2.0 ** -9 * vd.abs().max()


def test_refusals(cuda):
    from leankv_amd._lib import LeanKVError

    store = _store(2, 2, 128, device=cuda)
    k, v = _kv(cuda, 2, 2, 3, seed=1)
    lens = _ints(cuda, [3, 3])
    q = torch.randn(2, 4, D, device=cuda, dtype=F16)
    bad = [
        lambda: store.update(k[:1], v[:1], lens), lambda: store.update(k, v[:, :, :2], lens),
        lambda: store.update(k, v.float(), lens), lambda: store.update(k.long(), v.long(), lens),
        lambda: store.update(k.cpu(), v.cpu(), lens), lambda: store.update(k, v, lens.long()),
        lambda: store.update(k, v, lens[:1]), lambda: store.update(k, v, lens.cpu()),
        lambda: store.update(k, v, lens, _ints(cuda, [1, 2, 3])), lambda: store.update(k[..., :64], v[..., :64], lens),
        lambda: store.read(lens, 129), lambda: store.read(lens, 3, 4), lambda: store.read(lens, 3, -1),
        lambda: store.decode_attention(q[:, :3], lens), lambda: store.decode_attention(q.unsqueeze(2), lens),
        lambda: store.decode_attention(q.double(), lens), lambda: store.decode_attention(q, lens, max_len=129),
        lambda: store.decode_attention(q, lens, out=torch.empty(2, 4, D, device=cuda)),
        lambda: store.decode_attention(q, lens, out=torch.empty(2, 4, 2 * D, device=cuda, dtype=F16)[..., ::2]),
        lambda: store.prefill_attention(q, lens), lambda: store.prefill_attention(q.unsqueeze(2), lens, lens[:1]),
        lambda: store.decode_attention(q, lens, index=torch.zeros(2, 2, 1, device=cuda)),
        lambda: store.decode_attention(q, lens, index=torch.zeros(2, 2, 0, device=cuda, dtype=torch.int32)),
        lambda: store.select_blocks(q, lens, 0), lambda: store.select_blocks(q, lens, 2, 2, 1),
        lambda: store.select_blocks(q, lens, 2, -1, 1), lambda: store.sparse_decode_attention(q, lens, 1),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(LeanKVError):
            f()
            print("not refused:", i)
    # nothing to do
    store.update(k[:, :, :0], v[:, :, :0], lens)
    assert store.prefill_attention(q.unsqueeze(2)[:, :, :0], lens).shape == (2, 4, 0, D)
    assert store.read(lens, 0)[0].shape == (2, 2, 0, D)
