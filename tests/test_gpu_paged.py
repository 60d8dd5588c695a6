"""The 16-bit paged cache on the GPU: tables against a model in Python lists, attention against 64 bits with the bound that its
roundings give, and a run of all of it as a serving loop makes it."""

import math
import random

import pytest
import torch

from paged_ref import D, Tables, attention, check, packed

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lens, first=0):
    at = [first]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _rows(gen, n, heads, dtype, spread=1.0):
    x = torch.randn(n, heads, D, generator=gen)
    x[..., ::37] *= 3
    return (spread * x).to(dtype)


def _cache(gen, lens, kv, page, dtype, layers=1, spare=3, order=True, room=0):
    """A cache of sequences whose pages lie in no order, and its (k, v) rows per layer and sequence on the host.  What lies
    behind a sequence, and in free pages, is NaN."""
    from leankv_amd.paged import PagedKV

    width = max(1, -(-(max(lens) + room) // page))
    need = sum(-(-n // page) for n in lens)
    cache = PagedKV(layers, kv, need + spare, len(lens), width * page, page_size=page, dtype=dtype)
    ids = torch.randperm(need + spare, generator=gen).tolist() if order else list(range(need + spare))
    rows, at = [], 0
    for n in lens:
        m = -(-n // page)
        rows.append(ids[at:at + m])
        at += m
    pool = torch.full(cache.pool.shape, math.nan, dtype=dtype)
    held = []
    for layer in range(layers):
        held.append([])
        for s, n in enumerate(lens):
            k, v = _rows(gen, n, kv, dtype), _rows(gen, n, kv, dtype)
            held[-1].append((k, v))
            for j, p in enumerate(rows[s]):
                part = slice(j * page, min((j + 1) * page, n))
                m = part.stop - part.start
                pool[layer, p, 0, :, :m] = k[part].transpose(0, 1)
                pool[layer, p, 1, :, :m] = v[part].transpose(0, 1)
    cache.pool.copy_(pool)
    _set(cache, rows, lens)
    return cache, rows, held


def _set(cache, rows, lens):
    table = torch.full(cache.table.shape, -1, dtype=torch.int32)
    refs = torch.zeros(cache.num_pages, dtype=torch.int32)
    for s, row in enumerate(rows):
        table[s, :len(row)] = torch.tensor(row, dtype=torch.int32)
        for p in row:
            refs[p] += 1
    cache.table.copy_(table)
    cache.refs.copy_(refs)
    cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))


# -------------------------------------------------------------------------------------------------- packed prompts
LENS = [[1], [64], [65], [1, 0, 63, 64, 127], [257, 3, 0, 130], [40] * 20]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("heads,kv,dtype", [(4, 1, F16), (8, 8, BF16), (6, 1, BF16), (14, 2, F16), (16, 2, BF16), (20, 1, F16)])
def test_packed(cuda, lens, heads, kv, dtype):
    from leankv_amd.paged import packed_attention

    gen = torch.Generator().manual_seed(sum(lens) * 31 + heads)
    T = sum(lens)
    q, k, v = _rows(gen, T, heads, dtype, 1.3), _rows(gen, T, kv, dtype), _rows(gen, T, kv, dtype)
    at = _starts(lens)
    want, bound = packed(q, k, v, at)
    check(packed_attention(q.cuda(), k.cuda(), v.cuda(), _ints(at)), want, bound)
    got = packed_attention(q.cuda(), k.cuda(), v.cuda(), _ints(at), max_len=max(lens))
    check(got, want, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n,heads,kv", [(3000, 4, 1), (1500, 8, 8), (1111, 7, 1)])
def test_packed_long(cuda, n, heads, kv, dtype):
    """Few column tiles: their tokens are split and joined."""
    from leankv_amd.paged import packed_attention

    gen = torch.Generator().manual_seed(n)
    lens = [n, 70]
    q, k, v = (_rows(gen, sum(lens), h, dtype) for h in (heads, kv, kv))
    at = _starts(lens)
    want, bound = packed(q, k, v, at, scale=0.11)
    check(packed_attention(q.cuda(), k.cuda(), v.cuda(), _ints(at), scale=0.11), want, bound)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_packed_strides_and_rows_of_no_sequence(cuda, dtype):
    """q, k and v as slices of one projection, rows before the first sequence and behind the last."""
    from leankv_amd.paged import packed_attention

    gen = torch.Generator().manual_seed(5)
    lens, heads, kv = [70, 0, 129], 8, 2
    at = _starts(lens, first=3)
    T = at[-1] + 5
    x = _rows(gen, T, heads + 2 * kv, dtype)
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    want, bound = packed(q, k, v, at)
    y = x.cuda()
    parts = y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:]
    got = packed_attention(*parts, _ints(at))
    check(got, want, bound)
    assert not got[:3].any() and not got[at[-1]:].any()
    out = torch.full((heads, T, D), 7.0, dtype=dtype, device="cuda").transpose(0, 1)
    assert packed_attention(*parts, _ints(at), out=out) is out
    assert (out[:3] == 7).all() and (out[at[-1]:] == 7).all()
    assert torch.equal(out[3:at[-1]], got[3:at[-1]])
    # rows that are not aligned, heads before tokens, dims that are not dense: copied
    odd = torch.empty(T, heads, D + 1, dtype=dtype, device="cuda")[..., 1:].copy_(parts[0])
    k2 = parts[1].transpose(0, 1).contiguous().transpose(0, 1)
    v2 = parts[2].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(packed_attention(odd, k2, v2, _ints(at)), got)
    # in place of the queries
    z = y.clone()
    packed_attention(z[:, :heads], z[:, heads:heads + kv], z[:, heads + kv:], _ints(at), out=z[:, :heads])
    assert torch.equal(z[3:at[-1], :heads], got[3:at[-1]]) and torch.equal(z[:, heads:], y[:, heads:])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_packed_values_that_are_no_numbers(cuda, dtype):
    """A query's row is that of the tokens that it sees, whatever later ones hold."""
    from leankv_amd.paged import packed_attention

    gen = torch.Generator().manual_seed(6)
    lens, heads, kv = [200, 90], 4, 2
    at = _starts(lens)
    q, k, v = (_rows(gen, sum(lens), h, dtype) for h in (heads, kv, kv))
    want, bound = packed(q, k, v, at)
    v2, k2, q2 = v.clone(), k.clone(), q.clone()
    v2[100, 0, 5], v2[150, 0, 5], v2[120, 0, 9], v2[180, 1, 7] = math.inf, -math.inf, -math.inf, math.nan
    k2[290 - 10, 0, 3] = math.nan     # sequence 1, its token 80
    q2[200 + 40, 1, 0] = math.nan     # a query of sequence 1
    got = packed_attention(q2.cuda(), k2.cuda(), v2.cuda(), _ints(at)).cpu().double()
    mask = torch.zeros(got.shape, dtype=torch.bool)
    mask[100:200, :2, 5] = True
    mask[120:200, :2, 9] = True
    mask[180:200, 2:, 7] = True
    mask[280:290, :2] = True
    mask[240, 1] = True
    check(torch.where(mask, want, got), want, bound)
    assert (got[100:150, :2, 5] == math.inf).all() and got[150:200, :2, 5].isnan().all()
    assert (got[120:200, :2, 9] == -math.inf).all() and got[180:200, 2:, 7].isnan().all()
    assert got[280:290, :2].isnan().all() and got[240, 1].isnan().all()


def test_packed_large_scores(cuda):
    """Scores of thousands, rising and falling: the running offset follows."""
    from leankv_amd.paged import packed_attention

    gen = torch.Generator().manual_seed(7)
    n = 300
    for dtype in (F16, BF16):
        q, k, v = _rows(gen, n, 2, dtype), _rows(gen, n, 1, dtype), _rows(gen, n, 1, dtype)
        k = (k.float() * torch.linspace(0.1, 30, n).view(n, 1, 1)).to(dtype)
        want, bound = packed(q, k, v, [0, n])
        check(packed_attention(q.cuda(), k.cuda(), v.cuda(), _ints([0, n])), want, bound)


@pytest.mark.parametrize("max_len", [100, 300])
def test_packed_many_sequences(cuda, max_len):
    """More pieces a workgroup than are found at once: 2000 sequences alike give 2000 results alike."""
    from leankv_amd.paged import packed_attention

    gen = torch.Generator().manual_seed(31)
    n, B, heads = 100, 2000, 32
    q, k, v = _rows(gen, n, heads, F16), _rows(gen, n, 1, F16), _rows(gen, n, 1, F16)
    want, bound = packed(q, k, v, [0, n])
    at = torch.arange(0, n * B + 1, n, dtype=torch.int32, device="cuda")
    got = packed_attention(*(t.cuda().repeat(B, 1, 1) for t in (q, k, v)), at, max_len=max_len).view(B, n, heads, D)
    check(got[0], want, bound)
    assert bool((got == got[0]).all())


def test_packed_most_sequences(cuda):
    """Sequences of none to three tokens, as many as there may be; their stored rows in pages."""
    from leankv_amd.paged import PagedKV, packed_attention

    rng = random.Random(5)
    lens = [rng.randint(0, 3) for _ in range(2048)]
    gen = torch.Generator().manual_seed(32)
    at = _starts(lens)
    q, k, v = (_rows(gen, at[-1], h, BF16) for h in (2, 1, 1))
    want, bound = packed(q, k, v, at)
    check(packed_attention(q.cuda(), k.cuda(), v.cuda(), _ints(at), max_len=3), want, bound)
    cache = PagedKV(1, 1, 2100, 2048, 16, page_size=16, dtype=BF16)
    cache.extend(_ints(at))
    cache.store(0, k.cuda(), v.cuda(), _ints(at))
    kk, vv = cache.read(0, 3)
    for s in range(0, 2048, 7):
        assert torch.equal(kk[s, 0, :lens[s]].cpu(), k[at[s]:at[s + 1], 0]) and not kk[s, 0, lens[s]:].any()
        assert torch.equal(vv[s, 0, :lens[s]].cpu(), v[at[s]:at[s + 1], 0])
    check(cache.prefill_attention(0, q.cuda(), _ints(at), max_new=3), want, bound)
    q1 = _rows(gen, 2048, 2, BF16)
    some = [s for s in range(2048) if lens[s]][:300]
    got = cache.decode_attention(0, q1.cuda()).cpu()
    for s in some:
        for h in range(2):
            w, b = attention(q1[s, h:h + 1], k[at[s]:at[s + 1], 0], v[at[s]:at[s + 1], 0], torch.tensor([lens[s]]))
            check(got[s, h:h + 1], w, b)
    assert not got[[s for s in range(2048) if not lens[s]]].any()


# -------------------------------------------------------------------------------------------------- over pages
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("heads,kv,dtype", [(8, 2, F16), (7, 1, BF16)])
def test_prefill(cuda, page, heads, kv, dtype):
    gen = torch.Generator().manual_seed(page + heads)
    lens, new = [300, 64, 0, 17, 129], [70, 64, 2, 30, 1]  # (more rows than tokens: zeros)
    cache, _, held = _cache(gen, lens, kv, page, dtype, layers=2)
    at = _starts(new, first=1)
    q = _rows(gen, at[-1] + 2, heads, dtype)
    want, bound = packed(q, None, None, at, paged=lambda b: held[1][b])
    got = cache.prefill_attention(1, q.cuda(), _ints(at))
    check(got, want, bound)
    assert not got[0].any() and not got[at[-1]:].any()
    check(cache.prefill_attention(1, q.cuda(), _ints(at), max_new=70, max_len=300), want, bound)
    out = torch.full_like(got, 3.0)
    cache.prefill_attention(1, q.cuda(), _ints(at), out=out)
    assert torch.equal(out[1:at[-1]], got[1:at[-1]]) and (out[0] == 3).all() and (out[at[-1]:] == 3).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("heads,kv,new", [(4, 1, [5, 3]), (8, 8, [1, 1]), (6, 2, [40, 2])])
def test_prefill_few_rows_of_long_sequences(cuda, heads, kv, new, dtype):
    gen = torch.Generator().manual_seed(heads)
    cache, _, held = _cache(gen, [2500, 700], kv, 64, dtype)
    at = _starts(new)
    q = _rows(gen, at[-1], heads, dtype)
    want, bound = packed(q, None, None, at, paged=lambda b: held[0][b])
    check(cache.prefill_attention(0, q.cuda(), _ints(at), max_new=max(new)), want, bound)


@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("heads,kv,new,dtype", [(8, 2, 5, F16), (8, 2, 8, BF16), (4, 4, 32, F16), (14, 2, 3, BF16), (32, 2, 2, F16),
                                                (12, 1, 2, BF16), (20, 1, 1, F16)])
def test_prefill_few_rows(cuda, page, heads, kv, new, dtype):
    """Up to 32 columns of a kv head; more rows than max_new says, and longer sequences than max_len, are right too."""
    gen = torch.Generator().manual_seed(page + heads + new)
    lens = [1, 2, 0, 31, 33, 64, 130, 300, 700]
    news = [1, 3, 2, new, new, 0, 1, new, new]
    cache, _, held = _cache(gen, lens, kv, page, dtype, layers=2)
    at = _starts(news, first=2)
    q = _rows(gen, at[-1] + 1, heads, dtype)
    want, bound = packed(q, None, None, at, paged=lambda b: held[1][b])
    for kw in (dict(max_new=new), dict(max_new=1, max_len=40), dict(max_new=new, max_len=700), {}):
        got = cache.prefill_attention(1, q.cuda(), _ints(at), **kw)
        check(got, want, bound, str(kw))
        assert not got[:2].any() and not got[at[-1]:].any()
    out = torch.full_like(got, 5.0)
    cache.prefill_attention(1, q.cuda(), _ints(at), max_new=new, out=out)
    assert torch.equal(out[2:at[-1]], cache.prefill_attention(1, q.cuda(), _ints(at), max_new=new)[2:at[-1]])
    assert (out[:2] == 5).all() and (out[at[-1]:] == 5).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("max_new", [6, 40])
def test_prefill_values_that_are_no_numbers(cuda, dtype, max_new):
    """A drafted token's value has no part in the rows of the tokens before it, whatever it is."""
    gen = torch.Generator().manual_seed(41)
    n, m, page = 100, 6, 16
    cache, rows, held = _cache(gen, [n], 1, page, dtype)
    q = _rows(gen, m, 4, dtype)
    want, bound = packed(q, None, None, [0, m], paged=lambda b: held[0][b])
    mask = torch.zeros(want.shape, dtype=torch.bool)
    for i, d, x in ((2, 7, math.inf), (4, 7, -math.inf), (3, 9, -math.inf), (5, 3, math.nan), (1, 100, math.nan)):
        t = n - m + i
        cache.pool[0, rows[0][t // page], 1, 0, t % page, d] = x
        mask[i:, :, d] = True
    got = cache.prefill_attention(0, q.cuda(), _ints([0, m]), max_new=max_new).cpu().double()
    check(torch.where(mask, want, got), want, bound)
    assert (got[2:4, :, 7] == math.inf).all() and got[4:, :, 7].isnan().all() and (got[3:, :, 9] == -math.inf).all()
    assert got[5, :, 3].isnan().all() and got[1:, :, 100].isnan().all()


@pytest.mark.parametrize("new", [4, 100])
def test_results_over_their_queries(cuda, new):
    """q as out, also where rows are gone through again for a value that is no number."""
    from leankv_amd.paged import packed_attention

    gen = torch.Generator().manual_seed(57)
    n, page = 700, 64
    cache, rows, _ = _cache(gen, [n, n], 2, page, F16)
    t = n - new + new // 2
    cache.pool[0, rows[0][t // page], 1, 0, t % page, 5] = math.nan
    at = _ints([0, new, 2 * new])
    q = _rows(gen, 2 * new, 8, F16).cuda()
    want = cache.prefill_attention(0, q, at, max_new=new)
    assert want[new // 2:new, :4, 5].isnan().all() and not want[:new // 2].isnan().any() and not want[new:].isnan().any()
    over = q.clone()
    assert cache.prefill_attention(0, over, at, max_new=new, out=over) is over
    assert torch.equal(over.nan_to_num(9.0), want.nan_to_num(9.0))
    k, v = _rows(gen, 2 * new, 2, F16).cuda(), _rows(gen, 2 * new, 2, F16).cuda()
    v[new // 2, 1, 7] = math.inf
    want, over = packed_attention(q, k, v, at), q.clone()
    packed_attention(over, k, v, at, out=over)
    assert torch.equal(over.nan_to_num(9.0), want.nan_to_num(9.0))
    q1 = _rows(gen, 2, 8, F16).cuda()
    want, over = cache.decode_attention(0, q1), q1.clone()
    cache.decode_attention(0, over, out=over)
    assert torch.equal(over.nan_to_num(9.0), want.nan_to_num(9.0))


@pytest.mark.parametrize("new,kv,heads", [([0, 2], 4, 132), ([300], 1, 4), ([70, 0, 64], 2, 8)])
def test_rows_of_sequences_that_hold_nothing(cuda, new, kv, heads):
    """Rows are zeros where no sequence holds a token, whichever kernel takes them."""
    gen = torch.Generator().manual_seed(59)
    cache, _, _ = _cache(gen, [0] * len(new), kv, 16, F16, room=700)
    at = _starts(new, first=1)
    q = _rows(gen, at[-1] + 1, heads, F16).cuda()
    for kw in ({}, dict(max_new=max(new)), dict(max_new=1), dict(max_new=max(new), max_len=1)):
        out = torch.full_like(q, 5.0)
        cache.prefill_attention(0, q, _ints(at), out=out, **kw)
        assert not out[1:at[-1]].any() and (out[0] == 5).all() and (out[at[-1]:] == 5).all()
        assert not cache.prefill_attention(0, q, _ints(at), **kw).any()


def test_bounds_of_nothing(cuda):
    """max_len = 0 says that every sequence is empty (decode); for prefill bounds only divide the work."""
    gen = torch.Generator().manual_seed(58)
    cache, _, _ = _cache(gen, [100, 3], 2, 16, F16)
    assert not cache.decode_attention(0, _rows(gen, 2, 8, F16).cuda(), max_len=0).any()
    q, at = _rows(gen, 43, 8, F16).cuda(), _ints([0, 40, 43])
    want = cache.prefill_attention(0, q, at)
    for kw in (dict(max_new=0), dict(max_len=0), dict(max_new=0, max_len=0), dict(max_new=1, max_len=1)):
        err = (cache.prefill_attention(0, q, at, **kw).double() - want.double()).norm() / want.double().norm()
        assert err < 2 * 2.0 ** -11 + 2 * 2.0 ** -11, kw  # both round the weights and the result to float16


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("heads,kv,dtype", [(8, 2, F16), (3, 3, BF16), (7, 1, F16), (12, 1, BF16), (40, 2, F16), (16, 1, BF16)])
def test_decode(cuda, page, heads, kv, dtype):
    gen = torch.Generator().manual_seed(page * 3 + heads)
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 200, 700]
    cache, _, held = _cache(gen, lens, kv, page, dtype, layers=2)
    q = _rows(gen, len(lens), heads, dtype)
    at = _starts([1] * len(lens))
    want, bound = packed(q, None, None, at, paged=lambda b: held[1][b])
    check(cache.decode_attention(1, q.cuda()), want, bound)
    # a bound on the lengths, queries and result of other strides
    wide = torch.zeros(heads, len(lens), 2 * D, dtype=dtype, device="cuda")
    x = wide[..., :D].transpose(0, 1).copy_(q)
    got = cache.decode_attention(1, x, max_len=700, out=x)
    assert got is x
    check(got, want, bound)
    assert not wide[..., D:].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_long(cuda, dtype):
    gen = torch.Generator().manual_seed(9)
    cache, _, held = _cache(gen, [9000], 2, 16, dtype, room=30000)
    q = _rows(gen, 1, 8, dtype)
    want, bound = packed(q, None, None, [0, 1], paged=lambda b: held[0][b])
    check(cache.decode_attention(0, q.cuda()), want, bound)
    check(cache.decode_attention(0, q.cuda(), max_len=9000), want, bound)
    short = [(k[:1000], v[:1000]) for k, v in held[0]]
    want, bound = packed(q, None, None, [0, 1], paged=lambda b: short[b])
    check(cache.decode_attention(0, q.cuda(), max_len=1000), want, bound)


@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 2), (16, 2), (3, 1), (10, 1)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decode_shared_pages(cuda, heads, kv, dtype):
    """Sequences that name the same pages: the same rows as when each has pages of its own."""
    gen = torch.Generator().manual_seed(heads)
    page, prompt = 16, 600
    tails = [0, 0, 3, 20, 20, 0, 3, 40, 20, 0, 0, 1, 0, 0, 0, 0, 0, 25]
    lens = [prompt + t for t in tails] + [0, 5]
    cache, rows, held = _cache(gen, lens, kv, page, dtype, spare=5)
    n = prompt // page
    pool = cache.pool.cpu()
    for s in range(1, len(tails)):
        if s % 7:  # (two of them keep pages of their own)
            for side in (0, 1):
                held[0][s][side][:n * page] = held[0][0][side][:n * page]
            rows[s] = rows[0][:n] + rows[s][n:]
    _set(cache, rows, lens)
    q = _rows(gen, len(lens), heads, dtype)
    want, bound = packed(q, None, None, _starts([1] * len(lens)), paged=lambda b: held[0][b])
    check(cache.decode_attention(0, q.cuda()), want, bound)
    check(cache.decode_attention(0, q.cuda(), max_len=640), want, bound)
    assert torch.equal(torch.nan_to_num(cache.pool.cpu()), torch.nan_to_num(pool))


def test_decode_values_that_are_no_numbers(cuda):
    gen = torch.Generator().manual_seed(11)
    for dtype in (F16, BF16):
        cache, rows, held = _cache(gen, [100, 33], 1, 32, dtype)
        q = _rows(gen, 2, 4, dtype)
        q[1, 2, 5] = math.nan
        at = rows[0][99 // 32], 99 % 32
        cache.pool[0, at[0], 1, 0, at[1], 4] = math.inf  # the newest token's value
        held[0][0][1][99, 0, 4] = 0
        want, bound = packed(torch.nan_to_num(q), None, None, [0, 1, 2], paged=lambda b: held[0][b])
        got = cache.decode_attention(0, q.cuda()).cpu().double()
        assert (got[0, :, 4] == math.inf).all() and got[1, 2].isnan().all()
        got[0, :, 4] = want[0, :, 4]
        got[1, 2] = want[1, 2]
        check(got, want, bound)


# -------------------------------------------------------------------------------------------------- tables
def _same(cache, model, what):
    assert torch.equal(cache.table.cpu(), model.table()), what
    assert cache.lens.tolist() == model.lens, what
    assert cache.refs.tolist() == model.refs(), what
    assert cache.taken.tolist() == model.taken, what


@pytest.mark.parametrize("page,seqs,pages,width", [(16, 1, 9, 4), (16, 12, 60, 7), (32, 5, 30, 9), (64, 3, 5000, 2000),
                                                   (16, 1500, 6000, 3)])
def test_tables_follow_the_model(cuda, page, seqs, pages, width):
    """Random calls: growing (past the free pages and past max_len too), forking, cutting, freeing, compacting.  Tokens keep
    what was stored for them through all of it."""
    from leankv_amd.paged import PagedKV

    rng = random.Random(page * seqs + pages)
    layers, kv = 2, 1
    cache = PagedKV(layers, kv, pages, seqs, width * page, page_size=page, dtype=F16)
    model = Tables(pages, seqs, width, page)
    tokens = [[] for _ in range(seqs)]  # what every token is, in each sequence
    count = 0
    small = seqs <= 12 and width < 100
    for step in range(60 if small else 12):
        what = rng.choice(("extend", "extend", "one", "fork", "cut", "free", "compact"))
        if step == 0:
            what = "extend"
        if what in ("extend", "one"):
            if what == "one":
                new, cu = [1 if n else 0 for n in model.lens], None
            else:
                top = rng.choice((1, page, 2 * page, width * page))
                new = [rng.choice((0, rng.randint(0, top))) for _ in range(seqs)]
                cu = _ints(_starts(new))
            cache.extend(cu)
            model.extend(new)
            total = seqs if cu is None else sum(new)
            x = torch.zeros(total, dtype=torch.float32)
            for s in range(seqs):
                a = s if cu is None else sum(new[:s]) if small else None
                if a is None:
                    break
                for i in range(model.taken[s]):
                    count = count % 2000 + 1
                    x[a + i] = count
                    tokens[s].append(count)
            if small and total:
                for layer in range(layers):
                    k = (x + 0.5 * layer).view(-1, 1, 1).expand(-1, kv, D).half().cuda()
                    cache.store(layer, k, -k, cu)
        elif what == "fork":
            parent = [rng.randint(-1, seqs - 1) for _ in range(seqs)]
            cache.fork(_ints(parent))
            model.fork(parent)
            tokens = [list(tokens[p]) if p >= 0 else [] for p in parent]
        elif what == "cut":
            cut = [rng.randint(-1, width * page) for _ in range(seqs)]
            cache.truncate(_ints(cut))
            model.fork(None, cut)
            tokens = [t[:max(c, 0)] for t, c in zip(tokens, cut)]
        elif what == "free":
            which = [s for s in range(seqs) if rng.random() < 0.3]
            if rng.random() < 0.5:
                cache.free(which)
            else:
                mask = torch.zeros(seqs, dtype=torch.bool)
                mask[which] = True
                cache.free(mask.cuda())
            model.fork([-1 if s in which else s for s in range(seqs)])
            for s in which:
                tokens[s] = []
        else:
            taken = model.taken
            assert cache.compact().tolist() == [model.compact()]
            assert model.taken == taken
        _same(cache, model, "%s in step %d" % (what, step))
        if small:
            longest = max(model.lens)
            for layer in range(layers):
                k, v = cache.read(layer, longest)
                want = torch.zeros(seqs, longest)
                for s, t in enumerate(tokens):
                    want[s, :len(t)] = torch.tensor([x + 0.5 * layer for x in t])
                want = want.half().view(seqs, 1, longest, 1).expand(-1, kv, -1, D)
                assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), -want), "%s in step %d" % (what, step)


def test_extend_copies_only_what_others_need(cuda):
    """Of sequences on one page that is not full, the first keeps it where all of them grow; copies hold its tokens."""
    from leankv_amd.paged import PagedKV

    cache = PagedKV(3, 2, 12, 4, 64, page_size=16, dtype=BF16)
    cache.extend(_ints([0, 20, 20, 20, 20]))
    gen = torch.Generator().manual_seed(1)
    k = [_rows(gen, 20, 2, BF16).cuda() for _ in range(3)]
    for layer in range(3):
        cache.store(layer, k[layer], -k[layer], _ints([0, 20, 20, 20, 20]))
    cache.fork(_ints([0, 0, 0, -1]))
    assert cache.refs.tolist()[:2] == [3, 3]
    before = cache.snapshot()
    cache.extend()
    assert cache.table.tolist()[:3] == [[0, 1, -1, -1], [0, 2, -1, -1], [0, 3, -1, -1]]
    assert cache.refs.tolist()[:4] == [3, 1, 1, 1] and cache.lens.tolist() == [21, 21, 21, 0]
    for layer in range(3):
        kk, vv = cache.read(layer, 20)
        for s in range(3):
            assert torch.equal(kk[s].transpose(0, 1), k[layer]) and torch.equal(vv[s], -kk[s])
    cache.rollback(before)
    assert cache.lens.tolist() == [20, 20, 20, 0]
    cache.extend(_ints([0, 1, 2, 2, 2]))  # the third waits: the first two take copies
    assert cache.table.tolist()[:3] == [[0, 2, -1, -1], [0, 3, -1, -1], [0, 1, -1, -1]]


def test_extend_without_room(cuda):
    """The first sequence that does not fit and all behind it that need pages take nothing; others grow."""
    from leankv_amd.paged import PagedKV

    cache = PagedKV(1, 1, 4, 4, 64, page_size=16, dtype=F16)
    cache.extend(_ints([0, 16, 26, 26, 26]))
    assert cache.taken.tolist() == [16, 10, 0, 0]
    cache.extend(_ints([0, 40, 43, 50, 50]))  # 3 pages, none, 1 page
    assert cache.taken.tolist() == [0, 3, 0, 0] and cache.lens.tolist() == [16, 13, 0, 0]
    cache.extend(_ints([0, 32, 33, 34, 34]))
    assert cache.taken.tolist() == [32, 1, 0, 0] and cache.refs.tolist() == [1, 1, 1, 1]
    before = cache.pool.clone()
    cache.store(0, torch.ones(34, 1, D, dtype=F16, device="cuda"), torch.ones(34, 1, D, dtype=F16, device="cuda"),
                _ints([0, 32, 33, 34, 34]))
    assert int((cache.pool != before).any(-1).sum()) == 2 * 33
    cache.extend(_ints([0, 17, 17, 17, 17]))  # past max_len
    assert cache.taken.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_store_strides(cuda, dtype):
    from leankv_amd.paged import PagedKV

    gen = torch.Generator().manual_seed(3)
    kv, lens = 3, [40, 0, 25]
    cache = PagedKV(2, kv, 10, 3, 64, page_size=16, dtype=dtype)
    at = _starts(lens, first=2)
    x = _rows(gen, at[-1] + 4, 2 * kv, dtype).cuda()
    cache.extend(_ints(at))
    cache.store(1, x[:, :kv], x[:, kv:], _ints(at))
    k, v = cache.read(1, 40)
    for s, n in enumerate(lens):
        assert torch.equal(k[s, :, :n].transpose(0, 1), x[at[s]:at[s] + n, :kv]) and not k[s, :, n:].any()
        assert torch.equal(v[s, :, :n].transpose(0, 1), x[at[s]:at[s] + n, kv:])
    assert not cache.pool[0].any()


def test_resized(cuda):
    from leankv_amd._lib import LeanKVError

    gen = torch.Generator().manual_seed(4)
    cache, _, held = _cache(gen, [40, 100, 7], 2, 16, F16, layers=2, spare=20)
    k, v = cache.read(1, 100)
    cache.free([1])
    with pytest.raises(LeanKVError, match="in use"):
        cache.resized(1)
    n = int(cache.compact())
    assert n == 4
    for pages in (n, 50):
        other = cache.resized(pages)
        k2, v2 = other.read(1, 100)
        assert other.num_pages == pages and torch.equal(k2[0], k[0]) and torch.equal(v2[2], v[2]) and not k2[1].any()
        assert other.refs.tolist() == [1] * n + [0] * (pages - n)


# -------------------------------------------------------------------------------------------------- as it is used
def _step(cache, x, heads, kv):
    """One token of every sequence: q, k and v from a projection."""
    cache.extend()
    outs = []
    for layer in range(cache.num_layers):
        cache.store(layer, x[layer][:, heads:heads + kv], x[layer][:, heads + kv:])
        outs.append(cache.decode_attention(layer, x[layer][:, :heads]))
    return outs


def test_serving_loop(cuda):
    """Prompts stored and attended, chunks, forked beams, steps, sequences that end, a compacted pool, drafted tokens taken
    back: every result against 64 bits of the tokens that its sequence should hold."""
    from leankv_amd.paged import PagedKV, packed_attention

    for dtype in (F16, BF16):
        gen = torch.Generator().manual_seed(21)
        layers, heads, kv, seqs, page = 2, 8, 2, 6, 16
        cache = PagedKV(layers, kv, 60, seqs, 160, page_size=page, dtype=dtype)
        held = [[(torch.zeros(0, kv, D, dtype=dtype),) * 2 for _ in range(seqs)] for _ in range(layers)]

        def add(layer, x, at):
            for s in range(seqs):
                k, v = held[layer][s]
                new = x[at[s]:at[s + 1]]
                held[layer][s] = torch.cat([k, new[:, heads:heads + kv]]), torch.cat([v, new[:, heads + kv:]])

        def forward(new, prompt=False):
            at = _starts(new)
            cache.extend(_ints(at))
            for layer in range(layers):
                x = _rows(gen, at[-1], heads + 2 * kv, dtype)
                y = x.cuda()
                add(layer, x, at)
                cache.store(layer, y[:, heads:heads + kv], y[:, heads + kv:], _ints(at))
                want, bound = packed(x[:, :heads], None, None, at, paged=lambda b: held[layer][b])
                check(cache.prefill_attention(layer, y[:, :heads], _ints(at)), want, bound)
                if prompt:
                    check(packed_attention(y[:, :heads], y[:, heads:heads + kv], y[:, heads + kv:], _ints(at)), want, bound)

        def step():
            x = [_rows(gen, seqs, heads + 2 * kv, dtype) for _ in range(layers)]
            live = [held[0][s][0].shape[0] > 0 for s in range(seqs)]
            got = _step(cache, [y.cuda() for y in x], heads, kv)
            for layer in range(layers):
                for s in range(seqs):
                    if live[s]:
                        k, v = held[layer][s]
                        held[layer][s] = (torch.cat([k, x[layer][s:s + 1, heads:heads + kv]]),
                                          torch.cat([v, x[layer][s:s + 1, heads + kv:]]))
                want, bound = packed(x[layer][:, :heads], None, None, _starts([1] * seqs), paged=lambda b: held[layer][b])
                check(got[layer], want, bound)

        def fork(parent, cut=None):
            for layer in range(layers):
                held[layer] = [tuple(t[:None if cut is None else cut[s]] for t in held[layer][p]) if p >= 0
                               else (torch.zeros(0, kv, D, dtype=dtype),) * 2 for s, p in enumerate(parent)]

        forward([37, 0, 0, 50, 0, 1], prompt=True)
        forward([20, 0, 0, 3, 0, 15])
        cache.fork(_ints([0, 0, 0, 3, 3, 5]))
        fork([0, 0, 0, 3, 3, 5])
        for _ in range(18):
            step()
        cache.fork(_ints([1, 0, 1, 4, 3, -1]))
        fork([1, 0, 1, 4, 3, -1])
        step()
        cache.free([0])
        fork([-1, 1, 2, 3, 4, 5])
        n = int(cache.compact())
        assert (cache.refs[:n] > 0).all() and not cache.refs[n:].any()
        step()
        forward([9, 4, 0, 5, 4, 30])  # a new prompt, drafted tokens of others
        cut = [t[0].shape[0] - d for t, d in zip(held[0], (0, 3, 0, 5, 1, 0))]
        cache.truncate(_ints(cut))
        fork(range(seqs), cut)
        for _ in range(3):
            step()
        cache = cache.resized(70)
        step()


def test_graph(cuda):
    """A captured step of forking, growing, storing and attending, replayed with other parents between eager work."""
    from leankv_amd.paged import PagedKV

    gen = torch.Generator().manual_seed(22)
    heads, kv, seqs = 8, 2, 8
    caches = [PagedKV(1, kv, 80, seqs, 128, page_size=16, dtype=F16) for _ in range(2)]
    x = _rows(gen, 60, 2 * kv, F16).cuda()
    at = _ints([0, 30, 60, 60, 60, 60, 60, 60, 60])
    for c in caches:
        c.extend(at)
        c.store(0, x[:, :kv], x[:, kv:], at)
        c.fork(_ints([0, 1, 0, 1, 0, 1, 0, 1]))
    parent = torch.arange(seqs, dtype=torch.int32, device="cuda")
    y = _rows(gen, seqs, heads + 2 * kv, F16).cuda()

    def step(c):
        c.fork(parent)
        return _step(c, [y], heads, kv)[0]

    chunk = _ints([0, 2, 4, 4, 5, 8, 8, 9, 9])
    rows = _rows(gen, 9, heads + 2 * kv, F16).cuda()

    def draft(c):
        c.extend(chunk)
        c.store(0, rows[:, heads:heads + kv], rows[:, heads + kv:], chunk)
        out = c.prefill_attention(0, rows[:, :heads], chunk)
        return out, c.compact()

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        before = caches[0].snapshot()
        step(caches[0])
        draft(caches[0])
        caches[0].rollback(before)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0])
        drafted, used = draft(caches[0])
    # (the warm-up's tokens lie in pages that are free again; both caches start from the same tables)
    for i in range(5):
        parent.copy_(torch.tensor([(s * (i + 1)) % seqs for s in range(seqs)], dtype=torch.int32))
        y.copy_(_rows(gen, seqs, heads + 2 * kv, F16))
        rows.copy_(_rows(gen, 9, heads + 2 * kv, F16))
        graph.replay()
        want = step(caches[1])
        want_draft, want_used = draft(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(drafted, want_draft) and torch.equal(used, want_used)
        for name in ("table", "lens", "refs", "taken"):
            assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), (name, i)


def test_streams_and_repeats(cuda):
    """Another stream than the tensors' own; the same call gives the same bits."""
    from leankv_amd.paged import packed_attention

    gen = torch.Generator().manual_seed(23)
    q, k, v = (_rows(gen, 500, h, BF16).cuda() for h in (8, 2, 2))
    at = _ints([0, 200, 500])
    cache, _, _ = _cache(gen, [900, 100], 2, 64, BF16)
    q1 = _rows(gen, 2, 8, BF16).cuda()
    want = packed_attention(q, k, v, at), cache.decode_attention(0, q1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [(packed_attention(q, k, v, at), cache.decode_attention(0, q1)) for _ in range(3)]
    stream.synchronize()
    for a, b in got:
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_offsets_past_32_bits(cuda):
    """A pool of over 2^32 numbers."""
    from leankv_amd.paged import PagedKV

    gen = torch.Generator().manual_seed(24)
    kv, page = 8, 256
    pages = 2 ** 32 // (2 * kv * page * D) + 40
    cache = PagedKV(1, kv, pages, 2, 700, page_size=page, dtype=F16)
    cache.refs[:pages - 8] = 1  # (in use by nobody here)
    at = [0, 600, 630]
    x = _rows(gen, 630, 3 * kv, F16)
    y = x.cuda()
    cache.extend(_ints(at))
    p = pages - 8  # (600 tokens fill the three pages of a row, 30 one)
    assert cache.table.tolist() == [[p, p + 1, p + 2], [p + 3, -1, -1]]
    cache.store(0, y[:, kv:2 * kv], y[:, 2 * kv:], _ints(at))
    want, bound = packed(x[:, :kv], x[:, kv:2 * kv], x[:, 2 * kv:], at)
    check(cache.prefill_attention(0, y[:, :kv], _ints(at)), want, bound)
    got = cache.decode_attention(0, y[[599, 629], :kv])
    check(got, want[[599, 629]], bound[[599, 629]])
    cache.fork(_ints([0, 0]))
    cache.extend()
    k, _ = cache.read(0, 600)
    assert torch.equal(k[0], k[1]) and torch.equal(k[0].transpose(0, 1), y[:600, kv:2 * kv])
    del cache, y, k
    torch.cuda.empty_cache()


def test_backward_raises(cuda):
    from leankv_amd._lib import LeanKVError
    from leankv_amd.paged import PagedKV, packed_attention

    q = torch.randn(4, 2, D, dtype=F16, device="cuda", requires_grad=True)
    k = torch.randn(4, 1, D, dtype=F16, device="cuda")
    at = _ints([0, 4])
    out = packed_attention(q, k, k, at)
    with pytest.raises(LeanKVError, match="no backward"):
        out.sum().backward()
    with pytest.raises(LeanKVError, match="autograd"):
        packed_attention(q, k, k, at, out=torch.empty_like(q))
    with torch.no_grad():
        assert not packed_attention(q, k, k, at).requires_grad
    cache = PagedKV(1, 1, 4, 1, 64, dtype=F16)
    cache.extend(at)
    cache.store(0, k.clone().requires_grad_(), k, at)
    got = cache.prefill_attention(0, q.detach(), at)
    with pytest.raises(LeanKVError, match="no backward"):
        got.sum().backward()
    with pytest.raises(LeanKVError, match="autograd"):
        cache.decode_attention(0, q.detach()[:1], out=torch.empty(1, 2, D, dtype=F16, device="cuda"))
