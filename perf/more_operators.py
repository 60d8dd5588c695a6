"""Performance cases of the 16-bit paged KV cache and of the attention of prompts: storing tokens in pages, forking and
compacting the pages, attention of packed prompts, of chunks over pages, and of one new token over pages.

A pool holds pages of `page` tokens, K and V of [kv heads, page, 128] each, for every layer.  A sequence is a row of page ids
and a length; sequences that come from one prompt name the same pages until one of them writes.

  kind      entry points                                what it stands for
  store     PagedKV.extend + store                      room for new tokens of every sequence, and their K and V
  fork      PagedKV.fork + extend                       a beam step: every sequence goes on from a parent; shared last pages
                                                        are copied before they are written to
  compact   PagedKV.compact                             pages of the sequences that stay move to the front of the pool
  prompt    packed_attention                            causal attention of prompts that lie one behind the other
  chunk     PagedKV.prefill_attention                   new tokens of a prompt's chunk, or drafted ones, over the pages
  decode    PagedKV.decode_attention                    one new token of every sequence over the pages

`own` False computes the same from the definitions with torch operations; `exact` does so in 64 bits, apart from both.
"""

from __future__ import annotations

import math

import torch

own = False

D = 128  # head size
KINDS = ("store", "fork", "compact", "prompt", "chunk", "decode")
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # sixteen prompts of different lengths stored in one layer
        dict(name="store_16x1201", kind="store", seqs=16, kv=8, page=64, length=0, new=1201, ragged=True, dtype="bf16"),
        # one new token of sixty-four sequences: the smallest launches
        dict(name="append_64", kind="store", seqs=64, kv=8, page=64, length=1503, new=1, ragged=True, dtype="f16"),
        # a beam step of eight prompts with eight beams each, four layers
        dict(name="fork_8x8", kind="fork", prompts=8, beams=8, kv=8, page=64, length=2087, layers=4, dtype="bf16"),
        # half of the sequences have ended, four layers
        dict(name="compact_32", kind="compact", seqs=32, kv=8, page=64, length=2048, layers=4, dtype="f16"),
        # one long prompt
        dict(name="prompt_1x8192", kind="prompt", seqs=1, heads=32, kv=8, length=8192, ragged=False, dtype="bf16"),
        # sixteen prompts of different lengths
        dict(name="prompt_16_ragged", kind="prompt", seqs=16, heads=32, kv=8, length=1201, ragged=True, dtype="f16"),
        # sixty-four short requests
        dict(name="prompt_64_short", kind="prompt", seqs=64, heads=32, kv=8, length=150, ragged=True, dtype="bf16"),
        # chunks of four prompts over what is stored already
        dict(name="chunk_4x512", kind="chunk", seqs=4, heads=32, kv=8, page=64, length=8192, new=512, ragged=True,
             dtype="bf16"),
        # five drafted tokens of eight sequences checked in one pass
        dict(name="verify_8x5", kind="chunk", seqs=8, heads=32, kv=8, page=64, length=4096, new=5, ragged=False,
             dtype="f16"),
        # thirty-two sequences of mixed lengths
        dict(name="decode_32_mixed", kind="decode", seqs=32, beams=1, heads=32, kv=8, page=64, length=8192, ragged=True,
             dtype="bf16"),
        # one long sequence
        dict(name="decode_1x131072", kind="decode", seqs=1, beams=1, heads=32, kv=8, page=64, length=131072, ragged=False,
             dtype="f16"),
        # four prompts with eight beams each, which share the prompt's pages
        dict(name="decode_4x8_beams", kind="decode", seqs=32, beams=8, heads=32, kv=8, page=64, length=8192, ragged=False,
             dtype="f16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(KINDS)
    kv = rng.choice((1, 2, 3, 4, 8, 8))
    case = dict(kind=kind, kv=kv, dtype=rng.choice(("f16", "bf16")))
    if kind != "prompt":
        case["page"] = rng.choice((16, 32, 64, 64, 128))
    if kind == "store":
        seqs = _log_int(rng, 1, 64)
        if rng.random() < 0.4:
            return dict(case, seqs=seqs, length=_log_int(rng, 1, 4096), new=1, ragged=rng.random() < 0.5)
        return dict(case, seqs=seqs, length=rng.choice((0, _log_int(rng, 1, 512))), new=_log_int(rng, 2, 150000 // (seqs * kv)),
                    ragged=rng.random() < 0.5)
    if kind == "fork":
        return dict(case, prompts=_log_int(rng, 1, 8), beams=rng.randint(2, 8), length=_log_int(rng, 40, 2087),
                    layers=rng.randint(1, 4))
    if kind == "compact":
        return dict(case, seqs=rng.randint(2, 32), length=_log_int(rng, 100, 2048), layers=rng.randint(1, 4))
    heads = kv * rng.choice((1, 2, 4, 4, 6, 7, 8))
    seqs = _log_int(rng, 1, 32)
    case.update(seqs=seqs, heads=heads, ragged=rng.random() < 0.6)
    if kind == "prompt":
        # at most the pairs of the longest listed prompt
        return dict(case, length=_log_int(rng, 1, int(math.sqrt(32 * 8192 * 8192 / (heads * seqs)))))
    if kind == "chunk":
        new = _log_int(rng, 2, 2048)
        seqs = case["seqs"] = max(1, min(seqs, 2 ** 29 // (heads * new * new)))
        return dict(case, new=new, length=_log_int(rng, new, max(new, min(16384, 2 ** 29 // (heads * seqs * new),
                                                                         2 ** 18 // (seqs * kv)))))
    beams = rng.choice((1, 1, 2, 3, 4, 5, 8))
    return dict(case, seqs=max(seqs // beams, 1) * beams, beams=beams, length=_log_int(rng, 1, min(131072, 2 ** 20 // (seqs * kv))))


# ------------------------------------------------------------------------------------------------------- inputs
def _spread(top, n, low, ragged):
    """n lengths, the longest first; a ragged batch falls to a fifth of it."""
    if not ragged or n == 1:
        return [top] * n
    return [max(low, top - (top * 4 * i) // (5 * (n - 1)) - (i * 37) % 64 * (i > 0)) for i in range(n)]


def _shape(case):
    """(tokens that every sequence holds before the call, new tokens of each).  Beams, and what is compacted: no new ones."""
    kind = case["kind"]
    if kind == "store":
        if case["new"] == 1:
            return _spread(case["length"], case["seqs"], 1, case["ragged"]), [1] * case["seqs"]
        return [case["length"]] * case["seqs"], _spread(case["new"], case["seqs"], 1, case["ragged"])
    if kind == "fork":
        return [case["length"]] * (case["prompts"] * case["beams"]), [1] * (case["prompts"] * case["beams"])
    if kind == "compact":
        return _spread(case["length"], case["seqs"], 1, True), [0] * case["seqs"]
    if kind == "prompt":
        return [0] * case["seqs"], _spread(case["length"], case["seqs"], 1, case["ragged"])
    if kind == "chunk":
        new = [max(1, case["new"] - (i * case["new"]) // (2 * case["seqs"])) if case["ragged"] else case["new"]
               for i in range(case["seqs"])]
        return _spread(case["length"], case["seqs"], case["new"], case["ragged"]), new
    n, beams = case["seqs"], case["beams"]
    if beams == 1:
        return _spread(case["length"], n, 1, case["ragged"]), [1] * n
    # beams of a prompt, each some tokens into an answer of its own
    prompt = _spread(case["length"], n // beams, 1, case["ragged"])
    return [prompt[i // beams] + _tail(case) - (3 * (i % beams) if case["ragged"] else 0) for i in range(n)], [1] * n


def _tail(case):
    return 100 + 3 * case["beams"]


def _tables(case, gen):
    """(rows of page ids, pages of the pool).  Pages lie in no order, as in a pool that has been in use."""
    lens, new = _shape(case)
    page, kind = case["page"], case["kind"]
    rows = [0] * len(lens)
    at = 0
    for i, n in enumerate(lens):
        need = -(-n // page)
        own_from = 0
        if kind == "fork" and i % case["beams"]:
            own_from = n // page - min(n // page, 1)  # the beams of the step before: all but the last pages are the prompt's
        if kind == "decode" and case["beams"] > 1 and i % case["beams"]:
            own_from = (lens[i - i % case["beams"]] - _tail(case)) // page  # the whole pages of the prompt
        rows[i] = rows[i - 1][:own_from] + list(range(at, at + need - own_from)) if own_from else list(range(at, at + need))
        at += need - own_from
    room = sum(-(-(n + m) // page) for n, m in zip(lens, new)) + len(lens) if kind in ("store", "fork") else at
    pages = max(room, at) + at // 8 + 1
    order = torch.randperm(pages, generator=gen).tolist()
    return [[order[p] for p in row] for row in rows], pages


def _kv(gen, shape, dtype, heads_at, key):
    """Keys as a rotary model has them (channels of different spread and mean, a few large ones), or values."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=dtype)
    if key:
        side = [1] * len(shape)
        side[heads_at], side[-1] = shape[heads_at], D
        spread = torch.exp(0.3 * torch.randn(side, generator=gen, device="cuda"))
        spread[..., ::37] *= 4.0
        x.mul_(spread).add_(0.5 * torch.randn(side, generator=gen, device="cuda").to(dtype))
    return x


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    host = torch.Generator().manual_seed(seed * 104729 + 5)
    dtype, kv, kind = DTYPES[case["dtype"]], case["kv"], case["kind"]
    lens, new = _shape(case)
    x = dict(n_host=len(lens), new_host=new, lens_host=lens)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    x["cu"] = _ints(starts)
    total = starts[-1]
    if kind in ("prompt", "chunk", "decode"):
        x["q"] = (1.2 * torch.randn(total, case["heads"], D, generator=gen, device="cuda")).to(dtype)
    if kind in ("prompt", "store"):
        x["k"], x["v"] = _kv(gen, (total, kv, D), dtype, 1, True), _kv(gen, (total, kv, D), dtype, 1, False)
    if kind == "prompt":
        return x
    rows, pages = _tables(case, host)
    layers, page = case.get("layers", 1), case["page"]
    width = -(-max(n + m for n, m in zip(lens, new)) // page)
    x["table"] = _ints([row + [-1] * (width - len(row)) for row in rows])
    x["lens"] = _ints(lens)
    used = torch.tensor([p for row in rows for p in row], dtype=torch.int64)
    x["refs"] = torch.bincount(used, minlength=pages).int().cuda()
    x["pool"] = torch.empty(layers, pages, 2, kv, page, D, dtype=dtype, device="cuda")
    for side in (0, 1):
        x["pool"][:, :, side] = _kv(gen, (layers, pages, kv, page, D), dtype, 2, side == 0)
    if kind == "fork":  # some beams go on from another beam of their prompt
        pick = torch.randint(0, case["beams"], (len(lens),), generator=host).tolist()
        parent = [i - i % case["beams"] + (pick[i] if i % 3 else pick[i - i % case["beams"]]) for i in range(len(lens))]
        x["parent"] = _ints(parent)
    if kind == "compact":  # every second sequence has ended
        keep = torch.arange(len(lens), device="cuda") % 2 == 0
        gone = x["table"][~keep]
        x["refs"].index_add_(0, gone[gone >= 0].long(), torch.full_like(gone[gone >= 0], -1))
        x["table"][~keep] = -1
        x["lens"][~keep] = 0
    return x


# -------------------------------------------------------------------------------------------------- plain form
def _pages_of(lens, page):
    return (lens + page - 1) // page


def _plain_extend(pool, table, lens, refs, n):
    """Room for n new tokens of every sequence: (table, lens, refs); shared last pages are copied in the pool."""
    page, width, pages = pool.shape[4], table.shape[1], refs.shape[0]
    old, end = _pages_of(lens, page), _pages_of(lens + n, page)
    last = table.gather(1, (lens // page).clamp(max=width - 1).long().unsqueeze(1)).squeeze(1)
    part = (lens % page > 0) & (n > 0)
    at = torch.where(part, last, pages).long()
    writers = torch.zeros(pages + 1, dtype=torch.int32, device=at.device).index_add_(0, at, torch.ones_like(lens))
    uses = torch.cat([refs, refs.new_zeros(1)])[at]
    alike = (at.unsqueeze(0) == at.unsqueeze(1)) & part
    first = ~torch.tril(alike, -1).any(1)
    copy = part & (uses > 1) & ~(first & (writers[at] == uses))
    need = end - old + copy
    begin = torch.cumsum(need, 0) - need
    free = torch.sort((refs > 0).to(torch.uint8), stable=True).indices.int()
    j = torch.arange(width, device=at.device).unsqueeze(0)
    is_copy = copy.unsqueeze(1) & (j == (lens // page).unsqueeze(1))
    is_new = (j >= old.unsqueeze(1)) & (j < end.unsqueeze(1))
    place = begin.unsqueeze(1) + torch.where(is_copy, 0, copy.int().unsqueeze(1) + j - old.unsqueeze(1))
    got = free[place.clamp(0, pages - 1).long()]
    out = torch.where(is_copy | is_new, got, table)
    refs = refs.clone().index_add_(0, at[copy], torch.full_like(lens[copy], -1))
    taken = got[is_copy | is_new].long()
    refs.index_add_(0, taken, torch.ones_like(taken, dtype=torch.int32))
    src, dst = at[copy], out[is_copy].long()
    filled = (torch.arange(page, device=at.device) < (lens % page)[copy].unsqueeze(1)).view(1, -1, 1, 1, page, 1)
    pool[:, dst] = torch.where(filled, pool[:, src], pool[:, dst])
    return out, lens + n, refs


def _count(table, pages):
    at = torch.where(table >= 0, table, pages).long().flatten()
    return torch.zeros(pages + 1, dtype=torch.int32, device=at.device).index_add_(
        0, at, torch.ones_like(at, dtype=torch.int32))[:pages]


def _plain_store(state):
    x, page = state["x"], state["case"]["page"]
    n = x["cu"].diff()
    table, lens, refs = _plain_extend(x["pool"], x["table"], x["lens"], x["refs"], n)
    row = torch.arange(x["k"].shape[0], device=n.device, dtype=torch.int32)
    seq = torch.searchsorted(x["cu"], row, right=True) - 1
    pos = x["lens"][seq] + row - x["cu"][seq]
    at = table[seq, (pos // page).long()].long()
    slot = (pos % page).long()
    pool = x["pool"][0]
    pool[at, 0, :, slot] = x["k"]
    pool[at, 1, :, slot] = x["v"]
    return x["pool"], table, lens, refs


def _plain_fork(state):
    x = state["x"]
    parent = x["parent"].long()
    table, lens = x["table"][parent], x["lens"][parent]
    table, lens, refs = _plain_extend(x["pool"], table, lens, _count(table, x["refs"].shape[0]), torch.ones_like(lens))
    return x["pool"], table, lens, refs


def _plain_compact(state):
    x = state["x"]
    live = x["refs"] > 0
    n = live.sum(dtype=torch.int32)
    ids = torch.arange(live.shape[0], device=n.device, dtype=torch.int32)
    holes, movers = ids[~live & (ids < n)], ids[live & (ids >= n)]
    to = ids.clone()
    to[movers.long()] = holes
    table = torch.where(x["table"] >= 0, to[x["table"].clamp(min=0).long()], x["table"])
    refs = x["refs"].clone()
    refs[holes.long()] = refs[movers.long()]
    refs[movers.long()] = 0
    x["pool"][:, holes.long()] = x["pool"][:, movers.long()]
    return x["pool"], table, refs, n.view(1)


def _attend(q, k, v, first, seen):
    """softmax(q k^T / sqrt(D)) v in 32 bits of q [B, H, G, S, D] over k, v [B, H, n, D]: query i of row b sees the tokens
    below first[b] + i + 1, and below seen[b]; a query that sees none is zero."""
    B, H, G, S, _ = q.shape
    t = torch.arange(k.shape[2], device=k.device)
    s = q.reshape(B, H, G * S, D) @ k.transpose(2, 3).contiguous() / math.sqrt(D)
    i = torch.arange(S, device=k.device)
    ok = (t <= first.view(-1, 1, 1) + i.view(1, -1, 1)) & (t < seen.view(-1, 1, 1))  # [B, S, n]
    s = s.view(B, H, G, S, -1).masked_fill(~ok[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    v = torch.where((t < seen.view(-1, 1)).view(B, 1, -1, 1), v, 0.0)
    return (w.view(B, H, G * S, -1) @ v).view(B, H, G, S, D) / torch.where(total > 0, total, 1.0)


def _padded(x, cu, n):
    """Packed rows [T, heads, D] as fp32 [B, heads, n, D] (rows past a sequence repeat one)."""
    at = (cu[:-1].unsqueeze(1) + torch.arange(n, device=cu.device)).clamp(max=x.shape[0] - 1)
    return x[at.long()].float().transpose(1, 2)


def _packed(out, cu, total, like):
    """[B, H, G, S, D] back to packed rows."""
    row = torch.arange(total, device=cu.device, dtype=torch.int32)
    seq = torch.searchsorted(cu, row, right=True) - 1
    return out.permute(0, 3, 1, 2, 4)[seq, (row - cu[seq]).long()].reshape(like.shape).to(like.dtype)


def _plain_prompt(state):
    case, x = state["case"], state["x"]
    n, kv = max(x["new_host"]), case["kv"]
    q = _padded(x["q"], x["cu"], n).unflatten(1, (kv, -1))
    lens = x["cu"].diff()
    out = _attend(q, _padded(x["k"], x["cu"], n), _padded(x["v"], x["cu"], n), torch.zeros_like(lens), lens)
    return _packed(out, x["cu"], x["q"].shape[0], x["q"])


def _paged_kv(x):
    """K, V fp32 [S, H, n, D] of every sequence's pages."""
    kv = x["pool"][0][x["table"].clamp(min=0).long()]  # [S, M, 2, H, page, D]
    return tuple(kv[:, :, side].transpose(1, 2).flatten(2, 3).float() for side in (0, 1))


def _plain_chunk(state):
    case, x = state["case"], state["x"]
    q = _padded(x["q"], x["cu"], max(x["new_host"])).unflatten(1, (case["kv"], -1))
    k, v = _paged_kv(x)
    out = _attend(q, k, v, x["lens"] - x["cu"].diff(), x["lens"])
    return _packed(out, x["cu"], x["q"].shape[0], x["q"])


def _plain_decode(state):
    case, x = state["case"], state["x"]
    k, v = _paged_kv(x)
    q = x["q"].float().view(case["seqs"], case["kv"], -1, 1, D)
    return _attend(q, k, v, x["lens"] - 1, x["lens"]).reshape(x["q"].shape).to(x["q"].dtype)


# ------------------------------------------------------------------------------------------------------ the tools
def prepare(case, seed):
    x = _inputs(case, seed)
    state = dict(case=case, x=x)
    if own and case["kind"] != "prompt":
        from leankv_amd.paged import PagedKV

        pool = x["pool"]
        cache = PagedKV(pool.shape[0], case["kv"], pool.shape[1], x["n_host"], x["table"].shape[1] * case["page"],
                        page_size=case["page"], dtype=pool.dtype)
        for name in ("pool", "table", "lens", "refs"):
            getattr(cache, name).copy_(x.pop(name))
        # what a program that may go back keeps (a pass starts from the same pages each time)
        state.update(cache=cache, before=cache.snapshot())
    return state


def run(state):
    case, x = state["case"], state["x"]
    kind = case["kind"]
    if not own:
        return {"store": _plain_store, "fork": _plain_fork, "compact": _plain_compact, "prompt": _plain_prompt,
                "chunk": _plain_chunk, "decode": _plain_decode}[kind](state)
    if kind == "prompt":
        from leankv_amd.paged import packed_attention

        return packed_attention(x["q"], x["k"], x["v"], x["cu"], max_len=case["length"])
    cache = state["cache"]
    if kind == "decode":
        return cache.decode_attention(0, x["q"])
    if kind == "chunk":
        return cache.prefill_attention(0, x["q"], x["cu"], max_new=case["new"])
    cache.rollback(state["before"])
    if kind == "store":
        cu = None if case["new"] == 1 else x["cu"]
        cache.extend(cu)
        cache.store(0, x["k"], x["v"], cu)
        return cache.pool, cache.table, cache.lens, cache.refs
    if kind == "fork":
        cache.fork(x["parent"])
        cache.extend()
        return cache.pool, cache.table, cache.lens, cache.refs
    return cache.pool, cache.table, cache.refs, cache.compact()


def work(case):
    lens, new = _shape(case)
    row = case["kv"] * D * 2  # bytes of a token's keys (or values) in one layer
    if case["kind"] == "store":
        return {"bytes": 4 * row * sum(new), "flops": 0}
    if case["kind"] == "fork":  # every beam but one of those on a page copies its tokens
        copies = case["prompts"] * (case["beams"] - 1) if case["length"] % case["page"] else 0
        return {"bytes": 4 * row * case["layers"] * copies * (case["length"] % case["page"])
                + 8 * sum(-(-n // case["page"]) for n in lens), "flops": 0}
    if case["kind"] == "compact":
        held = [-(-n // case["page"]) for n in lens]
        live, pages = sum(held[::2]), sum(held) + sum(held) // 8 + 1
        return {"bytes": 4 * row * case["page"] * case["layers"] * live * (pages - live) // pages, "flops": 0}
    ends = 2 * 2 * case["heads"] * D * sum(new)  # queries and outputs
    if case["kind"] == "prompt":
        pairs = sum(n * (n + 1) // 2 for n in new)
        return {"bytes": ends + 2 * row * sum(new), "flops": 4 * case["heads"] * D * pairs}
    held = sum(lens)
    if case["kind"] == "decode" and case["beams"] > 1:  # a prompt's whole pages once
        whole = [(lens[i] - _tail(case)) // case["page"] * case["page"] for i in range(0, len(lens), case["beams"])]
        held -= (case["beams"] - 1) * sum(whole)
    pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, new))
    return {"bytes": ends + 2 * row * held, "flops": 4 * case["heads"] * D * pairs}


# ------------------------------------------------------------------------------------------------------- 64 bits
def _exact_extend(x, rows, lens, new):
    """Pages given out one sequence at a time, as lists; copies of shared last pages are made in the pool."""
    page, pool = x["pool"].shape[4], x["pool"]
    uses = [0] * pool.shape[1]
    for row in rows:
        for p in row:
            uses[p] += 1
    writers = {}
    for s, row in enumerate(rows):
        if new[s] and lens[s] % page:
            writers.setdefault(row[-1], []).append(s)
    free = [p for p, u in enumerate(uses) if not u][::-1]
    copied = []
    for s, row in enumerate(rows):
        if new[s] and lens[s] % page:
            p = row[-1]
            group = writers[p]
            if uses[p] > 1 and not (group[0] == s and len(group) == uses[p]):
                row[-1] = free.pop()
                copied.append((p, row[-1], lens[s] % page))
        lens[s] += new[s]
        while len(row) * page < lens[s]:
            row.append(free.pop())
    for p, q, filled in copied:
        pool[:, q, :, :, :filled] = pool[:, p, :, :, :filled]


def _exact_pages(case, x):
    page, pool = case["page"], x["pool"]
    rows = [[p for p in row if p >= 0] for row in x["table"].tolist()]
    lens = x["lens"].tolist()
    if case["kind"] == "compact":
        used = sorted({p for row in rows for p in row})
        n = len(used)
        holes = sorted(set(range(n)) - set(used))
        to = dict(zip([p for p in used if p >= n], holes))
        for p, q in to.items():
            pool[:, q] = pool[:, p]
        rows = [[to.get(p, p) for p in row] for row in rows]
    else:
        new = x["new_host"]
        if case["kind"] == "fork":
            parent = x["parent"].tolist()
            rows, lens = [list(rows[p]) for p in parent], [lens[p] for p in parent]
        before = list(lens)
        _exact_extend(x, rows, lens, new)
        if case["kind"] == "store":
            at = 0
            for s, row in enumerate(rows):
                for i in range(0, new[s]):
                    pool[0, row[(before[s] + i) // page], 0, :, (before[s] + i) % page] = x["k"][at]
                    pool[0, row[(before[s] + i) // page], 1, :, (before[s] + i) % page] = x["v"][at]
                    at += 1
    table = torch.full_like(x["table"], -1)
    refs = [0] * pool.shape[1]
    for s, row in enumerate(rows):
        table[s, :len(row)] = _ints(row)
        for p in row:
            refs[p] += 1
    if case["kind"] == "compact":
        return pool, table, _ints(refs), _ints([n])
    return pool, table, _ints(lens), _ints(refs)


def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "store" and sum(x["new_host"]) > 40000:
        return None
    if kind in ("store", "fork", "compact"):
        return _exact_pages(case, x)
    G = case["heads"] // case["kv"]
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    starts = x["cu"].tolist()
    for b, m in enumerate(x["new_host"]):
        a = starts[b]
        if kind == "prompt":
            n, keys, values = m, x["k"][a:a + m].transpose(0, 1), x["v"][a:a + m].transpose(0, 1)
        else:
            n = x["lens_host"][b]
            rows = torch.arange(n, device="cuda")
            at = x["table"][b].long()[rows // case["page"]]
            kv = x["pool"][0][at, :, :, rows % case["page"]]  # [n, 2, kv, D]
            keys, values = kv[:, 0].transpose(0, 1), kv[:, 1].transpose(0, 1)
        seen = n - m + 1 + torch.arange(m, device="cuda")
        hide = torch.arange(n, device="cuda").unsqueeze(0) >= seen.unsqueeze(1)
        for g in range(case["kv"]):
            k64, v64 = keys[g].double().t().contiguous(), values[g].double().contiguous()
            for h in range(g * G, g * G + G):
                s = x["q"][a:a + m, h].double() @ k64 * D ** -0.5
                s[hide] = -math.inf
                w = torch.exp(s - s.amax(1, keepdim=True))
                out[a:a + m, h] = (w @ v64) / w.sum(1, keepdim=True)
    return out
