"""Performance cases of the 8-bit block-scaled KV cache: its update and read-back, its attention for one new token and
for several, and the attention over the blocks that a score selects.

A cache layer keeps K and V of [batch, kv heads, tokens, 128].  Every finished block of 64 tokens of a head is held in
8 bits with one scale (amax / 127), the unfinished last block in fp16.  Keys also keep, for each finished block and
dimension, the lowest and the highest code: an upper bound of q.k over the block costs two short products.

  kind      entry points                                what it stands for
  store     KV8Store.update + read                      storing a prompt (or one token), and the K / V that any other
                                                        attention implementation then reads
  decode    KV8Store.decode_attention                   one new token of every sequence over its whole cache
  prefill   KV8Store.prefill_attention                  the new tokens of a prompt or of a chunk, causal over the cache
  sparse    KV8Store.sparse_decode_attention            one new token over the blocks with the highest score

`own` False computes the same from the formulas with torch operations; `exact` does so in 64 bits, apart from both.
"""

from __future__ import annotations

import math

import torch

own = False

D = 128       # head size
BLOCK = 64    # tokens of a block
F16_MAX = 65504.0
KINDS = ("store", "decode", "prefill", "sparse")
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one layer of a 4096-token prompt stored and handed on (the default mode of the framework's caches)
        dict(name="store_1x4096", kind="store", batch=1, kv=8, pos=0, new=4096, ragged=False, dtype="f16"),
        # sixteen padded prompts of different lengths, bfloat16
        dict(name="store_16x1201", kind="store", batch=16, kv=8, pos=0, new=1201, ragged=True, dtype="bf16"),
        # one new token of sixty-four sequences, which finishes a block of each: the smallest launches
        dict(name="append_64", kind="store", batch=64, kv=8, pos=4095, new=1, ragged=False, dtype="f16"),
        # one sequence at context 4096 and a little
        dict(name="decode_1x4133", kind="decode", batch=1, heads=32, kv=8, length=4133, ragged=False, dtype="f16"),
        # thirty-two sequences of mixed lengths, bfloat16
        dict(name="decode_32_mixed", kind="decode", batch=32, heads=32, kv=8, length=8192, ragged=True, dtype="bf16"),
        # one long sequence
        dict(name="decode_1x131072", kind="decode", batch=1, heads=32, kv=8, length=131072, ragged=False, dtype="f16"),
        # one layer of a 4096-token prompt
        dict(name="prefill_4096", kind="prefill", batch=1, heads=32, kv=8, length=4096, new=4096, ragged=False,
             dtype="f16"),
        # chunks of four prompts of different lengths over what is cached already, bfloat16
        dict(name="prefill_chunks", kind="prefill", batch=4, heads=32, kv=8, length=8192, new=512, ragged=True,
             dtype="bf16"),
        # five drafted tokens of eight sequences checked in one pass
        dict(name="verify_8x5", kind="prefill", batch=8, heads=32, kv=8, length=4096, new=5, ragged=False, dtype="f16"),
        # a sixteenth of a middling context: latency
        dict(name="sparse_1x8200", kind="sparse", batch=1, heads=32, kv=8, length=8200, blocks=8, ragged=False,
             dtype="f16"),
        # sixteen sequences of mixed lengths, bfloat16
        dict(name="sparse_16_mixed", kind="sparse", batch=16, heads=32, kv=8, length=32768, blocks=64, ragged=True,
             dtype="bf16"),
        # one long sequence, 4096 tokens of it
        dict(name="sparse_1x131072", kind="sparse", batch=1, heads=32, kv=8, length=131072, blocks=64, ragged=False,
             dtype="f16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(KINDS)
    kv = rng.choice((1, 2, 3, 4, 8, 8))
    case = dict(kind=kind, ragged=rng.random() < 0.5, dtype=rng.choice(("f16", "bf16")))
    if kind == "store":
        if rng.random() < 0.3:
            return dict(case, batch=_log_int(rng, 1, 64), kv=kv, pos=_log_int(rng, 1, 16384) - 1, new=1, ragged=False)
        batch = _log_int(rng, 1, 16)
        return dict(case, batch=batch, kv=kv, pos=0, new=_log_int(rng, 2, 19216 * 8 // (batch * kv)))
    batch = _log_int(rng, 1, 32)
    heads = kv * rng.choice((1, 2, 4, 4, 6, 7, 8))
    if kind == "prefill":
        new = _log_int(rng, 2, 4096)
        # at most the pairs of the whole 4096-token prompt, and a cache of at most 2^18 tokens of one head
        pairs = 32 * 4096 * 4096 // 2
        batch = max(1, min(batch, pairs // (heads * new * new)))
        length = max(new, min(16384, pairs // (heads * batch * new), 2 ** 18 // (batch * kv)))
        return dict(case, batch=batch, heads=heads, kv=kv, length=_log_int(rng, new, length), new=new)
    length = _log_int(rng, 1 if kind == "decode" else 64, min(131072, 2 ** 20 // (batch * kv)))
    case.update(batch=batch, heads=heads, kv=kv, length=length)
    if kind == "sparse":
        case["blocks"] = _log_int(rng, 2, 128)
    return case


# ------------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """Tokens of every sequence (store: new tokens), the longest first; a ragged batch falls to a fifth of it."""
    top, n = case["new"] if case["kind"] == "store" else case["length"], case["batch"]
    low = case["new"] if case["kind"] == "prefill" else 1
    if not case["ragged"] or n == 1:
        return [top] * n
    return [max(low, top - (top * 4 * i) // (5 * (n - 1)) - (i * 37) % 64 * (i > 0)) for i in range(n)]


def _q_lengths(case):
    """New tokens of every sequence that attend (prefill)."""
    n, new = case["batch"], case["new"]
    return [max(1, new - (i * new) // (2 * n)) for i in range(n)] if case["ragged"] else [new] * n


def _keys(gen, batch, kv, n, dtype):
    """Keys as a rotary model has them: channels of different spread and mean, a few large ones, and neighbouring tokens
    alike (a part that changes every 64 tokens)."""
    dev = torch.device("cuda")
    spread = torch.exp(0.3 * torch.randn(1, kv, 1, D, generator=gen, device=dev))
    spread[..., ::37] *= 4.0
    mean = 0.5 * torch.randn(1, kv, 1, D, generator=gen, device=dev)
    part = torch.randn(batch, kv, -(-n // 64), 1, D, generator=gen, device=dev).expand(-1, -1, -1, 64, -1)
    part = part.reshape(batch, kv, -1, D)[:, :, :n]
    out = torch.empty(batch, n, kv, D, dtype=dtype, device=dev)  # the projections' layout, seen as [batch, kv, n, D]
    for b in range(batch):
        x = torch.randn(kv, n, D, generator=gen, device=dev)
        out[b] = ((x + 0.7 * part[b]) * spread[0] + mean[0]).transpose(0, 1).to(dtype)
    return out.transpose(1, 2)


def _values(gen, batch, kv, n, dtype):
    out = torch.empty(batch, n, kv, D, dtype=dtype, device="cuda")
    for b in range(batch):
        out[b] = torch.randn(n, kv, D, generator=gen, device="cuda").to(dtype)
    return out.transpose(1, 2)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7919 + 11)
    dtype, B, kv = DTYPES[case["dtype"]], case["batch"], case["kv"]
    x = dict(lens=_lengths(case))
    if case["kind"] == "store":
        head = case["pos"] % BLOCK  # tokens of the unfinished block before the first new one
        n = head + case["new"]
    else:
        n = case["length"]
        S = case["new"] if case["kind"] == "prefill" else 1
        q = torch.randn(B, S, case["heads"], D, generator=gen, device="cuda") * 1.2
        x["q"] = q.to(dtype).transpose(1, 2)  # [B, heads, S, D]
        if case["kind"] == "prefill":
            x["q_lens"] = _q_lengths(case)
    x["k"], x["v"] = _keys(gen, B, kv, n, dtype), _values(gen, B, kv, n, dtype)
    return x


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# -------------------------------------------------------------------------------------------------- plain form
def _f16(x):
    return x.float().clamp(-F16_MAX, F16_MAX).half()


def _quantize(x):
    """(codes, scale) of finished blocks x [..., 64, 128] fp16: rint(x * (127 / amax)), amax / 127."""
    x = x.float()
    amax = x.abs().amax((-2, -1), keepdim=True)
    inv = torch.where(amax > 0, 127.0 / amax, torch.zeros_like(amax))
    return torch.round(x * inv).clamp(-127, 127).to(torch.int8), (amax / 127.0)[..., 0, 0]


def _blocks(x):
    """[batch, kv, n, D] -> codes [batch, kv, n // 64, 64, D] and scales of the finished blocks."""
    full = x.shape[2] // BLOCK * BLOCK
    return _quantize(_f16(x[:, :, :full]).reshape(*x.shape[:2], -1, BLOCK, D))


def _plain_cache(x):
    out = {}
    for name in ("k", "v"):
        t = x[name]
        codes, scales = _blocks(t)
        rest = []  # the unfinished block of every sequence
        for b, n in enumerate(x["lens"]):
            rest.append(_f16(t[b, :, n // BLOCK * BLOCK:n]))
        out[name] = (codes, scales, rest)
    codes = out["k"][0]
    out["lo"], out["hi"] = codes.amin(3), codes.amax(3)
    return out


def _full(cache, name, b, n, index=None):
    """fp32 [kv, tokens, D] of sequence b: its finished blocks (or those of index [kv, m]), then the unfinished one."""
    codes, scales, rest = cache[name]
    codes, scales = codes[b, :, :n // BLOCK], scales[b, :, :n // BLOCK]
    if index is not None:
        codes = codes.gather(1, index[:, :, None, None].expand(-1, -1, BLOCK, D))
        scales = scales.gather(1, index)
    head = codes.float() * scales[..., None, None]
    return torch.cat([head.reshape(codes.shape[0], -1, D), rest[b].float()], dim=1)


def _attend(q, k, v, first=None):
    """softmax(q k^T / sqrt(D)) v of q [kv, G, S, D] over k, v [kv, n, D]; query i sees keys below first + i + 1."""
    kv, G, S, _ = q.shape
    s = q.reshape(kv, G * S, D).float() @ k.transpose(1, 2).contiguous() / math.sqrt(D)
    if first is not None:
        seen = torch.arange(k.shape[1], device=k.device) <= first + torch.arange(S, device=k.device).unsqueeze(1)
        s = s.view(kv, G, S, -1).masked_fill(~seen, -math.inf).view(kv, G * S, -1)
    return (torch.softmax(s, -1) @ v).view(kv, G, S, D)


def _plain_store(state):
    x, out = state["x"], []
    for name in ("k", "v"):
        codes, scales = _blocks(x[name])
        head = (codes.float() * scales[..., None, None]).half().reshape(*codes.shape[:2], -1, D)
        y = _f16(x[name]).contiguous()
        at = torch.arange(y.shape[2], device=y.device).view(1, 1, -1, 1)
        held = state["held"].view(-1, 1, 1, 1)  # tokens of every sequence, from the unfinished block's first
        full = held // BLOCK * BLOCK
        m = head.shape[2]
        y[:, :, :m] = torch.where(at[:, :, :m] < full, head, y[:, :, :m])
        out.append(torch.where(at < held, y, torch.zeros_like(y)))
    return tuple(out)


def _plain_decode(state):
    case, x, cache = state["case"], state["x"], state["cache"]
    kv, q = case["kv"], x["q"]
    out = torch.zeros(case["batch"], case["heads"], D, dtype=q.dtype, device=q.device)
    for b, n in enumerate(x["lens"]):
        o = _attend(_f16(q[b]).view(kv, -1, 1, D), _full(cache, "k", b, n), _full(cache, "v", b, n))
        out[b] = o.reshape(-1, D).to(q.dtype)
    return out


def _plain_prefill(state):
    case, x, cache = state["case"], state["x"], state["cache"]
    kv, q, G = case["kv"], x["q"], case["heads"] // case["kv"]
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    for b, (n, m) in enumerate(zip(x["lens"], x["q_lens"])):
        k, v = _full(cache, "k", b, n), _full(cache, "v", b, n)
        for i in range(0, m, 1024):
            j = min(i + 1024, m)
            part = _f16(q[b, :, i:j]).view(kv, G, j - i, D)
            seen = n - m + j
            o = _attend(part, k[:, :seen], v[:, :seen], n - m + i)
            out[b, :, i:j] = o.reshape(-1, j - i, D).to(q.dtype)
    return out


def _plain_select(case, q, cache, b, n):
    """[kv, m] indices of the selected finished blocks, ascending.  Sums of products of codes are whole numbers below
    2^24, so the score's only roundings are its two products."""
    kv, nb = case["kv"], n // BLOCK
    q16 = _f16(q).float().view(kv, -1, D)
    amax = q16.abs().amax(-1, keepdim=True)
    inv = torch.where(amax > 0, 127.0 / amax, torch.zeros_like(amax))
    q8 = torch.round(q16 * inv).clamp(-127, 127)
    lo, hi = cache["lo"][b, :, :nb].float(), cache["hi"][b, :, :nb].float()
    dot = q8.clamp(min=0) @ hi.transpose(1, 2).contiguous() + q8.clamp(max=0) @ lo.transpose(1, 2).contiguous()
    score = (dot * (amax / 127.0)).amax(1) * cache["k"][1][b, :, :nb] + 0.0
    score[:, :1] = math.inf
    score[:, nb - 1:] = math.inf
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    return order[:, :case["blocks"]].sort(-1).values


def _plain_sparse(state):
    case, x, cache = state["case"], state["x"], state["cache"]
    kv, q = case["kv"], x["q"]
    out = torch.zeros(case["batch"], case["heads"], D, dtype=q.dtype, device=q.device)
    index = torch.full((case["batch"], kv, case["blocks"]), -1, dtype=torch.int32, device=q.device)
    for b, n in enumerate(x["lens"]):
        chosen = _plain_select(case, q[b, :, 0], cache, b, n)
        o = _attend(_f16(q[b]).view(kv, -1, 1, D), _full(cache, "k", b, n, chosen), _full(cache, "v", b, n, chosen))
        out[b] = o.reshape(-1, D).to(q.dtype)
        index[b, :, :chosen.shape[1]] = chosen.int()
    return out, index


# ------------------------------------------------------------------------------------------------------ the tools
def prepare(case, seed):
    x = _inputs(case, seed)
    state = dict(case=case, x=x)
    if not own:
        if case["kind"] == "store":
            state["held"] = _ints([case["pos"] % BLOCK + m for m in x["lens"]])
        else:
            state["cache"] = _plain_cache(x)
            del x["k"], x["v"]
        return state
    from leankv_amd.kv8 import KV8Store

    B, kv = case["batch"], case["kv"]
    if case["kind"] == "store":
        pos, head = case["pos"], case["pos"] % BLOCK
        store = KV8Store(B, kv, pos + case["new"], device="cuda")
        if head:  # the unfinished block that the new token joins
            store.update(x["k"][:, :, :head], x["v"][:, :, :head], _ints([pos - head] * B))
        state.update(pos=_ints([pos] * B), k=x["k"][:, :, head:], v=x["v"][:, :, head:], n_new=_ints(x["lens"]),
                     lens=_ints([pos + m for m in x["lens"]]))
    else:
        store = KV8Store(B, kv, case["length"], device="cuda")
        store.update(x["k"], x["v"], _ints([0] * B), _ints(x["lens"]))
        state.update(lens=_ints(x["lens"]), q=x["q"] if case["kind"] == "prefill" else x["q"][:, :, 0])
        if case["kind"] == "prefill":
            state["q_lens"] = _ints(x["q_lens"]) if case["ragged"] else None
        del x["k"], x["v"]
    state["store"] = store
    return state


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"store": _plain_store, "decode": _plain_decode, "prefill": _plain_prefill,
                "sparse": _plain_sparse}[kind](state)
    store = state["store"]
    if kind == "store":
        store.update(state["k"], state["v"], state["pos"], state["n_new"] if case["ragged"] else None)
        end = case["pos"] + case["new"]
        return store.read(state["lens"], end, first=case["pos"] // BLOCK * BLOCK)
    if kind == "decode":
        return store.decode_attention(state["q"], state["lens"])
    if kind == "prefill":
        return store.prefill_attention(state["q"], state["lens"], state["q_lens"])
    return store.sparse_decode_attention(state["q"], state["lens"], case["blocks"])


def work(case):
    kv, lens = case["kv"], _lengths(case)
    if case["kind"] == "store":
        new, head, B = sum(lens), case["pos"] % BLOCK, case["batch"]
        # new tokens in, the unfinished block's where it is finished, codes and the fp16 rest out, the values out
        held = [head + m for m in lens]
        joined = sum(head for n in held if n >= BLOCK)
        kept = sum(n // BLOCK * BLOCK + 2 * (n % BLOCK if n >= BLOCK else n - head) for n in held)
        rows = 2 * kv * D * (2 * (new + joined) + kept + 2 * B * (head + case["new"]))
        return {"bytes": rows, "flops": 2 * kv * D * new * 3}
    heads = case["heads"]
    S = case["new"] if case["kind"] == "prefill" else 1
    ends = 4 * case["batch"] * heads * S * D  # q and out
    rest = sum(n % BLOCK for n in lens) * kv * D * 4
    if case["kind"] == "sparse":
        chosen = [min(n // BLOCK, case["blocks"]) for n in lens]
        ranges = sum(n // BLOCK for n in lens) * kv * (2 * D + 4)
        return {"bytes": ranges + sum(chosen) * kv * (2 * BLOCK * D + 8) + rest + ends,
                "flops": 4 * heads * D * sum(c * BLOCK + n % BLOCK for c, n in zip(chosen, lens))
                + 4 * heads * D * sum(n // BLOCK for n in lens)}
    codes = sum(n // BLOCK for n in lens) * kv * (2 * BLOCK * D + 8)
    if case["kind"] == "decode":
        pairs = sum(lens)
    else:  # query i of m over n tokens sees n - m + i + 1
        pairs = sum(m * (n - m) + m * (m + 1) // 2 for n, m in zip(lens, _q_lengths(case)))
    return {"bytes": codes + rest + ends, "flops": 4 * heads * D * pairs}


# ------------------------------------------------------------------------------------------------------- 64 bits
def _exact_tokens(x, b, n):
    """fp64 [kv, n, D] of the stored tokens of sequence b, and the codes and scales of its finished blocks.  A code is
    the fp32 quotient's nearest whole number by definition; everything after it is in 64 bits."""
    t = x[b, :, :n].to(torch.float64).clamp(-F16_MAX, F16_MAX).to(torch.float16)
    nb = n // BLOCK
    blocks = t[:, :nb * BLOCK].reshape(t.shape[0], nb, BLOCK * D)
    top = blocks.abs().max(-1).values if nb else blocks.new_zeros(t.shape[0], 0)
    up = torch.where(top > 0, 127.0 / top.float(), top.float())
    codes = torch.round(blocks.float() * up.unsqueeze(-1))
    full = codes.double() * (top.double() / 127.0).unsqueeze(-1)
    return torch.cat([full.reshape(t.shape[0], nb * BLOCK, D), t[:, nb * BLOCK:].double()], dim=1), codes, top


def _exact_rows(q, k, v, seen):
    """Softmax attention in 64 bits of q [rows, D] over the first seen[i] tokens of k, v [n, D]."""
    s = (q.double() @ k.t()) / math.sqrt(D)
    hide = torch.arange(k.shape[0], device=k.device).view(1, -1) >= seen.view(-1, 1)
    s[hide] = -math.inf
    w = torch.exp(s - s.amax(1, keepdim=True))
    return (w @ v) / w.sum(1, keepdim=True)


def _exact_choice(q, codes, top, blocks):
    """Indices of the selected blocks of one kv head: q [G, D], codes [nb, 64 * D]; the score in the definition's fp32."""
    nb = codes.shape[0]
    c = codes.view(nb, BLOCK, D)
    lo, hi = c.min(1).values.double(), c.max(1).values.double()
    best = None
    for row in q:
        a = row.abs().max().float()
        r = torch.round(row.float() * (127.0 / a)).double() if a > 0 else row.double() * 0
        bound = torch.maximum(r * lo, r * hi).sum(-1).float() * (a / 127.0)
        best = bound if best is None else torch.maximum(best, bound)
    best = (best * (top.float() / 127.0) + 0.0).tolist()
    forced = [0, nb - 1]
    rank = sorted(range(nb), key=lambda j: (j not in forced, -best[j], j))
    return sorted(rank[:blocks])


def exact(case, seed):
    x = _inputs(case, seed)
    kind, kv, lens = case["kind"], case["kv"], x["lens"]
    if kind == "store":
        out = []
        for name in ("k", "v"):
            y = torch.zeros(x[name].shape, dtype=torch.float64, device="cuda")
            for b, m in enumerate(lens):
                n = case["pos"] % BLOCK + m
                y[b, :, :n] = _exact_tokens(x[name], b, n)[0]
            out.append(y)
        return tuple(out)
    G = case["heads"] // kv
    q = x["q"].double().clamp(-F16_MAX, F16_MAX).half()
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    index = torch.full((case["batch"], kv, case.get("blocks", 1)), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        k, codes, top = _exact_tokens(x["k"], b, n)
        v = _exact_tokens(x["v"], b, n)[0]
        m = x["q_lens"][b] if kind == "prefill" else 1
        for h in range(case["heads"]):
            g = h // G
            kk, vv, seen = k[g], v[g], n - m + 1 + torch.arange(m, device="cuda")
            if kind == "sparse" and n >= BLOCK:
                if h % G == 0:
                    pick = _exact_choice(q[b, g * G:(g + 1) * G, 0], codes[g], top[g], case["blocks"])
                    index[b, g, :len(pick)] = torch.tensor(pick, dtype=torch.int32, device="cuda")
                    rows = (torch.tensor(pick, device="cuda").view(-1, 1) * BLOCK
                            + torch.arange(BLOCK, device="cuda")).view(-1)
                    rows = torch.cat([rows, torch.arange(n // BLOCK * BLOCK, n, device="cuda")])
                kk, vv = kk[rows], vv[rows]
                seen = torch.tensor([rows.numel()], device="cuda")
            out[b, h, :m] = _exact_rows(q[b, h, :m], kk, vv, seen)
    if kind == "prefill":
        return out
    return out[:, :, 0] if kind == "decode" else (out[:, :, 0], index)
