"""The 8-bit block-scaled cache and its attention in 64 bits (codes in the fp32 steps that define them), on the CPU."""
import math

import torch

BLOCK, D = 64, 128


def stored(x):
    """What a key or value becomes before it is stored: fp16, finite, NaN as 0."""
    x = torch.nan_to_num(x.double(), nan=0.0, posinf=65504.0, neginf=-65504.0).clamp(-65504.0, 65504.0)
    return x.to(torch.float32).to(torch.float16) if x.dtype != torch.float64 else x.half()


def query(x):
    return x.double().clamp(-65504.0, 65504.0).half()


STEP = torch.tensor(1.0) / torch.tensor(127.0)  # fp32


def factor(amax):
    return torch.where(amax > 0, (torch.ones_like(amax) / amax) * 127.0, torch.zeros_like(amax))


def quantize(blocks):
    """(codes int, scale fp32) of fp16 blocks [..., 64, 128]."""
    x = blocks.float()
    amax = x.abs().amax((-2, -1))
    return torch.round(x * factor(amax)[..., None, None]).to(torch.int64), amax * STEP


class Ref:
    """One sequence and kv head: every token as stored, fp64."""

    def __init__(self, k, v):  # fp16 [n, 128], already stored()
        self.n = k.shape[0]
        nb = self.n // BLOCK
        self.nb = nb
        self.codes, self.scales, self.vals, self.vscale = {}, {}, {}, torch.ones(self.n, dtype=torch.float64)
        for name, x in (("k", k), ("v", v)):
            c, s = quantize(x[:nb * BLOCK].reshape(nb, BLOCK, D))
            self.codes[name], self.scales[name] = c, s
            full = (c.double() * s.double()[:, None, None]).reshape(-1, D)
            self.vals[name] = torch.cat([full, x[nb * BLOCK:].double()])
        self.vscale[:nb * BLOCK] = self.scales["v"].double().clamp(min=2.0 ** -31).repeat_interleave(BLOCK)

    def attend(self, q, seen, scale, out_eps, tokens=None):
        """(out, bound) of one query fp16 [128] over its first `seen` tokens (of `tokens`): fp64 softmax attention and how
        far a kernel that rounds as documented may be off, element by element."""
        k, v, vs = self.vals["k"], self.vals["v"], self.vscale
        if tokens is not None:
            k, v, vs = k[tokens], v[tokens], vs[tokens]
        k, v, vs = k[:seen], v[:seen], vs[:seen]
        if k.shape[0] == 0:
            return torch.zeros(D, dtype=torch.float64), torch.zeros(D, dtype=torch.float64)
        q = q.double()
        s = (k @ q) * scale
        w = torch.exp(s - s.max())
        w = w / w.sum()
        out = w @ v
        # scores: 128 products summed in fp32 and three more roundings of the sum of magnitudes; the exponent's argument
        # (log2 domain, up to the spread of the scores and 64 for the block scales) is rounded four times
        mag = (k.abs() @ q.abs()) * abs(scale)
        ds = 2.0 ** -24 * (131 * mag + 4 * (s.abs().max() + mag.max() + 64))
        dev = (v - out).abs()
        err = 2 * (w * ds) @ dev
        # weights rounded to fp16: half a step each, or for the smallest half of the smallest step, 2^-25 of an offset at
        # most 2^4 above the largest weight (weights carry the value scale)
        wv = w * vs
        small = torch.minimum(wv, 2.0 ** -21 * wv.max()) / vs
        err += (w * 2.0 ** -11 + small) @ v.abs()
        # fp32 sums over the tokens, and the hardware's exp2, log2 and reciprocal (2^-22 each)
        err += (k.shape[0] * 2.0 ** -24 + 6 * 2.0 ** -22) * (w @ v.abs())
        # the output's rounding (subnormal outputs: half of the smallest fp16 step)
        return out, err + out_eps / 2 * (out.abs() + err) + 2.0 ** -25


def choose(ref, q, n, sink, recent):
    """Selected finished blocks of one kv head for its queries fp16 [G, 128]: fp32 scores as defined."""
    nb = ref.nb
    if nb == 0:
        return []
    lo, hi = ref.codes["k"].amin(1), ref.codes["k"].amax(1)
    best = None
    for row in stored(q):
        amax = row.float().abs().max()
        q8 = torch.round(row.float() * factor(amax)).to(torch.int64)
        dot = torch.maximum(q8 * lo, q8 * hi).sum(1)
        sc = dot.float() * (amax * STEP)
        best = sc if best is None else torch.maximum(best, sc)
    score = (best * ref.scales["k"] + 0.0).tolist()
    forced = set(range(min(sink, nb))) | set(range(max(0, nb - recent), nb))
    return sorted(sorted(range(nb), key=lambda j: (j not in forced, -score[j], j))[:n])


def v_tokens():
    """Token of every value position of a block."""
    return [32 * ((p >> 3) & 1) + 16 * ((p >> 2) & 1) + 4 * (p >> 4) + (p & 3) for p in range(BLOCK)]


SCALE = 1.0 / math.sqrt(D)
