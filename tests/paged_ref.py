"""Plain 64-bit forms for the tests of the 16-bit paged cache: attention with the bound that the kernels' roundings give, and
a model of the page tables as Python lists."""

import math

import torch

D = 128


def attention(q, k, v, seen, scale=None):
    """(out, bound) of q [m, D] over k, v [n, D] in float64: row i sees tokens 0 .. seen[i] - 1; zeros where it sees none.

    bound: with u half a step of the type and p the softmax weights, A = sum p |v|: the weights are rounded in the numerator and
    in their sum, sum p (1 + e) v / sum p (1 + e) with |e| <= u, which is off by u sum p |v - out| <= u (A + |out|) <= 2 u A;
    the output's rounding gives u |out| <= u A (and 2^-25 where fp16 is subnormal); fp32 scores of 128 products are off by at most
    129 * 2^-24 * scale * sum |q||k|, the weights by that relative error (numerator and denominator) and 2^-22 of the
    exponential; fp32 sums over n tokens by n 2^-24 A; an fp16 weight below 2^-14 is off by 2^-25, the largest is at least 2^6
    (a quarter of that where partial sums move their offsets): n 2^-29 max|v|."""
    scale = 1 / math.sqrt(D) if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    q, k, v = q.double(), k.double(), v.double()
    n = k.shape[0]
    hide = torch.arange(n, device=q.device).unsqueeze(0) >= seen.unsqueeze(1)
    if n == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    s = (q @ k.t() * scale).masked_fill(hide, -math.inf)
    size = (q.abs() @ k.abs().t() * abs(scale)).masked_fill(hide, 0.0).amax(1, keepdim=True)
    top = s.amax(1, keepdim=True).clamp(min=-1e300)
    w = torch.exp(s - top).masked_fill(hide, 0.0)
    total = w.sum(1, keepdim=True)
    w = w / torch.where(total > 0, total, 1.0)
    out, A = w @ v, w @ v.abs()
    relative = 2 * (129 * 2.0 ** -24 * size + 2.0 ** -22)
    bound = (3 * u + relative + n * 2.0 ** -24) * A + tiny + n * 2.0 ** -29 * v.abs().amax()
    return out, bound


def packed(q, k, v, starts, scale=None, kv_lens=None, paged=None):
    """(out, bound) of packed rows [T, heads, D]; k, v packed too, or paged(b) gives (k, v) [tokens, kv heads, D]."""
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for b in range(len(starts) - 1):
        a, m = starts[b], starts[b + 1] - starts[b]
        kk, vv = (k[a:a + m], v[a:a + m]) if paged is None else paged(b)
        n, G = kk.shape[0], q.shape[1] // kk.shape[1]
        m = min(m, n)
        seen = n - m + 1 + torch.arange(m)
        for h in range(q.shape[1]):
            out[a:a + m, h], bound[a:a + m, h] = attention(q[a:a + m, h], kk[:, h // G], vv[:, h // G], seen, scale)
    return out, bound


def check(got, want, bound, what=""):
    got = got.cpu().double()
    assert got.shape == want.shape
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d outside the bound, worst %.3g over %.3g" % (
        what, int(bad.sum()), bad.numel(), float(torch.nan_to_num(off, nan=math.inf)[bad].max()),
        float(bound[bad].min()))


class Tables:
    """What extend, fork and compact do, one sequence after the other."""

    def __init__(self, pages, seqs, width, page):
        self.pages, self.width, self.page = pages, width, page
        self.rows, self.lens, self.taken = [[] for _ in range(seqs)], [0] * seqs, [0] * seqs
        self.copies, self.moves = [], {}

    def refs(self):
        r = [0] * self.pages
        for row in self.rows:
            for p in row:
                r[p] += 1
        return r

    def extend(self, new):
        page, refs = self.page, self.refs()
        cap = self.width * page
        new = [n if 0 < n <= cap - have else 0 for n, have in zip(new, self.lens)]
        writers = {}
        for s, n in enumerate(new):
            if n and self.lens[s] % page:
                writers.setdefault(self.rows[s][-1], []).append(s)
        free = [p for p, r in enumerate(refs) if r == 0]
        self.copies, at = [], 0
        for s, n in enumerate(new):
            have = self.lens[s]
            last = self.rows[s][-1] if n and have % page else None
            copy = last is not None and refs[last] > 1 and not (writers[last][0] == s and len(writers[last]) == refs[last])
            need = -(-(have + n) // page) - len(self.rows[s]) + copy
            begin, at = at, at + need
            if need and at > len(free):
                self.taken[s] = 0
                continue
            got = free[begin:at]
            if copy:
                self.copies.append((last, got[0], have % page))
                self.rows[s][-1] = got.pop(0)
            self.rows[s] += got
            self.lens[s] += n
            self.taken[s] = n

    def fork(self, parent=None, cut=None):
        rows, lens = [], []
        for s in range(len(self.rows)):
            p = s if parent is None else parent[s]
            n = self.lens[p] if 0 <= p < len(self.rows) else 0
            if cut is not None:
                n = min(n, max(cut[s], 0))
            rows.append(self.rows[p][:-(-n // self.page)] if n else [])
            lens.append(n)
        self.rows, self.lens, self.taken = rows, lens, [0] * len(lens)

    def compact(self):
        used = sorted({p for row in self.rows for p in row})
        n = len(used)
        holes = sorted(set(range(n)) - set(used))
        self.moves = dict(zip([p for p in used if p >= n], holes))
        self.rows = [[self.moves.get(p, p) for p in row] for row in self.rows]
        return n

    def table(self):
        return torch.tensor([row + [-1] * (self.width - len(row)) for row in self.rows], dtype=torch.int32)
