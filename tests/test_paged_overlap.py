"""Which buffers count as lying over each other, against the addresses of their numbers; no GPU."""

import random

import torch

from leankv_amd.paged.packed import apart, meet


def _numbers(t):
    """Where every eighth number of t lies (rows and strides are multiples of eight)."""
    return {t.storage_offset() + i * t.stride(0) + j * t.stride(1) + k
            for i in range(t.shape[0]) for j in range(t.shape[1]) for k in range(0, t.shape[2], 8)}


def test_parts_of_one_projection_are_apart():
    x = torch.zeros(9, 8, 128, dtype=torch.float16)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    for a, b in ((q, k), (q, v), (k, v)):
        assert not meet(a, b) and not meet(b, a) and apart(a, b) is a
    assert meet(q, x[:, 3:5]) and meet(q, q) and meet(q, x[:, 3:7]) and not meet(q[:4], q[4:]) and meet(q[:5], q[4:])
    assert not meet(x, torch.zeros_like(x)) and not meet(x[:0], x)
    y = apart(x, x)
    assert y.data_ptr() != x.data_ptr() and torch.equal(x, y)
    heads_first = torch.zeros(4, 9, 128, dtype=torch.float16).transpose(0, 1)
    assert meet(heads_first, heads_first) and not meet(heads_first, q)


def test_nothing_in_common_is_missed():
    """Random views of a buffer: those that have a number in common always meet."""
    rng = random.Random(3)
    base = torch.zeros(12000, dtype=torch.bfloat16)
    apart_too = 0
    for _ in range(1500):
        views = []
        same = rng.choice((None, 128 * rng.randint(1, 6)))
        for _ in range(2):
            n, h = rng.randint(1, 5), rng.randint(1, 4)
            r, hs = same or 8 * rng.randint(0, 90), rng.choice((128, 128, 8 * rng.randint(0, 60)))
            at = 8 * rng.randint(0, 1000)
            if at + r * (n - 1) + hs * (h - 1) + 128 <= base.numel():
                views.append(base.as_strided((n, h, 128), (r, hs, 1), at))
        if len(views) < 2:
            continue
        a, b = views
        if _numbers(a) & _numbers(b):
            assert meet(a, b) and meet(b, a), (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        else:
            apart_too += not meet(a, b)
    assert apart_too > 100
