"""extend where pages run out: what a sequence holds stays its own, whoever else names its last page."""

import random

import pytest
import torch

from paged_books import FULL, Books, Contents, random_calls

pytestmark = pytest.mark.gpu


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Both:
    """A PagedKV and the lists, through the same calls."""

    def __init__(self, pages, seqs, width, page, dtype):
        from leankv_amd.paged import PagedKV

        self.cache = PagedKV(2, 1, pages, seqs, width * page, page_size=page, dtype=dtype)
        self.lists = Contents(Books(pages, seqs, width, page))

    def call(self, name, *args):
        if name == "fork":
            self.cache.fork(*(None if a is None else _ints(a) for a in args))
            self.lists.fork(*args)
            return
        new = args[0]
        at = [sum(new[:s]) for s in range(len(new) + 1)]
        added = self.lists.extend(new)
        self.cache.extend(_ints(at))
        x = torch.zeros(at[-1])
        for s, tokens in enumerate(added):
            x[at[s]:at[s] + len(tokens)] = torch.tensor([float(t % 251) for t in tokens])
        for layer in range(2):
            k = (x + layer).to(self.cache.dtype).cuda().view(-1, 1, 1).expand(-1, 1, 128)
            self.cache.store(layer, k, -k, _ints(at))

    def compare(self, what):
        cache, t = self.cache, self.lists.tables
        assert cache.taken.tolist() == t.taken, what
        assert torch.equal(cache.table.cpu(), t.table()) and cache.lens.tolist() == t.lens, what
        assert cache.refs.tolist() == t.refs(), what
        for layer in range(2):
            k, v = cache.read(layer, cache.max_len)
            want = torch.zeros(cache.max_seqs, cache.max_len)
            for s, tokens in enumerate(self.lists.tokens):
                want[s, :len(tokens)] = torch.tensor([float(x % 251) + layer for x in tokens])
            assert torch.equal(k[:, 0, :, 3].cpu().float(), want) and torch.equal(v, -k), what


@pytest.mark.parametrize("case", range(len(FULL)))
def test_full_pools(cuda, case):
    pages, seqs, width, page, calls = FULL[case]
    both = Both(pages, seqs, width, page, torch.float16)
    for i, call in enumerate(calls):
        both.call(*call)
        both.compare((case, i, call))


@pytest.mark.parametrize("pages,seqs,width,page,dtype", [
    (3, 3, 2, 16, torch.float16), (5, 6, 3, 16, torch.bfloat16), (9, 8, 4, 32, torch.float16), (40, 40, 3, 16, torch.bfloat16)])
def test_walks_in_full_pools(cuda, pages, seqs, width, page, dtype):
    for seed in range(10):
        both = Both(pages, seqs, width, page, dtype)
        calls = random_calls(random.Random(100 * page + seed), pages, seqs, width, page, 25)
        next(calls)
        try:
            while True:
                call = calls.send(both.lists.tables.lens)
                both.call(*call)
                both.compare((seed, call))
        except StopIteration:
            pass


def test_free_takes_numbers(cuda):
    """A list of truth values is no list of sequences: [True, False] would be sequences 1 and 0."""
    from leankv_amd._lib import LeanKVError
    from leankv_amd.paged import PagedKV

    cache = PagedKV(1, 1, 8, 3, 64, page_size=16)
    cache.extend(_ints([0, 5, 10, 15]))
    for bad in ([True, False, True], True, [3], [-1], [0.0]):
        with pytest.raises(LeanKVError, match="sequence numbers"):
            cache.free(bad)
    assert cache.lens.tolist() == [5, 5, 5]
    cache.free([1, 1])
    cache.free(2)
    assert cache.lens.tolist() == [5, 0, 0]
