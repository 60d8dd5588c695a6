"""The lists that the paged cache's tables are compared with where pages run out: no call changes the tokens of a sequence that
it does not name; no GPU."""

import random

import pytest

from paged_books import FULL, Books, Contents, random_calls
from paged_ref import Tables


def _go(tables, calls):
    c = Contents(tables)
    for call in calls:
        c.extend(call[1]) if call[0] == "extend" else c.fork(*call[1:])
    return c


def _kept(c):
    return all(c.held(s) == c.tokens[s] for s in range(len(c.tokens)))


def test_full_pools():
    pages, seqs, width, page, calls = FULL[0]
    c = _go(Books(pages, seqs, width, page), calls)
    assert c.tables.taken == [0, 0] and c.tables.lens == [6, 10] and _kept(c)
    pages, seqs, width, page, calls = FULL[1]
    c = _go(Books(pages, seqs, width, page), calls[:3])
    assert c.tables.taken == [1, 0]  # (as long as each other: the first goes on)
    for pages, seqs, width, page, calls in FULL:
        assert _kept(_go(Books(pages, seqs, width, page), calls))
    # deciding before it is known who is refused loses tokens
    assert not _kept(_go(Tables(*FULL[0][:4]), FULL[0][4]))


@pytest.mark.parametrize("pages,seqs,width,page", [(3, 3, 2, 4), (5, 6, 3, 4), (9, 8, 4, 4), (2, 5, 2, 8)])
def test_walks_in_full_pools(pages, seqs, width, page):
    lost = 0
    for seed in range(60):
        kept = True
        books, before = Contents(Books(pages, seqs, width, page)), Contents(Tables(pages, seqs, width, page))
        calls = random_calls(random.Random(seed), pages, seqs, width, page, 40)
        next(calls)
        try:
            while True:
                call = calls.send(books.tables.lens)
                for c in (books, before):
                    c.extend(call[1]) if call[0] == "extend" else c.fork(*call[1:])
                assert _kept(books), (seed, call)
                kept = kept and _kept(before)
                assert sum(books.tables.refs()) == sum(len(r) for r in books.tables.rows)
        except StopIteration:
            pass
        lost += not kept
    assert lost, "the walks do not reach the case"
