"""The page tables as `extend` is to keep them where pages run out, and what the pages hold, as Python lists."""

from paged_ref import Tables


class Books(Tables):
    """Tables whose extend refuses, beside the sequences that there are no pages for, the one that would go on in a shared
    last page in their place: where one of them holds more tokens of that page, they are its own as before.  (Tables lets it
    write there; the two agree where nothing is refused.)"""

    def extend(self, new):
        before, had = [list(row) for row in self.rows], list(self.lens)
        super().extend(new)
        for s, n in enumerate(self.taken):
            if not n or not had[s] % self.page or self.rows[s][:len(before[s])] != before[s]:
                continue  # refused, at the end of a page, or with a copy of its own
            last, j = before[s][-1], len(before[s]) - 1
            for u, row in enumerate(before):
                asked = u < len(new) and 0 < new[u] <= self.width * self.page - had[u]
                if u != s and asked and not self.taken[u] and had[u] > had[s] and row[-1] == last and len(row) == j + 1:
                    self.rows[s], self.lens[s], self.taken[s] = before[s], had[s], 0
                    break


class Contents:
    """What the slots of the pages hold, beside what each sequence's tokens are."""

    def __init__(self, tables):
        self.tables, self.slots, self.count = tables, {}, 0
        self.tokens = [[] for _ in tables.rows]

    def extend(self, new):
        """Returns the new tokens of every sequence."""
        t = self.tables
        t.extend(new)
        for a, b, n in t.copies:
            for i in range(n):
                self.slots[b, i] = self.slots[a, i]
        added = []
        for s, n in enumerate(t.taken):
            added.append(list(range(self.count + 1, self.count + n + 1)))
            self.count += n
            for x in added[-1]:
                i = len(self.tokens[s])
                self.slots[t.rows[s][i // t.page], i % t.page] = x
                self.tokens[s].append(x)
        return added

    def fork(self, parent=None, cut=None):
        self.tables.fork(parent, cut)
        tokens = []
        for s in range(len(self.tokens)):
            p = s if parent is None else parent[s]
            kept = self.tokens[p] if 0 <= p < len(self.tokens) else []
            tokens.append(list(kept if cut is None else kept[:max(cut[s], 0)]))
        self.tokens = tokens

    def held(self, s):
        t = self.tables
        return [self.slots[t.rows[s][i // t.page], i % t.page] for i in range(t.lens[s])]


# (pages, max_seqs, width, page, calls): one page, its two sequences at 6 and 10 tokens, no other; the same after a step that had
# one of them wait and a fork that swaps them; three on a page of which the last waits; one that waits though another got a copy
FULL = [
    (1, 2, 1, 16, [("extend", [10, 0]), ("fork", [0, 0], [6, 10]), ("extend", [1, 1])]),
    (1, 2, 1, 16, [("extend", [5, 0]), ("fork", [0, 0], None), ("extend", [1, 1]), ("extend", [2, 0]), ("fork", [1, 0], None),
                   ("extend", [1, 1])]),
    (2, 3, 2, 16, [("extend", [12, 0, 0]), ("fork", [0, 0, 0], [3, 7, 12]), ("extend", [2, 1, 3])]),
    (3, 4, 2, 16, [("extend", [20, 0, 0, 0]), ("fork", [0, 0, 0, -1], [18, 20, 19, 0]), ("extend", [1, 1, 13, 0]),
                   ("extend", [1, 1, 1, 1])]),
]


def random_calls(rng, pages, seqs, width, page, steps):
    """Calls on a pool that is nearly full, with forks to different lengths: generator of (name, arguments), which is sent
    the present lengths."""
    lens = yield
    for _ in range(steps):
        what = rng.choice(("extend", "extend", "one", "fork", "fork", "cut"))
        if what == "one":
            call = "extend", [1 if n else 0 for n in lens]
        elif what == "extend":
            call = "extend", [rng.choice((0, 1, 1, rng.randint(0, 2 * page))) for _ in lens]
        elif what == "fork":
            kept = [rng.randint(-1 if rng.random() < 0.1 else 0, seqs - 1) for _ in lens]
            call = "fork", kept, [rng.randint(0, width * page) if rng.random() < 0.6 else width * page for _ in lens]
        else:
            call = "fork", None, [max(0, n - rng.randint(0, page)) for n in lens]
        lens = yield call
