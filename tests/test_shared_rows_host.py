"""What `reorder_beams` remembers of the ring rows that beams share: a stand-in for the kernel that leaves those rows out, on the CPU, and
the rows of every sequence checked against what was written for it."""
import pytest
import torch

from msa_b200.cache import RingSpec, SequenceStateCache, window_of


def row_of(pos, first, rows):
    return pos if pos < first else first + (pos - first) % (rows - first)


def held(n, first, rows):
    """Positions of n whose rows are still there."""
    return [p for p in range(n) if p < first or p >= n - (rows - first)]


def reorder(self, slot, parent, length, shared=None):
    """``SequenceStateCache.reorder``, position by position: those that `shared` names are not copied."""
    out = slot.clone()
    for q in range(slot.shape[0]):
        s, p, n = slot[q].tolist(), parent[q].tolist(), int(length[q])
        spare, seen = [i for i in range(len(s)) if i not in p], set()
        for j, x in enumerate(p):
            own = x if x >= 0 and x not in seen else spare.pop(0)
            seen.add(x)
            out[q, j] = s[own]
            if x >= 0 and own != x:
                for i, t in self.ring.items():
                    first = window_of((self.specs[i].window, self.specs[i].first), self.max_len)[1]
                    for pos in held(n, first, t.shape[1]):
                        if pos >= int(shared[q, own, x]):
                            t[s[own], row_of(pos, first, t.shape[1])] = t[s[x], row_of(pos, first, t.shape[1])]
    return out, shared


class Lives:
    """Sequences on rings, and what was written for each of them."""

    def __init__(self, names, specs=(RingSpec(1, 16),), max_len=400, device="cpu"):
        self.cache = SequenceStateCache(list(specs), len(names), max_len, device, torch.float32)
        self.said, self.count = {s: [] for s in names}, 0
        for s in names:
            self.cache.acquire(s)

    def grow(self, **n):
        for s, k in n.items():
            for _ in range(k):
                self.count += 1
                pos = self.cache.length(s)
                for i, t in self.cache.ring.items():
                    t[self.cache.slot(s), row_of(pos, self.first(i), t.shape[1])] = float(self.count)
                if self.said[s] is not None:
                    self.said[s].append(self.count)
                self.cache.advance(s, 1)

    def first(self, i):
        return window_of((self.cache.specs[i].window, self.cache.specs[i].first), self.cache.max_len)[1]

    def move(self, *pairs):
        """(names, parents) of every question; a beam that goes on from nobody is not looked at until it follows somebody."""
        old = dict(self.said)
        self.cache.reorder_beams([g for g, _ in pairs], [p for _, p in pairs])
        for g, p in pairs:
            self.said.update({s: None if x < 0 else list(old[g[x]]) for s, x in zip(g, p)})
        self.check()

    def check(self):
        for s, said in self.said.items():
            if said is None:
                continue
            assert self.cache.length(s) == len(said), s
            for i, t in self.cache.ring.items():
                rows, first = t.shape[1], self.first(i)
                got = [int(t[self.cache.slot(s), row_of(p, first, rows), 0]) for p in held(len(said), first, rows)]
                assert got == [said[p] for p in held(len(said), first, rows)], (s, i)


@pytest.fixture(autouse=True)
def rows(monkeypatch):
    monkeypatch.setattr(SequenceStateCache, "reorder", reorder)


def test_other_groups_in_between():
    """c is moved in a group of its own in between: what b and c had in common is over."""
    m = Lives("abc")
    m.grow(a=5)
    m.move(("abc", [0, 0, 0]))
    m.grow(a=4, b=4, c=4)
    m.move(("abc", [0, 1, 1]))
    m.move(("ac", [0, 0]))
    m.grow(a=1, b=1, c=1)
    m.move(("abc", [0, 1, 1]))


def test_a_member_that_another_question_takes_along():
    m = Lives("abc", [RingSpec(1, None)])
    m.grow(a=10, c=10)
    m.move(("ab", [0, 0]))
    m.move(("bc", [1, 1]))
    m.move(("ab", [0, 0]))


def test_the_same_sequences_in_another_order():
    m = Lives("abc")
    m.grow(a=6)
    m.move(("abc", [0, 0, 0]))
    m.grow(a=3, b=3, c=3)
    m.move(("abc", [1, 1, 2]))
    m.grow(a=2, b=2, c=2)
    m.move(("cab", [0, 0, 0]))
    m.grow(a=2, b=2, c=2)
    m.move(("abc", [0, 0, 2]))
    m.grow(a=20, b=20, c=20)
    m.move(("abc", [2, 0, 0]))


def test_only_what_a_call_names_is_forgotten():
    m = Lives("abcdef")
    m.grow(a=3, c=4, e=5)
    m.move(("ab", [0, 0]), ("cd", [0, 0]), ("ef", [0, 0]))
    m.move(("bc", [-1, 1]), ("ef", [1, 0]))
    assert set(m.cache._shared) == {("b", "c"), ("e", "f")} and m.cache._shared["e", "f"] == [[5, 5], [5, 5]]


@pytest.mark.parametrize("ahead", [3, 15, 30])
def test_a_beam_that_nobody_goes_on_from_is_ahead(ahead):
    """Its ring has written over rows that both had in common."""
    m = Lives("ab", [RingSpec(1, 16), RingSpec(1, 4, first=2), RingSpec(1, None)])
    m.grow(a=20)
    m.move(("ab", [0, 0]))
    m.grow(a=1, b=ahead)
    m.move(("ab", [0, 0]))


@pytest.mark.parametrize("lead", [-7, 9, 25])
def test_a_beam_of_another_length_is_left_and_then_taken(lead):
    """b goes on from nobody, its length becomes the question's, and only the step after that copies into its slot."""
    m = Lives("abc")
    m.grow(a=20)
    m.move(("abc", [0, 0, 0]))
    m.grow(a=max(1, 1 - lead), c=max(1, 1 - lead), b=max(1, 1 + lead))
    m.move(("abc", [0, -1, 2]))
    m.grow(a=1, b=1, c=1)
    m.move(("abc", [0, 2, 0]))


@pytest.mark.parametrize("seed", range(40))
def test_lives_of_every_kind(seed):
    """Groups of any members in any order, lengths that part and meet, beams that nobody goes on from."""
    import random
    rng = random.Random(seed)
    m = Lives("abcdef", [RingSpec(1, 7, first=3), RingSpec(1, 11), RingSpec(1, None)])
    m.grow(**{s: rng.randint(0, 9) for s in "abcdef"})
    groups = ["abc", "de", "f"]
    for _ in range(30):
        if rng.random() < 0.15:
            names, size = rng.sample("abcdef", 6), rng.randint(1, 3)
            groups = ["".join(names[at:at + size]) for at in range(0, 7 - size, size)]
        pairs = []
        for g in groups:
            n = m.cache.length(rng.choice(g))
            from_ = [i for i, s in enumerate(g) if m.said[s] is not None and m.cache.length(s) == n]
            pairs.append((g, [rng.choice(from_) if from_ and rng.random() < 0.8 else -1 for _ in g]))
        for size in {len(g) for g in groups}:
            m.move(*[p for p in pairs if len(p[0]) == size])
        one = rng.randint(0, 4)
        m.grow(**{s: one if rng.random() < 0.8 else rng.randint(0, 14) for s in "abcdef"})


def test_tables_moved_by_hand(monkeypatch):
    """`reorder` itself, whose slots only the device knows: nothing that was known by sequence counts behind it."""
    import contextlib
    from torch._subclasses.fake_tensor import FakeTensorMode
    from msa_b200 import _cabi_lm as A
    monkeypatch.undo()
    seen = []
    monkeypatch.setattr(A, "call", lambda name, *a: seen.append(name))
    monkeypatch.setattr(A, "stream_ptr", lambda device=None: 0)
    monkeypatch.setattr(A, "ptr", lambda t: 0)
    monkeypatch.setattr(A, "on_device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(SequenceStateCache, "_state_parts", lambda self: torch.empty((2, 6), dtype=torch.int64))
    with FakeTensorMode():
        c = SequenceStateCache([RingSpec(6, 8)], 4, 50, "cuda:0", torch.float32)
        c._shared["a", "b"] = [[3, 3], [3, 3]]
        t = torch.empty((1, 2), dtype=torch.int32, device="cuda:0")
        c.reorder(t, t, t[0, :1])
    assert seen == ["msa_lm_reorder"] and not c._shared
