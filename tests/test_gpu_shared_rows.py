"""Lives of sequences whose beams are regrouped, run ahead, and are moved by tables in between: the rows of every one, on the device."""
import random

import pytest
import torch

from msa_b200.cache import RingSpec
from tests.test_shared_rows_host import Lives

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("seed", range(6))
def test_lives(seed):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    rng = random.Random(seed)
    m = Lives("abcdef", [RingSpec(1, 7, first=3), RingSpec(1, 11), RingSpec(1, None)], device=DEV)
    m.grow(**{s: rng.randint(0, 9) for s in "abcdef"})
    groups = ["abc", "de", "f"]
    for _ in range(16):
        if rng.random() < 0.15:
            names, size = rng.sample("abcdef", 6), rng.randint(1, 3)
            groups = ["".join(names[at:at + size]) for at in range(0, 7 - size, size)]
        if rng.random() < 0.2:                                     # one by hand: y follows x
            x, y = rng.sample("abcdef", 2)
            if m.said[x] is not None and m.said[y] is not None and m.cache.length(x) == m.cache.length(y):
                i = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
                slot, _ = m.cache.reorder(i(m.cache.slot(x), m.cache.slot(y))[None], i(0, 0)[None], i(m.cache.length(x)))
                assert slot.tolist() == [[m.cache.slot(x), m.cache.slot(y)]]
                m.said[y] = list(m.said[x])
                m.check()
        pairs = []
        for g in groups:
            n = m.cache.length(rng.choice(g))
            from_ = [i for i, s in enumerate(g) if m.said[s] is not None and m.cache.length(s) == n]
            pairs.append((g, [rng.choice(from_) if from_ and rng.random() < 0.8 else -1 for _ in g]))
        for size in {len(g) for g in groups}:
            m.move(*[p for p in pairs if len(p[0]) == size])
        one = rng.randint(0, 4)
        m.grow(**{s: one if rng.random() < 0.8 else rng.randint(0, 14) for s in "abcdef"})
