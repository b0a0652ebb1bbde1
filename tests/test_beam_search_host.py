"""Beam search on the host: what a search remembers, how the scheduler runs it beside other requests, the bookkeeping of slots.  The
kernels are replaced by plain restatements; states are tensors on the CPU."""
import math
from types import SimpleNamespace

import pytest
import torch

from msa_b200 import beam as B, lm_ops as K
from msa_b200.cache import PackedStep, RecurrentSpec, RingSpec, SequenceStateCache
from msa_b200.scheduler import Scheduler, SequenceRequest
from tests.beam_util import plain_search, plain_topk


def plain_reorder(self, slot, parent, length, shared=None):
    """``SequenceStateCache.reorder`` by copying whole slots."""
    out = slot.clone()
    for q in range(slot.shape[0]):
        s, p = slot[q].tolist(), parent[q].tolist()
        spare, seen = [i for i in range(len(s)) if i not in p], set()
        for j, x in enumerate(p):
            own = x if x >= 0 and x not in seen else spare.pop(0)
            seen.add(x)
            out[q, j] = s[own]
            if x >= 0 and own != x:
                for d in (self.ring, self.state, self.conv, self.shift):
                    for t in d.values():
                        t[s[own]] = t[s[x]]
                self.last_token[s[own]] = self.last_token[s[x]]
    self.reordered.append((slot.tolist(), parent.tolist(), length.tolist(), shared.tolist()))
    return out, None


class HashModel:
    """Logits from everything a sequence was fed, kept in its slot's state alone: a slot mixed up, or a state that did not follow its
    beam, shows in the next scores."""
    device = torch.device("cpu")

    def __init__(self, vocab=13, seed=0):
        self.config = SimpleNamespace(vocab=vocab, windows=())
        self.mix = torch.randn(64, vocab, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 1.5

    def new_cache(self, n_slots, max_len):
        c = SequenceStateCache([RecurrentSpec(1, 1, 1), RingSpec(1, 8)], n_slots, max_len, "cpu", torch.float32)
        c.reordered = []
        return c

    def fed(self, state, token):
        return (state * 5 + token + 1) % 64

    def run(self, entries, cache):
        step = PackedStep(entries, cache, ())
        rows = []
        for s, toks, want in entries:
            t = cache.state[0][cache.slot(s)]
            if cache.length(s) == 0:
                t.zero_()
            for j, tok in enumerate(toks):
                t.fill_(self.fed(int(t), tok))
                if j in want:
                    rows.append(self.mix[int(t)])
        step.commit(cache)
        return torch.stack(rows).float() if rows else torch.zeros(0, self.config.vocab)

    def log_probs(self, prompt):
        def of(toks):
            state = 0
            for t in list(prompt) + list(toks):
                state = self.fed(state, t)
            return torch.log_softmax(self.mix[state].float().double(), 0)
        return of

    def check_status(self):
        pass


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(K, "beam_topk", plain_topk)
    monkeypatch.setattr(SequenceStateCache, "reorder", plain_reorder)


def same(request, want):
    assert [t for _, t in request.results] == [t for _, t in want]
    assert all(abs(a - b) < 1e-5 for (a, _), (b, _) in zip(request.results, want)) and request.output == want[0][1]


@pytest.mark.parametrize("beams", [2, 3, 7])
@pytest.mark.parametrize("stop,penalty", [((), 1.0), ((4,), 1.0), ((4, 9), 0.0), ((0, 5, 7), 2.0)])
def test_a_search_is_the_plain_one(plain, beams, stop, penalty):
    model = HashModel()
    s = Scheduler(model, max_batch=beams, max_len=40, portion=3)
    for prompt in ([3, 1, 4, 1, 5], [2]):
        r = SequenceRequest(prompt, 9, eos_token_ids=list(stop), beams=beams, length_penalty=penalty)
        s.submit(r)
        assert s.run() == [r] and r.finished and s.cache.free_slots == beams and not s.cache._shared
        same(r, plain_search(model.log_probs(prompt), beams, 9, stop, penalty))


def test_searches_run_beside_other_requests(plain):
    """Searches of several sizes, greedy requests and long prompts share steps; slots go from one to the next."""
    model = HashModel(seed=3)
    s = Scheduler(model, max_batch=9, max_len=40, portion=4, step_tokens=11)
    reqs = [SequenceRequest([i + 1] * n, k, beams=b, eos_token_ids=e) for i, (n, k, b, e) in enumerate(
        [(5, 6, 4, [2]), (3, 8, 1, []), (1, 5, 4, [2]), (9, 4, 2, []), (2, 7, 1, []), (4, 6, 3, [1, 2]), (1, 1, 5, []), (6, 5, 9, [0])])]
    for r in reqs:
        s.submit(r)
    done = s.run()
    assert sorted(r.id for r in done) == list(range(8)) and s.cache.free_slots == 9
    for r in reqs:
        if r.beams > 1:
            same(r, plain_search(model.log_probs(r.tokens), r.beams, r.max_new_tokens, r.eos_token_ids))
        else:
            assert r.output == plain_search(model.log_probs(r.tokens), 1, r.max_new_tokens)[0][1]
    assert any(len(slots) > 1 for slots, _, _, _ in s.cache.reordered)       # two searches of a size moved in one call


def test_cancelled_and_refused_searches(plain):
    model = HashModel()
    s = Scheduler(model, max_batch=4, max_len=40)
    r = SequenceRequest([1, 2], 9, beams=3)
    s.submit(r)
    s.step(), s.step()
    s.cancel(r.id)
    assert s.cache.free_slots == 4 and not s.busy and not s.cache._shared
    for bad in (SequenceRequest([1], 2, beams=0), SequenceRequest([1], 2, beams=5), SequenceRequest([1], 2, beams=2, temperature=0.5),
                SequenceRequest([1] * 39, 2, beams=2)):
        with pytest.raises(ValueError):
            s.submit(bad)
    s = Scheduler(model, max_batch=64, max_len=40)
    with pytest.raises(ValueError):
        s.submit(SequenceRequest([1], 2, beams=33))


def test_fewer_continuations_than_beams(plain):
    """A vocabulary smaller than the number of beams, and logits that leave one token: beams without a score run along and are not chosen."""
    model = HashModel(vocab=3)
    model.mix[:, 1:] = -math.inf
    s = Scheduler(model, max_batch=4, max_len=40)
    r = SequenceRequest([1], 4, beams=4)
    s.submit(r)
    s.run()
    assert [t for _, t in r.results] == [[0, 0, 0, 0]] and abs(r.results[0][0]) < 1e-6
    r = SequenceRequest([1], 4, beams=2, eos_token_ids=[0])               # nothing but the end
    s.submit(r)
    s.run()
    assert r.output == [0] and len(r.results) == 1
    model.mix[:] = -math.inf                                               # nothing at all
    r = SequenceRequest([1], 4, beams=2)
    s.submit(r)
    s.run()
    assert r.output == [] and r.results == [] and s.cache.free_slots == 4


def test_what_a_search_remembers():
    s = B.BeamSearch(2, 5, stop=[9, 9])
    assert s.stop == (9,) and s.choices == 4 and B.BeamSearch(32, 5, [1, 2]).choices == 64
    inf = math.inf
    assert not s.update([(-1.0, 0, 9), (-2.0, 0, 3), (-3.0, 0, 4), (-9.0, 0, 5)], [(-2.0, 0, 3), (-3.0, 0, 4)])
    assert s.ended == [(-1.0, [9])] and s.tokens == [[3], [4]] and s.parents == [0, 0] and s.next_tokens == [3, 4]
    # an end beyond the best two does not count; a beam that is gone goes on from nobody with any token
    assert not s.update([(-2.5, 0, 1), (-4.0, 1, 2), (-4.5, 1, 9)], [(-2.5, 0, 1), (-inf, -1, -1)])
    assert s.ended == [(-1.0, [9])] and s.parents == [0, -1] and s.next_tokens == [1, 0] and s.tokens == [[3, 1], []]
    # two ended, both rated above what the best live beam has by now
    assert s.update([(-2.6, 0, 9), (-4.0, 0, 2)], [(-4.0, 0, 2), (-inf, -1, -1)])
    assert [t for _, t in s.ended] == [[3, 1, 9], [9]]


def cache(n=8):
    c = SequenceStateCache([RingSpec(2, 6, first=1), RecurrentSpec(1, 2, 2)], n, 30, "cpu", torch.float32)
    c.reordered = []
    for d in (c.ring, c.state):
        for t in d.values():
            t.normal_(generator=torch.Generator().manual_seed(1))
    return c


def test_slots_follow_the_beams(plain):
    c = cache()
    a, b = [("a", j) for j in range(3)], [("b", j) for j in range(3)]
    for s in a + b:
        c.acquire(s)
    c.advance(a[0], 5), c.advance(b[0], 7)
    c.reorder_beams([a, b], [[0, 0, 0], [0, 0, 0]])
    assert [c.length(s) for s in a + b] == [5, 5, 5, 7, 7, 7] and c.reordered[-1][2:] == ([5, 7], [[[0] * 3] * 3] * 2)
    assert all(torch.equal(c.state[1][c.slot(s)], c.state[1][c.slot(a[0])]) for s in a)
    for s in a + b:
        c.advance(s, 1)
    before = [c.slot(s) for s in a]
    c.reorder_beams([a], [[2, 0, 2]])
    assert [c.slot(s) for s in a] == [before[2], before[0], before[1]] and c.reordered[-1][2:] == ([6], [[[5] * 3] * 3])
    for s in a:
        c.advance(s, 1)
    n = len(c.reordered)
    c.reorder_beams([a], [[0, 1, 2]])                                      # nobody moves: nothing is launched
    assert len(c.reordered) == n and c._shared[tuple(a)] == [[7, 5, 6], [5, 7, 5], [6, 5, 7]]
    for s in a:
        c.advance(s, 1)
    c.reorder_beams([a], [[0, -1, 1]])                                     # beam 1 goes on from nobody and takes the slot of beam 2
    held = [before[2], before[0], before[1]]
    assert [c.slot(s) for s in a] == [held[0], held[2], held[1]]
    assert c._shared[tuple(a)] == [[8, 6, 5], [6, 8, 5], [5, 5, 8]]
    c.release(a[1])
    assert tuple(a) not in c._shared and tuple(b) in c._shared
    c.reorder_beams([], [])


@pytest.mark.parametrize("bad", ["sizes", "parents", "parent range", "unknown", "twice", "lengths", "many", "count"])
def test_reordering_by_sequence_refuses(plain, bad):
    c = cache(40)
    a, b, p = ["a", "b"], ["c", "d"], [[0, 0], [1, 1]]
    for s in a + b:
        c.acquire(s)
    c.advance("a", 3)
    if bad == "sizes": b = ["c"]
    if bad == "parents": p = [[0, 0], [1]]
    if bad == "parent range": p = [[0, 2], [1, 1]]
    if bad == "unknown": b = ["c", "x"]
    if bad == "twice": b = ["c", "a"]
    if bad == "lengths": p = [[0, 1], [1, 1]]
    if bad == "many": a, b, p = [f"s{i}" for i in range(33)], None, [[0] * 33]
    if bad == "count": p = [[0, 0]]
    if bad == "many":
        for s in a:
            c.acquire(s)
    with pytest.raises(ValueError):
        c.reorder_beams([a, b] if b else [a], p)
    assert not c.reordered and c.length("a") == 3 and not c._shared


def test_engine_refuses_beams_over_a_memory(tmp_path):
    import json
    from msa_b200.engine import GenerateConfig, MSAEngine
    from msa_b200.memory import ModelConfig
    (tmp_path / "config.json").write_text(json.dumps({"architectures": ["MSAForCausalLM"], "msa_config": {}}))
    with pytest.raises(ValueError, match="num_beams"):
        MSAEngine(GenerateConfig(devices=[0], num_beams=2), ModelConfig(model_path=str(tmp_path)), start=False)


@pytest.mark.parametrize("rows,want", [([4], [4, 4, 4]), ([2, 3, 4], [2, 3, 4]), ([5, 1, 3], [5, 1, 3])])
def test_a_search_chooses_from_its_own_rows(rows, want, monkeypatch):
    """One row behind the prompt stands for every beam; later rows lie wherever the step put them."""
    from msa_b200 import beam
    seen = []

    def choose(x, scores, k, stop):
        seen.append(x.clone())
        table = lambda n: (torch.zeros((1, n)), torch.zeros((1, n), dtype=torch.int32), torch.zeros((1, n), dtype=torch.int32))
        return table(k) + table(3)
    monkeypatch.setattr(beam.K, "beam_topk", choose)
    logits = torch.arange(6.0)[:, None].expand(6, 8).contiguous()
    assert beam.advance(logits, [(beam.BeamSearch(3, 10), rows)]) == [False]
    assert seen[0][:, 0].tolist() == want
