"""Searches whose stop tokens are many or likely: the ends take no place from the beams that go on (no GPU, plain stand-ins)."""
import math

import pytest
import torch

from msa_b200 import beam as B, lm_ops as K
from msa_b200.cache import SequenceStateCache
from msa_b200.scheduler import Scheduler, SequenceRequest
from tests.beam_util import plain_search, plain_topk
from tests.test_beam_search_host import HashModel, plain_reorder, same


@pytest.fixture(autouse=True)
def plain(monkeypatch):
    def topk(logits, scores, k, stop=None):
        assert 1 <= k <= min(K.BEAM_MAX_K, scores.shape[1] * logits.shape[1]) and logits.shape[0] == scores.numel()
        return plain_topk(logits, scores, k, stop)
    monkeypatch.setattr(K, "beam_topk", topk)
    monkeypatch.setattr(SequenceStateCache, "reorder", plain_reorder)


@pytest.mark.parametrize("beams", [3, 24, 32])
@pytest.mark.parametrize("stop", [(4, 9), (0, 5, 7), (1, 2, 3, 4, 5, 6, 7, 8)])
@pytest.mark.parametrize("favour,penalty", [(1.0, 1.0), (1.0, 2.0), (6.0, 1.0)])
def test_likely_ends(beams, stop, favour, penalty):
    """Logits close to each other, the stop tokens' a little higher: they fill the best places, and the search goes on beside them."""
    model = HashModel(vocab=41, seed=beams)
    model.mix *= 0.3
    model.mix[:, list(stop)] += favour
    s = Scheduler(model, max_batch=2 * beams, max_len=40, portion=3)
    reqs = [SequenceRequest(p, 6, eos_token_ids=list(stop), beams=beams, length_penalty=penalty) for p in ([3, 1, 4, 1, 5], [2, 1])]
    for r in reqs:
        s.submit(r)
    s.run()
    for r in reqs:
        same(r, plain_search(model.log_probs(r.tokens), beams, 6, stop, penalty))


def test_one_choice_while_it_is_enough(monkeypatch):
    """A search whose stop tokens cannot fill the 64 places is one choice, from the logits as they are."""
    seen, topk = [], K.beam_topk
    monkeypatch.setattr(K, "beam_topk", lambda x, *a, **kw: seen.append(x) or topk(x, *a, **kw))
    x = torch.randn((32, 50), generator=torch.Generator().manual_seed(1))
    for beams, stop in ((32, [7]), (21, [7, 8]), (16, [1, 2, 3]), (32, [])):
        seen.clear()
        assert B.advance(x[:beams], [(B.BeamSearch(beams, 9, stop), range(beams))]) == [False]
        assert len(seen) == 1 and seen[0].data_ptr() == x.data_ptr()


@pytest.mark.parametrize("kind", ["nothing but ends", "no ends", "infinite", "nan", "outside"])
def test_rows_of_a_kind(kind):
    """Stop tokens that cannot come, that alone can come, that the vocabulary does not have; rows that count for nothing."""
    beams, stop = 32, [3, 4, 5]
    x = torch.randn((beams, 40), generator=torch.Generator().manual_seed(2))
    x[:, stop] += 6.0
    if kind == "nothing but ends":
        x[:, 6:] = x[:, :3] = -math.inf
    if kind == "no ends":
        x[:, 3:6] = -math.inf
    if kind == "infinite":
        x[1, 4] = math.inf
    if kind == "nan":
        x[1, 5] = math.nan
    if kind == "outside":
        stop = [-1, 3, 4, 40, 99]
    kept = x.clone()
    search = B.BeamSearch(beams, 9, stop)
    search.tokens, search.scores = [[0]] * beams, [-0.1 * i for i in range(beams)]
    over = B.advance(x, [(search, range(beams))])
    assert torch.equal(x.nan_to_num(7.0), kept.nan_to_num(7.0))                    # the logits stay as they were
    lp = torch.log_softmax(x.double(), 1)
    lp[lp.isnan().any(1) | (x == math.inf).any(1)] = -math.inf
    total = lp + torch.tensor(search_scores(beams), dtype=torch.float64)[:, None]
    cand = sorted([(-float(total[b, t]), b, t) for b in range(beams) for t in range(40) if total[b, t] > -math.inf])
    live = [(b, t) for _, b, t in cand if t not in stop][:beams]
    rates = [total[b, t] / 2 for _, b, t in cand[:beams] if t in stop]
    assert over == [not live or (len(rates) == beams and float(rates[-1]) >= float(total[live[0]]) / 2)]
    assert [(b, t) for b, t in zip(search.parents, search.next_tokens) if b >= 0] == live
    assert [t[-1] for _, t in search.ended] == [t for _, b, t in cand[:beams] if t in stop]


def search_scores(beams):
    return torch.tensor([-0.1 * i for i in range(beams)], dtype=torch.float32).tolist()


def test_places_without_a_continuation_do_not_end():
    """-1, which some tokenizers have for no end token, is what stands in places left over."""
    inf = math.inf
    s = B.BeamSearch(3, 5, stop=[-1, 2])
    left = (-inf, -1, -1)
    assert not s.update([(-1.0, 0, 1), left, left], [(-1.0, 0, 1), left, left]) and s.ended == []
    assert s.update([(-1.5, 0, 2), left, left], [left, left, left]) and s.ended == [(-0.75, [1, 2])]
