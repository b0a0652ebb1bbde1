"""Beam search over models on state slots: what a search remembers on the host.  The choice itself (``lm_ops.beam_topk``) and the moving
of states (``SequenceStateCache.reorder_beams``) are kernels; ``scheduler.Scheduler`` drives them beside its other requests."""
from __future__ import annotations

import math
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import lm_ops as K


class BeamSearch:
    """One prompt's beams: their tokens and scores (sums of log probabilities), and the continuations that ended.

    A continuation that ends counts while it is among the best ``beams``; an ended one is rated by its score divided by
    ``tokens ** length_penalty``.  The search is over when the ``beams`` best that ended are rated no lower than the best live beam
    would be by now, when no beam is left, or at ``max_new_tokens``, where live beams count as ended."""

    def __init__(self, beams: int, max_new_tokens: int, stop: Sequence[int] = (), length_penalty: float = 1.0):
        self.beams, self.max_new_tokens, self.length_penalty = beams, max_new_tokens, length_penalty
        self.stop: Tuple[int, ...] = tuple(sorted(set(stop)))
        self.tokens: List[List[int]] = [[] for _ in range(beams)]
        self.scores: List[float] = [0.0] + [-math.inf] * (beams - 1)      # one prompt: one beam to begin with
        self.ended: List[Tuple[float, List[int]]] = []                    # best first

    def _rate(self, score: float, n: int) -> float:
        return score / n ** self.length_penalty

    def _end(self, score: float, tokens: List[int]) -> None:
        self.ended.append((self._rate(score, len(tokens)), tokens))
        self.ended.sort(key=lambda e: -e[0])                               # stable: equals stay in the order they came
        del self.ended[self.beams:]

    def update(self, candidates, live) -> bool:
        """``candidates`` and ``live``: (score, beam, token) lists as ``beam_topk`` returns them.  True when the search is over; else
        ``parents`` and ``next_tokens`` say how the beams go on."""
        for score, beam, token in candidates[:self.beams]:
            if beam >= 0 and token in self.stop:                            # -1: a place without a continuation
                self._end(score, self.tokens[beam] + [token])
        self.parents = [beam for _, beam, _ in live]
        self.next_tokens = [max(token, 0) for _, _, token in live]          # beams that are gone run along with any token
        self.tokens = [self.tokens[beam] + [token] if beam >= 0 else [] for _, beam, token in live]
        self.scores = [score for score, _, _ in live]
        best = max(self.scores)
        n = max(len(t) for t in self.tokens)
        if best > -math.inf and n >= self.max_new_tokens:
            for score, tokens in zip(self.scores, self.tokens):
                if score > -math.inf:
                    self._end(score, tokens)
            return True
        return best == -math.inf or (len(self.ended) == self.beams and self.ended[-1][0] >= self._rate(best, n))

    @property
    def choices(self) -> int:
        """Continuations to ask for: enough for ``beams`` that do not end, if ``beam_topk`` gives that many (``choose`` sees to it
        that no more are needed)."""
        return min(K.BEAM_MAX_K, self.beams * (1 + len(self.stop)))


def choose(x: torch.Tensor, scores: torch.Tensor, k: int, stop: Sequence[int]):
    """``beam_topk`` of the ``k`` best, of which ``beams`` go on whatever the others are: stop tokens take at most ``len(stop)`` places a
    beam.  Where that is more than ``beam_topk`` gives, the best are chosen by themselves, and for the beams that go on a row's stop
    tokens are one of their joint probability: log softmax stays what it was (but for the rounding of that one logit), and one place
    a beam is enough; the first three tables then hold ``beams`` places.  ``stop`` is a list on the host."""
    beams, vocab = scores.shape[1], x.shape[1]
    ids = lambda tokens: torch.tensor(tokens, dtype=torch.int32, device=x.device)
    if k >= min(beams * (1 + len(stop)), beams * vocab):
        return K.beam_topk(x, scores, k, ids(stop))
    known = [t for t in stop if 0 <= t < vocab]
    one = x.float()
    if len(known) > 1:
        at = ids(known).long()
        joint = torch.logsumexp(one[:, at], 1)
        one = one.index_fill(1, at, -math.inf)
        one[:, known[0]] = joint
    live = K.beam_topk(one, scores, min(2 * beams, beams * vocab), ids(known[:1]))[3:]
    return (*K.beam_topk(x, scores, min(beams, k)), *live)


def advance(logits: torch.Tensor, searches: Sequence[Tuple[BeamSearch, Sequence[int]]]) -> List[bool]:
    """Lets every search choose from its rows of ``logits`` (one row after the prompt, one per beam later); True where it is over."""
    groups: Dict[tuple, list] = {}
    for i, (s, _) in enumerate(searches):
        groups.setdefault((s.beams, s.stop, s.choices), []).append(i)
    over: List[Optional[bool]] = [None] * len(searches)
    for (beams, stop, k), members in groups.items():
        rows = [r for i in members for r in (list(searches[i][1]) * beams)[:beams]]
        if rows == list(range(rows[0], rows[0] + len(rows))):
            x = logits[rows[0]:rows[0] + len(rows)]
        elif len(set(rows)) == 1:
            x = logits[rows[0]:rows[0] + 1].expand(beams, -1)
        else:
            x = logits[torch.tensor(rows, device=logits.device)]
        scores = torch.tensor([searches[i][0].scores for i in members], dtype=torch.float32).to(logits.device)
        out = choose(x, scores, min(k, beams * x.shape[1]), stop)
        flat = torch.cat([t.view(torch.int32) for t in out], dim=1).cpu()          # one copy to the host
        parts = flat.split([t.shape[1] for t in out], dim=1)
        lists = [p.contiguous().view(torch.float32).tolist() if j % 3 == 0 else p.tolist() for j, p in enumerate(parts)]
        for n, i in enumerate(members):
            over[i] = searches[i][0].update(list(zip(*(p[n] for p in lists[:3]))), list(zip(*(p[n] for p in lists[3:]))))
    return over
