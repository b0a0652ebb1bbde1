"""The rows' sums behind a choice of beams, against 64 bits: at the ends of a row's range, and what they mean for candidates of two beams that are close."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# A term's exponential is good to 2^-22 (`ex2`) and its argument's fraction to 2^-26 (times log 2); five sums of 32 bits lie between the terms of a lane's
# sixteen logits, and 64 bits behind them.  Beyond 1e6, where logits are 2^-4 apart and more: `expf`, two steps of 2^-23, and fifteen sums.
SUM, FAR_SUM = 2.0 ** -22 + 2.0 ** -26 + 5 * 2.0 ** -24, 2 * 2.0 ** -23 + 15 * 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def rows(kind, g, n, vocab):
    x = torch.randn((n, vocab), generator=g, device=DEV)
    if kind == "flat": x.zero_()
    if kind == "wide": x *= 12
    if kind == "pair": x[:, 2:] = -90.0
    if kind == "tail": x -= 16.0
    if kind == "far tail": x -= 70.0
    if kind == "falling": x = -torch.arange(vocab, device=DEV, dtype=torch.float32).expand(n, -1) / 7 + x / 100
    if kind == "rising": x = torch.arange(vocab, device=DEV, dtype=torch.float32).expand(n, -1) / 7 + x / 100
    if kind == "few": x[:, 5:] = -math.inf
    if kind == "steps": x = (x * 40).round() / 8
    x[:, 3] = x.max(dim=1).values + torch.rand(n, generator=g, device=DEV)          # the one that is looked at: the best
    return x


@pytest.mark.parametrize("offset", [0.0, 79.0, -81.0, 1e4, -9.9e5, 9.9e5, 1.1e6, -3e7])
@pytest.mark.parametrize("kind", ["normal", "flat", "wide", "pair", "tail", "far tail", "falling", "rising", "few", "steps"])
def test_sums_at_the_ends_of_the_range(kind, offset):
    """The best logit's score, which is minus the log of the sum relative to it."""
    from msa_b200 import lm_ops as K
    for n, vocab in ((1, 700), (5, 4097), (24, 20001)):
        x = rows(kind, torch.Generator(device=DEV).manual_seed(vocab), n, vocab) + offset
        scores = torch.zeros((n, 1), device=DEV)
        score, beam, token = K.beam_topk(x, scores, 1)
        want = torch.log_softmax(x.double(), 1).max(dim=1).values
        error = (score[:, 0].double() - want).abs()
        bound = (SUM if abs(offset) + 4000 < 1e6 else FAR_SUM) + want.abs() * 2.0 ** -24
        assert bool((error <= bound).all()), (float(error.max()), n, vocab)
        assert bool((beam == 0).all()) and torch.equal(x.gather(1, token.long()), x.max(dim=1, keepdim=True).values)


def test_candidates_of_two_beams_that_are_close():
    """Further apart than the two sums' errors they are in the order of 64 bits, alone and among other questions."""
    from msa_b200 import lm_ops as K
    g = torch.Generator(device=DEV).manual_seed(5)
    n, vocab = 400, 3001
    x = torch.randn((n, 2, vocab), generator=g, device=DEV) * 2
    x[:, :, 7] = 14 + torch.rand((n, 2), generator=g, device=DEV)
    best = torch.log_softmax(x.double(), 2)[:, :, 7]
    gap = (torch.rand(n, generator=g, device=DEV).double() * 2 - 1) * 6e-6
    scores = torch.stack([torch.zeros(n, device=DEV), (best[:, 0] - best[:, 1] - gap).float()], 1)      # some 1e-2: a step of 2^-30
    total = best + scores.double()
    gap = total[:, 0] - total[:, 1]
    order = torch.where(gap > 0, 0, 1)
    clear = gap.abs() > 2 * SUM
    assert 150 < int(clear.sum()) < n
    score, beam, token = K.beam_topk(x.view(2 * n, vocab), scores, 2)
    assert bool((token == 7).all()) and bool((beam.sort(1).values == torch.tensor([0, 1], device=DEV)).all())
    assert torch.equal(beam[clear, 0].long(), order[clear])
    for i in clear.nonzero()[:, 0].tolist()[:40]:
        assert int(K.beam_topk(x[i], scores[i:i + 1], 2)[1][0, 0]) == int(order[i])
