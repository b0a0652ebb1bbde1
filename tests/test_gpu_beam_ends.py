"""A search's choice where its stop tokens could fill all places: the kernels against 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


@pytest.mark.parametrize("beams,stop,vocab", [(32, (3, 700, 5), 4001), (24, (0, 9), 50001), (17, tuple(range(40, 80)), 1000), (32, (-1, 3, 9, 70000), 700)])
@pytest.mark.parametrize("favour", [0.0, 9.0])
def test_beams_that_go_on(beams, stop, vocab, favour):
    from msa_b200 import beam as B
    g = torch.Generator(device=DEV).manual_seed(beams)
    known = [t for t in stop if 0 <= t < vocab]
    x = torch.randn((2 * beams, vocab), generator=g, device=DEV) * 2
    x[:, known] += favour
    kept, searches = x.clone(), []
    for _ in range(2):
        s = B.BeamSearch(beams, 9, stop)
        s.tokens, s.scores = [[0]] * beams, (-torch.rand(beams, generator=g, device=DEV)).tolist()
        searches.append(s)
    scores = [list(s.scores) for s in searches]
    B.advance(x, [(s, range(i * beams, (i + 1) * beams)) for i, s in enumerate(searches)])
    assert torch.equal(x, kept)
    for i, s in enumerate(searches):
        total = torch.log_softmax(x[i * beams:(i + 1) * beams].double(), 1) + torch.tensor(scores[i], dtype=torch.float64, device=DEV)[:, None]
        ends = torch.sort(total.flatten(), descending=True)
        want_ends = [float(v) for a, v in zip(ends.indices[:beams], ends.values[:beams]) if int(a) % vocab in stop]
        total[:, known] = -math.inf
        best = torch.sort(total.flatten(), descending=True)
        # A row's sum is good to 6.2e-7 (its exponentials to 2^-22 and 2^-25, six sums of 32 bits) and the joint logit of its stop tokens, up to 16,
        # to half a step, 5e-7: two scores closer than twice that may change places.
        close = 2 * (6.2e-7 + 5e-7)
        at = [b * vocab + t for b, t in zip(s.parents, s.next_tokens)]
        chosen = total.flatten()[at]
        assert len(set(at)) == beams and float((chosen - best.values[:beams]).abs().max()) < close
        # and the rounding of scores of up to 16
        assert float((torch.tensor(s.scores, dtype=torch.float64, device=DEV) - chosen).abs().max()) < close / 2 + 5e-7
        assert len(s.ended) == len(want_ends)
        got = torch.tensor([r * 2 for r, _ in s.ended], dtype=torch.float64)
        assert got.numel() == 0 or float((got - torch.tensor(want_ends, dtype=torch.float64)).abs().max()) < 6.2e-7 + 5e-7
