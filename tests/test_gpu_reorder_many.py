"""Reordering of more copies times tensors than the copying blocks keep prefix sums of (4095), and of as many."""
import pytest
import torch

from tests.test_gpu_beams import DEV, plain_reorder, table, tensors

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rings,batch,beams", [(90, 5, 10), (63, 8, 9), (100, 6, 9), (40, 30, 32)], ids=["4095", "4096", "4848", "4428"])
def test_many_copies_of_many_tensors(rings, batch, beams):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from msa_b200.cache import RingSpec, SequenceStateCache
    specs = [RingSpec(8 + i % 3, 3 + i % 5, first=i % 4) for i in range(rings)]
    n_slots, max_len = batch * beams + 1, 12
    caches = []
    for _ in range(2):
        c = SequenceStateCache(specs, n_slots, max_len, DEV, torch.bfloat16)
        g = torch.Generator(device=DEV).manual_seed(4)
        for t in c.ring.values():
            t.normal_(generator=g)
        c.last_token.random_(0, 1000, generator=g)
        caches.append(c)
    a, b = caches
    g = torch.Generator().manual_seed(rings)
    slots = torch.randperm(n_slots, generator=g)[:batch * beams].view(batch, beams).tolist()
    lengths = torch.randint(5, max_len + 1, (batch,), generator=g).tolist()
    parents = [[int(torch.randint(0, beams, (1,), generator=g))] * beams for _ in range(batch)]        # every other beam copies
    if beams == 32:                                                                             # the oracle row by row: few of these questions move
        parents = [p if q in (0, 13, 29) else list(range(beams)) for q, p in enumerate(parents)]
        parents[7] = [5] * 16 + list(range(16, beams))
    want, _ = plain_reorder(a, slots, parents, lengths)
    got, _ = b.reorder(table(slots), table(parents), table(lengths))
    assert got.tolist() == want
    for x, y in zip(tensors(a), tensors(b)):
        assert torch.equal(x, y)
