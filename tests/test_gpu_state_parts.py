"""Reordering over the tensors that a cache has now."""
import pytest
import torch

from tests.test_gpu_beams import DEV, filled, plain_reorder, table, tensors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


def test_tensors_put_in_the_place_of_others():
    a, b = filled("odd", 6, 30, torch.float32, 2), filled("odd", 6, 30, torch.float32, 2)
    old = tensors(b)
    kept = [t.clone() for t in old]
    b.ring[0], b.state[2], b.last_token = b.ring[0].clone(), b.state[2].clone(), b.last_token.clone()
    for parents, lengths in (([[1, 1, 0]], [30]), ([[2, 0, 0]], [11])):
        want, _ = plain_reorder(a, [[4, 0, 3]], parents, lengths)
        got, _ = b.reorder(table([[4, 0, 3]]), table(parents), table(lengths))
        assert got.tolist() == want and all(torch.equal(x, y) for x, y in zip(tensors(a), tensors(b)))
    now = tensors(b)
    replaced = [i for i, (x, y) in enumerate(zip(old, now)) if x is not y]
    assert len(replaced) == 3 and all(torch.equal(old[i], kept[i]) for i in replaced)
