"""What the kernels know of a cache's tensors follows them (no GPU)."""
import pytest
import torch

from msa_b200.cache import RecurrentSpec, RingSpec, SequenceStateCache


def cache():
    return SequenceStateCache([RingSpec(24, 8, 10, 4, first=3), RecurrentSpec(2, 4, 4, 6, 1, shift=12), RingSpec(5, None)], 2, 50, "cpu", torch.bfloat16)


def bases(c):
    from msa_b200 import _cabi_lm as A
    return [A.StatePart.from_buffer_copy(bytes(p.numpy().tobytes())).base for p in c._state_parts()]


@pytest.mark.parametrize("name,run", [("ring", 0), ("ring", 2), ("conv", 0), ("state", 1), ("shift", 1)])
def test_a_tensor_put_in_the_place_of_another(name, run):
    c = cache()
    before, table = bases(c), getattr(c, name)
    old = table[run]
    table[run] = old.clone()
    after = bases(c)
    assert [b for a, b in zip(before, after) if a != b] == [table[run].data_ptr()]
    assert before[after.index(table[run].data_ptr())] == old.data_ptr()


def test_the_last_tokens_and_all_rings_at_once():
    c = cache()
    bases(c)
    c.last_token = c.last_token.clone()
    c.ring = {i: t.clone() for i, t in c.ring.items()}
    got = bases(c)
    assert got[-1] == c.last_token.data_ptr() and {t.data_ptr() for t in c.ring.values()} <= set(got)


def test_the_table_is_made_once():
    c = cache()
    assert c._state_parts() is c._state_parts()


@pytest.mark.parametrize("bad", ["few slots", "order", "device"])
def test_a_tensor_that_is_no_state_is_refused(bad):
    from msa_b200 import _cabi_lm as A
    c = cache()
    bases(c)
    t = c.ring[0]
    c.ring[0] = {"few slots": t[:1], "order": t.transpose(1, 2).contiguous().transpose(1, 2), "device": t.to("meta")}[bad]
    with pytest.raises(A.MsaError):
        c._state_parts()
    c.ring[0] = t.clone()
    assert c.ring[0].data_ptr() in bases(c)
