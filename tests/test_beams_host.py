"""Beam search's operators: what they refuse, and what they take, before anything is launched (no GPU)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32
pytestmark = pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")


@pytest.fixture
def launches(monkeypatch):
    """Names of the calls that would have been made, on fake CUDA tensors."""
    import contextlib
    from msa_b200 import _cabi_lm as A
    seen = []
    monkeypatch.setattr(A, "call", lambda name, *a: seen.append(name))
    monkeypatch.setattr(A, "stream_ptr", lambda device=None: 0)
    monkeypatch.setattr(A, "ptr", lambda t: 0)
    monkeypatch.setattr(A, "on_device", lambda d: contextlib.nullcontext())
    with FakeTensorMode():
        yield seen


def new(*shape, dtype=F32, device="cuda:0"):
    return torch.empty(shape, dtype=dtype, device=device)


def test_choice_shapes(launches):
    from msa_b200 import lm_ops as K
    out = K.beam_topk(new(12, 100), new(3, 4), 8, new(2, dtype=I32))
    assert [tuple(t.shape) for t in out] == [(3, 8)] * 3 + [(3, 4)] * 3 and [t.dtype for t in out] == [F32, I32, I32] * 2
    assert len(K.beam_topk(new(12, 100, dtype=BF16), new(3, 4), 1)) == 3 and launches == ["msa_lm_beam_topk"] * 2
    assert K.beam_topk(new(0, 100), new(0, 4), 8)[0].shape == (0, 8) and len(launches) == 2            # nothing to choose from: no launch
    K.beam_topk(new(12, 200)[:, ::1][:, 50:150], new(3, 4), 8)
    K.beam_topk(new(12, 1), new(3, 4), 4, new(0, dtype=I32))


@pytest.mark.parametrize("bad", ["rank", "scores rank", "rows", "beams", "no beams", "k 0", "k 65", "k of few", "logits type", "scores type", "columns", "scores order",
                                 "scores device", "stop type", "stop rank", "stop order", "no columns"])
def test_choice_refuses(launches, bad):
    from msa_b200 import lm_ops as K
    x, s, k, stop = new(12, 100), new(3, 4), 8, new(4, dtype=I32)
    if bad == "rank": x = new(3, 4, 100)
    if bad == "scores rank": s = new(12)
    if bad == "rows": x = new(11, 100)
    if bad == "beams": x, s = new(33, 100), new(1, 33)
    if bad == "no beams": x, s = new(0, 100), new(3, 0)
    if bad == "k 0": k = 0
    if bad == "k 65": k = 65
    if bad == "k of few": x, k = new(12, 2), 9
    if bad == "logits type": x = x.double()
    if bad == "scores type": s = s.to(BF16)
    if bad == "columns": x = new(100, 12).t()
    if bad == "scores order": s = new(4, 3).t()
    if bad == "scores device": s = new(3, 4, device="cuda:1")
    if bad == "stop type": stop = stop.long()
    if bad == "stop rank": stop = new(2, 2, dtype=I32)
    if bad == "stop order": stop = new(8, dtype=I32)[::2]
    if bad == "no columns": x = new(12, 0)
    with pytest.raises(K.A.MsaError):
        K.beam_topk(x, s, k, stop)
    assert not launches


def test_host_tensors_are_refused():
    from msa_b200 import lm_ops as K
    from msa_b200.cache import RingSpec, SequenceStateCache
    with pytest.raises(K.A.MsaError, match="CUDA"):
        K.beam_topk(torch.zeros(4, 10), torch.zeros(1, 4), 2)
    c = SequenceStateCache([RingSpec(6, 8)], 4, 50, "cpu", F32)
    t = torch.zeros((1, 4), dtype=I32)
    with pytest.raises(K.A.MsaError, match="CUDA"):
        c.reorder(t, t, t[:, 0])


@pytest.mark.parametrize("bad", ["rank", "beams", "no beams", "parent shape", "length shape", "shared shape", "type", "order", "device"])
def test_reorder_refuses(launches, bad, monkeypatch):
    from msa_b200 import _cabi_lm as A
    from msa_b200.cache import RingSpec, SequenceStateCache
    monkeypatch.setattr(SequenceStateCache, "_state_parts", lambda self: torch.empty((2, 6), dtype=torch.int64))
    c = SequenceStateCache([RingSpec(6, 8)], 16, 50, "cuda:0", F32)
    i = lambda *s, **kw: new(*s, dtype=I32, **kw)
    slot, parent, length, shared = i(3, 4), i(3, 4), i(3), i(3, 4, 4)
    got = c.reorder(slot, parent, length, shared)
    assert [tuple(t.shape) for t in got] == [(3, 4), (3, 4, 4)] and launches == ["msa_lm_reorder"]
    assert c.reorder(slot, parent, length)[1] is None and c.reorder(i(0, 4), i(0, 4), i(0))[0].shape == (0, 4) and len(launches) == 2
    if bad == "rank": slot = parent = i(12)
    if bad == "beams": slot = parent = i(3, 33)
    if bad == "no beams": slot = parent = i(3, 0)
    if bad == "parent shape": parent = i(3, 5)
    if bad == "length shape": length = i(3, 1)
    if bad == "shared shape": shared = i(3, 4)
    if bad == "type": parent = parent.long()
    if bad == "order": parent = i(4, 3).t()
    if bad == "device": length = i(3, device="cuda:1")
    with pytest.raises(A.MsaError):
        c.reorder(slot, parent, length, shared)
    assert len(launches) == 2


def test_what_a_slot_holds():
    """Ring rows, the halves of convolution inputs, whole states; the widest pieces that fit every address."""
    from msa_b200 import _cabi_lm as A
    from msa_b200.cache import RecurrentSpec, RingSpec, SequenceStateCache
    c = SequenceStateCache([RingSpec(24, 8, 10, 4, first=3), RingSpec(5, 60, first=2), RecurrentSpec(2, 4, 4, 6, 1, shift=12)], 2, 50, "cpu", BF16)
    parts = [A.StatePart.from_buffer_copy(bytes(p.numpy().tobytes())) for p in c._state_parts()]
    ring, conv, odd, state, shift, last = parts
    assert (ring.base, ring.slot_bytes, ring.bytes, ring.rows, ring.first, ring.kind, ring.align) == (c.ring[0].data_ptr(), 11 * 48, 48, 11, 3, A.STATE_RING, 16)
    assert (conv.slot_bytes, conv.bytes, conv.kind, conv.align) == (2 * 3 * 10 * 2, 60, A.STATE_HALF, 4)
    assert (odd.bytes, odd.rows, odd.first, odd.align) == (10, 50, 0, 2)           # the cache holds everything: one window
    assert (state.bytes, state.kind) == (2 * 4 * 4 * 4, A.STATE_ALL) and shift.bytes == 24 and (last.base, last.bytes) == (c.last_token.data_ptr(), 4)


def test_entry_points_refuse():
    """The C functions' own checks; the pointers here lead nowhere."""
    from msa_b200 import _cabi_lm as A
    lib, p = A.lib(), 1 << 12

    def choice(dtype=0, batch=2, beams=4, vocab=100, k=8, n_stop=0, stop=None, work=p, live=(None, None, None), logits=p):
        return lib.msa_lm_beam_topk(logits, 100, dtype, p, batch, beams, vocab, k, stop, n_stop, work, p, p, p, *live, None)
    ok = A.dtype_code(F32)
    for kw in (dict(dtype=7), dict(dtype=ok, beams=0), dict(dtype=ok, beams=33), dict(dtype=ok, vocab=0), dict(dtype=ok, k=0), dict(dtype=ok, k=65), dict(dtype=ok, vocab=1, k=5),
               dict(dtype=ok, vocab=2 ** 31 - 1, beams=1), dict(dtype=ok, vocab=2 ** 29, beams=4), dict(dtype=ok, n_stop=2), dict(dtype=ok, n_stop=-1), dict(dtype=ok, work=p + 4),
               dict(dtype=ok, live=(p, None, p)), dict(dtype=ok, logits=None), dict(dtype=ok, batch=-1)):
        assert choice(**kw) != 0 and b"beam_topk" in lib.msa_last_error()
    assert choice(dtype=ok, batch=0) == 0
    assert lib.msa_lm_beam_topk_workspace(0, 4, 100, 8) == 0 and lib.msa_lm_beam_topk_workspace(2, 4, 100, 8) >= 2 * 4 * 16

    def reorder(batch=2, beams=4, n_slots=9, n_part=1, slot=p, slot_out=p + 64, shared=None, shared_out=None, work=p):
        return lib.msa_lm_reorder(slot, p, p, shared, batch, beams, n_slots, p, n_part, slot_out, shared_out, work, None)
    for kw in (dict(batch=-1), dict(beams=0), dict(beams=33), dict(n_slots=0), dict(n_part=0), dict(slot=None), dict(slot_out=p), dict(shared_out=p), dict(shared=p, shared_out=p),
               dict(work=p + 8), dict(work=None), dict(batch=2 ** 26, beams=32)):
        assert reorder(**kw) != 0 and b"reorder" in lib.msa_last_error()
    assert reorder(batch=0) == 0
