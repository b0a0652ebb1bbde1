"""What the C functions refuse comes to the caller as one and the same error, from native code and from Python."""
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF16, I32 = "cuda:0", torch.bfloat16, torch.int32


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


class Refuses:
    """Stands in for the native side: takes no operands."""

    def __getattr__(self, name):
        return lambda *a: None


def shifted(*shape):
    """Rows that begin two bytes behind a 16-byte boundary."""
    n = 1
    for d in shape:
        n *= d
    return torch.zeros(n + 8, dtype=BF16, device=DEV)[1:n + 1].view(shape)


def zeros(*shape):
    return torch.zeros(shape, dtype=BF16, device=DEV)


def ints(*values):
    return torch.tensor(values, dtype=I32, device=DEV)


def portions(dim=64, vdim=64, first=0, window=32, scale=0.125, q=None):
    from msa_b200 import lm_ops as K
    q = zeros(5, 4, dim) if q is None else q
    K.window_attn_tc(q, None, zeros(5, 2, dim), None, zeros(5, 2, vdim), zeros(5, 4, vdim), row0=0, status=ints(0, 0, 0, 0), first=first, scale=scale,
                     window=window, start=ints(0), cu=ints(0, 5), seq0=0, seq1=1, max_len=5, ctx_off=ints(0, 5))


def tokens(dim=64, vdim=64, first=0, window=32, rows=40, q=None, heads=4):
    from msa_b200 import lm_ops as K
    step = SimpleNamespace(slot=ints(0, 1), start=ints(3, 3))
    q = zeros(2, heads, dim) if q is None else q
    K.group_decode(q, zeros(2, rows, 2 * (dim + vdim)), 2, step, zeros(2, heads, vdim), window=window, first=first, scale=0.125, sink=True, gate=None)


CALLS = {
    "portions: head size": lambda: portions(dim=96), "portions: value size": lambda: portions(vdim=80), "portions: window": lambda: portions(window=0),
    "portions: scale": lambda: portions(scale=-1.0), "portions: address": lambda: portions(q=shifted(5, 4, 64)),
    "portions, first: head size": lambda: portions(dim=96, first=4), "portions, first: address": lambda: portions(q=shifted(5, 4, 64), first=4),
    "portions, first: span": lambda: portions(first=0x7ffffff0), "portions, first: negative": lambda: portions(first=-1),
    "tokens: head size": lambda: tokens(dim=96), "tokens: window": lambda: tokens(window=0), "tokens: address": lambda: tokens(q=shifted(2, 4, 64)),
    "tokens: groups": lambda: tokens(heads=3), "tokens, first: head size": lambda: tokens(dim=96, first=4),
    "tokens, first: no room": lambda: tokens(first=9), "tokens, first: address": lambda: tokens(q=shifted(2, 4, 64), first=4),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_one_error_either_way(name, monkeypatch):
    from msa_b200 import _cabi_lm as A
    before = A.launches
    with pytest.raises(A.MsaError) as native:
        CALLS[name]()
    monkeypatch.setattr(A, "_native", Refuses())
    with pytest.raises(A.MsaError) as plain:
        CALLS[name]()
    assert type(native.value) is type(plain.value) is A.MsaError and str(native.value) == str(plain.value)
    assert "failed (" in str(plain.value) and A.launches == before


def test_calls_go_on_behind_a_refusal():
    with pytest.raises(RuntimeError):
        tokens(window=0)
    tokens(), tokens(first=4), portions(), portions(first=4)
    torch.cuda.synchronize()


@torch.no_grad()
def test_the_memory_models_calls_too():
    """The first library's launches from native code: angles without a frequency."""
    from msa_b200 import _cabi
    with pytest.raises(_cabi.MsaError, match="msa_rope_table failed"):
        _cabi.native().angles(torch.zeros((1, 3), dtype=torch.int64, device=DEV), torch.zeros(0, dtype=torch.float32, device=DEV), 1.0)
