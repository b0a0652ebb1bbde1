"""The native side takes the calls that it is there for: every one of them, not only with the same results."""
import pytest
import torch

from tests.test_gpu_lm_native import CALLS, DEV

pytestmark = pytest.mark.gpu
FUNCTIONS = {"choice": "beam_topk", "states": "reorder", "tokens": "group_decode", "portions": "window_attn_tc"}


class Recorder:
    def __init__(self, native):
        self.native, self.seen = native, []

    def __getattr__(self, name):
        f = getattr(self.native, name)

        def call(*a):
            got = f(*a)
            self.seen.append((name, got is not None and got is not False))
            return got
        return call


@pytest.mark.parametrize("name", list(CALLS))
def test_native_code_takes_the_call(name, monkeypatch):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from msa_b200 import _cabi_lm as A
    run = CALLS[name](torch.Generator(device=DEV).manual_seed(1))
    recorder = Recorder(A.native())
    monkeypatch.setattr(A, "_native", recorder)
    before = A.launches
    run()
    assert recorder.seen == [(FUNCTIONS[name], True)] * (A.launches - before) and recorder.seen
