"""Portions of a step over plain windows take nothing from each other's contexts: grouped heads, and latent heads with a shared rotated part."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, BF16 = "cuda:0", torch.bfloat16
PORTIONS = [(100, "5@0,2@3,130@0,64@300,128@0"), (130, "3@0,70@0,260@500,2@7"), (300, "128@0,384@0,129@129,1@1"), (4000, "31@0,17@0,47@1,300@700,63@65,16@0")]


@pytest.fixture(scope="module", autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("window,portions", PORTIONS, ids=[str(w) for w, _ in PORTIONS])
@pytest.mark.parametrize("dim,rot,vdim,heads,kv", [(64, 0, 64, 4, 4), (64, 0, 128, 8, 2), (128, 0, 64, 6, 2), (128, 0, 128, 2, 1), (64, 64, 64, 3, 3), (128, 64, 128, 2, 2)])
def test_portions_take_nothing_from_each_other(window, portions, dim, rot, vdim, heads, kv, bad):
    """What lies in the others' contexts, or in unused rows behind the last one, does not reach a portion's rows: not a bit of them."""
    from msa_b200 import lm_ops as K
    from msa_b200.cache import PackedStep, RingSpec, SequenceStateCache
    parts = [tuple(map(int, p.split("@"))) for p in portions.split(",")]
    cache = SequenceStateCache([RingSpec(8, window)], len(parts), 5000, DEV, BF16)
    for i, (_, s) in enumerate(parts):
        cache.acquire(i)
        cache.advance(i, s)
    step = PackedStep([(i, [0] * n, []) for i, (n, _) in enumerate(parts)], cache, (window,))
    nd = step.n_decode                                     # single tokens come first and are not for this kernel
    view, status = step.views[window], torch.zeros(4, dtype=torch.int32, device=DEV)
    order = [i for i, (n, _) in enumerate(parts) if n > 1]
    g = torch.Generator(device=DEV).manual_seed(window)
    rand = lambda *shape: torch.randn(shape, generator=g, device=DEV).to(BF16)
    q = rand(step.n_tok, heads, dim + rot)[nd:]
    rows = [rand(view.n_ctx + 300, kv, dim), rand(view.n_ctx + 300, kv, vdim)] + ([rand(view.n_ctx + 300, 1, rot)] if rot else [])

    def run(k, v, r=None):
        out = torch.empty((q.shape[0], heads, vdim), dtype=BF16, device=DEV)
        K.window_attn_tc(q[:, :, :dim], q[:, :, dim:] if rot else None, k[:view.n_ctx], r[:view.n_ctx] if rot else None, v[:view.n_ctx], out, row0=nd, status=status,
                         scale=(dim + rot) ** -0.5, window=view.window, start=step.start, cu=step.cu, seq0=nd, seq1=step.n_seq, max_len=step.max_len,
                         ctx_off=view.ctx_off)
        return out
    want, cu, off = run(*rows), step.cu.tolist(), view.ctx_off.tolist()
    assert bool(want.isfinite().all())
    for j, i in enumerate(order):
        mixed = [torch.full_like(t, bad) for t in rows]
        for t, m in zip(rows, mixed):
            m[off[j]:off[j + 1]] = t[off[j]:off[j + 1]]
        a, b = cu[nd + j] - nd, cu[nd + j + 1] - nd
        assert b - a == parts[i][0] and torch.equal(run(*mixed)[a:b], want[a:b]), parts[i]
    assert status.tolist() == [0, 0, 0, 0]
