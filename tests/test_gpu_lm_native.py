"""The short calls of the layered decoders from native code and from Python: the same bits, the same refusals, any stream, captured too."""
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


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV).to(BF16)


def choice(g):
    from msa_b200 import lm_ops as K
    x = torch.randn((6, 1003), generator=g, device=DEV) * 3
    s = -torch.rand((2, 3), generator=g, device=DEV)
    stop = torch.tensor([5, 900], dtype=I32, device=DEV)
    return lambda: [*K.beam_topk(x, s, 9, stop=stop), *K.beam_topk(x[:, :7].to(BF16), s, 5), *K.beam_topk(x[:1].expand(6, -1), s, 4, stop=stop[:0])]


def states(g):
    from msa_b200.cache import RecurrentSpec, RingSpec, SequenceStateCache
    slot = torch.randperm(8, generator=g, device=DEV).to(I32).view(2, 4)
    parent = torch.tensor([[1, 1, 0, 3], [2, -1, 2, 2]], dtype=I32, device=DEV)
    length = torch.tensor([9, 30], dtype=I32, device=DEV)
    shared = torch.full((2, 4, 4), 5, dtype=I32, device=DEV)

    def run():
        cache = SequenceStateCache([RingSpec(24, 11, 16, 3, first=2), RecurrentSpec(2, 8, 8, 24, 4, 16)], 8, 64, DEV, BF16)
        fill = torch.Generator(device=DEV).manual_seed(3)
        tables = [t for d in (cache.ring, cache.state, cache.conv, cache.shift) for t in d.values()]
        for t in tables:
            t.normal_(generator=fill)
        a, b = cache.reorder(slot, parent, length, shared)
        c, none = cache.reorder(a, parent, length)
        assert none is None
        return [a, b, c, *tables]
    return run


def tokens(g):
    from types import SimpleNamespace
    from msa_b200 import lm_ops as K
    q, gate = randn(g, 3, 8, 64), randn(g, 3, 8)
    step = SimpleNamespace(slot=torch.tensor([2, 0, 1], dtype=I32, device=DEV), start=torch.tensor([4, 700, 9000], dtype=I32, device=DEV))
    rings = [(window, first, randn(g, 3, window + first, 2 * 192)) for window, first in ((300, 0), (300, 4), (6000, 4))]     # merge, cluster, merge

    def run():
        outs = []
        for window, first, ring in rings:
            for gate_ in (gate, None):
                out = torch.zeros((3, 8, 128), dtype=BF16, device=DEV)
                K.group_decode(q, ring, 2, step, out, window=window, first=first, scale=0.125, sink=True, gate=gate_)
                outs.append(out)
        return outs
    return run


def portions(g):
    from msa_b200.cache import PackedStep, RingSpec, SequenceStateCache
    from msa_b200.hybrid import portion_attention
    parts, made = [(70, 0), (130, 250)], []
    for key in ((100, 4), 100):                          # windows with and without first tokens
        window, first = key if isinstance(key, tuple) else (key, 0)
        cache = SequenceStateCache([RingSpec(8, window, first=first)], 2, 900, DEV, BF16)
        for i, (_, s) in enumerate(parts):
            cache.acquire(i)
            cache.advance(i, s)
        step = PackedStep([(i, [0] * n, []) for i, (n, _) in enumerate(parts)], cache, (key,))
        view = step.views[key]
        made.append((step, view, randn(g, 200, 8, 64), randn(g, view.n_ctx, 2 * 192), randn(g, 200, 8)))
    status = torch.zeros(4, dtype=I32, device=DEV)

    def run():
        outs = []
        for step, view, q, ctx, gate in made:
            for gate_ in (gate, None):
                out = torch.zeros((200, 8, 128), dtype=BF16, device=DEV)
                k, v = ctx[:, :128].unflatten(1, (2, 64)), ctx[:, 128:].unflatten(1, (2, 128))
                portion_attention((q, None, k, None, v, out), True, status, step, view, 0.125, sink=gate_ is None, gate=gate_)
                outs.append(out)
        return outs
    return run


CALLS = {f.__name__: f for f in (choice, states, tokens, portions)}


@pytest.mark.parametrize("name", list(CALLS))
def test_the_same_from_native_code_and_from_python(name, monkeypatch):
    from msa_b200 import _cabi_lm as A
    run = CALLS[name](torch.Generator(device=DEV).manual_seed(1))
    before = A.launches
    native, made = run(), None
    made = A.launches - before
    with monkeypatch.context() as m:
        m.setattr(A, "_native", Refuses())
        before = A.launches
        plain = run()
        assert A.launches - before == made > 0                       # counted alike
    assert len(native) == len(plain) and all(a.dtype == b.dtype and a.is_contiguous() and torch.equal(a, b) for a, b in zip(native, plain))


@pytest.mark.parametrize("name", ["choice", "tokens", "portions"])
def test_on_a_stream_of_its_own_and_captured(name):
    run = CALLS[name](torch.Generator(device=DEV).manual_seed(2))
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):                                               # two graphs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    for graph, _ in graphs * 2:
        graph.replay()
    assert all(torch.equal(a, b) for _, out in graphs for a, b in zip(out, want))


def test_results_have_sizes_of_their_own():
    run = choice(torch.Generator(device=DEV).manual_seed(4))
    first = run()
    kept = [t.clone() for t in first]
    for _ in range(20):
        run()
    assert all(torch.equal(a, b) for a, b in zip(first, kept))
    first[0].fill_(7.0)                                              # a table that is written to leaves the others alone
    assert all(torch.equal(a, b) for a, b in zip(first[1:], kept[1:]))


@pytest.mark.parametrize("bad", ["beams", "k", "dtype", "rows", "stop", "strided"])
def test_refusals_stay(bad):
    from msa_b200 import _cabi as A, lm_ops as K
    x, s, k, stop = torch.zeros((6, 50), device=DEV), torch.zeros((2, 3), device=DEV), 4, torch.zeros(1, dtype=I32, device=DEV)
    if bad == "beams":
        x, s = torch.zeros((33, 50), device=DEV), torch.zeros((1, 33), device=DEV)
    elif bad == "k":
        k = 65
    elif bad == "dtype":
        x = x.half()
    elif bad == "rows":
        x = x[:5]
    elif bad == "stop":
        stop = stop.long()
    else:
        x = torch.zeros((50, 6), device=DEV).t()
    with pytest.raises(A.MsaError):
        K.beam_topk(x, s, k, stop=stop)
