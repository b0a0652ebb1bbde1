"""Attention over a window with first tokens that stay visible, on the GPU: whole layers against the oracle in 64 bits at every cut,
the tensor-core kernels element by element, and a model with such layers."""
import pytest
import torch

from oracle import hybrid_oracle as O
from tests import hybrid_util as U

pytestmark = pytest.mark.gpu
DEV, BF16, F64 = "cuda:0", torch.bfloat16, torch.float64


@pytest.fixture(scope="module", autouse=True)
def exact_products():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    torch.set_float32_matmul_precision("highest")


DTYPES = pytest.mark.parametrize("dtype", [torch.float32, BF16], ids=["f32", "bf16"])


def attention(heads, kv_heads, dim, vdim, window, first, rot, conv):
    m = U.attention(heads, kv_heads, dim, vdim, window, rot, conv)
    m["mask"]["first"] = first
    return m


# ------------------------------------------------------------------------------------------ layers against the oracle
class Layer:
    """One attention layer over hand-made inputs: what the model's step does around it."""

    def __init__(self, spec, width, dtype, seed=5):
        from msa_b200 import hybrid as H, hybrid_config as C
        cfg = U.config(width, 8, [U.layer("attention", spec, None)])
        w = {k[len("l0.mix."):]: v for k, v in U.make_weights(cfg, seed).items() if k.startswith("l0.mix.")}
        self.s, self.dtype = C.GroupedAttentionSpec.parse(spec), dtype
        self.mixer = H.GroupedAttention(self.s, H.Weights({"m." + k: v for k, v in w.items()}, DEV, dtype), "m.", width, 1e-5)
        self.oracle = lambda h: O.MIXERS["attention"](h.double(), {k: v.double() for k, v in w.items()}, spec, 1e-5)

    def cache(self, n_slots, max_len):
        from msa_b200.cache import SequenceStateCache
        return SequenceStateCache([self.mixer.state_spec], n_slots, max_len, DEV, self.dtype)

    def run(self, cache, entries):
        from msa_b200 import lm_ops as K
        from msa_b200.cache import PackedStep
        step = PackedStep([(s, [0] * h.shape[0], range(h.shape[0])) for s, h in entries], cache, (self.s.span,))
        packed = torch.empty((step.n_tok, entries[0][1].shape[1]), dtype=self.dtype, device=DEV)
        packed[step.want_rows.long()] = torch.cat([h for _, h in entries]).to(DEV, self.dtype)
        y = K.matmul(self.mixer.forward(packed, step, cache, 0), self.mixer.w_o)
        step.commit(cache)
        return list(y[step.want_rows.long()].float().cpu().split([h.shape[0] for _, h in entries]))


def rows(n, width, seed):
    return torch.randn(n, width, generator=torch.Generator().manual_seed(seed)).to(BF16).float()


def close(got, want, dtype):
    """The bounds of every other layer (``test_gpu_hybrid``): rounded projections, scores and outputs against 64 bits."""
    e = U.row_errors(got, want)
    if dtype == torch.float32:
        assert float(e.max()) < 5e-5, (float(e.max()), int(e.argmax()))
    else:
        assert float(e.max()) < 0.1 and (len(e) < 10 or float(e.median()) < 0.015), (float(e.max()), int(e.argmax()), float(e.median()))


LAYERS = {
    "uneven": (attention(6, 2, 20, 28, 17, 3, 12, 3), 72),
    "odd": (attention(3, 1, 7, 5, 6, 5, 2, 2), 33),
    "window1": (attention(4, 2, 8, 8, 1, 4, 8, 4), 32),
    "many-first": (attention(4, 2, 16, 8, 9, 100, 6, 6), 40),
    "64": (attention(8, 2, 64, 64, 100, 4, 32, 4), 128),
    "64-128": (attention(8, 1, 64, 128, 40, 70, 32, 1), 128),
    "128": (attention(24, 2, 128, 128, 64, 1, 128, 4), 128),
    "padded": (attention(6, 3, 96, 40, 64, 64, 30, 3), 96),
    "192": (attention(2, 1, 192, 160, 30, 7, 64, 2), 64),
}


@DTYPES
@pytest.mark.parametrize("case", list(LAYERS))
def test_layer_at_every_cut(case, dtype):
    """Whole, in portions down to single tokens, and a mixed batch of unequal sequences; a cache with room to spare, one that the
    window and the first tokens just fill, and one that holds everything."""
    spec, width = LAYERS[case]
    m = Layer(spec, width, dtype)
    h = [rows(n, width, 10 + n) for n in (300, 131, 1)]
    want = [m.oracle(x) for x in h]
    for max_len in (320, 300):
        cache = m.cache(4, max_len)
        for cuts in ((300,), (2, 3), (64, 1, 7), (97, 65, 2, 1, 128)):
            cache.acquire("s")
            out, at, k = [], 0, 0
            while at < 300:
                n = min(cuts[k % len(cuts)], 300 - at)
                out.append(m.run(cache, [("s", h[0][at:at + n])])[0])
                at, k = at + n, k + 1
            cache.release("s")
            close(torch.cat(out), want[0], dtype)
    for i in range(3):
        cache.acquire(i)
    at, out = [0, 0, 0], [[], [], []]
    for plan in ((40, 1, 1), (1, 70, 0), (150, 1, 0), (1, 1, 0), (2, 57, 0), (106, 1, 0)):
        entries = [(i, h[i][at[i]:at[i] + n]) for i, n in enumerate(plan) if n]
        for (i, x), y in zip(entries, m.run(cache, entries)):
            out[i].append(y)
            at[i] += x.shape[0]
    for i in range(3):
        close(torch.cat(out[i]), want[i], dtype)
    span = m.s.window + m.s.first                     # a cache one position longer than what is seen, and one of just that length
    for max_len in (span + 1, span):
        if max_len <= 131:
            cache = m.cache(1, max_len)
            cache.acquire("t")
            got = [m.run(cache, [("t", h[1][:max_len - 1])])[0], m.run(cache, [("t", h[1][max_len - 1:max_len])])[0]] if max_len > 1 else m.run(cache, [("t", h[1][:1])])
            close(torch.cat(got), want[1][:max_len], dtype)


# ------------------------------------------------------------------------------------------ kernels element by element
def attend(q, k, v, seen, scale, sink, gate):
    """64 bits; q [n, heads, d], k and v [m, kv heads, ..]; the outputs and, per output, what a relative error of the weights moves
    at most: the weighted sum of the values' sizes."""
    g = q.shape[1] // k.shape[1]
    q, k, v = q.to(F64), k.to(F64).repeat_interleave(g, 1), v.to(F64).repeat_interleave(g, 1)
    s = (torch.einsum("ihd,jhd->hij", q, k) * scale).masked_fill(~seen, float("-inf"))
    m = s.amax(-1, keepdim=True)
    m = m.clamp(min=0) if sink else m
    e = torch.exp(s - m)
    w = e / (e.sum(-1, keepdim=True) + (torch.exp(-m) if sink else 0))
    f = 1 if gate is None else torch.sigmoid(gate.to(F64))[..., None]
    return torch.einsum("hij,jhd->ihd", w, v) * f, torch.einsum("hij,jhd->ihd", w, v.abs()) * f


def within(got, want, size):
    """Weights are rounded to bf16 (2^-8 of each), and so is the output (2^-8 of it).  Scores: sums of 128 products in fp32, off by
    128 * 2^-24 of the sum of their sizes, about 150 here, times the scale 0.09: 1e-4 in the exponent, twice for numerator and
    denominator; 3e-4 of the weighted sizes with the fp32 rest."""
    bound = 2 ** -8 * want.abs() + (2 ** -8 + 3e-4) * size
    over = (got.to(F64) - want).abs() - bound
    assert float(over.max()) <= 0, float(over.max())


def randn(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(BF16)


def seen_of(i, j, window, first):
    back = i[:, None] - j[None]
    return (back >= 0) & ((back < window) | (j[None] < first))


PORTIONS = [
    # window, first, portions (tokens@position)
    (100, 4, "300@0"), (100, 4, "2@0,3@1,257@99,130@100,64@103,65@104,5@2000"), (1, 1, "200@0,70@50"), (1, 64, "400@7,33@64,2@65"),
    (64, 65, "513@0,300@128,129@129"), (130, 128, "700@3,100@5000"), (37, 200, "600@0,260@100,90@237,41@100000"), (1000, 1, "1100@0,256@999"),
    (5, 63, "256@60,256@67,256@68"),
]


@pytest.mark.parametrize("dim,vdim,group", [(64, 64, 1), (64, 128, 4), (128, 64, 3), (128, 128, 2)])
@pytest.mark.parametrize("window,first,portions", PORTIONS, ids=[f"{w}+{f}" for w, f, _ in PORTIONS])
def test_portions_on_the_tensor_cores(window, first, portions, dim, vdim, group):
    from msa_b200.cache import PackedStep, RingSpec, SequenceStateCache
    from msa_b200.hybrid import portion_attention
    parts = [tuple(map(int, p.split("@"))) for p in portions.split(",")]
    kv, g = 2, torch.Generator(device=DEV).manual_seed(window + first)
    cache = SequenceStateCache([RingSpec(8, window, first=first)], len(parts), max(n + s for n, s in parts) + window + first, DEV, BF16)
    for i, (_, s) in enumerate(parts):
        cache.acquire(i)
        cache.advance(i, s)
    step = PackedStep([(i, [0] * n, []) for i, (n, _) in enumerate(parts)], cache, ((window, first),))
    view, status = step.views[window, first], torch.zeros(4, dtype=torch.int32, device=DEV)
    q = randn(g, step.n_tok, kv * group, dim, scale=1.5)
    ctx = randn(g, view.n_ctx, kv * (dim + vdim))
    for sink, gate in ((False, None), (True, randn(g, step.n_tok, kv * group))):
        k, v = ctx[:, :kv * dim].unflatten(1, (kv, dim)), ctx[:, kv * dim:].unflatten(1, (kv, vdim))
        wide = torch.full((step.n_tok + 3, kv * group * vdim), 7.0, dtype=BF16, device=DEV)          # rows behind the last one stay
        out = wide[:step.n_tok].unflatten(1, (kv * group, vdim))
        portion_attention((q, None, k, None, v, out), True, status, step, view, dim ** -0.5, sink=sink, gate=gate)
        row, at = 0, 0
        for n, s in parts:
            lo = max(0, s - window + 1)
            j = torch.cat([torch.arange(min(first, lo)), torch.arange(lo, s + n)]).to(DEV)
            rows_ = slice(row, row + n)
            want, size = attend(q[rows_], k[at:at + len(j)], v[at:at + len(j)], seen_of(torch.arange(s, s + n, device=DEV), j, window, first), dim ** -0.5,
                                sink, None if gate is None else gate[rows_])
            within(out[rows_], want, size)
            row, at = row + n, at + len(j)
        assert at == view.n_ctx and bool((wide[step.n_tok:] == 7.0).all())
    assert status.tolist() == [0, 0, 0, 0]


@pytest.mark.parametrize("dim,vdim,kv,group", [(64, 64, 3, 1), (64, 128, 1, 8), (128, 64, 2, 5), (128, 128, 2, 20)])
@pytest.mark.parametrize("window,first", [(100, 4), (1, 1), (1, 70), (64, 64), (700, 3), (33, 129), (16, 15)])
def test_tokens_over_the_rings(window, first, dim, vdim, kv, group):
    """Sequences at every place where the window leaves the first tokens or the ring turns; rings longer than needed too."""
    from types import SimpleNamespace
    from msa_b200 import lm_ops as K
    g = torch.Generator(device=DEV).manual_seed(window * 31 + first)
    span = window + first
    pos = sorted({0, 1, first - 1, first, window - 1, window, span - 2, span - 1, span, span + 1, span + window - 1, span + window, 3 * span + 5, 40 * span + 7} - {-1})
    n, scale = len(pos), dim ** -0.5
    for extra in (0, 37):
        ring_rows = span + extra
        ring = randn(g, n + 2, ring_rows, kv * (dim + vdim))
        slot = torch.randperm(n + 2, generator=g, device=DEV)[:n].to(torch.int32)
        step = SimpleNamespace(slot=slot, start=torch.tensor(pos, dtype=torch.int32, device=DEV))
        q = randn(g, n, kv * group, dim, scale=1.5)
        for sink, gate in ((True, randn(g, n, kv * group)), (False, None)):
            wide = torch.full((n + 1, kv * group, vdim), 7.0, dtype=BF16, device=DEV)
            K.group_decode(q, ring, kv, step, wide[:n], window=window, first=first, scale=scale, sink=sink, gate=gate)
            for i, p in enumerate(pos):
                j = [x for x in range(p + 1) if x < first or p - x < window]
                at = [x if x < first else first + (x - first) % (ring_rows - first) for x in j]
                r = ring[int(slot[i]), at]
                want, size = attend(q[i:i + 1], r[:, :kv * dim].unflatten(1, (kv, dim)), r[:, kv * dim:].unflatten(1, (kv, vdim)),
                                    torch.ones((1, len(j)), dtype=torch.bool, device=DEV), scale, sink, None if gate is None else gate[i:i + 1])
                within(wide[i:i + 1], want, size)
            assert bool((wide[n] == 7.0).all())


@pytest.mark.parametrize("n,window,splits", [(2, 5000, 64), (150, 120, 1), (40, 400, 3), (3, 3000, 8)])
def test_tokens_in_every_number_of_splits(n, window, splits):
    """One block a sequence, a cluster of blocks, and more blocks than a cluster holds."""
    from types import SimpleNamespace
    from msa_b200 import lm_ops as K
    first, kv, group, dim = 4, 2, 4, 64
    rows_ = window + first
    got = K.group_decode_splits(n, kv * group, kv, rows_)
    assert (min(got, K.GROUP_CLUSTER) if K.splits_join(got, rows_) else got) == splits
    g = torch.Generator(device=DEV).manual_seed(n)
    ring = randn(g, n, rows_, kv * 2 * dim)
    pos = torch.randint(0, 3 * window, (n,), generator=g, device=DEV).to(torch.int32)
    pos[0], pos[-1] = 0, 50 * window                                 # one row for all the splits; all of them full
    step = SimpleNamespace(slot=torch.randperm(n, generator=g, device=DEV).to(torch.int32), start=pos)
    q, gate, out = randn(g, n, kv * group, dim, scale=1.5), randn(g, n, kv * group), torch.empty((n, kv * group, dim), dtype=BF16, device=DEV)
    for sink in (True, False):
        K.group_decode(q, ring, kv, step, out, window=window, first=first, scale=dim ** -0.5, sink=sink, gate=gate)
        for i, p in enumerate(pos.tolist()):
            j = torch.arange(p + 1, device=DEV)
            j = j[(j < first) | (p - j < window)]
            r = ring[int(step.slot[i]), torch.where(j < first, j, first + (j - first) % window)]
            want, size = attend(q[i:i + 1], r[:, :kv * dim].unflatten(1, (kv, dim)), r[:, kv * dim:].unflatten(1, (kv, dim)),
                                torch.ones((1, len(j)), dtype=torch.bool, device=DEV), dim ** -0.5, sink, gate[i:i + 1])
            within(out[i:i + 1], want, size)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("window,first,portions", [(100, 4, "5@0,2@3,130@0,64@300,128@0"), (130, 200, "3@0,70@0,260@500,2@7"), (300, 1, "128@0,384@0,129@129")])
def test_portions_take_nothing_from_each_other(window, first, portions, bad):
    """What lies in the others' contexts, or in unused rows behind the last one, does not reach a portion's rows: not a bit of them."""
    from msa_b200.cache import PackedStep, RingSpec, SequenceStateCache
    from msa_b200.hybrid import portion_attention
    parts = [tuple(map(int, p.split("@"))) for p in portions.split(",")]
    kv, group, dim, vdim = 2, 4, 64, 128
    cache = SequenceStateCache([RingSpec(8, window, first=first)], len(parts), max(n + s for n, s in parts) + window + first, DEV, BF16)
    for i, (_, s) in enumerate(parts):
        cache.acquire(i)
        cache.advance(i, s)
    step = PackedStep([(i, [0] * n, []) for i, (n, _) in enumerate(parts)], cache, ((window, first),))
    view, status = step.views[window, first], torch.zeros(4, dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(window)
    q, rows_ = randn(g, step.n_tok, kv * group, dim, scale=1.5), randn(g, view.n_ctx + 300, kv * (dim + vdim))

    def run(all_rows):
        ctx, out = all_rows[:view.n_ctx], torch.empty((step.n_tok, kv * group, vdim), dtype=BF16, device=DEV)
        k, v = ctx[:, :kv * dim].unflatten(1, (kv, dim)), ctx[:, kv * dim:].unflatten(1, (kv, vdim))
        portion_attention((q, None, k, None, v, out), True, status, step, view, dim ** -0.5)
        return out
    want, cu, off = run(rows_), step.cu.tolist(), view.ctx_off.tolist()
    assert bool(want.isfinite().all())
    for i in range(len(parts)):
        mixed = torch.full_like(rows_, bad)
        mixed[off[i]:off[i + 1]] = rows_[off[i]:off[i + 1]]
        assert torch.equal(run(mixed)[cu[i]:cu[i + 1]], want[cu[i]:cu[i + 1]]), parts[i]
    assert status.tolist() == [0, 0, 0, 0]


# ------------------------------------------------------------------------------------------ a model with such layers
CONFIG = U.parallel(256, 320, [
    U.layer("attention", attention(8, 2, 64, 128, 40, 4, 32, 4), U.dense(256)),
    U.layer("mamba2", U.mamba2(6, 64, 128, 2, 3, 4), U.dense(192)),
    U.layer("attention", attention(20, 2, 128, 64, 60, 3, 64, 1), U.dense(256)),
    U.layer("attention", attention(4, 4, 64, 64, 40, 0, 64, 3), None),
], bigram=(127, 11, 3), cap=20.0)


@DTYPES
def test_model_in_portions_and_from_a_graph(dtype):
    from msa_b200.hybrid import GraphedDecode, HybridForCausalLM
    from msa_b200.hybrid_config import HybridConfig
    w = U.make_weights(CONFIG, 3)
    m = HybridForCausalLM(HybridConfig.parse(CONFIG), w, DEV, dtype)
    assert m.config.windows == ((40, 4), (60, 3), 40)
    toks = U.tokens_of(CONFIG, 150, 1)
    want = O.forward(CONFIG, w, toks)

    def check(got, at=0):
        e = U.row_errors(got, want[at:at + got.shape[0]])
        if dtype == torch.float32:
            assert float(e.max()) < 2e-4
        else:
            assert float(e.quantile(0.8)) < 0.06
    cache = m.new_cache(2, 150)
    for cuts in ((150,), (70, 1), (33, 5, 64, 2, 1, 9)):
        cache.acquire("a")
        out, at, k = [], 0, 0
        while at < 150:
            n = min(cuts[min(k, len(cuts) - 1)], 150 - at)
            out.append(m.run([("a", toks[at:at + n], range(n))], cache))
            at, k = at + n, k + 1
        cache.release("a")
        check(torch.cat(out))
    slot = cache.acquire("b")
    m.run([("b", toks[:80], [])], cache)
    graph = GraphedDecode(m, cache, 1)
    check(torch.cat([graph.run([t], [80 + i], [slot]).clone() for i, t in enumerate(toks[80:])]), 80)
    m.check_status()
