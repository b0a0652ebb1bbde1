"""Beam search's two operators on the GPU: the choice of continuations against 64 bits, and the reordering of sequence states against
a plain restatement, slot by slot."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV, F32, BF16, F64, I32 = "cuda:0", torch.float32, torch.bfloat16, torch.float64, torch.int32


@pytest.fixture(scope="module", autouse=True)
def needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")


# ------------------------------------------------------------------------------------------ choice
def wanted(logits, scores, k, stop):
    """Lists of (score, beam, token) per question: the k best, and the first that do not stop."""
    batch, beams = scores.shape
    out, live = [], []
    for q in range(batch):
        cand = []
        for b in range(beams):
            s, x = float(scores[q, b]), logits[q * beams + b].to(F64).cpu()
            if not math.isfinite(s) or bool(x.isnan().any()) or bool((x == math.inf).any()) or bool((x == -math.inf).all()):
                continue
            total = s + (x - torch.logsumexp(x, 0))
            best = torch.sort(x, descending=True, stable=True).indices[:k + 1]
            cand += [(float(total[t]), b, int(t), float(x[t])) for t in best if x[t] > -math.inf]
        cand.sort(key=lambda c: (-c[0], c[1], -c[3], c[2]))
        cand = [c[:3] for c in cand[:k]]
        on = [c for c in cand if c[2] not in stop][:beams]
        out.append(cand + [(-math.inf, -1, -1)] * (k - len(cand)))
        live.append(on + [(-math.inf, -1, -1)] * (beams - len(on)))
    return out, live


def agree(got, want):
    score, beam, token = (t.cpu() for t in got)
    for q, rows in enumerate(want):
        assert beam[q].tolist() == [r[1] for r in rows] and token[q].tolist() == [r[2] for r in rows], q
        for s, r in zip(score[q].tolist(), rows):
            # rounded to fp32 once (2^-24 of the value); the row's sum in terms of 2^-22 each (the exponential), averaged at worst: 2.4e-7
            assert s == r[0] or abs(s - r[0]) <= 2 ** -24 * abs(r[0]) + 3e-7, (q, s, r)


def check(logits, scores, k, stop=()):
    from msa_b200 import lm_ops as K
    stop_t = torch.tensor(list(stop), dtype=I32, device=DEV)
    got = K.beam_topk(logits, scores, k, stop_t)
    cand, live = wanted(logits, scores, k, set(stop))
    agree(got[:3], cand)
    agree(got[3:], live)
    plain = K.beam_topk(logits, scores, k)
    assert len(plain) == 3 and all(torch.equal(a, b) for a, b in zip(plain, got))
    return got


def inputs(batch, beams, vocab, dtype=F32, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((batch * beams, vocab), generator=g, device=DEV) * spread
    s = -torch.rand((batch, beams), generator=g, device=DEV) * 5
    return x.to(dtype), s


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("batch,beams,vocab,k", [
    (1, 1, 1, 1), (3, 2, 1, 2), (1, 1, 64, 64), (2, 4, 7, 28), (1, 4, 100, 8), (2, 32, 2, 64), (5, 3, 4095, 6), (2, 5, 4096, 10), (3, 2, 4097, 5),
    (1, 7, 8191, 14), (2, 32, 12289, 64), (1, 4, 151936, 8), (150, 5, 5000, 10), (1, 1, 300001, 1), (700, 1, 999, 3)])
def test_choice_over_sizes(batch, beams, vocab, k, dtype):
    x, s = inputs(batch, beams, vocab, dtype, seed=vocab + k)
    check(x, s, k, stop=(0, vocab // 2) if vocab > 4 else ())


def test_choice_of_rows_with_a_stride():
    x, s = inputs(3, 4, 5003, seed=1)
    wide = torch.full((12, 5013), float("nan"), device=DEV)
    wide[:, 5:5008] = x
    a, b = check(wide[:, 5:5008], s, 8, (3,)), check(x, s, 8, (3,))
    assert all(torch.equal(p, q) for p, q in zip(a, b))                # wherever a row starts in memory, the same bits
    same = x[:1].expand(12, -1)                                        # a broadcast row: equals go to the lowest beam and token
    check(same, torch.zeros((3, 4), device=DEV), 8)


@pytest.mark.parametrize("k", [1, 8, 64])
def test_equal_logits(k):
    for x in (torch.zeros((4, 9001), device=DEV), torch.full((4, 9001), torch.finfo(F32).min, device=DEV),
              torch.randint(0, 3, (4, 9001), generator=torch.Generator().manual_seed(k)).float().to(DEV)):
        check(x, torch.tensor([[-1.0, -1.0], [-2.0, -1.5]], device=DEV), k)


@pytest.mark.parametrize("k", [3, 33, 64])
@pytest.mark.parametrize("kind", ["up", "down", "block", "lanes", "few", "lowest", "spikes"])
def test_rows_in_an_order(kind, k):
    """Rows that are sorted, masked in blocks, or masked so that some warps of a tile see nothing at all."""
    n = 12345
    x, s = inputs(2, 3, n, seed=k)
    t = torch.arange(n, device=DEV)
    if kind == "up":
        x = x.sort(1).values
    elif kind == "down":
        x = x.sort(1, descending=True).values
    elif kind == "block":
        x[:, (t < 5000) | (t > 5100)] = -math.inf
    elif kind == "lanes":                                              # one warp's tokens masked, all others close together
        x[:, t % 256 < 32] = -math.inf
        x = x * 1e-3
        x[::2] = x[::2].sort(1).values
    elif kind == "few":
        x[:, t % 1021 > 0] = -math.inf
        x[1] = -math.inf
    elif kind == "lowest":
        x[:, t % 1021 > 0] = torch.finfo(F32).min
    else:
        x[:, ::4096] += 50
    check(x, s, k, (0, 4096))


def test_values_at_the_ends_of_the_range():
    x, s = inputs(6, 2, 6000, seed=4)
    x[0, 17] = math.inf
    x[1, 18] = float("nan")
    x[2] = -math.inf
    x[3] = x[3] * 1e30
    x[4] = x[4] + 2e6
    x[5] = -3e38
    x[6, 0], x[6, 1:] = 88.0, -3e38
    x[7] = x[7] * 1e-30
    s[4, 0], s[4, 1] = -math.inf, float("nan")
    s[5, 0] = math.inf
    x[10, 5], x[8, 4] = float("nan"), float("nan")                     # in rows that do not count
    check(x, s, 12)


def test_a_row_in_parts_is_as_good_as_one():
    """The same rows in a small and in a large batch, which cuts them into other parts."""
    from msa_b200 import lm_ops as K
    x, s = inputs(1, 4, 151936, seed=9)
    one = K.beam_topk(x, s, 8)
    many = K.beam_topk(x.repeat(200, 1), s.repeat(200, 1), 8)
    assert torch.equal(one[1], many[1][:1]) and torch.equal(one[2], many[2][:1])
    assert all(torch.equal(t, t[:1].expand_as(t)) for t in many)
    assert float((one[0] - many[0][:1]).abs().max()) <= 3e-7 + 2 ** -23 * float(one[0].abs().max())


def test_choice_in_a_graph_and_on_another_stream():
    from msa_b200 import lm_ops as K
    a, b = inputs(2, 4, 30000, seed=1), inputs(2, 4, 30000, seed=2)
    stop = torch.tensor([5], dtype=I32, device=DEV)
    want = [K.beam_topk(*i, 8, stop) for i in (a, b)]
    x, s = (t.clone() for t in a)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.beam_topk(x, s, 8, stop)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want[0]))
    with torch.cuda.graph(graph):
        got = K.beam_topk(x, s, 8, stop)
    for i, w in ((b, want[1]), (a, want[0])):
        x.copy_(i[0])
        s.copy_(i[1])
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(got, w))


# ------------------------------------------------------------------------------------------ reordering
def specs(kind):
    from msa_b200.cache import RecurrentSpec as R, RingSpec as W
    return {"rings": [W(64, 20, first=3), W(40, None, 24, 3), W(8, 100), W(16, 1, first=1), W(24, 9, first=60)],
            "odd": [W(13, 20, 7, 4, first=5), W(1, 6), R(3, 5, 7, 9, 2, shift=11), W(3, 2, first=1)],
            "states": [R(4, 16, 16, 48, 4), R(2, 64, 32, shift=128), R(1, 8, 8, 16, 1)]}[kind]


def filled(kind, n_slots, max_len, dtype, seed):
    from msa_b200.cache import SequenceStateCache
    c = SequenceStateCache(specs(kind), n_slots, max_len, DEV, dtype)
    g = torch.Generator(device=DEV).manual_seed(seed)
    for d in (c.ring, c.state, c.conv, c.shift):
        for t in d.values():
            t.normal_(generator=g)
    c.last_token.random_(0, 1000, generator=g)
    return c


def tensors(c):
    return [t for d in (c.ring, c.state, c.conv, c.shift) for _, t in sorted(d.items())] + [c.last_token]


def plain_reorder(c, slots, parents, lengths):
    """Slot by slot on copies of the cache's tensors; the new slots, and whose slot every beam took."""
    from msa_b200.cache import window_of
    new_slots, owners = [], []
    for s, p, n in zip(slots, parents, lengths):
        named = {x for x in p if 0 <= x < len(s)}
        spare = [i for i in range(len(s)) if i not in named]
        own, seen = [], set()
        for x in p:
            first = x in named and x not in seen
            own.append(x if first else spare.pop(0))
            seen.add(x)
        for x, o in zip(p, own):
            if x not in named or o == x:
                continue
            src, dst = s[x], s[o]
            for i, spec in enumerate(c.specs):
                if i in c.ring:
                    first, rows = window_of((spec.window, spec.first), c.max_len)[1], c.ring[i].shape[1]
                    for pos in range(n):
                        at = pos if pos < first else first + (pos - first) % (rows - first)
                        c.ring[i][dst, at] = c.ring[i][src, at]
                if i in c.conv:
                    c.conv[i][dst, n % 2] = c.conv[i][src, n % 2]
                for d in (c.state, c.shift):
                    if i in d:
                        d[i][dst] = d[i][src]
            c.last_token[dst] = c.last_token[src]
        new_slots.append([s[o] for o in own])
        owners.append([x if x in named else o for x, o in zip(p, own)])
    return new_slots, owners


def table(x):
    return torch.tensor(x, dtype=I32, device=DEV)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("kind", ["rings", "odd", "states"])
@pytest.mark.parametrize("batch,beams", [(1, 1), (1, 2), (3, 4), (2, 7), (5, 32), (70, 3)])
def test_reorder(kind, batch, beams, dtype):
    g = torch.Generator().manual_seed(batch * 100 + beams)
    max_len, n_slots = 75, batch * beams + 2
    lengths = torch.randint(0, max_len + 1, (batch,), generator=g).tolist()
    lengths[0] = 75
    if batch > 2:
        lengths[1], lengths[2] = 0, 1
    slots = torch.randperm(n_slots, generator=g)[:batch * beams].view(batch, beams).tolist()
    for low in (0, -1):                                                # with and without beams that go on from nobody
        a, b = filled(kind, n_slots, max_len, dtype, 3), filled(kind, n_slots, max_len, dtype, 3)
        parents = torch.randint(low, beams, (batch, beams), generator=g).tolist()
        parents[-1] = [beams - 1] * beams
        want, _ = plain_reorder(a, slots, parents, lengths)
        got, shared = b.reorder(table(slots), table(parents), table(lengths))
        assert got.tolist() == want and shared is None
        for x, y in zip(tensors(a), tensors(b)):
            assert torch.equal(x, y)                                   # scratch and foreign slots among them


@pytest.mark.parametrize("kind", ["rings", "odd", "states"])
def test_a_life_of_many_steps_with_shared_rows(kind):
    """Beams that begin from one prompt and go on for many steps: copying only what two slots do not share comes to the same states as
    copying everything, and the table says no more than is true."""
    from msa_b200.cache import window_of
    g = torch.Generator().manual_seed(5)
    batch, beams, max_len = 3, 5, 75
    slots = torch.randperm(batch * beams, generator=g).view(batch, beams).tolist()
    lengths = [6, 1, 40]
    a, b = filled(kind, batch * beams, max_len, BF16, 1), filled(kind, batch * beams, max_len, BF16, 1)
    shared, b_slots = torch.zeros((batch, beams, beams), dtype=I32, device=DEV), table(slots)
    parents = [[0] * beams] * batch
    for step in range(34):
        slots, _ = plain_reorder(a, slots, parents, lengths)
        b_slots, shared = b.reorder(b_slots, table(parents), table(lengths), shared)
        assert b_slots.tolist() == slots
        live = [s for q in slots for s in q]
        for i, spec in enumerate(a.specs):                             # what a later step reads
            if i in a.ring:
                first, rows = window_of((spec.window, spec.first), max_len)[1], a.ring[i].shape[1]
                for q in range(batch):
                    n = lengths[q]
                    at = sorted({p if p < first else first + (p - first) % (rows - first) for p in range(n)})
                    assert torch.equal(a.ring[i][slots[q]][:, at], b.ring[i][slots[q]][:, at]), (step, i, q)
                    t = shared[q].tolist()
                    held = lambda j, p: b.ring[i][slots[q][j], p if p < first else first + (p - first) % (rows - first)]
                    for x in range(beams):
                        for y in range(beams):
                            keep = [p for p in range(t[x][y]) if p < first or p >= n - (rows - first)]
                            assert t[x][y] <= n and all(torch.equal(held(x, p), held(y, p)) for p in keep[-3:] + keep[:3])
        for x, y in zip(tensors(a)[len(a.ring):], tensors(b)[len(b.ring):]):
            assert torch.equal(x[live], y[live])
        # every beam goes on by one token: new rows, new states, the same in both
        for c in (a, b):
            h = torch.Generator(device=DEV).manual_seed(100 + step)
            for i, spec in enumerate(c.specs):
                for q in range(batch):
                    for s in slots[q]:
                        if i in c.ring:
                            first, rows = window_of((spec.window, spec.first), max_len)[1], c.ring[i].shape[1]
                            p = lengths[q]
                            c.ring[i][s, p if p < first else first + (p - first) % (rows - first)].normal_(generator=h)
                        if i in c.conv:
                            c.conv[i][s, (lengths[q] + 1) % 2].normal_(generator=h)
                        for d in (c.state, c.shift):
                            if i in d:
                                d[i][s].normal_(generator=h)
        lengths = [n + 1 for n in lengths]
        parents = torch.randint(0, beams, (batch, beams), generator=g).tolist()
        if step % 5 == 4:
            parents = [list(range(beams)) for _ in range(batch)]       # nobody moves


def test_slots_outside_the_cache_are_left_alone():
    """Entries of a table that name no slot: nothing is copied to or from them, the others are served."""
    a, b = filled("odd", 6, 30, F32, 2), filled("odd", 6, 30, F32, 2)
    for bad in (-1, 6, 7, 2 ** 31 - 1, -2 ** 31):
        got, _ = b.reorder(table([[0, bad], [2, 3], [bad, 5]]), table([[0, 0], [1, 1], [0, 0]]), table([30, 30, 30]))
        assert got.tolist() == [[0, bad], [3, 2], [bad, 5]]
    plain_reorder(a, [[2, 3]], [[1, 1]], [30])
    for x, y in zip(tensors(a), tensors(b)):
        assert torch.equal(x, y)
    b.reorder(table([[0, 1]]), table([[2 ** 31 - 1, -2 ** 31]]), table([30]))
    b.reorder(table([[0, 1]]), table([[0, 1]]), table([-5]), table([[[9, -3], [2 ** 31 - 1, 4]]]))
    for x, y in zip(tensors(a), tensors(b)):
        assert torch.equal(x, y)


def test_reorder_in_a_graph_and_on_another_stream():
    tabs = [(table([[0, 1, 2], [5, 4, 3]]), table(p), table([20, 31])) for p in ([[2, 2, 2], [0, 1, 1]], [[0, 0, 1], [2, 0, 0]])]
    want = []
    for t in tabs:
        c = filled("odd", 6, 40, BF16, 8)
        slots, _ = c.reorder(*t)
        want.append((slots, [x.clone() for x in tensors(c)]))
    c = filled("odd", 6, 40, BF16, 8)
    start = [x.clone() for x in tensors(c)]
    ins = [t.clone() for t in tabs[0]]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = c.reorder(*ins)
    side.synchronize()
    assert torch.equal(got, want[0][0]) and all(torch.equal(x, y) for x, y in zip(tensors(c), want[0][1]))
    with torch.cuda.graph(graph):
        got, _ = c.reorder(*ins)
    for t, (slots, after) in ((tabs[1], want[1]), (tabs[0], want[0])):
        for x, y in zip(ins, t):
            x.copy_(y)
        for x, y in zip(tensors(c), start):
            x.copy_(y)
        graph.replay()
        assert torch.equal(got, slots) and all(torch.equal(x, y) for x, y in zip(tensors(c), after))
