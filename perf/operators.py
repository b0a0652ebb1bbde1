"""Operators of beam search over the layered decoders' cache, measured alone: attention over a window with first tokens that stay
visible (portions of prompts, and decode tokens over the rings), the choice of the next beams from the logits, and the reordering of
the sequence states that the choice asks for.

Three restatements of each.  ``run`` with ``own`` false is the plain form in 32 bits (64 for the sums behind an order), with
``own`` true the package's kernels, and ``exact`` the definition in 64 bits.  Everything random comes from the seed, drawn on
the GPU in a fixed order, so that all of them see the same inputs.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


def listed():
    return [
        # a short portion in a small layer: the window cuts inside it
        dict(name="portion-small", kind="portion", heads=8, kv=2, dim=64, vdim=128, window=100, first=3, sink=True, gate=True, portions="150@0"),
        # prompts of a lightly loaded server, a window of a quarter of their length
        dict(name="portion-prompts", kind="portion", heads=16, kv=4, dim=128, vdim=128, window=512, first=4, sink=False, gate=False,
             portions="2048@0,1500@0,1911@0,777@0"),
        # the largest: long portions of longer prompts, the wide layers of the benchmark's larger design
        dict(name="portion-long", kind="portion", heads=32, kv=8, dim=128, vdim=128, window=2048, first=4, sink=True, gate=True,
             portions="2048@0,2048@2048,2048@9000,2048@31007"),
        # one token of one sequence whose window has moved on long ago: latency
        dict(name="token-one", kind="token", heads=16, kv=4, dim=128, vdim=128, window=1024, first=4, sink=True, gate=True, batch=1, shortest=30000, longest=30000),
        # a decode step of a busy server, sequences of all lengths
        dict(name="token-batch", kind="token", heads=32, kv=8, dim=128, vdim=128, window=2048, first=64, sink=True, gate=True, batch=128,
             shortest=1, longest=9000),
        # narrow heads, eight query heads to a key head, no gate
        dict(name="token-narrow", kind="token", heads=32, kv=4, dim=64, vdim=64, window=4095, first=1, sink=False, gate=False, batch=33,
             shortest=500, longest=20000),
        # one question searched with four beams
        dict(name="choice-one", kind="choice", batch=1, beams=4, vocab=32768, k=8, stops=1, dtype="float32"),
        # many questions at once over a wide vocabulary
        dict(name="choice-many", kind="choice", batch=48, beams=4, vocab=151936, k=12, stops=2, dtype="float32"),
        # wide beams over an odd vocabulary, logits as 16-bit products leave them
        dict(name="choice-wide", kind="choice", batch=8, beams=32, vocab=50001, k=64, stops=1, dtype="bfloat16"),
        # one question of a small model
        dict(name="states-one", kind="states", batch=1, beams=4, kept=2, rings=2, width=512, window=512, first=4, mats=2, heads=8, dim=64, vdim=64,
             channels=1536, taps=4, shift=512, prompt=400, grown=20, max_len=2048, dtype="bfloat16"),
        # the states of a design that mixes windowed attention with recurrences: whole matrices move
        dict(name="states-mixed", kind="states", batch=16, beams=4, kept=2, rings=4, width=1024, window=1024, first=4, mats=3, heads=64, dim=128, vdim=64,
             channels=6144, taps=4, shift=0, prompt=2000, grown=300, max_len=4096, dtype="bfloat16"),
        # rings that keep everything behind a long prompt that all beams share
        dict(name="states-long", kind="states", batch=8, beams=8, kept=3, rings=4, width=2048, window=0, first=0, mats=0, heads=0, dim=0, vdim=0,
             channels=8192, taps=3, shift=0, prompt=5000, grown=700, max_len=6144, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _one(rng):
    kind = rng.choice(["portion", "token", "choice", "states"])
    if kind in ("portion", "token"):
        kv = rng.choice([1, 2, 4, 8])
        case = dict(kind=kind, heads=kv * rng.choice([1, 2, 3, 4, 5, 8]), kv=kv, dim=rng.choice([64, 128]), vdim=rng.choice([64, 128]),
                    window=_log(rng, 1, 4096), first=rng.choice([1, 2, 3, 4, 5, 16, 64, 100]), sink=rng.random() < 0.5, gate=rng.random() < 0.5)
        if kind == "token":
            longest = _log(rng, 2, 40000)
            return dict(case, batch=_log(rng, 1, 128), shortest=rng.randint(1, longest), longest=longest)
        return dict(case, portions=",".join(f"{_log(rng, 2, 2048)}@{rng.choice([0, _log(rng, 1, 20000)])}" for _ in range(rng.randint(1, 5))))
    if kind == "choice":
        beams = rng.randint(1, 32)
        return dict(kind=kind, batch=_log(rng, 1, 64), beams=beams, vocab=_log(rng, 200, 200000), k=rng.randint(beams, 2 * beams), stops=rng.randint(0, 3),
                    dtype=rng.choice(["float32", "bfloat16"]))
    beams, window = rng.randint(2, 16), rng.choice([0, _log(rng, 16, 2048)])
    mats, prompt, grown = rng.randint(0, 3), _log(rng, 1, 3000), _log(rng, 1, 1000)
    return dict(kind=kind, batch=_log(rng, 1, 16), beams=beams, kept=rng.randint(1, beams), rings=rng.randint(1, 4), width=8 * _log(rng, 4, 256),
                window=window, first=rng.choice([0, 1, 4, 64]) if window else 0, mats=mats, heads=rng.choice([4, 8, 32]), dim=rng.choice([64, 128]),
                vdim=rng.choice([64, 128]), channels=8 * _log(rng, 8, 800), taps=rng.randint(2, 4), shift=rng.choice([0, 1024]), prompt=prompt,
                grown=grown, max_len=prompt + grown + rng.randint(0, 500), dtype=rng.choice(["float32", "bfloat16"]))


def _cost(case):
    """Seconds of the work at round rates (a floor under small calls, so that these compare as equals)."""
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / 1.4e15, 1e-6)


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        case = _one(rng)
        if _cost(case) <= top and _memory(case) < 12e9:
            return case


# ---------------------------------------------------------------------------------------------------- sizes
def _portions(case):
    return [tuple(int(x) for x in p.split("@")) for p in case["portions"].split(",")]


def _lengths(case):
    """Positions of the tokens: spread over shortest .. longest, in no order."""
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [lo - 1 + (hi - lo) * ((i * 37 + 11) % n) // max(n - 1, 1) for i in range(n)]


def _seen(pos, case):
    """Rows that position ``pos`` sees."""
    lo = max(0, pos - case["window"] + 1)
    return min(case["first"], lo) + pos - lo + 1


def _ring_rows(case):
    return case["max_len"] if not case["window"] else min(case["window"] + case["first"], case["max_len"])


def _moved_rows(case):
    """Ring rows of the positions prompt .. prompt + grown - 1 that are still held."""
    n, rows, first = case["prompt"] + case["grown"], _ring_rows(case), case["first"]
    oldest = max(first, n - (rows - first)) if n > rows else 0
    return sum(1 for p in range(case["prompt"], n) if p < first or p >= oldest)


def _esize(case):
    return 2 if case.get("dtype", "bfloat16") == "bfloat16" else 4


def _memory(case):
    if case["kind"] == "states":
        slots = case["batch"] * case["beams"] + 1
        return slots * (case["rings"] * _ring_rows(case) * case["width"] * _esize(case) + case["mats"] * case["heads"] * case["dim"] * case["vdim"] * 4)
    if case["kind"] == "choice":
        return case["batch"] * case["beams"] * case["vocab"] * 20          # what the plain form spreads
    if case["kind"] == "token":
        return case["batch"] * (case["window"] + case["first"]) * case["kv"] * (case["dim"] + case["vdim"]) * 8
    return max(n * min(n + s, case["window"] + case["first"] + n) for n, s in _portions(case)) * case["heads"] // case["kv"] * 12


def work(case):
    kind = case["kind"]
    if kind == "portion":
        span = case["window"] + case["first"]
        pairs = sum(_seen(s + i, case) for n, s in _portions(case) for i in range(n))
        rows, ctx = sum(n for n, _ in _portions(case)), sum(min(s, span - 1) + n for n, s in _portions(case))
        per = case["dim"] + case["vdim"]
        return dict(bytes=2 * per * (rows * case["heads"] + ctx * case["kv"]), flops=2 * per * pairs * case["heads"])
    if kind == "token":
        seen, per = sum(_seen(p, case) for p in _lengths(case)), case["dim"] + case["vdim"]
        return dict(bytes=2 * per * (case["batch"] * case["heads"] + seen * case["kv"]), flops=2 * per * seen * case["heads"])
    if kind == "choice":
        n = case["batch"] * case["beams"] * case["vocab"]
        return dict(bytes=n * _esize(case) + case["batch"] * (4 * case["beams"] + 12 * (case["k"] + case["beams"])), flops=3 * n)
    e = _esize(case)
    one = (case["rings"] * (_moved_rows(case) * case["width"] + (case["taps"] - 1) * case["channels"]) * e
           + case["mats"] * (case["heads"] * case["dim"] * case["vdim"] * 4 + (case["taps"] - 1) * case["channels"] * e + case["shift"] * e) + 4)
    return dict(bytes=2 * one * case["batch"] * (case["beams"] - case["kept"]), flops=0)


# ---------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _attention_inputs(case, g, n):
    q = _randn(g, n, case["heads"], case["dim"], scale=1.5)
    gate = _randn(g, n, case["heads"]) if case["gate"] else None
    return q, gate


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "portion":
        parts, span = _portions(case), case["window"] + case["first"]
        n = sum(x for x, _ in parts)
        q, gate = _attention_inputs(case, g, n)
        width = case["kv"] * (case["dim"] + case["vdim"])
        ctx = _randn(g, sum(min(s, span - 1) + x for x, s in parts), width)
        st = dict(case=case, q=q, gate=gate, ctx=ctx, out=torch.empty((n, case["heads"], case["vdim"]), dtype=BF16, device=DEV))
        if own:
            from msa_b200.cache import PackedStep, RingSpec, SequenceStateCache
            cache = SequenceStateCache([RingSpec(8, case["window"], first=case["first"])], len(parts), max(s + x for x, s in parts) + span, DEV, BF16)
            for i, (_, s) in enumerate(parts):
                cache.acquire(i)
                cache.advance(i, s)
            key = (case["window"], case["first"])
            st["step"] = PackedStep([(i, [0] * x, []) for i, (x, _) in enumerate(parts)], cache, (key,))
            st["view"], st["status"] = st["step"].views[key], torch.zeros(4, dtype=I32, device=DEV)
        return st
    if kind == "token":
        n, rows = case["batch"], case["window"] + case["first"]
        q, gate = _attention_inputs(case, g, n)
        ring = _randn(g, n + 1, rows, case["kv"] * (case["dim"] + case["vdim"]))
        slot = torch.randperm(n, generator=g, device=DEV).to(I32)
        pos = torch.tensor(_lengths(case), dtype=I32, device=DEV)
        st = dict(case=case, q=q, gate=gate, ring=ring, slot=slot, pos=pos, out=torch.empty((n, case["heads"], case["vdim"]), dtype=BF16, device=DEV))
        if own:
            from msa_b200.cache import DecodeStep, RingSpec, SequenceStateCache
            key = (case["window"], case["first"])
            cache = SequenceStateCache([RingSpec(ring.shape[2], case["window"], first=case["first"])], n, case["longest"] + rows, DEV, BF16)
            cache.ring[0].copy_(ring)
            st["ring"], st["step"] = cache.ring[0], DecodeStep(n, cache, (key,))
            st["step"].slot.copy_(slot)
            st["step"].pos.copy_(pos)
            st["view"] = st["step"].views[key]
        return st
    if kind == "choice":
        rows, vocab = case["batch"] * case["beams"], case["vocab"]
        logits = torch.randn((rows, vocab), generator=g, device=DEV) * 2.5
        likely = torch.randint(0, vocab, (rows, 24), generator=g, device=DEV)         # what the context makes likely
        logits.scatter_add_(1, likely, torch.rand((rows, 24), generator=g, device=DEV) * 9)
        stop = torch.randperm(vocab, generator=g, device=DEV)[:case["stops"]].to(I32)
        if case["stops"]:
            logits[:, stop.long()] += torch.rand((rows, case["stops"]), generator=g, device=DEV) * 12
        scores = -(torch.rand((case["batch"], case["beams"]), generator=g, device=DEV) * 6).cumsum(1) * (4 / case["beams"]) - 10
        return dict(case=case, logits=logits.to(getattr(torch, case["dtype"])), scores=scores, stop=stop)
    return _prepare_states(case, g)


def _prepare_states(case, g):
    batch, beams, n, dt = case["batch"], case["beams"], case["prompt"] + case["grown"], getattr(torch, case["dtype"])
    slots, rows, first = batch * beams, _ring_rows(case), case["first"]
    if own:
        from msa_b200.cache import RecurrentSpec, RingSpec, SequenceStateCache
        specs = [RingSpec(case["width"], case["window"] or None, case["channels"], case["taps"], first=first)] * case["rings"]
        specs += [RecurrentSpec(case["heads"], case["dim"], case["vdim"], case["channels"], case["taps"], case["shift"])] * case["mats"]
        cache = SequenceStateCache(specs, slots, case["max_len"], DEV, dt)
        by_run = lambda d: [d[i] for i in sorted(d)]
        st = dict(cache=cache, ring=by_run(cache.ring), state=by_run(cache.state), conv=by_run(cache.conv), shift=by_run(cache.shift), last=cache.last_token)
    else:
        new = lambda k, *shape, dtype=dt: [torch.empty((slots + 1, *shape), dtype=dtype, device=DEV) for _ in range(k)]
        st = dict(ring=new(case["rings"], rows, case["width"]), state=new(case["mats"], case["heads"], case["dim"], case["vdim"], dtype=F32),
                  conv=new(case["rings"] + case["mats"], 2, case["taps"] - 1, case["channels"]),
                  shift=new(case["mats"] if case["shift"] else 0, case["shift"]), last=torch.empty(slots + 1, dtype=I32, device=DEV))
    for name in ("ring", "state", "conv", "shift"):
        for t in st[name]:
            t.normal_(generator=g)
    st["last"].random_(0, 30000, generator=g)
    st["slot"] = torch.randperm(slots, generator=g, device=DEV).to(I32).view(batch, beams)
    # beams of one question hold the same rows for its prompt
    pos = torch.arange(case["prompt"], device=DEV)
    if n > rows:
        pos = pos[(pos < first) | (pos >= n - (rows - first))]
    at = torch.where(pos < first, pos, first + (pos - first) % max(rows - first, 1))
    for t in st["ring"]:
        for e in range(batch):
            s = st["slot"][e].long()
            t[s[1:, None], at[None, :]] = t[s[0], at][None]
    # `kept` beams live on, each at least once
    order = torch.rand((batch, beams), generator=g, device=DEV).argsort(1)
    pick = torch.cat([torch.arange(case["kept"], device=DEV).expand(batch, -1),
                      torch.randint(0, case["kept"], (batch, beams - case["kept"]), generator=g, device=DEV)], dim=1)
    pick = pick.gather(1, torch.rand((batch, beams), generator=g, device=DEV).argsort(1))
    st["parent"] = order.gather(1, pick).to(I32)
    st["length"] = torch.full((batch,), n, dtype=I32, device=DEV)
    st["shared"] = torch.full((batch, beams, beams), case["prompt"], dtype=I32, device=DEV)
    return dict(st, case=case)


# ---------------------------------------------------------------------------------------------------- plain forms
def _softmax_rows(s, seen, sink):
    """Weights of the seen entries along the last axis; with ``sink`` one more entry of score 0 shares the sum."""
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    if sink:
        m = m.clamp(min=0)
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    return e / (total + torch.exp(-m) if sink else total)


def _gated(o, gate):
    return o if gate is None else o / (1 + torch.exp(-gate.to(o.dtype)))[..., None]


def _context_positions(start, n, case):
    """Positions of the rows of a portion's context: the first tokens, the window before the portion, the portion."""
    lo = max(0, start - case["window"] + 1)
    return torch.cat([torch.arange(min(case["first"], lo), device=DEV), torch.arange(lo, start + n, device=DEV)])


def _plain_portion(st):
    case, row, at = st["case"], 0, 0
    out, kv, d, dv = st["out"], case["kv"], case["dim"], case["vdim"]
    group, scale = case["heads"] // kv, d ** -0.5
    for n, start in _portions(case):
        j = _context_positions(start, n, case)
        i = torch.arange(start, start + n, device=DEV)[:, None]
        seen = (j <= i) & ((i - j < case["window"]) | (j < case["first"]))
        ctx = st["ctx"][at:at + len(j)].float()
        for h in range(kv):
            k, v = ctx[:, h * d:(h + 1) * d], ctx[:, kv * d + h * dv:kv * d + (h + 1) * dv]
            q = st["q"][row:row + n, h * group:(h + 1) * group].float().transpose(0, 1)
            o = (_softmax_rows(q @ k.t() * scale, seen, case["sink"]) @ v).transpose(0, 1)
            gate = None if st["gate"] is None else st["gate"][row:row + n, h * group:(h + 1) * group]
            out[row:row + n, h * group:(h + 1) * group] = _gated(o, gate).to(BF16)
        row, at = row + n, at + len(j)
    return out


def _plain_token(st):
    case = st["case"]
    n, kv, d, dv, window, first = case["batch"], case["kv"], case["dim"], case["vdim"], case["window"], case["first"]
    pos = st["pos"].long()
    lo = (pos - window + 1).clamp(min=0)
    front = lo.clamp(max=first)
    c = torch.arange(window + first, device=DEV)
    j = torch.where(c[None] < front[:, None], c[None], (lo - front)[:, None] + c[None])
    seen = j <= pos[:, None]
    at = torch.where(j < first, j, first + (j - first) % window)
    rows = st["ring"][st["slot"].long()[:, None], at].float()
    k = rows[..., :kv * d].unflatten(-1, (kv, d)).permute(0, 2, 3, 1)
    v = rows[..., kv * d:].unflatten(-1, (kv, dv)).transpose(1, 2)
    q = st["q"].float().view(n, kv, case["heads"] // kv, d)
    o = _softmax_rows(q @ k * d ** -0.5, seen[:, None, None], case["sink"]) @ v
    st["out"].copy_(_gated(o.reshape(n, case["heads"], dv), st["gate"]))
    return st["out"]


def _first_of(keep, score, beam, token, n):
    """The first ``n`` kept candidates of every row; places without one are (-inf, -1, -1)."""
    order = torch.sort((~keep).to(I32), dim=1, stable=True).indices[:, :n]
    kept = keep.gather(1, order)
    pick = lambda t, no: torch.where(kept, t.gather(1, order), torch.full_like(t[:, :1], no))
    return pick(score, -math.inf), pick(beam, -1), pick(token, -1)


def _plain_choice(st):
    case = st["case"]
    batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
    x = st["logits"].to(F64)                         # the order of close candidates hangs on the long sums
    m = x.amax(1, keepdim=True)
    total = st["scores"].to(F64).view(-1, 1) + (x - (m + torch.log(torch.exp(x - m).sum(1, keepdim=True))))
    score, at = torch.sort(total.view(batch, beams * vocab), dim=1, descending=True, stable=True)
    score, at = score[:, :case["k"]], at[:, :case["k"]]
    none = ~(score > -math.inf)
    beam, token = (at // vocab).to(I32).masked_fill(none, -1), (at % vocab).to(I32).masked_fill(none, -1)
    score = score.to(F32)
    keep = ~none & ~(token[..., None] == st["stop"]).any(-1)
    return (score, beam, token, *_first_of(keep, score, beam, token, beams))


def _plain_states(st):
    case = st["case"]
    batch, beams, first = case["batch"], case["beams"], case["first"]
    parent, slot, length = st["parent"].long(), st["slot"], st["length"].long()
    earlier = torch.ones((beams, beams), dtype=torch.bool, device=DEV).tril(-1)
    copied = ((parent[:, :, None] == parent[:, None, :]) & earlier).any(2)           # somebody before it took the parent's slot
    free = ~(parent[:, :, None] == torch.arange(beams, device=DEV)).any(1)           # beams that nobody continues
    spare = torch.sort((~free).to(I32), dim=1, stable=True).indices                  # those first, in order
    to = torch.where(copied, spare.gather(1, (copied.cumsum(1) - 1).clamp(min=0)), parent)
    slot_out = slot.gather(1, to)
    e, j = copied.nonzero(as_tuple=True)
    src, dst = slot.long()[e, parent[e, j]], slot_out.long()[e, j]
    n = length[e]
    for t in st["ring"]:
        held = torch.arange(t.shape[1], device=DEV)[None] < n[:, None]               # rows that have been written
        t[dst] = torch.where(held[..., None], t[src], t[dst])
    for t in st["state"] + st["shift"] + [st["last"]]:
        t[dst] = t[src]
    for t in st["conv"]:
        t[dst, n & 1] = t[src, n & 1]
    b = torch.arange(batch, device=DEV)[:, None, None]
    shared = torch.where(parent[:, :, None] == parent[:, None, :], st["length"][:, None, None], st["shared"][b, parent[:, :, None], parent[:, None, :]])
    return [slot_out, shared, st["last"]] + st["ring"] + st["state"] + st["conv"] + st["shift"]


# ---------------------------------------------------------------------------------------------------- one pass
def run(st):
    case = st["case"]
    kind = case["kind"]
    if not own:
        return {"portion": _plain_portion, "token": _plain_token, "choice": _plain_choice, "states": _plain_states}[kind](st)
    from msa_b200 import lm_ops as K
    if kind == "portion":
        from msa_b200.hybrid import portion_attention
        kv, d, dv = case["kv"], case["dim"], case["vdim"]
        k, v = st["ctx"][:, :kv * d].unflatten(1, (kv, d)), st["ctx"][:, kv * d:].unflatten(1, (kv, dv))
        portion_attention((st["q"], None, k, None, v, st["out"]), True, st["status"], st["step"], st["view"], d ** -0.5, sink=case["sink"], gate=st["gate"])
        return st["out"]
    if kind == "token":
        view = st["view"]
        K.group_decode(st["q"], st["ring"], case["kv"], st["step"], st["out"], window=view.window, first=view.first, scale=case["dim"] ** -0.5,
                       sink=case["sink"], gate=st["gate"])
        return st["out"]
    if kind == "choice":
        return K.beam_topk(st["logits"], st["scores"], case["k"], stop=st["stop"])
    slot, shared = st["cache"].reorder(st["slot"], st["parent"], st["length"], st["shared"])
    return [slot, shared, st["last"]] + st["ring"] + st["state"] + st["conv"] + st["shift"]


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _attend(q, k, v, seen, scale, sink):
    """q [n, h, d], k [m, h, d], v [m, h, dv], seen [n, m]."""
    s = torch.einsum("ihd,jhd->hij", q, k) * scale
    s = s.masked_fill(~seen, -math.inf)
    if sink:
        s = torch.cat([s, s.new_zeros(s.shape[0], s.shape[1], 1)], dim=2)
        v = torch.cat([v, v.new_zeros(1, v.shape[1], v.shape[2])])
    return torch.einsum("hij,jhd->ihd", torch.softmax(s, dim=-1), v)


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    kind = case["kind"]
    if kind in ("portion", "token"):
        def visible(start, n):                       # positions that some token of start .. start + n - 1 sees
            j = torch.arange(start + n, device=DEV)
            return j[(j < case["first"]) | (start - j < case["window"])]
        kv, d, dv = case["kv"], case["dim"], case["vdim"]
        split = lambda rows: (rows[:, :kv * d].view(-1, kv, d).double(), rows[:, kv * d:].view(-1, kv, dv).double())
        out = torch.empty(st["out"].shape, dtype=F64, device=DEV)
        if kind == "portion":
            jobs, row, at = [], 0, 0
            for n, s in _portions(case):
                j = visible(s, n)
                jobs.append((row, s, n, j, st["ctx"][at:at + len(j)]))
                row, at = row + n, at + len(j)
        else:
            jobs = []
            for b, (p, s) in enumerate(zip(_lengths(case), st["slot"].tolist())):
                j = visible(p, 1)
                row_of = [x if x < case["first"] else case["first"] + (x - case["first"]) % case["window"] for x in j.tolist()]
                jobs.append((b, p, 1, j, st["ring"][s, row_of]))
        for row, start, n, j, rows in jobs:
            k, v = split(rows)
            q = st["q"][row:row + n].double()
            for i0 in range(0, n, 512):              # rows at a time
                i1 = min(i0 + 512, n)
                i = torch.arange(start + i0, start + i1, device=DEV)
                back = i[:, None] - j[None, :]
                seen = (back >= 0) & ((back < case["window"]) | (j[None, :] < case["first"]))
                for h in range(kv):                  # a key head at a time
                    hs = slice(h * (case["heads"] // kv), (h + 1) * (case["heads"] // kv))
                    g = case["heads"] // kv
                    out[row + i0:row + i1, hs] = _attend(q[i0:i1, hs], k[:, h:h + 1].expand(-1, g, -1), v[:, h:h + 1].expand(-1, g, -1), seen, d ** -0.5,
                                                         case["sink"])
        return out if st["gate"] is None else out * torch.sigmoid(st["gate"].double())[..., None]
    if kind == "choice":
        score, beam, token, live = [], [], [], []
        stop = set(st["stop"].tolist())
        for e in range(case["batch"]):
            rows = st["logits"][e * case["beams"]:(e + 1) * case["beams"]].double()
            flat = (torch.log_softmax(rows, dim=1) + st["scores"][e].double()[:, None]).flatten()
            best = torch.topk(flat, min(4 * case["k"] + 64, flat.numel())).indices.sort().values
            best = best[torch.sort(flat[best], descending=True, stable=True).indices[:case["k"]]]
            s, b, t = flat[best].tolist(), (best // case["vocab"]).tolist(), (best % case["vocab"]).tolist()
            on = [x for x in zip(s, b, t) if x[2] not in stop][:case["beams"]]
            on += [(-math.inf, -1, -1)] * (case["beams"] - len(on))
            score.append(s), beam.append(b), token.append(t), live.append(on)
        whole = lambda x: torch.tensor(x, dtype=I32, device=DEV)
        part = lambda i: [[x[i] for x in on] for on in live]
        return (torch.tensor(score, dtype=F64, device=DEV), whole(beam), whole(token), torch.tensor(part(0), dtype=F64, device=DEV), whole(part(1)), whole(part(2)))
    # states: beam by beam
    slots, parents, lengths, table = st["slot"].tolist(), st["parent"].tolist(), st["length"].tolist(), st["shared"].tolist()
    new_slots, new_shared = [], []
    for s, p, n, sh in zip(slots, parents, lengths, table):
        spare = [s[i] for i in range(len(s)) if i not in p]
        mine = []
        for i, x in enumerate(p):
            if x not in p[:i]:
                mine.append(s[x])
                continue
            mine.append(spare.pop(0))
            for t in st["ring"]:
                t[mine[-1], :n] = t[s[x], :n]
            for t in st["state"] + st["shift"] + [st["last"]]:
                t[mine[-1]] = t[s[x]]
            for t in st["conv"]:
                t[mine[-1], n % 2] = t[s[x], n % 2]
        new_slots.append(mine)
        new_shared.append([[n if a == b else sh[a][b] for b in p] for a in p])
    whole = lambda x: torch.tensor(x, dtype=I32, device=DEV)
    return [whole(new_slots), whole(new_shared), st["last"]] + st["ring"] + st["state"] + st["conv"] + st["shift"]
