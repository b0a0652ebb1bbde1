"""A plain beam search over any function from a token list to log probabilities, and plain stand-ins for the two kernels."""
import math

import torch


def plain_search(log_probs, beams, max_new, stop=(), length_penalty=1.0):
    """[(rating, tokens)], best first.  ``log_probs(tokens so far)``: 64-bit scores of every next token."""
    live, ended = [(0.0, [])], []
    rate = lambda s, t: s / len(t) ** length_penalty
    while True:
        cand = []
        for b, (s, toks) in enumerate(live):
            lp = log_probs(toks)
            cand += [(s + float(lp[t]), b, t) for t in range(len(lp)) if lp[t] > -math.inf]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        for s, b, t in cand[:beams]:
            if t in stop:
                ended.append((rate(s, live[b][1] + [t]), live[b][1] + [t]))
        ended.sort(key=lambda e: -e[0])
        ended = ended[:beams]
        live = [(s, live[b][1] + [t]) for s, b, t in cand if t not in stop][:beams]
        if not live:
            return ended
        if len(live[0][1]) >= max_new:
            return sorted(ended + [(rate(s, t), t) for s, t in live], key=lambda e: -e[0])[:beams]
        if len(ended) == beams and ended[-1][0] >= rate(*live[0]):
            return ended


def plain_topk(logits, scores, k, stop=None):
    """``lm_ops.beam_topk`` in plain torch."""
    batch, beams = scores.shape
    vocab = logits.shape[1]
    total = (scores.double().view(-1, 1) + torch.log_softmax(logits.double(), 1)).view(batch, beams * vocab)
    total = torch.where(total.isnan(), -math.inf, total)
    s, at = torch.sort(total, dim=1, descending=True, stable=True)
    s, at = s[:, :k], at[:, :k]
    none = s == -math.inf
    out = [s.float(), (at // vocab).int().masked_fill(none, -1), (at % vocab).int().masked_fill(none, -1)]
    if stop is None:
        return tuple(out)
    rows = []
    for q in range(batch):
        on = [c for c in zip(*(t[q].tolist() for t in out)) if c[0] > -math.inf and c[2] not in stop.tolist()][:beams]
        rows.append(on + [(-math.inf, -1, -1)] * (beams - len(on)))
    return tuple(out) + tuple(torch.tensor([[c[i] for c in r] for r in rows], dtype=(torch.float32, torch.int32, torch.int32)[i]) for i in range(3))
