"""Stand-ins for the kernels of adapters and beam search, with torch on the CPU, beside those of
emulated_kernels.py; and a plain beam search over whole forwards, which shares no code with the engine."""
from __future__ import annotations

import numpy as np
import torch

import emulated_kernels


def beam_select(logits, scores, picked, parents, tokens):
    B, W = scores.shape
    V, K = logits.shape[1], picked.shape[1]
    picked.fill_(float("-inf"))
    parents.fill_(-1)
    tokens.fill_(-1)
    for b in range(B):
        found = []
        for w in range(W):
            if not torch.isfinite(scores[b, w]):
                continue                              # such a beam's row is not looked at
            v = scores[b, w].double() + torch.log_softmax(logits[b * W + w].double(), 0)
            order = v.argsort(descending=True, stable=True)[:K].tolist()
            found += [(-float(v[i]), w, i) for i in order if v[i] > -float("inf")]
        for k, (v, w, i) in enumerate(sorted(found)[:K]):
            picked[b, k], parents[b, k], tokens[b, k] = -v, w, i


def reorder_rows(tensors, index, parents, axis=0):
    for t in tensors:
        old = t.clone()
        for row, par in zip(index.tolist(), parents.tolist()):
            for w, p in enumerate(par):
                if p != w and 0 <= p < len(row) and min(row[w], row[p]) >= 0 and max(row[w], row[p]) < t.shape[axis]:
                    t.select(axis, row[w]).copy_(old.select(axis, row[p]))


def low_rank_add(x, y, a, b, scale, ids, widths, interleaved=False, out=None):
    out = y if out is None else out
    new = y.double().clone()
    col = (torch.arange(sum(widths)) // 8) % 2 if interleaved else \
        torch.repeat_interleave(torch.arange(len(widths)), torch.tensor(widths))
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero().flatten()
        for s in range(len(widths)):
            at = (col == s).nonzero().flatten()
            d = (x[rows].double() @ a[i, s].double().T) @ b[i][at].double().T
            new[rows.unsqueeze(1), at] += scale[i].double() * d
    out.copy_(new.to(out.dtype))


def install(monkeypatch):
    from tgo_b200.kernels import ops
    emulated_kernels.install(monkeypatch)
    for name in ("beam_select", "reorder_rows", "low_rank_add"):
        monkeypatch.setattr(ops, name, globals()[name])


# --------------------------------------------------------------------- a plain search


def random_adapter(spec, names, rank, seed, size=0.3):
    """{matrix: (A, B)} for some of a model's matrices, given {matrix: [out, in]}."""
    g = torch.Generator().manual_seed(seed)
    return {n: (torch.randn(rank, spec[n][1], generator=g) * spec[n][1] ** -0.5,
                torch.randn(spec[n][0], rank, generator=g) * size * rank ** -0.5) for n in names}


def with_adapter(weights, matrices, scale):
    """The plain implementation's weights with an adapter's product added to its matrices."""
    out = dict(weights)
    for n, (a, b) in matrices.items():
        out[n] = out[n] + scale * (b.double().numpy() @ a.double().numpy()).astype(np.float32)
    return out


def plain_beam_search(last_logits, prompt, beams, max_tokens, stop_ids=(), length_penalty=1.0):
    """last_logits(tokens) -> the logits behind the last of them. [(tokens, score, stopped)], best first."""
    def worth(s, n):
        return s / max(n, 1) ** length_penalty
    live, done = [([], 0.0)], []
    finished = False
    for _ in range(max_tokens):
        found = []
        for w, (t, s) in enumerate(live):
            x = np.asarray(last_logits(prompt + t), dtype=np.float64)
            lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
            found += [(-(s + lp[i]), w, i) for i in np.argsort(-lp, kind="stable")[:2 * beams]]
        new = []
        for k, (v, w, i) in enumerate(sorted(found)[:2 * beams]):
            if len(new) == beams:
                break
            if int(i) in stop_ids:
                if k < beams:
                    done = sorted(done + [(worth(-v, len(live[w][0])), live[w][0], -v, True)], key=lambda h: -h[0])[:beams]
                continue
            new.append((live[w][0] + [int(i)], -v))
        live = new
        if not live or (len(done) == beams and worth(live[0][1], len(live[0][0])) <= done[-1][0]):
            finished = True
            break
    if not finished:
        done = sorted(done + [(worth(s, len(t)), t, s, False) for t, s in live], key=lambda h: -h[0])[:beams]
    return [(t, s, stopped) for _, t, s, stopped in done]
