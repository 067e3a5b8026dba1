"""From rows of logits on the device to token ids, with one small read-back.

`sample_rows(logits, requests)` applies each request's Policy: biases, penalties and masks of allowed
tokens edit the rows in place, one launch for all that ask for them, then one kernel launch
samples every row (greedy rows take the argmax branch inside it), and the ids come back
as one int32 copy. Every row consumes one draw of its request's stream, greedy or not.
A policy that asks for log probabilities gets them from the same launch: the kernel that
draws also reports the drawn token's share and the most likely alternatives, so the draw
is the same with and without the report (decode.go:263-318).
"""
from __future__ import annotations

from collections import Counter
from typing import List, Optional, Sequence

import numpy as np
import torch

from ..kernels import ops
from .policy import DrawStream, Policy, TokenProb


def penalty_counts(history: Sequence[int], window: int):
    """Distinct tokens of the last `window` tokens of history (0: all) with their counts: for `adjust_row`."""
    h = list(history)
    if window > 0 and len(h) > window:
        h = h[-window:]
    c = Counter(h)
    ids = sorted(c)
    return ids, [c[i] for i in ids]


def adjust_row(row: torch.Tensor, policy: Policy, history: Sequence[int]) -> None:
    """One row edited from counts made on the host: the plain form that the tests hold `constrain` to."""
    dev = row.device
    bias_ids = bias = ids = counts = None
    if policy.logit_bias:
        keys = sorted(policy.logit_bias)
        bias_ids = torch.tensor(keys, dtype=torch.int32, device=dev)
        bias = torch.tensor([policy.logit_bias[k] for k in keys], dtype=torch.float32, device=dev)
    if policy.repetition_penalty not in (0.0, 1.0) or policy.presence_penalty != 0 or \
            policy.frequency_penalty != 0:
        i, c = penalty_counts(history, policy.penalty_window)
        if i:
            ids = torch.tensor(i, dtype=torch.int32, device=dev)
            counts = torch.tensor(c, dtype=torch.int32, device=dev)
    ops.logits_adjust(row, bias_ids, bias, ids, counts, policy.repetition_penalty,
                      policy.presence_penalty, policy.frequency_penalty)


def constrain(logits: torch.Tensor, policies: Sequence[Policy], histories: Sequence[Sequence[int]], masks: Sequence = (),
              owner: Optional[Sequence[int]] = None, drafts: Optional[tuple] = None) -> None:
    """Edit rows of logits in place as the policies ask: row r is the request's owner[r] (None: r), masks[r] an array of
    uint32 (Policy.allowed_words) or None. `drafts` as for `ops.logits_constrain`: what a row's request has
    drafted up to it comes behind its history."""
    Q, R = len(policies), logits.shape[0]
    masks = list(masks) or [None] * R
    edits = [p.edits_logits for p in policies]
    if not any(edits) and all(m is None for m in masks):
        return
    biases = [sorted(p.logit_bias.items()) for p in policies]
    said = []
    for p, h in zip(policies, histories or [()] * Q):
        if not p.penalises:
            h = ()
        elif p.penalty_window > 0:
            h = h[-p.penalty_window:]
        said.append(np.asarray(h, dtype=np.int32))
    # one buffer of 32-bit numbers, one copy: starts, owners and ids, then what is no whole number
    first_bias = np.concatenate([[0], np.cumsum([len(b) for b in biases])]).astype(np.int32)
    first_said = np.concatenate([[0], np.cumsum([s.size for s in said])]).astype(np.int32)
    kept = [m for m in masks if m is not None]
    which = np.cumsum([m is not None for m in masks]) - 1
    parts = [np.array([q if edits[q] else -1 for q in (owner if owner is not None else range(R))], dtype=np.int32),
             np.array([-1 if m is None else w for m, w in zip(masks, which)], dtype=np.int32),
             np.array([min(p.penalty_window, 2 ** 31 - 1) for p in policies], dtype=np.int32), first_bias, first_said, np.concatenate(said),
             np.array([i for b in biases for i, _ in b], dtype=np.int32),
             np.array([v for b in biases for _, v in b], dtype=np.float32),
             np.array([[p.repetition_penalty, p.presence_penalty, p.frequency_penalty] for p in policies], dtype=np.float32),
             np.stack(kept) if kept else np.empty((0, 0), dtype=np.uint32)]
    host = torch.from_numpy(np.concatenate([x.ravel().view(np.int32) for x in parts]))
    dev, at = host.to(logits.device), 0
    views = []
    for x in parts:
        views.append(dev[at:at + x.size].view(x.shape))
        at += x.size
    owners, rows, windows, b0, h0, tokens, b_ids, b_values, penalties, words = views
    floats = [t.view(torch.float32) for t in (b_values, penalties)]
    ops.logits_constrain(logits, owners, bias=(b0, b_ids, floats[0]) if b_ids.numel() else None,
                         history=(h0, tokens), penalties=floats[1], windows=windows, drafts=drafts,
                         allowed=words if kept else None, allowed_rows=rows if kept else None)


def sample_batch(logits: torch.Tensor, policies: Sequence[Policy], draws: Sequence[float],
                 histories: Sequence[Sequence[int]] = (),
                 reports: Optional[list] = None, masks: Sequence = (), edited: bool = False) -> torch.Tensor:
    """Token ids (int32, on the device) for each row. With `reports` (a list), it is
    filled with one entry per row: a TokenProb for a policy with logprobs, else None. `masks`: each row's
    Policy.allowed_words. `edited`: the rows have been through `constrain` already."""
    n = logits.shape[0]
    assert len(policies) == n and len(draws) == n
    if not edited:
        constrain(logits, policies, histories, masks)
    out = torch.empty(n, dtype=torch.int32, device=logits.device)
    asked = reports is not None and any(p.logprobs for p in policies)
    if reports is not None:
        reports[:] = [None] * n
    if all(p.greedy for p in policies) and not asked:
        ops.argmax(logits, out)
        return out
    dev = logits.device
    packed = torch.tensor([[p.temperature for p in policies], [p.top_p for p in policies],
                           list(draws)], dtype=torch.float32).to(dev)
    ks = torch.tensor([p.top_k for p in policies], dtype=torch.int32).to(dev)
    if not asked:
        ops.sample(logits, packed[0], ks, packed[1], packed[2], out)
        return out
    wants = [p.top_logprobs if p.logprobs else -1 for p in policies]
    width = max(max(wants), 0)
    report = torch.tensor(wants, dtype=torch.int32).to(dev)
    lp = torch.empty(n, dtype=torch.float32, device=dev)
    top_ids = torch.full((n, width), -1, dtype=torch.int32, device=dev) if width else None
    top_lp = torch.empty((n, width), dtype=torch.float32, device=dev) if width else None
    ops.sample(logits, packed[0], ks, packed[1], packed[2], out, report, lp, top_ids, top_lp)
    ids, lps = out.tolist(), lp.tolist()
    alt_ids = top_ids.tolist() if width else None
    alt_lps = top_lp.tolist() if width else None
    for r, w in enumerate(wants):
        if w < 0:
            continue
        top = [TokenProb(i, v) for i, v in zip(alt_ids[r][:w], alt_lps[r][:w]) if i >= 0] \
            if w else []
        reports[r] = TokenProb(ids[r], lps[r], top)
    return out


def sample_rows(logits: torch.Tensor, requests) -> List[int]:
    """The Runner's sampling hook: requests carry `.policy`, `.sampler` (a DrawStream),
    `.prompt`, `.output` and `.logprobs` (a TokenProb is appended for every sampled token of a
    policy that asks; the Runner drops a stop token's)."""
    policies, draws, histories, masks = [], [], [], []
    for req in requests:
        if req.sampler is None:
            req.sampler = DrawStream(req.policy.seed)
        policies.append(req.policy)
        draws.append(req.sampler.next())
        histories.append(req.prompt + req.output if req.policy.edits_logits else ())
        masks.append(req.policy.allowed_words(req.output, logits.shape[1]))
    reports: list = []
    ids = sample_batch(logits, policies, draws, histories, reports, masks).tolist()
    for req, rep in zip(requests, reports):
        if rep is not None:
            req.logprobs.append(rep)
    return ids
