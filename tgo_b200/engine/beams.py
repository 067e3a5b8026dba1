"""Beam search above the step function: every request keeps `beams` hypotheses, and a step runs all of
them as one decode batch.

A prompt is run once; its other beams then share its pages (`Engine.follow`). Each turn selects, on the
device, the best continuations over a request's beams and the vocabulary
(`ops.beam_select`: summed log probabilities, equal ones by beam and token), (1 + stop ids) x beams of them,
so that `beams` remain however many of the others end in a stop id, and reads back those few numbers. Where
these are more than a selection gives, it is made for each beam alone, beams + stop ids of each, and the host
puts them in order. In their order, a continuation that ends in a stop id becomes a finished hypothesis (if it is
among the first `beams`: a worse one would not be kept), any other the next live beam, until there are
`beams` of them; the beams then take over the pages and states of the ones they continue, in place.

A finished hypothesis is worth its score / length ** length_penalty, its length counting the generated
tokens and not the stop id. A request is done when it has `beams` finished ones and no live beam, at its
present length, would be worth more than the worst of them; or when it has generated `max_tokens`, and its
live beams then count as finished.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional, Sequence

import numpy as np
import torch

from ..kernels import ops
from .step import Engine, StepEntry


@dataclass
class Hypothesis:
    tokens: List[int]
    score: float                      # sum of the tokens' log probabilities (and the stop id's)
    worth: float                      # score / length ** length_penalty
    stopped: bool                     # a stop id ended it


@dataclass
class _Search:
    """One request's search. Beams that have died (fewer continuations than beams) keep score -inf: they
    run along on token 0 and no selection looks at them."""
    rids: List[object]
    tokens: List[List[int]]
    scores: List[float]
    finished: List[Hypothesis] = field(default_factory=list)
    done: bool = False


class BeamSearch:
    def __init__(self, engine: Engine, beams: int, max_tokens: int, stop_ids: Sequence[int] = (),
                 length_penalty: float = 1.0, chunk: int = 2048):
        if not 0 < beams <= ops.BEAM_MAX:
            raise ValueError(f"beam search: {beams} beams; 1 to {ops.BEAM_MAX}")
        if max_tokens <= 0:
            raise ValueError(f"beam search: max_tokens {max_tokens}; it must be positive")
        if chunk <= 0:
            raise ValueError(f"beam search: the prompt chunk is {chunk}")
        self.engine, self.beams, self.max_tokens = engine, beams, max_tokens
        self.stop_ids = set(int(t) for t in stop_ids if 0 <= int(t) < engine.model.spec.vocab_size)
        self.length_penalty, self.chunk = float(length_penalty), chunk
        self._runs = 0

    def run(self, prompts: Sequence[Sequence[int]], adapters: Optional[Sequence[Optional[str]]] = None
            ) -> List[List[Hypothesis]]:
        """Every prompt's hypotheses, the one worth most first, at most `beams` of them."""
        adapters = list(adapters) if adapters is not None else [None] * len(prompts)
        if len(adapters) != len(prompts):
            raise ValueError(f"beam search: {len(adapters)} adapters for {len(prompts)} prompts")
        prompts = [[int(t) for t in p] for p in prompts]
        if any(not p for p in prompts):
            raise ValueError("beam search: a prompt is empty; there is nothing to condition on")
        if not prompts:
            return []
        self._runs += 1
        live, searches = set(), []
        try:
            for q, (prompt, adapter) in enumerate(zip(prompts, adapters)):
                s = _Search([("beam", self._runs, q, w) for w in range(self.beams)],
                            [[] for _ in range(self.beams)], [0.0] + [-np.inf] * (self.beams - 1))
                for w, rid in enumerate(s.rids):
                    self.engine.admit(rid, len(prompt) if w == 0 else 0, adapter=adapter)
                    live.add(rid)
                searches.append(s)
            logits = self._prompts(searches, prompts)
            self.engine.follow([s.rids for s in searches], [[0] * self.beams for _ in searches])
            for turn in range(self.max_tokens):
                going = [s for s in searches if not s.done]
                parents = self._advance(going, logits)
                for s in searches:
                    if s.done:
                        for rid in s.rids:
                            if rid in live:
                                self.engine.finish(rid)
                                live.discard(rid)
                pairs = [(s, p) for s, p in zip(going, parents) if not s.done]
                if not pairs or turn + 1 == self.max_tokens:
                    break
                self.engine.follow([s.rids for s, _ in pairs], [p for _, p in pairs])
                logits = self.engine.step([StepEntry(rid, [t[-1] if t else 0], [0]) for s, _ in pairs
                                           for rid, t in zip(s.rids, s.tokens)])
            self.engine.check_kernels()
        finally:
            for rid in live:
                self.engine.finish(rid)
        return [self._ranked(s) for s in searches]

    # ------------------------------------------------------------------------ pieces
    def _prompts(self, searches, prompts) -> torch.Tensor:
        """Run every prompt through its first beam; logits [requests x beams, vocabulary], of which the
        first beams' rows hold something (the others' scores are -inf: nobody reads them)."""
        V = self.engine.model.spec.vocab_size
        logits = torch.empty((len(searches) * self.beams, V), dtype=torch.float32, device=self.engine.device)
        for q, (s, prompt) in enumerate(zip(searches, prompts)):
            for o in range(0, len(prompt), self.chunk):
                part = prompt[o:o + self.chunk]
                last = o + len(part) == len(prompt)
                got = self.engine.step([StepEntry(s.rids[0], part, [len(part) - 1] if last else [])])
            logits[q * self.beams] = got[0]
        return logits

    def _select(self, searches, logits) -> List[list]:
        """Every search's continuations (value, parent, token), the best first: `beams` that end in no stop id
        are among them if there are as many. (A selection for one beam holds 64: with more than 64 - beams stop
        ids, continuations are missed of a beam whose 64 best are nearly all of them stop ids.)"""
        B, W, n = len(searches), self.beams, len(self.stop_ids)
        groups, beams, K = B, W, (1 + n) * W
        if K > ops.BEAM_MAX_PICKS:
            groups, beams, K = B * W, 1, min(W + n, ops.BEAM_MAX_PICKS)
        scores = torch.tensor([s.scores for s in searches], dtype=torch.float32).to(logits.device)
        picks = torch.empty((3, groups, K), dtype=torch.int32, device=logits.device)
        ops.beam_select(logits, scores.view(groups, beams), picks[0].view(torch.float32), picks[1], picks[2])
        host = picks.cpu().numpy()
        values = host[0].view(np.float32).tolist()
        from_beam, token = host[1].tolist(), host[2].tolist()
        found = []
        for q in range(B):
            own = [q] if groups == B else range(q * W, (q + 1) * W)
            one = [(v, p + g - own[0], t) for g in own for v, p, t in zip(values[g], from_beam[g], token[g]) if p >= 0]
            found.append(one if groups == B else sorted(one, key=lambda c: -c[0]))      # equal ones stay by beam and token
        return found

    def _advance(self, searches, logits) -> List[List[int]]:
        """Select, and bring every search a token further; the parents of its beams."""
        W = self.beams
        parents = []
        for s, found in zip(searches, self._select(searches, logits)):
            parent, tokens, scores = [], [], []
            for k, (v, p, t) in enumerate(found):
                if len(parent) == W:
                    break
                if t in self.stop_ids:
                    if k < W:
                        self._finish(s, s.tokens[p], v, True)
                    continue
                parent.append(p)
                tokens.append(s.tokens[p] + [t])
                scores.append(v)
            for w in range(len(parent), W):              # fewer continuations than beams
                parent.append(w)
                tokens.append([])
                scores.append(-np.inf)
            s.tokens, s.scores = tokens, scores
            s.done = self._is_done(s)
            parents.append(parent)
        return parents

    def _worth(self, score: float, length: int) -> float:
        return score / max(length, 1) ** self.length_penalty

    def _finish(self, s: _Search, tokens: List[int], score: float, stopped: bool) -> None:
        s.finished.append(Hypothesis(list(tokens), score, self._worth(score, len(tokens)), stopped))
        s.finished.sort(key=lambda h: -h.worth)
        del s.finished[self.beams:]

    def _is_done(self, s: _Search) -> bool:
        best = max(s.scores)
        if best == -np.inf:
            return True
        if len(s.finished) < self.beams:
            return False
        length = max(len(t) for t in s.tokens)
        return self._worth(best, length) <= s.finished[-1].worth

    def _ranked(self, s: _Search) -> List[Hypothesis]:
        if not s.done:
            for tokens, score in zip(s.tokens, s.scores):
                if score > -np.inf:
                    self._finish(s, tokens, score, False)
        return s.finished
