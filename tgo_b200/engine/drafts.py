"""Generation with drafted tokens: several tokens a step where a cheap guess at what comes next is right.

A drafter proposes a tree of continuations for every request; the engine runs all the trees as one batch
(`Engine.draft_step`: every token attends over its request's cache and its own path), a token is chosen behind each of
their tokens by the request's policy, and each request keeps the drafts that were chosen, and the token behind the last
of them. A token is chosen with the draw that it would have had without drafts, and its history, its penalties and its
grammar's mask are those of its path, so the result does not depend on the drafts (but for rounding: steps of
other sizes run other kernels).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import numpy as np

from ..cache.pages import PagesExhausted, SlotsExhausted
from ..kernels import ops
from ..sampling.policy import DrawStream
from ..sampling.sampler import constrain, sample_batch, sample_rows
from .scheduler import ContextExhausted, Request
from .step import DraftEntry, Engine, StepEntry


class NgramDrafter:
    """Continuations of earlier places in the request's own tokens that ended as it ends now: the longest
    endings first (of `longest` tokens, then fewer, down to `shortest`), the latest places first."""

    def __init__(self, longest: int = 4, shortest: int = 1, depth: int = 8):
        if not 1 <= shortest <= longest or depth < 1:
            raise ValueError(f"drafter: endings of {shortest} to {longest} tokens, continuations of {depth}")
        self.longest, self.shortest, self.depth = longest, shortest, depth

    def propose(self, tokens: Sequence[int], nodes: int) -> Tuple[List[int], List[int]]:
        """At most `nodes` drafted tokens behind `tokens`, and for each the place it continues: 0 is the last of `tokens`,
        i the drafted token i - 1."""
        t = np.asarray(tokens)
        drafted: List[int] = []
        parents: List[int] = []
        children: Dict[Tuple[int, int], int] = {}
        seen = set()
        for n in range(min(self.longest, len(t) - 1), self.shortest - 1, -1):
            ends = np.arange(n - 1, len(t) - 1)              # an ending's last place, with a token behind it
            for k in range(n):
                ends = ends[t[ends - k] == t[len(t) - 1 - k]]
            for e in ends[::-1].tolist():
                if len(drafted) >= nodes:
                    return drafted, parents
                if e in seen:
                    continue
                seen.add(e)
                at = 0
                for token in t[e + 1:e + 1 + self.depth].tolist():
                    nxt = children.get((at, token))
                    if nxt is None:
                        if len(drafted) >= nodes:
                            break
                        drafted.append(token)
                        parents.append(at)
                        nxt = children[(at, token)] = len(drafted)
                    at = nxt
        return drafted, parents


@dataclass
class _Live:
    request: Request
    rid: object


class DraftedGeneration:
    """Requests through an engine with drafted tokens: a prompt is run when its request is admitted, then every turn is one
    step of all live requests' trees, or a decode step where no request has a draft. When pages run out, a turn goes
    without drafts, and if that does not help the request that was admitted last gives its pages back and is run again later."""

    def __init__(self, engine: Engine, drafter=None, nodes: int = 16, chunk: int = 2048, stop_ids: Sequence[int] = ()):
        why = engine.takes_drafts()
        if why:
            raise ValueError(f"drafted generation: not with this model: {why}")
        if not 1 <= nodes <= ops.TREE_NODES:
            raise ValueError(f"drafted generation: trees of {nodes} tokens; 1 to {ops.TREE_NODES}")
        if chunk <= 0:
            raise ValueError(f"drafted generation: the prompt chunk is {chunk}")
        self.engine, self.drafter, self.nodes, self.chunk = engine, drafter or NgramDrafter(), nodes, chunk
        self.stop_ids = set(int(t) for t in stop_ids)
        self.steps = self.drafted = self.accepted = self.evictions = 0
        self._runs = 0

    def run(self, requests: Sequence[Request]) -> None:
        V = self.engine.model.spec.vocab_size
        for r in requests:
            r.policy.check(V)
            if not r.prompt:
                raise ValueError("drafted generation: a prompt is empty; there is nothing to condition on")
            if r.policy.max_tokens <= 0:
                raise ValueError("drafted generation: give every policy a positive max_tokens")
            if not self.engine.cache.can_hold(len(r.prompt) + r.policy.max_tokens, min(self.chunk, len(r.prompt))):
                raise ContextExhausted(f"drafted generation: a {len(r.prompt)}-token prompt and {r.policy.max_tokens} tokens "
                                       "need more pages than the pool holds")
        waiting, live = list(requests), []
        try:
            while waiting or live:
                self._admit(waiting, live)
                if live:
                    self._turn(waiting, live)
            if hasattr(self.engine, "check_kernels"):
                self.engine.check_kernels()
        finally:
            for one in live:
                self.engine.finish(one.rid)

    # ------------------------------------------------------------------------ pieces
    def _admit(self, waiting: List[Request], live: List[_Live]) -> None:
        """Requests while there is room, each through its prompt to its next token."""
        while waiting:
            req = waiting[0]
            text = req.prompt + req.output
            self._runs += 1
            rid = ("drafted", id(self), self._runs)
            try:
                self.engine.admit(rid, len(text) + 1, adapter=req.adapter)
            except (PagesExhausted, SlotsExhausted):
                if not live:
                    raise
                return
            try:
                for o in range(0, len(text), self.chunk):
                    part = text[o:o + self.chunk]
                    last = o + len(part) == len(text)
                    logits = self.engine.step([StepEntry(rid, part, [len(part) - 1] if last else [])])
            except BaseException as e:
                self.engine.finish(rid)
                if isinstance(e, PagesExhausted) and live:
                    return
                raise
            waiting.pop(0)
            one = _Live(req, rid)
            live.append(one)
            self._take(one, [int(t) for t in sample_rows(logits, [req])], live)

    def _take(self, one: _Live, tokens: Sequence[int], live: List[_Live]) -> None:
        """A request's next tokens: its output, up to a stop id or its budget."""
        req = one.request
        for t in tokens:
            if t in self.stop_ids:
                req.finished, req.finish_reason = True, "stop"
            else:
                req.output.append(t)
                if len(req.output) >= req.policy.max_tokens:
                    req.finished, req.finish_reason = True, "length"
            if req.finished:
                del req.logprobs[len(req.output):]           # parallel to the output
                self.engine.finish(one.rid)
                live.remove(one)
                return

    def _trees(self, live: List[_Live], longest: int) -> List[DraftEntry]:
        entries = []
        for one in live:
            req = one.request
            # the last token of the budget is the one behind a path
            room = min(longest, req.policy.max_tokens - len(req.output)) - 1
            tokens, parents, depth = [req.output[-1]], [-1], [0]
            if room > 0 and self.nodes > 1:
                place = {0: 0}                               # a drafter's places among those that are kept
                V = self.engine.model.spec.vocab_size
                for i, (t, p) in enumerate(zip(*self.drafter.propose(req.prompt + req.output, self.nodes - 1)), 1):
                    if len(tokens) < self.nodes and p in place and p < i and depth[place[p]] < room and 0 <= int(t) < V:
                        place[i] = len(tokens)
                        tokens.append(int(t))
                        parents.append(place[p])
                        depth.append(depth[place[p]] + 1)
            entries.append(DraftEntry(one.rid, tokens, parents))
        return entries

    def _turn(self, waiting: List[Request], live: List[_Live]) -> None:
        longest = self.engine._longest_path()
        entries, reports, stuck = self._trees(live, longest), [], {}
        while True:
            reqs = [one.request for one in live]
            try:
                if any(len(e.tokens) > 1 for e in entries):
                    got = self.engine.draft_step(entries, lambda logits, ctx: self._choose(logits, ctx, reqs, entries, reports, stuck))
                else:                                         # a decode step as any other, from a graph where there is one
                    got, logits = None, self.engine.step([StepEntry(e.request_id, e.tokens, [0]) for e in entries])
                break
            except PagesExhausted:
                if any(len(e.tokens) > 1 for e in entries):
                    entries = [DraftEntry(e.request_id, e.tokens[:1], e.parents[:1]) for e in entries]
                    continue
                if len(live) <= 1:
                    raise
                gone = live.pop()
                self.engine.finish(gone.rid)
                gone.request.evictions += 1
                self.evictions += 1
                waiting.insert(0, gone.request)
                entries.pop()
        self.steps += 1
        if got is None:
            for one, t in zip(list(live), sample_rows(logits, reqs)):
                self._take(one, [int(t)], live)
            return
        at = 0
        for one, e, a in zip(list(live), entries, got):
            req = one.request
            path = a.path
            # a grammar's failure counts where the request comes first; what was chosen from there on had no mask
            failed = next((k for k, i in enumerate(path) if at + i in stuck), None)
            if failed is not None:
                path = path[:failed + 1]
            along = [e.tokens[i] for i in path[1:]]
            chosen = path if failed is None else path[:-1]   # where a token was chosen that the request gets
            self.drafted += len(e.tokens) - 1
            self.accepted += len(along)
            req.sampler.index += len(chosen)
            req.logprobs.extend(r for r in (reports[at + i] for i in chosen) if r is not None)
            if failed is not None:
                req.output.extend(along)
                raise stuck[at + path[-1]]
            at += len(e.tokens)
            self._take(one, along + [a.following], live)

    def _choose(self, logits, ctx, reqs: Sequence[Request], entries: Sequence[DraftEntry], reports: list, stuck: dict):
        """A token behind every token of every tree, as its request's policy chooses it there. `stuck` gets the rows where a
        grammar failed behind drafts, and how: that matters if the request comes there."""
        V = logits.shape[1]
        policies, draws, masks, owner = [], [], [], []
        for q, (req, e) in enumerate(zip(reqs, entries)):
            if req.sampler is None:
                req.sampler = DrawStream(req.policy.seed)
            first = len(masks)
            said: List[List[int]] = []                       # drafted tokens up to each one
            reached: List[bool] = []                         # not behind a token that is forbidden or ends the request,
            for i, p in enumerate(e.parents):                # where a grammar cannot be asked: nobody comes there
                t = e.tokens[i]
                said.append(said[p] + [t] if i else [])
                over = masks[first + p] if i else None
                reached.append(i == 0 or reached[p] and first + p not in stuck and t not in self.stop_ids and
                               (over is None or bool(int(over[t // 32]) >> t % 32 & 1)))
                policies.append(req.policy)
                draws.append(req.sampler.ahead(len(said[i])))
                masks.append(None)
                owner.append(q)
                if reached[i] and req.policy.allowed is not None:
                    try:
                        masks[-1] = req.policy.allowed_words(req.output + said[i], V)
                    except Exception as error:
                        if i == 0:
                            raise
                        stuck[first + i] = error
        constrain(logits, [r.policy for r in reqs], [r.prompt + r.output[:-1] if r.policy.penalises else () for r in reqs],
                  masks, owner, (ctx.q_start, ctx.token_ids, ctx.seen))
        return sample_batch(logits, policies, draws, reports=reports, edited=True)
