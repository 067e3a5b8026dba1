"""Pages of steps of drafted tokens: what the request does not keep goes back to the pool; no GPU."""
import random

import pytest
import torch

from plain_cache import CacheManager
from test_beam_search import cpu_model, tiny_model
from test_cache import make_manager
from test_drafting import emulated, prompts_of                                # noqa: F401  (a fixture)
from tgo_b200.cache.pages import PagesExhausted, SlotsExhausted
from tgo_b200.engine.drafts import DraftedGeneration
from tgo_b200.engine.scheduler import Request
from tgo_b200.engine.step import DraftEntry, StepEntry
from tgo_b200.sampling.policy import Policy


class Wrong:
    """Drafts that are never right, all of them behind the last token."""

    def __init__(self, texts, vocab):
        self.texts, self.vocab = texts, vocab

    def propose(self, tokens, nodes):
        text = next(t for t in self.texts if t[:len(tokens)] == list(tokens))
        nxt = text[len(tokens)] if len(tokens) < len(text) else 0
        return [(nxt + 1 + i % (self.vocab - 1)) % self.vocab for i in range(nodes)], [0] * nodes


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("pages", [20, 22, 24, 26, 30, 34])
def test_wrong_drafts_need_no_more_pages_than_none(emulated, tmp_path, name, pages):        # noqa: F811
    """Steps, evictions and admissions of a pool that just holds everybody: those of generation without drafts."""
    d, cfg, run = tiny_model(tmp_path, name)
    V = cfg["vocab_size"]
    prompts = prompts_of(V, [9, 6, 7], seed=4)
    model = cpu_model(d, cfg)
    texts = [p + t for p, t in zip(prompts, model.generate(prompts, Policy(max_tokens=18), page_size=4))]
    seen = []
    for nodes in (1, 64):
        runner = DraftedGeneration(model.new_engine(page_size=4, num_pages=pages, num_slots=3), Wrong(texts, V), nodes=nodes)
        reqs = [Request(p, Policy(max_tokens=18)) for p in prompts]
        runner.run(reqs)
        assert [p + r.output for p, r in zip(prompts, reqs)] == texts
        seen.append((runner.evictions, runner._runs, runner.steps))
        assert all(p.free_count == p.num_pages for p in runner.engine.cache.pools)
    assert seen[0] == seen[1] and seen[0][0] == 0, seen


def test_a_step_keeps_the_pages_of_what_it_keeps(emulated, tmp_path):        # noqa: F811
    d, cfg, run = tiny_model(tmp_path, "B")                  # full layers, and windows of 24
    eng = cpu_model(d, cfg).new_engine(page_size=4, num_pages=24, num_slots=3)
    eng.admit("a")
    eng.admit("b", reserve_tokens=30)
    for r in "ab":
        eng.step([StepEntry(r, [1, 2, 3, 4, 5, 6], [])])
    held = lambda: [[p.num_pages - p.free_count for p in eng.cache.pools], [len(eng.cache.requests[r].held(g)) for r in "ab"    # noqa: E731
                                                                            for g in range(len(eng.cache.pools))]]
    before = held()
    bad = lambda logits, ctx: torch.zeros(logits.shape[0], dtype=torch.int32)       # noqa: E731
    tree = [DraftEntry(r, [7] + [8] * 12, [-1] + [0] * 12) for r in "ab"]
    got = eng.draft_step(tree, bad)
    assert [len(a.path) for a in got] == [1, 1] and eng.length("a") == 7
    assert held() == before
    eng.cache.check_invariants()

    def fails(logits, ctx):
        raise RuntimeError("no choice")
    with pytest.raises(RuntimeError):
        eng.draft_step(tree, fails)
    assert held() == before and eng.length("a") == 7
    with pytest.raises(PagesExhausted):                        # the first request's tree fits, both do not
        eng.draft_step([DraftEntry(r, [7] + [8] * 52, [-1] + [0] * 52) for r in "ab"], bad)      # 15 pages each of 24
    assert held() == before
    eng.cache.check_invariants()
    # the places are there again, for drafts that are right too
    got = eng.draft_step([DraftEntry("a", list(range(7, 20)), list(range(-1, 12)))],
                         lambda logits, ctx: torch.arange(8, 21, dtype=torch.int32))
    assert len(got[0].path) == 13 and eng.length("a") == 20
    assert [len(eng.cache.requests["a"].held(g)) for g in range(len(eng.cache.pools))] == [5, 5]
    for r in "ab":
        eng.finish(r)
    assert all(p.free_count == p.num_pages for p in eng.cache.pools)


class Trimmed(CacheManager):
    """The plain books with a tail that goes back: what neither the length nor, where every key is kept, the reservation needs."""

    def admit(self, request_id, reserve_tokens=0):
        req = super().admit(request_id, reserve_tokens)
        req.reserved = reserve_tokens
        return req

    def trim(self, request_ids):
        for rid in request_ids:
            req = self.requests[rid]
            for g, grp in enumerate(self.groups):
                keep = self.pages_for(max(req.length, req.reserved if grp.kind == "full" else 0))
                gone = [p for p in req.tables[g][keep:] if p]
                del req.tables[g][keep:]
                if gone:
                    self.pools[g].give(gone)


@pytest.mark.parametrize("keep", [0, 6])
@pytest.mark.parametrize("seed", range(4))
def test_native_books_follow_the_plain_ones_when_tails_go_back(seed, keep):
    rng = random.Random(seed)
    plain = Trimmed(make_manager("plain", keep_first=keep).groups, 4, [30, 30], 4)
    native = make_manager("native", pages=(30, 30), page=4, slots=4, window=10, keep_first=keep)
    live, n = {}, 0

    def both(call, *args):
        out = []
        for cm in (plain, native):
            try:
                getattr(cm, call)(*args)
                out.append("ok")
            except (PagesExhausted, SlotsExhausted) as e:
                out.append(type(e).__name__)
        assert out[0] == out[1], (call, args, out)
        return out[0] == "ok"

    for turn in range(500):
        action = rng.random()
        if action < 0.2:
            n += 1
            if both("admit", n, rng.choice([0, 5, 17])):
                live[n] = 0
        elif action < 0.7 and live:
            for r in rng.sample(list(live), rng.randint(1, len(live))):
                e = rng.choice([1, 2, 7, 20])
                if both("grow", r, live[r] + e):
                    live[r] += rng.randint(0, e)             # what is kept of a tree
                    both("commit", r, live[r])
        elif action < 0.9 and live:
            both("trim", rng.sample(list(live), rng.randint(1, len(live))))
        elif live:
            r = rng.choice(list(live))
            both("finish", r)
            del live[r]
        plain.check_invariants()
        native.check_invariants()
        for r in live:
            a, b = plain.requests[r], native.requests[r]
            assert a.tables == b.tables and a.length == b.length
            for p in range(live[r]):
                native.slot_of(b, 0, p)
            for p in range(max(0, live[r] - 9), live[r]):
                native.slot_of(b, 1, p)
    with pytest.raises(KeyError):
        native.trim(["nobody"])
