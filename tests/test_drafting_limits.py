"""Models that drafted steps do not take are refused by name before anything runs; no GPU."""
import pytest

import tiny
from emulated_drafts import Oracle
from test_beam_search import cpu_model
from test_drafting import emulated                                # noqa: F401  (a fixture)
from tgo_b200.engine.drafts import DraftedGeneration
from tgo_b200.engine.step import DraftEntry
from tgo_b200.sampling.policy import Policy


@pytest.mark.parametrize("dim,taken", [(64, True), (256, True), (258, False), (320, False), (512, False)])
def test_heads_wider_than_the_attention_of_trees_takes(emulated, tmp_path, dim, taken):        # noqa: F811
    cfg = dict(tiny.TINIES["A"][0], head_dim=dim)
    d = tiny.make_model_dir(tmp_path / "m", cfg, 1, 0.05)
    model = cpu_model(d, cfg)
    eng = model.new_engine(page_size=8, max_tokens=100, num_slots=1)
    if taken:
        assert eng.takes_drafts() is None
        return
    assert str(dim) in eng.takes_drafts()
    with pytest.raises(ValueError, match=f"heads of {dim}"):
        DraftedGeneration(eng)
    with pytest.raises(ValueError, match=f"heads of {dim}"):
        model.generate_drafted([[1, 2]], Policy(max_tokens=3))
    eng.admit("a")
    with pytest.raises(ValueError, match=f"heads of {dim}"):
        eng.draft_step([DraftEntry("a", [1], [-1])], None)
    assert eng.cache.requests["a"].held(0) == []
    assert len(model.generate([[1, 2]], Policy(max_tokens=3))[0]) == 3


@pytest.mark.parametrize("nodes,wrong,steps", [(1, 0, 19), (2, 0, 10), (2, 1, 19), (5, 0, 4), (4, 1, 10), (64, 0, 1)])
def test_steps_that_right_drafts_take(emulated, tmp_path, nodes, wrong, steps):        # noqa: F811
    """20 tokens, the first of them from the prompt: a step gives as many as its path has. Beside a right draft `wrong`
    others come first, with one behind the last of them."""
    d = tiny.make_model_dir(tmp_path / "m", tiny.TINIES["A"][0], 1, 0.2)
    model = cpu_model(d, tiny.TINIES["A"][0])
    prompt = [5, 9, 11, 3]
    text = prompt + model.generate([prompt], Policy(max_tokens=20), page_size=4)[0]
    got = model.generate_drafted([prompt], Policy(max_tokens=20), nodes=nodes, page_size=4,
                                 drafter=Oracle([text], 30, wrong, tiny.TINIES["A"][0]["vocab_size"]))
    assert prompt + got[0] == text and model.last_drafts.steps == steps


class NowAndThen:
    """Drafts every so often."""

    def __init__(self, every):
        self.every, self.asked = every, 0

    def propose(self, tokens, nodes):
        self.asked += 1
        return ([1, 2], [0, 1]) if self.asked % self.every == 0 else ([], [])


@pytest.mark.parametrize("drafter", ["never", "now and then"])
def test_turns_without_drafts_are_decode_steps(emulated, tmp_path, monkeypatch, drafter):        # noqa: F811
    """They go through `Engine.step`, which has captured graphs, with the same draws, reports and ends."""
    from tgo_b200.engine.step import Engine
    cfg = tiny.TINIES["A"][0]
    model = cpu_model(tiny.make_model_dir(tmp_path / "m", cfg, 1, 0.05), cfg)
    prompts = [[5, 9, 11, 3], [7, 8]]
    policies = [Policy(max_tokens=15, temperature=0.9, seed=2, logprobs=True, repetition_penalty=1.3),
                Policy(max_tokens=10, allowed=lambda out: range(3, cfg["vocab_size"]))]
    want = model.generate(prompts, policies, page_size=4, stop_ids=[4])
    reports = [[p.id for p in r.logprobs] for r in model.last_requests]
    kinds = []
    step, draft_step = Engine.step, Engine.draft_step
    monkeypatch.setattr(Engine, "step", lambda self, entries: (kinds.append("step"), step(self, entries))[1])
    monkeypatch.setattr(Engine, "draft_step", lambda self, entries, choose: (kinds.append([len(e.tokens) for e in entries]), draft_step(self, entries, choose))[1])
    got = model.generate_drafted(prompts, policies, page_size=4, stop_ids=[4], drafter=NowAndThen(3 if drafter == "now and then" else 10 ** 9))
    assert got == want and [[p.id for p in r.logprobs] for r in model.last_requests] == reports
    trees = [k for k in kinds if k != "step"]
    assert all(max(k) > 1 for k in trees) and bool(trees) == (drafter == "now and then")
    assert model.last_drafts.steps == len(kinds) - 2                            # two prompts
