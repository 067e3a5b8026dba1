"""Grammars that fail on a request's way, with and without drafts, and through a session; no GPU."""
import copy

import pytest

from emulated_drafts import Oracle
from test_beam_search import cpu_model, tiny_model
from test_drafting import emulated, prompts_of                                # noqa: F401  (a fixture)
from tgo_b200.engine.drafts import DraftedGeneration
from tgo_b200.engine.scheduler import Request, Runner
from tgo_b200.sampling.policy import Policy
from tgo_b200.sampling.sampler import sample_rows


@pytest.mark.parametrize("right", [1, 2, 3, 4, 5, 6, 8, 11])
@pytest.mark.parametrize("at", [1, 5, 10])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_a_grammar_that_fails_on_the_way(emulated, tmp_path, right, at, temperature):        # noqa: F811
    """The error comes where it comes without drafts, however deep the drafts confirmed behind that place go and whatever is
    allowed there; the request holds what it held then."""
    d, cfg, run = tiny_model(tmp_path, "B")
    V = cfg["vocab_size"]
    prompts = prompts_of(V, [6, 7], seed=8)
    model = cpu_model(d, cfg)
    free = Policy(max_tokens=12, temperature=temperature, seed=5, logprobs=True)
    text = model.generate(prompts[:1], free, page_size=8)[0]
    fails = copy.copy(free)
    fails.allowed = lambda out: [] if len(out) == at else None

    plain = Request(prompts[0], fails)
    runner = Runner(model.new_scheduler(1, reserve=12, pool_tokens=160, page_size=8), sample_rows)
    runner.submit(plain)
    with pytest.raises(ValueError, match="no token"):
        runner.run()
    assert plain.output == text[:at]

    mine, other = Request(prompts[0], fails), Request(prompts[1], Policy(max_tokens=12))
    drafts = DraftedGeneration(model.new_engine(page_size=8, num_pages=40, num_slots=2), Oracle([prompts[0] + text], right, 1, V), nodes=40)
    with pytest.raises(ValueError, match="no token"):
        drafts.run([mine, other])
    assert mine.output == plain.output and mine.sampler.index == at             # a draw a token, to run on from
    assert [p.id for p in mine.logprobs] == [p.id for p in plain.logprobs] == text[:at]
    assert not drafts.engine.cache.requests and drafts.accepted <= drafts.drafted

