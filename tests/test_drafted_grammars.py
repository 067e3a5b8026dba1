"""Grammars that fail on a request's way, with and without drafts, and through a session; no GPU."""
import copy

import numpy as np
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



@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_a_bias_and_a_grammar_that_leave_nothing(emulated, tmp_path, temperature):        # noqa: F811
    """Allowed ids that a bias of -inf takes out do not come; when that is all of them, no token may."""
    d, cfg, run = tiny_model(tmp_path, "A")
    V = cfg["vocab_size"]
    model = cpu_model(d, cfg)
    out = -float("inf")
    pol = Policy(max_tokens=6, temperature=temperature, logit_bias={3: out, 4: out, 7: 2.0},
                 allowed=lambda done: [3, 4, 9, V - 1] if len(done) < 4 else [4, 3])
    for call in (lambda: model.generate([[1, 2]], pol, page_size=8), lambda: model.generate_drafted([[1, 2]], pol, page_size=8),
                 lambda: list(model.new_session(64, page_size=8).complete([1, 2], pol))):
        with pytest.raises(ValueError, match="no token is allowed"):
            call()
    words = pol.allowed_words([], V)
    assert [i for i in range(V) if words[i // 32] >> i % 32 & 1] == [9, V - 1]
    fine = copy.copy(pol)
    fine.max_tokens = 4
    for got in (model.generate([[1, 2]], fine, page_size=8)[0], list(model.new_session(64, page_size=8).complete([1, 2], fine))):
        assert set(got) <= {9, V - 1} and len(got) == 4


def test_a_session_under_a_grammar(emulated, tmp_path):        # noqa: F811
    """The tokens of `generate`, the grammar asked with what came so far; stop ids and failures end it."""
    d, cfg, run = tiny_model(tmp_path, "A")
    V = cfg["vocab_size"]
    model = cpu_model(d, cfg)
    asked = []

    def odd(done):
        asked.append(list(done))
        return [i for i in range(V) if (i + len(done)) % 2] if len(done) < 8 else [5]

    for temperature in (0.0, 0.9):
        pol = Policy(max_tokens=12, temperature=temperature, seed=3, allowed=odd, repetition_penalty=1.2)
        want = model.generate([[1, 2, 3]], pol, page_size=8)[0]
        asked.clear()
        got = list(model.new_session(64, page_size=8).complete([1, 2, 3], pol))
        assert got == want and asked == [want[:n] for n in range(12)]
        assert all((t + i) % 2 for i, t in enumerate(got[:8])) and got[8:] == [5] * 4
        session = model.new_session(64, page_size=8)
        session.stop_ids = {5}
        assert list(session.complete([1, 2, 3], pol)) == want[:next(i for i, t in enumerate(want) if t == 5)]


@pytest.mark.parametrize("got", [[True, False, True], np.array([True, False]), (np.bool_(True),)])
def test_truth_values_are_no_ids(got):
    with pytest.raises(ValueError, match="truth values"):
        Policy(allowed=lambda done: got).allowed_words([], 70)
    assert Policy(allowed=lambda done: range(2)).allowed_words([], 70).tolist() == [3, 0, 0]
    assert Policy(allowed=lambda done: np.array([1, 64])).allowed_words([], 70).tolist() == [2, 0, 1]
