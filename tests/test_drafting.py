"""Drafted generation without a GPU: the engine's host side with torch stand-ins for the kernels, against
generation without drafts and against plain whole forwards."""
import random

import numpy as np
import pytest
import torch

import emulated_drafts
import plain_qwen3 as plain
import tiny
from emulated_drafts import Noise, Oracle
from test_beam_search import cpu_model, some_adapters, tiny_model
from tgo_b200.cache.pages import PagesExhausted
from tgo_b200.engine.drafts import DraftedGeneration, NgramDrafter
from tgo_b200.engine.scheduler import ContextExhausted, Request
from tgo_b200.engine.step import DraftEntry, StepEntry
from tgo_b200.sampling.policy import DrawStream, Policy


@pytest.fixture()
def emulated(monkeypatch):
    emulated_drafts.install(monkeypatch)


def prompts_of(V, lengths, seed=7):
    return list(tiny.random_requests(V, lengths, seed=seed).values())


# ------------------------------------------------------------------------------- steps


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_a_tree_gives_what_its_paths_give(emulated, tmp_path, name):
    """Logits behind every token of a tree: those of the request's text and the token's path."""
    d, cfg, run = tiny_model(tmp_path, name)
    pcfg, w = plain.load_model_dir(d)
    V = cfg["vocab_size"]
    eng = cpu_model(d, cfg).new_engine(page_size=run["page_size"], max_tokens=400, num_slots=3)
    prompts, rng = prompts_of(V, [5, 30, 16]), random.Random(1)
    for i, p in enumerate(prompts):
        eng.admit(i)
        eng.step([StepEntry(i, p, [])])
    texts = [list(p) for p in prompts]
    for turn in range(4):
        entries, kept = [], []
        for i in range(3):
            n = rng.choice([1, 4, 9])
            entries.append(DraftEntry(i, [rng.randrange(V) for _ in range(n)], [-1] + [rng.randrange(max(0, j - 3), j) for j in range(1, n)]))
        seen = {}

        def choose(logits, ctx):
            seen["logits"] = logits.clone()
            chosen = logits.argmax(1).to(torch.int32)
            at = 0
            for e in entries:                                # now and then the drafts are right
                for j in range(1, len(e.tokens)):
                    if rng.random() < 0.6:
                        chosen[at + e.parents[j]] = e.tokens[j]
                at += len(e.tokens)
            seen["chosen"] = chosen
            return chosen
        got = eng.draft_step(entries, choose)
        at = 0
        for i, (e, a) in enumerate(zip(entries, got)):
            paths = []
            for j, p in enumerate(e.parents):
                paths.append((paths[p] if j else []) + [e.tokens[j]])
                want = plain.forward(pcfg, w, texts[i] + paths[j])[-1]
                assert np.allclose(seen["logits"][at + j].numpy(), want, rtol=0, atol=2e-4 * max(1.0, float(np.abs(want).max())))
            assert a.path[0] == 0 and all(e.parents[y] == x for x, y in zip(a.path, a.path[1:]))
            assert a.following == int(seen["chosen"][at + a.path[-1]])
            texts[i] += [e.tokens[j] for j in a.path]
            assert eng.length(i) == len(texts[i])
            at += len(e.tokens)
    # what the cache holds now is the accepted text
    lg = eng.step([StepEntry(i, [3], [0]) for i in range(3)])
    for i in range(3):
        want = plain.forward(pcfg, w, texts[i] + [3])[-1]
        assert np.allclose(lg[i].numpy(), want, rtol=0, atol=2e-4 * max(1.0, float(np.abs(want).max())))
    eng.cache.check_invariants()


def test_steps_that_are_refused(emulated, tmp_path):
    d, cfg, run = tiny_model(tmp_path, "B")                  # windows of 24
    V = cfg["vocab_size"]
    eng = cpu_model(d, cfg).new_engine(page_size=4, max_tokens=60, num_slots=2)
    eng.admit("a")
    eng.step([StepEntry("a", [1, 2, 3], [])])
    none = lambda logits, ctx: torch.zeros(logits.shape[0], dtype=torch.int32)       # noqa: E731
    for tokens, parents, match in [([1, 2], [-1], "parent per token"), ([1, 2], [0, 0], "continues"), ([1, 2], [-1, 1], "continues"),
                                   ([1, 2], [-1, -1], "continues"), ([1, V], [-1, 0], "vocabulary"), ([], [], "no tokens"),
                                   ([1] * 65, [-1] + [0] * 64, "at most 64"), ([1] * 25, list(range(-1, 24)), "longer than 24")]:
        with pytest.raises(ValueError, match=match):
            eng.draft_step([DraftEntry("a", tokens, parents)], none)
    with pytest.raises(KeyError):
        eng.draft_step([DraftEntry("b", [1], [-1])], none)
    with pytest.raises(ValueError, match="twice"):
        eng.draft_step([DraftEntry("a", [1], [-1])] * 2, none)
    with pytest.raises(ValueError, match="empty"):
        eng.draft_step([], none)
    with pytest.raises(PagesExhausted):
        eng.draft_step([DraftEntry("a", [1] * 60, [-1] + [0] * 59)], none)

    def fails(logits, ctx):
        raise RuntimeError("no choice")
    with pytest.raises(RuntimeError, match="no choice"):
        eng.draft_step([DraftEntry("a", [1, 2], [-1, 0])], fails)
    assert eng.length("a") == 3
    assert len(eng.draft_step([DraftEntry("a", [1] * 24, list(range(-1, 23)))], none)) == 1


def test_models_with_states_are_refused(emulated, tmp_path):
    import gafonex_tiny
    from test_engine_emulated import cpu_model as make
    cfg, page = gafonex_tiny.CONFIGS["G1"]
    d = str(tmp_path / "g")
    gafonex_tiny.write_model_dir(d, cfg, gafonex_tiny.make_weights(cfg, 3))
    eng = make(d, cfg).new_engine(page_size=page, max_tokens=100, num_slots=2)
    assert eng.takes_drafts() is not None
    with pytest.raises(ValueError, match="drafted"):
        DraftedGeneration(eng)
    with pytest.raises(ValueError, match="drafted"):
        eng.draft_step([DraftEntry("a", [1], [-1])], None)


# -------------------------------------------------------------------------- generation


@pytest.mark.parametrize("name", ["A", "B", "C"])
@pytest.mark.parametrize("drafter", ["ngram", "right", "half right", "noise"])
def test_greedy_text_does_not_depend_on_the_drafts(emulated, tmp_path, name, drafter):
    d, cfg, run = tiny_model(tmp_path, name)
    pcfg, w = plain.load_model_dir(d)
    V = cfg["vocab_size"]
    prompts = [p + p[-3:] + p[:4] for p in prompts_of(V, [6, 15, 11])]
    want = [plain.greedy_generate(pcfg, w, p, 14) for p in prompts]
    texts = [p + t for p, t in zip(prompts, want)]
    made = {"ngram": NgramDrafter(), "right": Oracle(texts, 5, 0), "half right": Oracle(texts, 3, 2, V), "noise": Noise(V)}[drafter]
    model = cpu_model(d, cfg)
    got = model.generate_drafted(prompts, Policy(max_tokens=14), nodes=12, drafter=made, page_size=run["page_size"], chunk=7,
                                 slots=2)
    assert got == want
    stats = model.last_drafts
    if drafter == "right":
        assert stats.accepted == stats.drafted and stats.steps < 14
    if drafter == "half right":
        assert 0 < stats.accepted < stats.drafted
    assert not stats.engine.cache.requests and all(p.free_count == p.num_pages for p in stats.engine.cache.pools)


@pytest.mark.parametrize("nodes", [1, 2, 64])
def test_numbers_of_drafts(emulated, tmp_path, nodes):
    d, cfg, run = tiny_model(tmp_path, "A")
    pcfg, w = plain.load_model_dir(d)
    prompts = prompts_of(cfg["vocab_size"], [6, 9])
    want = [plain.greedy_generate(pcfg, w, p, 20) for p in prompts]
    model = cpu_model(d, cfg)
    oracle = Oracle([p + t for p, t in zip(prompts, want)], 30, 1, cfg["vocab_size"])
    assert model.generate_drafted(prompts, Policy(max_tokens=20), nodes=nodes, drafter=oracle, page_size=4) == want
    assert model.last_drafts.steps == {1: 19, 2: 19, 64: 1}[nodes] or nodes == 2


def test_samples_are_drawn_as_without_drafts(emulated, tmp_path):
    """Temperature, truncation, penalties over windows, biases, grammars and reports: the same draws behind the
    same text give the same tokens."""
    d, cfg, run = tiny_model(tmp_path, "A", 0.05)
    V = cfg["vocab_size"]
    prompts = [p + p for p in prompts_of(V, [4, 7, 12, 5])]
    odd = lambda out: [i for i in range(V) if (i + len(out)) % 2] if len(out) % 3 else None       # noqa: E731
    words = np.full((V + 31) // 32, 0x7F7F7F7F, dtype=np.uint32)
    policies = [Policy(max_tokens=12, temperature=0.9, seed=3, logprobs=True, top_logprobs=3),
                Policy(max_tokens=15, temperature=1.2, top_k=7, seed=4, repetition_penalty=1.4, frequency_penalty=0.3, penalty_window=6),
                Policy(max_tokens=9, temperature=0.7, top_p=0.8, seed=5, logit_bias={3: 4.0, 5: float("-inf")}, presence_penalty=0.5),
                Policy(max_tokens=12, temperature=0.8, seed=6, allowed=odd, repetition_penalty=1.2, logprobs=True)]
    model = cpu_model(d, cfg)
    want = model.generate(prompts, policies, page_size=4)
    asked = model.last_requests
    texts = [p + t for p, t in zip(prompts, want)]
    for drafter in (Oracle(texts, 4, 2, V), Noise(V, 3), NgramDrafter()):
        got = model.generate_drafted(prompts, policies, nodes=14, drafter=drafter, page_size=4, slots=3)
        assert got == want
        for r, s in zip(model.last_requests, asked):
            assert len(r.logprobs) == len(s.logprobs) and [p.id for p in r.logprobs] == [p.id for p in s.logprobs]
            assert np.allclose([p.logprob for p in r.logprobs], [p.logprob for p in s.logprobs], atol=1e-3)
    masked = model.generate_drafted(prompts[:1], Policy(max_tokens=10, allowed=lambda out: words), drafter=Noise(V), page_size=4)[0]
    assert all(t % 8 != 7 for t in masked)


def test_a_grammar_that_ends_on_a_path_nobody_takes(emulated, tmp_path):
    """What a grammar says behind drafts matters where the request comes there, and then as without drafts."""
    d, cfg, run = tiny_model(tmp_path, "B")
    V = cfg["vocab_size"]
    prompts = prompts_of(V, [6, 7], seed=8)
    model = cpu_model(d, cfg)
    free = model.generate(prompts, Policy(max_tokens=12), page_size=8)
    texts = [p + t for p, t in zip(prompts, free)]
    asked = []

    def along(out):                          # nothing comes next but on the texts' way
        asked.append(list(out))
        return list(range(V)) if any(t[:len(out)] == out for t in free) else []

    pol = Policy(max_tokens=12, allowed=along)
    assert model.generate_drafted(prompts, pol, nodes=20, drafter=Oracle(texts, 4, 3, V), page_size=8) == free
    assert model.last_drafts.accepted > 0 and any(all(t[:len(o)] != o for t in free) for o in asked)
    early = Policy(max_tokens=12, allowed=lambda out: list(range(V)) if len(out) < 5 else [])
    with pytest.raises(ValueError, match="no token"):
        model.generate(prompts[:1], early, page_size=8)
    runner = DraftedGeneration(model.new_engine(page_size=8, num_pages=20, num_slots=1), Oracle(texts, 4, 3, V), nodes=20)
    req = Request(prompts[0], early)
    with pytest.raises(ValueError, match="no token"):
        runner.run([req])
    assert req.output == free[0][:5]


def test_a_grammar_is_asked_once_a_node(emulated, tmp_path):
    d, cfg, run = tiny_model(tmp_path, "A")
    V = cfg["vocab_size"]
    prompts = prompts_of(V, [6], seed=3)
    model = cpu_model(d, cfg)
    calls = []
    pol = Policy(max_tokens=20, allowed=lambda out: calls.append(len(out)))
    text = prompts[0] + model.generate(prompts, Policy(max_tokens=20), page_size=8)[0]
    model.generate_drafted(prompts, pol, nodes=12, drafter=Oracle([text], 8, 1, V), page_size=8)
    assert len(calls) <= 1 + model.last_drafts.steps + model.last_drafts.drafted


def test_stop_ids_end_a_path(emulated, tmp_path):
    d, cfg, run = tiny_model(tmp_path, "B")
    V = cfg["vocab_size"]
    prompts = prompts_of(V, [5, 8, 13, 4], seed=2)
    model = cpu_model(d, cfg)
    free = model.generate(prompts, Policy(max_tokens=16), page_size=8)
    stop = sorted({t[k] for t, k in zip(free, (0, 3, 7))})
    want = model.generate(prompts, Policy(max_tokens=16), page_size=8, stop_ids=stop)
    oracle = Oracle([p + t for p, t in zip(prompts, free)], 6, 1, V)
    assert model.generate_drafted(prompts, Policy(max_tokens=16), nodes=20, drafter=oracle, page_size=8, stop_ids=stop) == want
    assert [r.finish_reason for r in model.last_requests] == ["stop" if len(t) < 16 else "length" for t in want]


def test_a_tight_pool(emulated, tmp_path):
    """Drafts are given up, then requests, and run again later."""
    d, cfg, run = tiny_model(tmp_path, "A")
    pcfg, w = plain.load_model_dir(d)
    V = cfg["vocab_size"]
    prompts = prompts_of(V, [9, 6, 7], seed=4)
    want = [plain.greedy_generate(pcfg, w, p, 18) for p in prompts]
    eng = cpu_model(d, cfg).new_engine(page_size=4, num_pages=10, num_slots=3)
    runner = DraftedGeneration(eng, Oracle([p + t for p, t in zip(prompts, want)], 3, 2, V), nodes=10)
    reqs = [Request(p, Policy(max_tokens=18)) for p in prompts]
    runner.run(reqs)
    assert [r.output for r in reqs] == want and runner.evictions > 0
    assert not eng.cache.requests and all(p.free_count == p.num_pages for p in eng.cache.pools)
    with pytest.raises(ContextExhausted):
        runner.run([Request(prompts[0], Policy(max_tokens=60))])


def test_adapted_requests(emulated, tmp_path):
    d, cfg, run = tiny_model(tmp_path, "A")
    _, w = plain.load_model_dir(d)
    model = cpu_model(d, cfg)
    model.load_adapters(some_adapters(w))
    prompts = prompts_of(cfg["vocab_size"], [5, 8, 6], seed=9)
    which = ["all", None, "first layer"]
    want = model.generate(prompts, Policy(max_tokens=10), adapters=which, page_size=4)
    oracle = Oracle([p + t for p, t in zip(prompts, want)], 4, 1, cfg["vocab_size"])
    assert model.generate_drafted(prompts, Policy(max_tokens=10), adapters=which, drafter=oracle, page_size=4) == want
    assert model.last_drafts.accepted > 0


def test_runs_that_are_refused(emulated, tmp_path):
    d, cfg, run = tiny_model(tmp_path, "A")
    model = cpu_model(d, cfg)
    eng = model.new_engine(page_size=4, max_tokens=100, num_slots=2)
    for bad in (dict(nodes=0), dict(nodes=65), dict(chunk=0)):
        with pytest.raises(ValueError):
            DraftedGeneration(eng, **bad)
    for bad in (dict(longest=0), dict(shortest=0), dict(shortest=5, longest=4), dict(depth=0)):
        with pytest.raises(ValueError):
            NgramDrafter(**bad)
    with pytest.raises(ValueError, match="max_tokens"):
        model.generate_drafted([[1, 2]], Policy())
    with pytest.raises(ValueError, match="empty"):
        model.generate_drafted([[]], Policy(max_tokens=3))
    with pytest.raises(ValueError, match="2 policies"):
        model.generate_drafted([[1]], [Policy(max_tokens=3)] * 2)
    assert model.generate_drafted([], Policy(max_tokens=3)) == []


# ----------------------------------------------------------------------- small pieces


def test_ngram_drafts():
    d = NgramDrafter(longest=3, shortest=1, depth=4)
    assert d.propose([1, 2, 3], 8) == ([], [])
    # the longest ending first, the latest place first, shared beginnings once
    tokens = [7, 1, 2, 3, 9, 1, 2, 3, 8, 8, 5, 2, 3, 4, 1, 2, 3]
    drafted, parents = d.propose(tokens, 64)
    assert (drafted[:4], parents[:4]) == ([8, 8, 5, 2], [0, 1, 2, 3])          # behind 1 2 3 at places 5..7
    assert (drafted[4:8], parents[4:8]) == ([9, 1, 2, 3], [0, 5, 6, 7])        # behind 1 2 3 at places 1..3
    assert drafted[8:12] == [4, 1, 2, 3] and parents[8] == 0                   # behind 2 3 at places 11..12
    assert all(0 <= p <= i for i, p in enumerate(parents))
    for n in (0, 1, 5):
        assert d.propose(tokens, n) == (drafted[:n], parents[:n])
    assert d.propose([5], 3) == ([], []) and d.propose([], 3) == ([], [])
    assert NgramDrafter(1, 1, 2).propose([4, 4, 4, 4], 9)[0] == [4, 4]


def test_draws_ahead_are_those_that_come():
    a, b = DrawStream(11), DrawStream(11)
    ahead = [a.ahead(n) for n in range(6)]
    assert [b.next() for _ in range(6)] == ahead and a.index == 0


def test_grammar_masks():
    V = 70
    pol = Policy(allowed=lambda out: {0: [0, 69, 33], 1: None, 2: []}.get(len(out), [V]))
    w = pol.allowed_words([], V)
    assert w.tolist() == [1, 2, 32] and pol.allowed_words([5], V) is None
    with pytest.raises(ValueError, match="no token"):
        pol.allowed_words([1, 2], V)
    with pytest.raises(ValueError, match="outside"):
        pol.allowed_words([1, 2, 3], V)
    full = Policy(allowed=lambda out: np.full(5, -1, dtype=np.int32))
    assert full.allowed_words([], V).tolist() == [2 ** 32 - 1, 2 ** 32 - 1, 63]
    with pytest.raises(ValueError, match="mask of 1 words"):
        Policy(allowed=lambda out: np.ones(1, dtype=np.uint32)).allowed_words([], V)
    with pytest.raises(ValueError, match="called"):
        Policy(allowed=[1, 2]).check(V)
    assert Policy().allowed_words([], V) is None


def test_the_command(emulated, tmp_path, capsys):
    import io
    from tgo_b200 import cli
    d, cfg, run = tiny_model(tmp_path, "A")
    outs = {}
    for drafts in ("0", "8"):
        out, err = io.StringIO(), io.StringIO()
        rc = cli.main(["run", "--prompt", "1 2 3 1 2 3 1 2", "--prompt", "4 5 6", "--max-tokens", "9", "--stop-ids", "none",
                       "--drafts", drafts, "--context", "64", d], out=out, err=err, opener=lambda *a, **k: cpu_model(d, cfg))
        assert rc == 0
        outs[drafts] = out.getvalue()
        assert ("drafts accepted" in err.getvalue()) == (drafts != "0")
    assert outs["0"] == outs["8"]
    err = io.StringIO()
    assert cli.main(["run", "--drafts", "65", d], out=io.StringIO(), err=err, opener=lambda *a, **k: cpu_model(d, cfg)) == 2
