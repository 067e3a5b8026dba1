"""Beam search and adapters through the engine on the GPU: against plain searches over whole forwards
(true float32), and adapted requests in bfloat16 decode graphs against merged weights."""
import numpy as np
import pytest
import torch

import plain_qwen3 as plain
import tiny
from emulated_beams import plain_beam_search, random_adapter, with_adapter

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def matrices_of(w):
    return {n: tuple(m.shape) for n, m in w.items() if m.ndim == 2 and ".layers." in n}


def adapters_for(w, rank=12):
    from tgo_b200.weights.adapters import Adapter
    shapes = matrices_of(w)
    names = sorted(shapes)
    return {"all": Adapter(random_adapter(shapes, names, rank, seed=1), 2.0),
            "attention": Adapter(random_adapter(shapes, [n for n in names if "self_attn" in n], 4, seed=2), 1.5),
            "second layer": Adapter(random_adapter(shapes, [n for n in names if ".layers.1." in n and "up_proj" not in n], 7,
                                                   seed=3), 1.0)}


def same(got, want, atol):
    assert [h.tokens for h in got] == [t for t, _, _ in want]
    assert [h.stopped for h in got] == [s for _, _, s in want]
    assert np.allclose([h.score for h in got], [s for _, s, _ in want], rtol=0, atol=atol)


@pytest.mark.parametrize("name,beams,length_penalty", [("A", 4, 1.0), ("B", 3, 0.0), ("B", 6, 1.5), ("C", 2, 1.0)])
def test_adapted_searches_match_plain(tmp_path, name, beams, length_penalty):
    import tgo_b200
    cfg, run = tiny.TINIES[name]
    d = tiny.make_model_dir(tmp_path / name, cfg, run["seed"], 0.2)
    pcfg, w = plain.load_model_dir(d)
    model, adapters = tgo_b200.open(d, dtype="float32", device=DEV), adapters_for(w)
    model.load_adapters(adapters)
    prompts = list(tiny.random_requests(cfg["vocab_size"], [5, 16, 31, 8], seed=3).values())
    which = ["all", None, "attention", "second layer"]
    stop = list(range(0, cfg["vocab_size"], 9))
    got = model.beam_search(prompts, beams=beams, max_tokens=20, adapters=which, stop_ids=stop, chunk=7,
                            length_penalty=length_penalty, page_size=run["page_size"])
    for g, p, a in zip(got, prompts, which):
        ww = w if a is None else with_adapter(w, adapters[a].matrices, adapters[a].scale)
        same(g, plain_beam_search(lambda t: plain.forward(pcfg, ww, t)[-1], p, beams, 20, set(stop), length_penalty), 2e-3)


@pytest.mark.parametrize("name", ["G1", "G2"])
def test_searches_reorder_states(tmp_path, name):
    """Retention layers: each beam's float32 state follows it."""
    import gafonex_tiny
    import plain_gafonex
    import tgo_b200
    cfg, page = gafonex_tiny.CONFIGS[name]
    W = gafonex_tiny.make_weights(cfg, 3)
    d = str(tmp_path / "m")
    gafonex_tiny.write_model_dir(d, cfg, W)
    model = tgo_b200.open(d, dtype="float32", device=DEV)
    vocab = model.spec.vocab_size
    prompts = [np.random.default_rng(i).integers(0, vocab, n).tolist() for i, n in enumerate([4, 19])]
    got = model.beam_search(prompts, beams=4, max_tokens=12, page_size=page)
    for g, p in zip(got, prompts):
        same(g, plain_beam_search(lambda t: plain_gafonex.forward(cfg, W, t)[-1], p, 4, 12), 2e-3)


def test_one_beam_is_greedy_and_pages_come_back(tmp_path):
    import tgo_b200
    from tgo_b200.engine.beams import BeamSearch
    cfg, run = tiny.TINIES["B"]
    d = tiny.make_model_dir(tmp_path / "b", cfg, run["seed"], 0.2)
    pcfg, w = plain.load_model_dir(d)
    model = tgo_b200.open(d, dtype="float32", device=DEV)
    prompts = list(tiny.random_requests(cfg["vocab_size"], [12, 40], seed=5).values())
    eng = model.new_engine(page_size=8, max_tokens=600, num_slots=6)
    got = BeamSearch(eng, 1, 14).run(prompts)
    assert [g[0].tokens for g in got] == [plain.greedy_generate(pcfg, w, p, 14) for p in prompts]
    first = BeamSearch(eng, 3, 14).run(prompts)
    for g in range(len(eng.cache.pools)):                       # what nobody holds cannot be read
        eng.storage.poison_pages(g, [p for p in range(1, eng.cache.pools[g].num_pages + 1)])
    again = BeamSearch(eng, 3, 14).run(prompts)
    assert [[h.tokens for h in q] for q in first] == [[h.tokens for h in q] for q in again]
    assert all(p.free_count == p.num_pages for p in eng.cache.pools) and eng.cache.slots.free_count == 6


@pytest.mark.parametrize("name", ["B", "C", "D"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_adapted_requests_match_merged_weights(tmp_path, name, dtype):
    """Prompts and then decode steps (captured as graphs) of adapted and plain requests in one batch."""
    import tgo_b200
    from tgo_b200.engine.step import StepEntry
    cfg, run = {**tiny.TINIES, "D": (tiny.TINY_D, tiny.TINY_D_RUN)}[name]
    d = tiny.make_model_dir(tmp_path / name, cfg, run["seed"], run["sigma"])
    pcfg, w = plain.load_model_dir(d)
    model, adapters = tgo_b200.open(d, dtype=dtype, device=DEV), adapters_for(w, rank=16)
    model.load_adapters(adapters)
    reqs = tiny.random_requests(cfg["vocab_size"], [20, 47, 33, 70, 12], seed=6)
    which = dict(zip(reqs, ["all", None, "attention", "second layer", "all"]))
    eng = model.new_engine(page_size=run["page_size"], max_tokens=600, num_slots=5)
    for r in reqs:
        eng.admit(r, adapter=which[r])
    got = {}
    heads = {r: len(t) - 9 for r, t in reqs.items()}
    logits = eng.step([StepEntry(r, t[:heads[r]], list(range(heads[r]))) for r, t in reqs.items()]).cpu().numpy()
    at = 0
    for r in reqs:
        for p in range(heads[r]):
            got[(r, p)] = logits[at]
            at += 1
    for j in range(9):
        rows = eng.step([StepEntry(r, [t[heads[r] + j]], [0]) for r, t in reqs.items()]).cpu().numpy()
        for i, r in enumerate(reqs):
            got[(r, heads[r] + j)] = rows[i]
    assert any(k[2] for k in eng._graphs)
    merged = {r: w if a is None else with_adapter(w, adapters[a].matrices, adapters[a].scale) for r, a in which.items()}
    want = {r: plain.forward(pcfg, merged[r], t) for r, t in reqs.items()}
    rounded = {r: plain.forward_rounded(pcfg, merged[r], t) for r, t in reqs.items()} if dtype == "bfloat16" else None
    worst, where, allowed = tiny.compare(got, want, cfg, dtype, f"adapters/{name}/{dtype}", rounded)
    assert worst <= allowed, (worst, where, allowed)


def test_plain_requests_keep_their_bits_when_adapters_are_loaded(tmp_path):
    import tgo_b200
    from tgo_b200.sampling.policy import Policy
    cfg, run = tiny.TINIES["C"]
    d = tiny.make_model_dir(tmp_path / "c", cfg, run["seed"], 0.2)
    _, w = plain.load_model_dir(d)
    prompts = list(tiny.random_requests(cfg["vocab_size"], [300, 300, 21], seed=8).values())

    def logits_of(model):
        from tgo_b200.engine.step import StepEntry
        eng = model.new_engine(page_size=16, max_tokens=1000, num_slots=3)
        out = []
        for i, p in enumerate(prompts):
            eng.admit(i)
            out.append(eng.step([StepEntry(i, p, [len(p) - 1])]).clone())
        for t in (3, 4):
            out.append(eng.step([StepEntry(i, [t], [0]) for i in range(3)]).clone())
        return torch.cat(out)
    model = tgo_b200.open(d, dtype="bfloat16", device=DEV)
    before, text = logits_of(model), model.generate(prompts, Policy(max_tokens=5))
    model.load_adapters(adapters_for(w))
    assert torch.equal(logits_of(model), before)
    assert model.generate(prompts, Policy(max_tokens=5)) == text


@pytest.mark.parametrize("name,adapter", [("B", None), ("C", "all")])
def test_searches_in_bfloat16_read_their_own_pages(tmp_path, name, adapter):
    """What every beam of a bfloat16 search sees behind each prefix of its hypothesis, through pages that the beams share,
    copy and give up, is what a whole forward over that text gives."""
    import tgo_b200
    from tgo_b200.engine.beams import BeamSearch
    cfg, run = tiny.TINIES[name]
    d = tiny.make_model_dir(tmp_path / name, cfg, run["seed"], run["sigma"])
    pcfg, w = plain.load_model_dir(d)
    model = tgo_b200.open(d, dtype="bfloat16", device=DEV)
    if adapter:
        adapters = adapters_for(w, rank=16)
        model.load_adapters(adapters)
        w = with_adapter(w, adapters[adapter].matrices, adapters[adapter].scale)
    prompts = list(tiny.random_requests(cfg["vocab_size"], [13, 40], seed=9).values())
    seen = {}

    class Watched(BeamSearch):
        def _advance(self, searches, logits):
            rows = logits.cpu().numpy()
            for i, s in enumerate(searches):
                for k, (t, score) in enumerate(zip(s.tokens, s.scores)):
                    if score > -np.inf:
                        seen[(s.rids[0][2], tuple(t))] = rows[i * self.beams + k]
            return super()._advance(searches, logits)
    eng = model.new_engine(page_size=4, max_tokens=600, num_slots=8)
    found = Watched(eng, 4, 22).run(prompts, [adapter] * 2)
    assert all(len(q) == 4 and all(len(h.tokens) == 22 for h in q) for q in found)
    got, want, rounded = {}, {}, {}
    for q, p in enumerate(prompts):
        for i, h in enumerate(found[q]):
            text = p + h.tokens
            want[(q, i)], rounded[(q, i)] = plain.forward(pcfg, w, text), plain.forward_rounded(pcfg, w, text)
            for n in range(22):
                got[((q, i), len(p) - 1 + n)] = seen[(q, tuple(h.tokens[:n]))]
    worst, where, allowed = tiny.compare(got, want, cfg, "bfloat16", f"bfloat16 search/{name}", rounded)
    assert worst <= allowed, (worst, where, allowed)
