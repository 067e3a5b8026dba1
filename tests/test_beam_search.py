"""Beam search and adapters without a GPU: the books of shared pages, and the engine's host side with
torch stand-ins for the kernels, against plain searches over whole forwards."""
import json
import os
import random

import numpy as np
import pytest
import torch

import emulated_beams
import plain_qwen3 as plain
import tiny
from emulated_beams import plain_beam_search, random_adapter, with_adapter
from tgo_b200.cache.native import NativeCacheManager
from tgo_b200.cache.pages import NULL_PAGE, GroupLayout, PagesExhausted
from tgo_b200.weights.adapters import Adapter, AdapterError, read_adapter


@pytest.fixture()
def emulated(monkeypatch):
    emulated_beams.install(monkeypatch)


# --------------------------------------------------------------------- books of shared pages


def books(pages=(60, 60), page=4, slots=12, window=10, keep_first=0):
    groups = [GroupLayout("full", None, 2, (2, 8), [0]), GroupLayout("window", window, 2, (2, 8), [1], keep_first=keep_first)]
    return NativeCacheManager(groups, page, list(pages), slots)


def write(cm, store, rid, text):
    """Run a step's tokens: each token's row of each group gets the token's name."""
    r = cm.requests[rid]
    cm.grow(rid, r.length + len(text))
    for j, c in enumerate(text):
        for g in range(2):
            store[g][cm.slot_of(r, g, r.length + j)] = c
    cm.commit(rid, r.length + len(text))


def follow(cm, store, rids, parents):
    pages = cm.follow(rids, parents)
    ps = cm.page_size
    for g in range(2):
        old = dict(store[g])
        for i, p in enumerate(parents):
            if p != i and pages[g][i] >= 0:
                for o in range(ps):
                    store[g][int(pages[g][i]) * ps + o] = old.get(int(pages[g][p]) * ps + o)


def read(cm, store, rid, g, live_from=0):
    r = cm.requests[rid]
    return [store[g][cm.slot_of(r, g, p)] for p in range(live_from, r.length)]


@pytest.mark.parametrize("keep", [0, 6])
@pytest.mark.parametrize("seed", range(6))
def test_random_searches_keep_the_books(seed, keep):
    """Groups of beams that write, follow one another and end, in any order: every table finds its own
    history, no page is lost or counted wrongly, and all of them come back."""
    rng = random.Random(seed)
    cm, store = books(keep_first=keep), [{}, {}]
    searches, history, counter = [], {}, 0
    for _ in range(120):
        what = rng.random()
        if what < 0.2 and len(searches) < 3:
            W = rng.choice([2, 3, 4])
            rids = [(counter, w) for w in range(W)]
            counter += 1
            for w, r in enumerate(rids):
                cm.admit(r, rng.choice([0, 7]) if w == 0 else 0)
                history[r] = []
            prompt = [f"p{counter}.{i}" for i in range(rng.randint(1, 13))]
            write(cm, store, rids[0], prompt)
            history[rids[0]] += prompt
            follow(cm, store, rids, [0] * W)
            for r in rids:
                history[r] = list(prompt)
            searches.append(rids)
        elif searches and what < 0.9:
            rids = rng.choice(searches)
            for r in rids:
                counter += 1
                write(cm, store, r, [f"t{counter}"])
                history[r].append(f"t{counter}")
            if rng.random() < 0.8:
                parents = [rng.randrange(len(rids)) for _ in rids]
                follow(cm, store, rids, parents)
                old = {r: list(history[r]) for r in rids}
                for i, p in enumerate(parents):
                    history[rids[i]] = list(old[rids[p]])
        elif searches:
            rids = searches.pop(rng.randrange(len(searches)))
            for r in rids:
                for g, page in cm.finish(r):
                    assert not cm.pools[g].is_held(page)
                    for o in range(4):
                        store[g].pop(page * 4 + o, None)
                del history[r]
        cm.check_invariants()
        for rids in searches:
            for r in rids:
                n = len(history[r])
                assert cm.requests[r].length == n
                assert read(cm, store, r, 0) == history[r]
                first = max(0, n - 10 + 1)
                assert read(cm, store, r, 1, first) == history[r][first:]
                assert [store[1][cm.slot_of(cm.requests[r], 1, p)] for p in range(min(keep, n))] == history[r][:min(keep, n)]
    for rids in searches:
        for r in rids:
            cm.finish(r)
    assert all(p.free_count == p.num_pages for p in cm.pools) and cm.slots.free_count == 12


def test_full_pages_are_shared_and_part_pages_are_not():
    cm, store = books(), [{}, {}]
    for r in "abc":
        cm.admit(r)
    write(cm, store, "a", list("0123456789"))
    follow(cm, store, ["a", "b", "c"], [0, 0, 0])
    a, b, c = (cm.requests[r].table(0) for r in "abc")
    assert a[:2] == b[:2] == c[:2] and len({a[2], b[2], c[2]}) == 3
    assert cm.pools[0].held_count == 5
    gone = cm.finish("a")
    assert (0, a[0]) not in gone and (0, a[2]) in gone          # the shared ones stay
    assert cm.pools[0].held_count == 4
    cm.check_invariants()
    cm.finish("b")
    assert (0, a[0]) in cm.finish("c")
    # whole pages: nothing to copy
    cm.admit("d"), cm.admit("e")
    write(cm, store, "d", list("01234567"))
    assert (cm.follow(["d", "e"], [0, 0]) == -1).all()
    cm.check_invariants()


def test_follow_is_all_or_nothing_and_refuses():
    cm, store = books(pages=(4, 60)), [{}, {}]
    for r in "abcd":
        cm.admit(r)
    write(cm, store, "a", list("0123456789"))                   # 3 of 4 pages
    before = [cm.requests[r].tables for r in "abc"]
    with pytest.raises(PagesExhausted) as e:
        cm.follow(["a", "b", "c"], [0, 0, 0])                   # two part pages, one page free
    assert e.value.group == 0
    assert [cm.requests[r].tables for r in "abc"] == before and [cm.requests[r].length for r in "abc"] == [10, 0, 0]
    cm.check_invariants()
    for rids, parents, text in [(["a", "a"], [0, 0], "twice"), (["a", "b"], [0, 2], "among"), (["a", "b"], [1, 1], "longer"),
                                (["a", "b", "c"], [0, 0, 1], "shorter")]:
        with pytest.raises(ValueError, match=text):
            cm.follow(rids, parents)
    with pytest.raises(ValueError):
        cm.follow(["a", "b"], [0])
    with pytest.raises(KeyError):
        cm.follow(["a", "z"], [0, 0])
    cm.check_invariants()
    assert NULL_PAGE not in cm.requests["a"].table(0)


# ------------------------------------------------------------------------------ searches


def cpu_model(model_dir, cfg):
    from test_engine_emulated import cpu_model as make
    return make(model_dir, cfg)


def tiny_model(tmp_path, name, sigma=0.2):
    cfg, run = tiny.TINIES[name]
    d = tiny.make_model_dir(tmp_path / name, cfg, run["seed"], sigma)
    return d, cfg, run


def same(got, want, atol):
    assert [h.tokens for h in got] == [t for t, _, _ in want]
    assert [h.stopped for h in got] == [s for _, _, s in want]
    assert np.allclose([h.score for h in got], [s for _, s, _ in want], rtol=0, atol=atol)


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("beams,length_penalty", [(1, 1.0), (3, 1.0), (4, 0.0), (5, 2.0)])
def test_searches_match_plain(emulated, tmp_path, name, beams, length_penalty):
    d, cfg, run = tiny_model(tmp_path, name)
    pcfg, w = plain.load_model_dir(d)
    prompts = list(tiny.random_requests(cfg["vocab_size"], [5, 16, 31], seed=3).values())
    stop = list(range(0, cfg["vocab_size"], 9))                 # many stop ids: searches end early and late
    got = cpu_model(d, cfg).beam_search(prompts, beams=beams, max_tokens=9, stop_ids=stop, chunk=7,
                                        length_penalty=length_penalty, page_size=run["page_size"])
    for g, p in zip(got, prompts):
        same(g, plain_beam_search(lambda t: plain.forward(pcfg, w, t)[-1], p, beams, 9, set(stop), length_penalty), 1e-3)


def search_over_everything(last_logits, prompt, beams, max_tokens, stop_ids, length_penalty):
    """A search whose turns put every continuation of every beam in order, none left out. [(tokens, score, stopped)]."""
    def worth(s, n):
        return s / max(n, 1) ** length_penalty
    live, done = [([], 0.0)], []
    for _ in range(max_tokens):
        found = []
        for w, (t, s) in enumerate(live):
            x = np.asarray(last_logits(prompt + t), dtype=np.float64)
            lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
            found += [(-(s + v), w, i) for i, v in enumerate(lp)]
        found.sort()
        ends = [(worth(-v, len(live[w][0])), live[w][0], -v, True) for v, w, i in found[:beams] if i in stop_ids]
        done = sorted(done + ends, key=lambda h: -h[0])[:beams]
        live = [(live[w][0] + [i], -v) for v, w, i in found if i not in stop_ids][:beams]
        assert len(live) == beams                # the vocabulary has enough of them
        if len(done) == beams and worth(live[0][1], len(live[0][0])) <= done[-1][0]:
            return [h[1:] for h in done]
    return [h[1:] for h in sorted(done + [(worth(s, len(t)), t, s, False) for t, s in live], key=lambda h: -h[0])[:beams]]


@pytest.mark.parametrize("stops,beams", [(1, 4), (2, 1), (2, 3), (3, 2), (3, 4), (5, 8), (2, 32), (13, 5), (40, 4)])
def test_stop_ids_leave_no_beam_without_continuations(emulated, tmp_path, stops, beams):
    """However many of the best continuations end in one of the stop ids, `beams` others go on."""
    from tgo_b200.engine.beams import BeamSearch
    d, cfg, run = tiny_model(tmp_path, "A")
    pcfg, w = plain.load_model_dir(d)
    V = cfg["vocab_size"]
    stop = np.random.default_rng(stops).choice(V, stops, replace=False).tolist()
    more = np.zeros(V, dtype=np.float32)
    more[stop] = 4.0
    eng = cpu_model(d, cfg).new_engine(page_size=4, max_tokens=4000, num_slots=2 * beams)
    step = eng.step
    eng.step = lambda entries: step(entries) + torch.from_numpy(more)
    prompts = list(tiny.random_requests(V, [5, 9], seed=7).values())
    got = BeamSearch(eng, beams, 5, stop + [V + 7], length_penalty=2.0).run(prompts)
    for g, p in zip(got, prompts):
        same(g, search_over_everything(lambda t: plain.forward(pcfg, w, t)[-1] + more, p, beams, 5, set(stop), 2.0), 1e-3)
        assert len(g) == beams


def test_one_beam_is_greedy(emulated, tmp_path):
    d, cfg, run = tiny_model(tmp_path, "B")
    pcfg, w = plain.load_model_dir(d)
    prompt = list(tiny.random_requests(cfg["vocab_size"], [12], seed=5).values())[0]
    got = cpu_model(d, cfg).beam_search([prompt], beams=1, max_tokens=12, page_size=8)
    assert got[0][0].tokens == plain.greedy_generate(pcfg, w, prompt, 12)


def test_more_beams_than_first_tokens(emulated, tmp_path):
    """Beams that find no continuation die and the search goes on without them."""
    from tgo_b200.engine.beams import BeamSearch
    d, cfg, run = tiny_model(tmp_path, "A")
    loaded = cpu_model(d, cfg)
    V = cfg["vocab_size"]
    eng = loaded.new_engine(page_size=4, max_tokens=400, num_slots=8)
    step, allowed = eng.step, [7, 11, 13]
    mask = torch.ones(V, dtype=torch.bool)
    mask[allowed] = False
    eng.step = lambda entries: step(entries).masked_fill(mask, float("-inf"))
    got = BeamSearch(eng, 8, 3).run([[1, 2, 3]])[0]
    assert len(got) == 8 and all(len(h.tokens) == 3 and set(h.tokens) <= set(allowed) for h in got)
    assert len({tuple(h.tokens) for h in got}) == 8
    assert all(p.free_count == p.num_pages for p in eng.cache.pools) and not eng.cache.requests


def test_a_search_that_fails_gives_everything_back(emulated, tmp_path):
    from tgo_b200.engine.beams import BeamSearch
    d, cfg, run = tiny_model(tmp_path, "A")
    eng = cpu_model(d, cfg).new_engine(page_size=4, num_pages=5, num_slots=3)
    with pytest.raises(PagesExhausted):
        BeamSearch(eng, 3, 40).run([[1, 2, 3, 4, 5]])
    assert not eng.cache.requests and all(p.free_count == p.num_pages for p in eng.cache.pools)
    for bad in (dict(beams=0), dict(beams=33), dict(max_tokens=0), dict(chunk=0)):
        with pytest.raises(ValueError):
            BeamSearch(eng, **{**dict(beams=2, max_tokens=4), **bad})
    with pytest.raises(ValueError, match="empty"):
        BeamSearch(eng, 2, 4).run([[]])
    assert BeamSearch(eng, 2, 4).run([]) == []


# ------------------------------------------------------------------------------ adapters


def matrices_of(w):
    return {n: tuple(m.shape) for n, m in w.items() if m.ndim == 2 and ".layers." in n}


def some_adapters(w, layers=2):
    shapes = matrices_of(w)
    names = sorted(shapes)
    return {"all": Adapter(random_adapter(shapes, names, 3, seed=1), 2.0),
            "q and down": Adapter(random_adapter(shapes, [n for n in names if "q_proj" in n or "down" in n], 8, seed=2), 0.5),
            "first layer": Adapter(random_adapter(shapes, [n for n in names if ".layers.0." in n and "k_proj" not in n],
                                                  1, seed=3), 1.0)}


@pytest.mark.parametrize("name", ["A", "B"])
def test_adapted_requests_beside_plain_ones(emulated, tmp_path, name):
    """Requests of three adapters and of none in the same steps: each as its own merged model gives it."""
    from tgo_b200.sampling.policy import Policy
    d, cfg, run = tiny_model(tmp_path, name)
    pcfg, w = plain.load_model_dir(d)
    loaded, adapters = cpu_model(d, cfg), some_adapters(w)
    loaded.load_adapters(adapters)
    prompts = list(tiny.random_requests(cfg["vocab_size"], [5, 16, 31, 9, 9], seed=3).values())
    prompts[4] = prompts[3]
    which = ["all", None, "q and down", "first layer", None]
    got = loaded.generate(prompts, Policy(max_tokens=6), slots=5, chunk=7, page_size=run["page_size"], adapters=which)
    for g, p, a in zip(got, prompts, which):
        ww = w if a is None else with_adapter(w, adapters[a].matrices, adapters[a].scale)
        assert g == plain.greedy_generate(pcfg, ww, p, 6)
    beams = loaded.beam_search(prompts[:3], beams=3, max_tokens=4, adapters=which[:3], page_size=run["page_size"])
    for g, p, a in zip(beams, prompts, which):
        ww = w if a is None else with_adapter(w, adapters[a].matrices, adapters[a].scale)
        same(g, plain_beam_search(lambda t: plain.forward(pcfg, ww, t)[-1], p, 3, 4), 1e-3)
    session = loaded.new_session(context=64, page_size=run["page_size"])
    assert list(session.complete(prompts[0], Policy(max_tokens=6), adapter="all")) == got[0]
    # an engine gives a finished request's name back without its adapter
    eng = loaded.new_engine(page_size=4, max_tokens=64, num_slots=2)
    eng.admit("r", adapter="all")
    eng.finish("r")
    eng.admit("r")
    assert not eng._adapter_of


@pytest.mark.parametrize("parents", [[1, 0, 2], [0, 0, 1], [2, 0, 1], [1, 2, 2], [2, 2, 0]])
def test_adapters_follow_what_the_parents_held(emulated, tmp_path, parents):
    """Requests of one group with unlike adapters: exchanges and chains take the parents' old ones, as they take their rows."""
    from tgo_b200.engine.step import StepEntry
    d, cfg, run = tiny_model(tmp_path, "A")
    pcfg, w = plain.load_model_dir(d)
    loaded, adapters = cpu_model(d, cfg), some_adapters(w)
    loaded.load_adapters(adapters)
    which, text = ["all", None, "first layer"], [[3, 1, 4, 1, 5], [9, 2, 6, 5, 3], [5, 8, 9, 7, 9]]
    eng = loaded.new_engine(page_size=4, max_tokens=96, num_slots=3)
    for r, name in enumerate(which):
        eng.admit(r, adapter=name)
    eng.step([StepEntry(r, text[r], []) for r in range(3)])
    eng.follow([[0, 1, 2]], [parents])
    got = eng.step([StepEntry(r, [7], [0]) for r in range(3)]).numpy()
    for r, p in enumerate(parents):
        ww = w if which[p] is None else with_adapter(w, adapters[which[p]].matrices, adapters[which[p]].scale)
        assert np.allclose(got[r], plain.forward(pcfg, ww, text[p] + [7])[-1], rtol=0, atol=1e-3), r


def write_folder(path, config, tensors):
    from tgo_b200.weights.safetensors import write_safetensors
    os.makedirs(path)
    with open(path / "adapter_config.json", "w") as f:
        json.dump(config, f)
    write_safetensors(str(path / "adapter_model.safetensors"), tensors)
    return str(path)


def test_adapters_from_folders(emulated, tmp_path):
    d, cfg, run = tiny_model(tmp_path, "A")
    pcfg, w = plain.load_model_dir(d)
    ad = some_adapters(w)["all"]
    tensors = {}
    for i, (n, (a, b)) in enumerate(ad.matrices.items()):
        stem = ("base_model.model." if i % 2 else "") + n[:-len(".weight")]
        tensors[stem + ".lora_A.weight"], tensors[stem + ".lora_B.weight"] = a, b
    folder = write_folder(tmp_path / "x", {"r": 3, "lora_alpha": 6, "bias": "none"}, tensors)
    got = read_adapter(folder)
    assert got.scale == 2.0 and set(got.matrices) == set(ad.matrices)
    assert all(torch.equal(got.matrices[n][0], ad.matrices[n][0]) for n in got.matrices)
    assert read_adapter(write_folder(tmp_path / "y", {"r": 4, "lora_alpha": 6, "use_rslora": True}, tensors)).scale == 3.0
    loaded = cpu_model(d, cfg)
    loaded.load_adapters({"x": folder})
    from tgo_b200.sampling.policy import Policy
    assert loaded.generate([[1, 2, 3]], Policy(max_tokens=5), adapters="x")[0] == \
        plain.greedy_generate(pcfg, with_adapter(w, ad.matrices, 2.0), [1, 2, 3], 5)
    for i, (config, text) in enumerate([({"r": 0, "lora_alpha": 1}, "r is 0"), ({"r": 3, "lora_alpha": None}, "lora_alpha"),
                                        ({"r": 3, "lora_alpha": 1, "use_dora": True}, "use_dora"),
                                        ({"r": 3, "lora_alpha": 1, "bias": "all"}, "bias")]):
        with pytest.raises(AdapterError, match=text):
            read_adapter(write_folder(tmp_path / f"bad{i}", config, tensors))
    some = next(iter(tensors))
    with pytest.raises(AdapterError, match="only one"):
        read_adapter(write_folder(tmp_path / "half", {"r": 3, "lora_alpha": 1}, {some: tensors[some]}))
    with pytest.raises(AdapterError, match="no half"):
        read_adapter(write_folder(tmp_path / "odd", {"r": 3, "lora_alpha": 1}, {"x.weight": tensors[some]}))


def test_adapters_are_checked(emulated, tmp_path):
    d, cfg, run = tiny_model(tmp_path, "A")
    pcfg, w = plain.load_model_dir(d)
    loaded = cpu_model(d, cfg)
    n = "model.layers.0.self_attn.q_proj.weight"
    out, inp = w[n].shape
    for matrices, text in [({}, "no matrices"), ({"model.embed_tokens.weight": (torch.zeros(2, 64), torch.zeros(256, 2))}, "no product"),
                           ({n: (torch.zeros(2, inp + 1), torch.zeros(out, 2))}, "for a matrix of"),
                           ({n: (torch.zeros(2, inp), torch.zeros(out, 3))}, "for a matrix of"),
                           ({n: (torch.full((2, inp), float("nan")), torch.zeros(out, 2))}, "not finite")]:
        with pytest.raises(AdapterError, match=text):
            loaded.load_adapters({"bad": Adapter(matrices)})
    with pytest.raises(AdapterError, match="no adapters"):
        loaded.load_adapters({})
    assert loaded.model.adapter_names == []
    loaded.load_adapters({"good": Adapter({n: (torch.ones(2, inp), torch.ones(out, 2))})})
    with pytest.raises(AdapterError, match="loaded already"):
        loaded.load_adapters({"good": Adapter({n: (torch.ones(2, inp), torch.ones(out, 2))})})
    eng = loaded.new_engine(page_size=4, max_tokens=64, num_slots=2)
    with pytest.raises(KeyError, match="not loaded"):
        eng.admit("r", adapter="other")
    assert not eng.cache.requests
    with pytest.raises(KeyError, match="not loaded"):
        loaded.generate([[1]], adapters=["other"])
    with pytest.raises(ValueError, match="2 adapters for 1"):
        loaded.beam_search([[1]], adapters=["good", "good"])


@pytest.mark.parametrize("dtype,number", [("float32", 1e39), ("bfloat16", 3.4e38)])
def test_adapters_that_the_engine_cannot_hold(emulated, tmp_path, dtype, number):
    """Numbers that are finite on disk and would be infinite in the bank, and a scale that would be."""
    d, cfg, run = tiny_model(tmp_path, "A")
    _, w = plain.load_model_dir(d)
    loaded = cpu_model(d, cfg)
    loaded.model.dtype = getattr(torch, dtype)
    n = "model.layers.0.self_attn.q_proj.weight"
    out, inp = w[n].shape
    a, b = torch.ones(2, inp, dtype=torch.float64), torch.ones(out, 2, dtype=torch.float64)
    for big_a, big_b, scale, text in [(number, 1.0, 1.0, "not finite"), (1.0, -number, 1.0, "not finite"), (1.0, 1.0, 1e39, "scale")]:
        with pytest.raises(AdapterError, match=text):
            loaded.load_adapters({"big": Adapter({n: (a * big_a, b * big_b)}, scale)})
    assert loaded.model.adapter_names == []
    loaded.load_adapters({"large": Adapter({n: (a * number / 1e3, b)}, 1e30)})


@pytest.mark.parametrize("begun,fine", [(True, True), (False, True), ("gaussian", True), ("pissa", False), ("pissa_niter_4", False),
                                        ("olora", False), ("loftq", False)])
def test_adapters_of_changed_matrices_are_refused(tmp_path, begun, fine):
    """Halves that were begun from parts of the model's matrices are added to what was left of those."""
    halves = {"x.lora_A.weight": torch.ones(2, 4), "x.lora_B.weight": torch.ones(4, 2)}
    folder = write_folder(tmp_path / "a", {"r": 2, "lora_alpha": 2, "init_lora_weights": begun}, halves)
    if fine:
        assert set(read_adapter(folder).matrices) == {"x.weight"}
    else:
        with pytest.raises(AdapterError, match="init_lora_weights"):
            read_adapter(folder)
