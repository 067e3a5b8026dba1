"""Drafted generation on the GPU: the text is that of generation without drafts in true float32; in bfloat16 the logits
behind a tree's tokens are those of its paths, and what the cache holds afterwards is the accepted text."""
import random

import numpy as np
import pytest
import torch

import plain_qwen3 as plain
import tiny
from emulated_drafts import Noise, Oracle
from test_beam_search_gpu import adapters_for
from tgo_b200.sampling.policy import Policy

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def tiny_model(tmp_path, name, dtype, sigma=0.2):
    import tgo_b200
    cfg, run = tiny.TINIES[name]
    d = tiny.make_model_dir(tmp_path / name, cfg, run["seed"], sigma)
    return tgo_b200.open(d, dtype=dtype, device=DEV), d, cfg, run


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_float32_text_does_not_depend_on_the_drafts(tmp_path, name):
    from tgo_b200.engine.drafts import NgramDrafter
    model, d, cfg, run = tiny_model(tmp_path, name, "float32")
    pcfg, w = plain.load_model_dir(d)
    V = cfg["vocab_size"]
    prompts = [p + p[-3:] + p[:4] for p in tiny.random_requests(V, [6, 40, 17, 90], seed=3).values()]
    want = [plain.greedy_generate(pcfg, w, p, 24) for p in prompts]
    texts = [p + t for p, t in zip(prompts, want)]
    for drafter in (NgramDrafter(), Oracle(texts, 5, 0), Oracle(texts, 4, 2, V), Noise(V)):
        got = model.generate_drafted(prompts, Policy(max_tokens=24), nodes=20, drafter=drafter, page_size=run["page_size"], chunk=33,
                                     slots=3)
        assert got == want
    oracle = Oracle(texts, 60, 0)
    assert model.generate_drafted(prompts, Policy(max_tokens=24), nodes=64, drafter=oracle, page_size=run["page_size"]) == want
    assert model.last_drafts.steps <= 2


def test_float32_samples_are_drawn_as_without_drafts(tmp_path):
    model, d, cfg, run = tiny_model(tmp_path, "A", "float32", 0.05)
    V = cfg["vocab_size"]
    prompts = [p + p for p in tiny.random_requests(V, [4, 30, 12], seed=5).values()]
    odd = lambda out: [i for i in range(V) if (i + len(out)) % 2]       # noqa: E731
    policies = [Policy(max_tokens=20, temperature=0.9, seed=3, logprobs=True, top_logprobs=3),
                Policy(max_tokens=25, temperature=1.2, top_k=7, seed=4, repetition_penalty=1.4, frequency_penalty=0.3, penalty_window=6,
                       logit_bias={3: 2.0}),
                Policy(max_tokens=22, temperature=0.8, seed=6, allowed=odd, presence_penalty=0.2)]
    want = model.generate(prompts, policies, page_size=16)
    texts = [p + t for p, t in zip(prompts, want)]
    assert all((t + i) % 2 for i, t in enumerate(want[2]))
    for drafter in (Oracle(texts, 6, 1, V), Noise(V, 3)):
        assert model.generate_drafted(prompts, policies, nodes=16, drafter=drafter, page_size=16) == want


def test_adapted_drafts_in_float32(tmp_path):
    model, d, cfg, run = tiny_model(tmp_path, "C", "float32")
    _, w = plain.load_model_dir(d)
    model.load_adapters(adapters_for(w))
    prompts = list(tiny.random_requests(cfg["vocab_size"], [5, 33, 8], seed=9).values())
    which = ["all", None, "attention"]
    want = model.generate(prompts, Policy(max_tokens=16), adapters=which, page_size=16)
    oracle = Oracle([p + t for p, t in zip(prompts, want)], 4, 1, cfg["vocab_size"])
    assert model.generate_drafted(prompts, Policy(max_tokens=16), adapters=which, drafter=oracle, page_size=16) == want
    assert model.last_drafts.accepted > 0


@pytest.mark.parametrize("dim,windows", [(128, True), (128, False), (64, True), (64, False)])
def test_bfloat16_trees_give_what_their_paths_give(tmp_path, dim, windows):
    """Trees on the tensor cores: the logits behind their tokens are those of whole plain forwards of their paths, within
    the bound of every bfloat16 run of this engine: twice what rounding the activations to bfloat16 does to the plain
    forwards of the same texts (`tiny.tolerance`). What the cache holds afterwards is the accepted text."""
    import tgo_b200
    from tgo_b200.engine.step import DraftEntry, StepEntry
    cfg = dict(tiny.TINY_C, head_dim=dim, num_attention_heads=8, num_key_value_heads=2, max_position_embeddings=1024)
    if not windows:
        cfg.update(sliding_window=None, layer_types=["full_attention"] * 2)
    d = tiny.make_model_dir(tmp_path / "m", cfg, 5, 0.05)
    pcfg, w = plain.load_model_dir(d)
    model = tgo_b200.open(d, dtype="bfloat16", device=DEV)
    V, rng = cfg["vocab_size"], random.Random(3)
    eng = model.new_engine(page_size=16, max_tokens=2000, num_slots=2)
    texts = [[rng.randrange(V) for _ in range(n)] for n in (260, 77)]
    for i, t in enumerate(texts):
        eng.admit(i)
        eng.step([StepEntry(i, t, [])])
    mine, ran = [], []
    for turn in range(2):
        entries = [DraftEntry(i, [rng.randrange(V) for _ in range(n)], [-1] + [rng.randrange(max(0, j - 3), j) for j in range(1, n)])
                   for i, n in ((0, 40), (1, 9))]
        seen = {}

        def choose(logits, ctx):
            seen["logits"] = logits.cpu().numpy()
            chosen, at = logits.argmax(1).to(torch.int32), 0
            for e in entries:
                for j in range(1, len(e.tokens), 2):
                    chosen[at + e.parents[j]] = e.tokens[j]
                at += len(e.tokens)
            return chosen
        got = eng.draft_step(entries, choose)
        at = 0
        for i, (e, a) in enumerate(zip(entries, got)):
            paths = []
            for j, p in enumerate(e.parents):
                paths.append((paths[p] if j else []) + [e.tokens[j]])
            for j in (0, len(paths) // 2, len(paths) - 1):
                mine.append(seen["logits"][at + j])
                ran.append(texts[i] + paths[j])
            texts[i] += [e.tokens[j] for j in a.path]
            assert eng.length(i) == len(texts[i]) and len(a.path) > 1
            at += len(e.tokens)
    lg = eng.step([StepEntry(i, [3], [0]) for i in range(2)]).cpu().numpy()
    for i in range(2):
        mine.append(lg[i])
        ran.append(texts[i] + [3])
    want = np.stack([plain.forward(pcfg, w, t)[-1] for t in ran])
    rounded = np.stack([plain.forward_rounded(pcfg, w, t)[-1] for t in ran])
    assert np.abs(np.stack(mine) - want).max() <= tiny.tolerance(cfg, "bfloat16", want, rounded)
    eng.check_kernels()


def test_drafts_beside_decode_graphs(tmp_path):
    """Steps of drafts, of single tokens through graphs and of prompts in one engine, in turn."""
    from tgo_b200.engine.step import DraftEntry, StepEntry
    model, d, cfg, run = tiny_model(tmp_path, "A", "float32")
    pcfg, w = plain.load_model_dir(d)
    V, rng = cfg["vocab_size"], random.Random(2)
    eng = model.new_engine(page_size=16, max_tokens=1000, num_slots=3)
    texts = {}
    for turn in range(12):
        if len(texts) < 3:
            p = [rng.randrange(V) for _ in range(rng.randint(1, 30))]
            eng.admit(turn)
            eng.step([StepEntry(turn, p, [])])
            texts[turn] = p
        for i in texts:
            texts[i] = texts[i] + [turn % V]
        if turn % 3:
            lg = eng.step([StepEntry(i, [turn % V], [0]) for i in texts])
        else:
            out = []
            got = eng.draft_step([DraftEntry(i, [turn % V, 5, 6, 7], [-1, 0, 0, 1]) for i in texts],
                                 lambda logits, ctx: (out.append(logits.clone()), torch.tensor([5, 7, 9, 4] * len(texts), dtype=torch.int32,
                                                                                              device=DEV))[1])
            assert all(a.path == [0, 1, 3] and a.following == 4 for a in got)
            lg = out[0][0::4]
        for k, i in enumerate(texts):
            want = plain.forward(pcfg, w, texts[i])[-1]
            assert np.allclose(lg[k].cpu().numpy(), want, rtol=0, atol=2e-3 * max(1.0, float(np.abs(want).max())))
            if turn % 3 == 0:
                texts[i] = texts[i] + [5, 7]
