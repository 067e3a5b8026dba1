"""The operators of adapted and beam-searched decoding, measured one call at a time.

Three operators. `low_rank`: each row of a batch adds its own adapter's low-rank product to the rows of a
shared projection (q, k and v joined; gate and up rows in eights; an output projection into the float32
stream). `beam_select`: the best continuations over the beams and the vocabulary. `reorder`: rows of a cache
or of a state taken from the beams they continue, in place. Sizes are those of the 8B shape (width 4096, 32
heads over 8, feed-forward 12288, vocabulary 151936) and of the smaller ones the measured cases use.

Inputs come from the seed alone. `exact` states each operator in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda:0"
BF = torch.bfloat16


def listed():
    return [
        # one user's decode step through an adapted output projection, added to the float32 stream
        dict(name="adapter_single", op="low_rank", dtype="bfloat16", stream=True, requests=1, tokens=1, spread=0.0,
             adapters=4, bare=0, rank=16, width=2048, columns="2048", interleaved=False),
        # a serving batch, many adapters, some requests without: joined q, k, v of the 8B shape
        dict(name="adapter_batch", op="low_rank", dtype="bfloat16", stream=False, requests=96, tokens=1, spread=0.0,
             adapters=24, bare=7, rank=16, width=4096, columns="4096+1024+1024", interleaved=False),
        # the true float32 path: short prompts of unlike, odd lengths
        dict(name="adapter_float32", op="low_rank", dtype="float32", stream=False, requests=3, tokens=151, spread=0.7,
             adapters=3, bare=0, rank=8, width=2048, columns="2048+512+512", interleaved=False),
        # prompts of several requests through adapted gate and up projections, rows in eights
        dict(name="adapter_prompts", op="low_rank", dtype="bfloat16", stream=False, requests=5, tokens=611, spread=0.9,
             adapters=4, bare=5, rank=32, width=4096, columns="12288+12288", interleaved=True),
        # a long prompt batch with large adapters on q, k, v
        dict(name="adapter_long", op="low_rank", dtype="bfloat16", stream=False, requests=4, tokens=2048, spread=0.0,
             adapters=3, bare=0, rank=64, width=4096, columns="4096+1024+1024", interleaved=False),
        # one request with four beams over a small vocabulary
        dict(name="beams_single", op="beam_select", requests=1, beams=4, live=4, vocab=32768, masked=0.0),
        # the first step after the prompts: one live beam each
        dict(name="beams_first", op="beam_select", requests=12, beams=5, live=1, vocab=151936, masked=0.0),
        # a batch of sixteen requests, a constrained vocabulary (a third of the tokens masked)
        dict(name="beams_masked", op="beam_select", requests=16, beams=4, live=4, vocab=151936, masked=0.33),
        # a large batch with eight beams each
        dict(name="beams_batch", op="beam_select", requests=64, beams=8, live=8, vocab=151936, masked=0.0),
        # the pages four beams of one request are writing, eight layers
        dict(name="pages_single", op="reorder", what="pages", requests=1, beams=4, moved=2, sources=1, layers=8,
             kv_heads=4, dim=128),
        # the pages of sixteen requests' beams, the 8B shape's 36 layers
        dict(name="pages_batch", op="reorder", what="pages", requests=16, beams=4, moved=3, sources=2, layers=36,
             kv_heads=8, dim=128),
        # float32 states of recurrent layers: two megabytes a layer and beam
        dict(name="states_batch", op="reorder", what="states", requests=8, beams=4, moved=3, sources=2, layers=8,
             kv_heads=16, dim=128),
    ]


def draw(rng):
    """One more case of the listed ranges."""
    def log_between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["low_rank", "low_rank", "low_rank", "beam_select", "beam_select", "reorder"])
    if op == "low_rank":
        wide = rng.random() < 0.5
        width, ff = (4096, 12288) if wide else (2048, 6144)
        qkv = "4096+1024+1024" if wide else "2048+512+512"
        float32 = rng.random() < 0.2
        columns, inter = rng.choice([(qkv, False), (f"{ff}+{ff}", True), (str(width), False)])
        rank = rng.choice([8, 16, 16, 32, 64] if not float32 else [4, 8, 16])
        if rng.random() < 0.4:
            requests, tokens, spread = log_between(1, 200), 1, 0.0
        else:
            requests = rng.choice([1, 2, 3, 5, 8])
            most = 600 if float32 else 3000 if inter else 8000
            tokens, spread = max(1, log_between(20, most) // requests), round(rng.uniform(0, 0.9), 2)
        return dict(op="low_rank", dtype="float32" if float32 else "bfloat16",
                    stream=not inter and not float32 and columns == str(width), requests=requests, tokens=tokens,
                    spread=spread, adapters=log_between(1, 32), bare=rng.choice([0, 0, 2, 5]), rank=rank, width=width,
                    columns=columns, interleaved=inter)
    if op == "beam_select":
        beams = rng.choice([2, 3, 4, 5, 8, 12])
        return dict(op="beam_select", requests=log_between(1, 512 // beams), beams=beams, live=rng.choice([1, beams, beams]),
                    vocab=log_between(4000, 151936), masked=rng.choice([0.0, 0.0, round(rng.uniform(0.1, 0.9), 2)]))
    beams = rng.choice([2, 3, 4, 6, 8])
    moved = rng.randint(1, beams - 1)
    what = rng.choice(["pages", "pages", "states"])
    return dict(op="reorder", what=what, requests=log_between(1, 64 // beams if what == "pages" else 32 // beams),
                beams=beams, moved=moved, sources=rng.randint(1, moved),
                layers=rng.randint(1, 36 if what == "pages" else 8), kv_heads=rng.choice([2, 4, 8]),
                dim=rng.choice([64, 96, 128]))


# --------------------------------------------------------------------------------- inputs


def _generator(seed, salt):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)


def _extents(case):
    n, r, s = case["tokens"], case["requests"], case["spread"]
    return [max(1, round(n * (1.0 - s * i / r))) for i in range(r)]


def _adapter_of(case):
    """The adapter of each request: in turn, every `bare`-th without one (-1)."""
    bare = case["bare"]
    return [-1 if bare and i % bare == bare - 1 else i % case["adapters"] for i in range(case["requests"])]


def _columns(case):
    return [int(c) for c in case["columns"].split("+")]


def _slice_of_columns(case):
    """The slice that each column of y belongs to."""
    widths = _columns(case)
    if case["interleaved"]:
        return (torch.arange(sum(widths), device=DEV) // 8) % 2
    return torch.repeat_interleave(torch.arange(len(widths), device=DEV), torch.tensor(widths, device=DEV))


def _low_rank_inputs(case, seed):
    g = _generator(seed, 1)
    dt = torch.float32 if case["dtype"] == "float32" else BF
    widths, K, r, n = _columns(case), case["width"], case["rank"], case["adapters"]
    N, S = sum(widths), len(widths)
    normal = lambda *s: torch.randn(s, generator=g, device=DEV)             # noqa: E731
    extents, which = _extents(case), _adapter_of(case)
    order = torch.randperm(len(which), generator=g, device=DEV)            # requests lie in any order in a batch
    ids = torch.repeat_interleave(torch.tensor(which, dtype=torch.int32, device=DEV)[order],
                                  torch.tensor(extents, device=DEV)[order])
    T = ids.numel()
    y = normal(T, N) if case["stream"] else normal(T, N).to(dt)
    return dict(op="low_rank", x=normal(T, K).to(dt), y=y, out=torch.empty_like(y),
                a=(normal(n, S, r, K) * K ** -0.5).to(dt), b=(normal(n, N, r) * 0.25 * r ** -0.5).to(dt),
                scale=0.5 + 1.5 * torch.rand((n,), generator=g, device=DEV), ids=ids, widths=tuple(widths),
                interleaved=case["interleaved"], columns=_slice_of_columns(case))


def _beam_inputs(case, seed):
    """Logits as a language model's head gives them, scores of the hypotheses so far. Candidates that
    would lie within 1e-3 of a better one are moved down: which of two equal ones wins would hang on the
    last bits of a sum."""
    g = _generator(seed, 2)
    B, W, V = case["requests"], case["beams"], case["vocab"]
    logits = torch.randn((B * W, V), generator=g, device=DEV) * 2.5
    if case["masked"]:
        logits.masked_fill_(torch.rand((B * W, V), generator=g, device=DEV) < case["masked"], float("-inf"))
    steps = -1.0 - 3.0 * torch.rand((B, W), generator=g, device=DEV)
    scores = steps.cumsum(1) - 10.0
    scores[:, case["live"]:] = float("-inf")
    K, gap = 2 * W, 1e-3
    C = min(4 * K, V)
    for _ in range(3):
        lse = torch.cat([p.double().logsumexp(1) for p in logits.split(64)]).view(B, W, 1)
        best, at = logits.view(B, W, V).topk(C, dim=2)
        value = (scores.double().unsqueeze(2) + best.double() - lse).view(B, W * C)
        value, where = value.sort(dim=1, descending=True)
        value, where = value[:, :C], where[:, :C]
        ramp = torch.arange(C, dtype=torch.float64, device=DEV) * gap
        down = value - ((value + ramp).cummin(1).values - ramp)
        down = torch.where(torch.isfinite(value), down, torch.zeros_like(down))
        rows = torch.arange(B, device=DEV).view(B, 1) * W + where // C
        cols = at.reshape(B, W * C).gather(1, where).long()
        logits[rows, cols] = (logits[rows, cols].double() - down).float()
    return dict(op="beam_select", logits=logits, scores=scores,
                picked=torch.empty((B, K), dtype=torch.float32, device=DEV),
                parents=torch.empty((B, K), dtype=torch.int32, device=DEV),
                tokens=torch.empty((B, K), dtype=torch.int32, device=DEV))


def _row_floats(case):
    return case["kv_heads"] * 16 * case["dim"] if case["what"] == "pages" else case["kv_heads"] * case["dim"] * 256


def _reorder_inputs(case, seed):
    """A pool twice as large as what the beams hold (pages of 16 tokens, keys and values per layer; or a
    state row per slot and layer), the rows the beams hold in no order, and for `moved` beams of each
    request another beam, out of `sources`, that they continue."""
    g = _generator(seed, 3)
    B, W, m, s = case["requests"], case["beams"], case["moved"], case["sources"]
    rows = 2 * B * W + 1
    if case["what"] == "pages":
        t = torch.randn((case["layers"], 2, rows, case["kv_heads"], 16, case["dim"]), generator=g, device=DEV).to(BF)
    else:
        t = torch.randn((case["layers"], rows, case["kv_heads"], case["dim"], 256), generator=g, device=DEV)
    index = (torch.randperm(rows - 1, generator=g, device=DEV)[:B * W] + 1).view(B, W).to(torch.int32)
    who = torch.rand((B, W), generator=g, device=DEV).argsort(1)
    # the last m of `who` move, the first s are continued: one beam may be both (a chain)
    turn = (torch.arange(m, device=DEV) + torch.randint(0, s, (B, 1), generator=g, device=DEV)) % s
    moves, source = who[:, W - m:], who.gather(1, turn)
    source = torch.where(source == moves, who.gather(1, (turn + 1) % s), source)
    parents = torch.arange(W, device=DEV).repeat(B, 1).scatter_(1, moves, source)
    return dict(op="reorder", rows=t, axis=t.dim() - 4, index=index, parents=parents.to(torch.int32))


def prepare(case, seed):
    if case["op"] == "low_rank":
        return _low_rank_inputs(case, seed)
    if case["op"] == "beam_select":
        return _beam_inputs(case, seed)
    return _reorder_inputs(case, seed)


# ------------------------------------------------------------------------------ one pass


def run(s):
    if own:
        from tgo_b200.kernels import ops
        if s["op"] == "low_rank":
            ops.low_rank_add(s["x"], s["y"], s["a"], s["b"], s["scale"], s["ids"], s["widths"], s["interleaved"],
                             out=s["out"])
            return s["out"]
        if s["op"] == "beam_select":
            ops.beam_select(s["logits"], s["scores"], s["picked"], s["parents"], s["tokens"])
            return s["picked"], s["parents"], s["tokens"]
        ops.reorder_rows([s["rows"]], s["index"], s["parents"], axis=s["axis"])
        return s["rows"]
    if s["op"] == "low_rank":
        return _plain_low_rank(s)
    if s["op"] == "beam_select":
        return _plain_beam_select(s)
    return _plain_reorder(s)


def _plain_low_rank(s):
    """Every adapter's u for every row, the rows' own kept, one product with all the adapters' b."""
    x, y, a, b, ids = s["x"].float(), s["y"].float(), s["a"].float(), s["b"].float(), s["ids"].long()
    n, S, r, K = a.shape
    own_one = (ids.unsqueeze(1) == torch.arange(n, device=DEV)).float() * s["scale"]          # [T, n]
    u = (x @ a.reshape(n * S * r, K).T).view(-1, n, S, r) * own_one.view(-1, n, 1, 1)
    in_slice = (s["columns"].unsqueeze(0) == torch.arange(S, device=DEV).unsqueeze(1)).float()   # [S, N]
    full = (b.permute(0, 2, 1).unsqueeze(1) * in_slice.view(1, S, 1, -1)).reshape(n * S * r, -1)
    return (y + u.reshape(-1, n * S * r) @ full).to(s["y"].dtype)


def _plain_beam_select(s):
    logits, scores = s["logits"], s["scores"]
    B, W = scores.shape
    V, K = logits.shape[1], s["picked"].shape[1]
    top = logits.max(dim=1, keepdim=True).values
    lse = top + torch.log(torch.exp(logits - top).sum(dim=1, keepdim=True))
    value = (scores.view(B * W, 1) + (logits - lse)).view(B, W * V)
    picked, flat = value.topk(K, dim=1)
    none = picked == float("-inf")
    parents = torch.where(none, -1, flat // V).to(torch.int32)
    tokens = torch.where(none, -1, flat % V).to(torch.int32)
    return picked, parents, tokens


def _plain_reorder(s):
    t, index = s["rows"], s["index"].long()
    source = index.gather(1, s["parents"].long())
    t.index_copy_(s["axis"], index.reshape(-1), t.index_select(s["axis"], source.reshape(-1)))
    return t


# ---------------------------------------------------------------------------- definitions


def work(case):
    """What a call cannot do without: each input it needs once, each output once."""
    if case["op"] == "low_rank":
        extents, which = _extents(case), _adapter_of(case)
        widths, K, r = _columns(case), case["width"], case["rank"]
        N, S, T = sum(widths), len(widths), sum(extents)
        adapted = sum(n for n, i in zip(extents, which) if i >= 0)
        used = len(set(which) - {-1})
        e = 4 if case["dtype"] == "float32" else 2
        ey = 4 if case["stream"] else e
        return {"bytes": adapted * K * e + 2 * T * N * ey + used * r * (S * K + N) * e + 4 * T + 4 * used,
                "flops": 2.0 * adapted * r * (S * K + N)}
    if case["op"] == "beam_select":
        B, W, V = case["requests"], case["beams"], case["vocab"]
        rows = B * case["live"]
        return {"bytes": 4 * rows * V + 4 * B * W + 12 * B * 2 * W, "flops": 3.0 * rows * V}
    rows = case["layers"] * (2 if case["what"] == "pages" else 1) * _row_floats(case) * \
        (2 if case["what"] == "pages" else 4)
    return {"bytes": case["requests"] * (case["moved"] + case["sources"]) * rows + 8 * case["requests"] * case["beams"],
            "flops": 0}


def exact(case, seed):
    """The operators in 64 bits from the same inputs, a request or an adapter at a time."""
    s = prepare(case, seed)
    if s["op"] == "low_rank":
        out = s["y"].double()
        starts = [sum(s["widths"][:i]) for i in range(len(s["widths"]) + 1)]
        for i in range(case["adapters"]):
            rows = (s["ids"] == i).nonzero().flatten()
            if not rows.numel():
                continue
            x = s["x"][rows].double()
            for k in range(len(s["widths"])):
                cols = torch.arange(starts[k], starts[k + 1], device=DEV)
                if s["interleaved"]:
                    j = torch.arange(s["widths"][k], device=DEV)
                    cols = j // 8 * 16 + k * 8 + j % 8
                d = (x @ s["a"][i, k].double().T) @ s["b"][i][cols].double().T
                out[rows.unsqueeze(1), cols.unsqueeze(0)] += s["scale"][i].double() * d
        return out
    if s["op"] == "beam_select":
        B, W = s["scores"].shape
        K, picked, parents, tokens = s["picked"].shape[1], [], [], []
        for q in range(B):
            rows = s["logits"][q * W:(q + 1) * W].double()
            v = s["scores"][q].double().unsqueeze(1) + torch.log_softmax(rows, dim=1)
            order = v.flatten().argsort(descending=True, stable=True)[:K]
            got = v.flatten()[order]
            some = got > float("-inf")
            picked.append(got)
            parents.append(torch.where(some, order // rows.shape[1], -1).int())
            tokens.append(torch.where(some, order % rows.shape[1], -1).int())
        return torch.stack(picked), torch.stack(parents), torch.stack(tokens)
    t = s["rows"]
    new = t.clone()
    for q in range(case["requests"]):
        for w, p in enumerate(s["parents"][q].tolist()):
            if p != w:
                new.select(s["axis"], int(s["index"][q, w])).copy_(t.select(s["axis"], int(s["index"][q, p])))
    return new
