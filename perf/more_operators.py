"""The operators of steps that verify drafted tokens, measured one call at a time.

A request brings a tree of drafted tokens to a step: node 0 is the token that is certain, every other node
continues an earlier one. Four operators. `attention_tree`: every node attends over its request's cache and over
the nodes on its own path. `logits_constrain`: biases, penalties for repeated tokens (a node's history ends in its own
path) and masks of allowed tokens on rows of logits. `tree_accept`: the path that the tokens chosen from the logits
confirm. `tree_keep`: the accepted nodes' rows of the cache moved together. Head counts and vocabulary are those of the
8B shape (32 heads over 8, 128 wide, 36 layers, 151936 tokens, pages of 16) and of the smaller ones that the other
measured cases use.

Inputs come from the seed alone. `exact` states each operator in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda:0"
BF = torch.bfloat16
PAGE = 16


def listed():
    return [
        # one user, a short answer over a short prompt: latency
        dict(name="tree_single", op="attention", dtype="bfloat16", requests=1, nodes=8, context=489, spread=0.0,
             heads=16, kv_heads=4, dim=128, window=0),
        # eight users of the 8B shape, contexts of unlike, odd lengths
        dict(name="tree_batch", op="attention", dtype="bfloat16", requests=8, nodes=16, context=4099, spread=0.8,
             heads=32, kv_heads=8, dim=128, window=0),
        # two long documents, the widest trees
        dict(name="tree_long", op="attention", dtype="bfloat16", requests=2, nodes=64, context=32703, spread=0.1,
             heads=32, kv_heads=8, dim=128, window=0),
        # sliding windows, narrow heads, eight query heads a kv head, an odd number of nodes
        dict(name="tree_window", op="attention", dtype="bfloat16", requests=12, nodes=23, context=5003, spread=0.5,
             heads=16, kv_heads=2, dim=64, window=1024),
        # the true float32 path
        dict(name="tree_float32", op="attention", dtype="float32", requests=3, nodes=12, context=1501, spread=0.7,
             heads=16, kv_heads=4, dim=128, window=0),
        # one row: a grammar and penalties, one user's step
        dict(name="constrain_single", op="constrain", requests=1, nodes=1, vocab=151936, history=700, window=0, bias=12,
             masked=True, tight=3),
        # the nodes of eight trees, each with its own path and its own grammar state
        dict(name="constrain_trees", op="constrain", requests=8, nodes=16, vocab=151936, history=1801, window=512, bias=0,
             masked=True, tight=1),
        # a decode batch of 64 with penalties over whole histories and many biases, no grammar
        dict(name="constrain_batch", op="constrain", requests=64, nodes=1, vocab=151936, history=4001, window=0, bias=300,
             masked=False, tight=0),
        # following one small tree
        dict(name="accept_single", op="accept", requests=1, nodes=8),
        # following the widest trees of a large batch
        dict(name="accept_batch", op="accept", requests=64, nodes=64),
        # the accepted rows of one request, a small model
        dict(name="keep_single", op="keep", dtype="bfloat16", requests=1, nodes=13, layers=8, kv_heads=4, dim=128, most=4),
        # the accepted rows of 48 requests, the 8B shape's 36 layers
        dict(name="keep_batch", op="keep", dtype="bfloat16", requests=48, nodes=33, layers=36, kv_heads=8, dim=128, most=6),
    ]


def draw(rng):
    """One more case of the listed ranges."""
    def log_between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["attention", "attention", "attention", "attention", "constrain", "constrain", "accept", "keep"])
    if op == "attention":
        float32 = rng.random() < 0.2
        nodes = log_between(1, 16 if float32 else 64)
        heads, kv_heads, dim = rng.choice([(32, 8, 128), (16, 4, 128), (40, 8, 128), (16, 2, 64), (8, 8, 64), (12, 12, 128)])
        # keys of all requests together
        keys = 4000 if float32 else 65000 * 8 // max(kv_heads, 8) // max(1, heads * nodes // 2048)
        requests = log_between(1, 3 if float32 else 64)
        context = log_between(17, max(18, keys // requests))
        return dict(op="attention", dtype="float32" if float32 else "bfloat16", requests=requests, nodes=nodes,
                    context=context, spread=round(rng.uniform(0, 0.9), 2), heads=heads, kv_heads=kv_heads, dim=dim,
                    window=rng.choice([0, 0, 0, log_between(16, 2048)]))
    if op == "constrain":
        nodes = log_between(1, 32)
        masked = rng.random() < 0.6
        return dict(op="constrain", requests=log_between(1, max(1, 128 // nodes)), nodes=nodes,
                    vocab=log_between(4000, 151936), history=log_between(1, 4000),
                    window=rng.choice([0, 0, log_between(8, 2048)]), bias=rng.choice([0, 0, log_between(1, 300)]),
                    masked=masked, tight=rng.randint(1, 5) if masked else 0)
    if op == "accept":
        return dict(op="accept", requests=log_between(1, 64), nodes=log_between(1, 64))
    return dict(op="keep", dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), requests=log_between(1, 24),
                nodes=log_between(9, 64), layers=rng.randint(1, 36), kv_heads=rng.choice([2, 4, 8]),
                dim=rng.choice([64, 96, 128]), most=rng.randint(2, 6))


# --------------------------------------------------------------------------------- inputs


def _generator(seed, salt):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)


def _contexts(case):
    n, r, s = case["context"], case["requests"], case["spread"]
    return [max(1, round(n * (1.0 - s * i / r))) for i in range(r)]


def _tree(rng, n):
    """Parents of n nodes in the order a drafter adds them: mostly long branches off a trunk."""
    parents = [-1]
    for i in range(1, n):
        parents.append(i - 1 if rng.random() < 0.6 else rng.randrange(max(0, i - 8), i))
    return parents


def _seen(parents):
    """For each node the bits of the nodes on its path, itself among them, as a signed 64-bit number."""
    bits = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def _ints(values, kind=torch.int32):
    return torch.tensor(values, dtype=kind, device=DEV)


def _starts(case):
    return [case["nodes"] * i for i in range(case["requests"] + 1)]


def _attention_inputs(case, seed):
    g, rng = _generator(seed, 1), random.Random(int(seed) * 7 + 1)
    dt = torch.float32 if case["dtype"] == "float32" else BF
    H, Hkv, D, n, B = case["heads"], case["kv_heads"], case["dim"], case["nodes"], case["requests"]
    lens = [c + n for c in _contexts(case)]
    pages = [-(-x // PAGE) for x in lens]
    total = sum(pages)
    normal = lambda *s: torch.randn(s, generator=g, device=DEV)             # noqa: E731
    kv = torch.empty((2, total + 1, Hkv, PAGE, D), dtype=dt, device=DEV)
    for plane in kv:
        plane.copy_(normal(total + 1, Hkv, PAGE, D))
    kv[:, 0] = float("nan")                                                # the page that nobody holds
    order = (torch.randperm(total, generator=g, device=DEV) + 1).to(torch.int32)
    tables = torch.zeros((B, max(pages)), dtype=torch.int32, device=DEV)
    at = 0
    for b, p in enumerate(pages):
        tables[b, :p] = order[at:at + p]
        kv[:, int(order[at + p - 1]), :, lens[b] - (p - 1) * PAGE:] = float("nan")    # places not written yet
        at += p
    qkv = (normal(B * n, (H + 2 * Hkv) * D) * 1.5).to(dt)
    seen = sum([_seen(_tree(rng, n)) for _ in range(B)], [])
    return dict(op="attention", q=qkv[:, :H * D], out=torch.empty((B * n, H * D), dtype=dt, device=DEV), k=kv[0], v=kv[1],
                tables=tables, lens=_ints(lens), q_start=_ints(_starts(case)), seen=_ints(seen, torch.int64),
                heads=H, kv_heads=Hkv, dim=D, window=case["window"], scale=D ** -0.5, nodes=n, longest=max(lens))


def _constrain_inputs(case, seed):
    g, rng = _generator(seed, 2), random.Random(int(seed) * 7 + 2)
    B, n, V, L = case["requests"], case["nodes"], case["vocab"], case["history"]
    R = B * n
    rand = lambda *s: torch.rand(s, generator=g, device=DEV)                # noqa: E731
    logits = torch.randn((R, V), generator=g, device=DEV) * 2.5
    lengths = [max(1, round(L * (1.0 - 0.6 * i / B))) for i in range(B)]
    starts = [sum(lengths[:i]) for i in range(B + 1)]
    tokens = (rand(starts[-1]).pow(3) * V).to(torch.int32)                 # some tokens come again and again
    state = dict(op="constrain", logits=logits, out=torch.empty_like(logits),
                 owner=torch.arange(B, dtype=torch.int32, device=DEV).repeat_interleave(n),
                 history=(_ints(starts), tokens),
                 penalties=torch.stack([1.05 + 0.3 * rand(B), 0.4 * rand(B), 0.2 * rand(B)], 1).contiguous(),
                 windows=torch.full((B,), case["window"], dtype=torch.int32, device=DEV),
                 drafts=None, bias=None, allowed=None, allowed_rows=None, longest=max(lengths))
    if n > 1:
        seen = sum([_seen(_tree(rng, n)) for _ in range(B)], [])
        state["drafts"] = (_ints(_starts(case)), (rand(R).pow(2) * V).to(torch.int32), _ints(seen, torch.int64))
    if case["bias"]:
        m = min(case["bias"], V)
        ids = torch.stack([torch.randperm(V, generator=g, device=DEV)[:m] for _ in range(B)])
        state["bias"] = (_ints([m * i for i in range(B + 1)]), ids.flatten().to(torch.int32),
                         torch.randn((B * m,), generator=g, device=DEV) * 3.0)
    if case["masked"]:
        words = torch.full((R, (V + 31) // 32), -1, dtype=torch.int32, device=DEV)
        for _ in range(case["tight"]):
            words &= torch.randint(-2 ** 31, 2 ** 31, words.shape, generator=g, device=DEV).to(torch.int32)
        state["allowed"], state["allowed_rows"] = words, torch.randperm(R, generator=g, device=DEV).to(torch.int32)
    return state


def _accept_inputs(case, seed):
    """Trees whose drafts are right about seven times in ten: what was chosen at a node is mostly one of its
    children's tokens."""
    rng = random.Random(int(seed) * 7 + 3)
    parents, tokens, chosen = [], [], []
    for _ in range(case["requests"]):
        p = _tree(rng, case["nodes"])
        t = [rng.randrange(151936) for _ in p]
        for i in range(1, len(p)):
            if rng.random() < 0.1 and any(p[j] == p[i] for j in range(1, i)):
                t[i] = t[next(j for j in range(1, i) if p[j] == p[i])]      # a drafter may draft a token twice
        for i in range(len(p)):
            children = [j for j in range(i + 1, len(p)) if p[j] == i]
            chosen.append(t[rng.choice(children)] if children and rng.random() < 0.7 else rng.randrange(151936))
        parents += p
        tokens += t
    T = len(tokens)
    return dict(op="accept", tokens=_ints(tokens), parents=_ints(parents), chosen=_ints(chosen), q_start=_ints(_starts(case)),
                path=torch.empty(T, dtype=torch.int32, device=DEV), nodes=case["nodes"],
                counts=torch.empty(case["requests"], dtype=torch.int32, device=DEV),
                following=torch.empty(case["requests"], dtype=torch.int32, device=DEV))


def _kept(case, seed):
    """Accepted nodes of each request. None is moved from a place that another is moved to, so that the call gives the
    same when it is made again."""
    rng = random.Random(int(seed) * 7 + 4)
    paths = []
    for _ in range(case["requests"]):
        c = rng.randint(2, case["most"])
        behind = sorted(rng.sample(range(c, case["nodes"]), min(c - 1, case["nodes"] - c)))
        stay = c - len(behind)                                               # the first nodes of a path may lie in place
        paths.append(list(range(stay)) + behind)
    return paths


def _keep_inputs(case, seed):
    g = _generator(seed, 4)
    dt = torch.float32 if case["dtype"] == "float32" else BF
    B, n, Hkv, D = case["requests"], case["nodes"], case["kv_heads"], case["dim"]
    per = -(-n // PAGE) + 1
    pages = B * per + 1
    kv = torch.randn((case["layers"], 2, pages, Hkv, PAGE, D), generator=g, device=DEV).to(dt)
    order = (torch.randperm(pages - 1, generator=g, device=DEV) + 1).view(B, per)
    first = torch.randint(0, PAGE, (B, 1), generator=g, device=DEV)          # where in its first page a request's nodes begin
    place = first + torch.arange(n, device=DEV)
    slots = (order.gather(1, place // PAGE) * PAGE + place % PAGE).flatten().to(torch.int32)
    paths = _kept(case, seed)
    flat = sum([p + [-1] * (n - len(p)) for p in paths], [])
    return dict(op="keep", rows=kv, slots=slots, q_start=_ints(_starts(case)), path=_ints(flat),
                counts=_ints([len(p) for p in paths]), nodes=n)


def prepare(case, seed):
    return {"attention": _attention_inputs, "constrain": _constrain_inputs, "accept": _accept_inputs,
            "keep": _keep_inputs}[case["op"]](case, seed)


# ------------------------------------------------------------------------------ one pass


def run(s):
    if own:
        from tgo_b200.kernels import ops
        if s["op"] == "attention":
            ops.attention_tree(s["q"], s["out"], s["heads"], s["kv_heads"], s["dim"], s["k"], s["v"], PAGE, s["tables"],
                               s["lens"], s["q_start"], s["seen"], s["scale"], s["window"], s["nodes"], s["longest"])
            return s["out"]
        if s["op"] == "constrain":
            ops.logits_constrain(s["logits"], s["owner"], bias=s["bias"], history=s["history"], penalties=s["penalties"],
                                 windows=s["windows"], drafts=s["drafts"], allowed=s["allowed"],
                                 allowed_rows=s["allowed_rows"], out=s["out"])
            return s["out"]
        if s["op"] == "accept":
            ops.tree_accept(s["tokens"], s["parents"], s["chosen"], s["q_start"], s["path"], s["counts"], s["following"])
            return s["path"], s["counts"], s["following"]
        ops.tree_keep([s["rows"]], s["slots"], s["q_start"], s["path"], s["counts"], axis=2)
        return s["rows"]
    return {"attention": _plain_attention, "constrain": _plain_constrain, "accept": _plain_accept,
            "keep": _plain_keep}[s["op"]](s)


def _bits(words, n):
    """[rows, n] truth values of the lowest n bits of 64-bit numbers."""
    return (words.unsqueeze(1) >> torch.arange(n, device=DEV)) & 1 != 0


def _plain_attention(s):
    """All requests at once, keys gathered through the tables and padded to the longest request's."""
    H, Hkv, D, n = s["heads"], s["kv_heads"], s["dim"], s["nodes"]
    B, L = s["lens"].numel(), s["longest"]
    outs = []
    key = torch.arange(L, device=DEV)
    see = _bits(s["seen"], n).view(B, n, n)
    place = see.sum(2) - 1
    base = (s["lens"] - n).long()
    step = max(1, int(2 ** 28 // (H * n * L)))                              # requests whose scores are held at a time
    for b in range(0, B, step):
        e = min(b + step, B)
        t = s["tables"][b:e].long()
        k = s["k"][t].float().permute(0, 2, 1, 3, 4).reshape(e - b, Hkv, -1, D)[:, :, :L]
        v = s["v"][t].float().permute(0, 2, 1, 3, 4).reshape(e - b, Hkv, -1, D)[:, :, :L]
        there = (key < s["lens"][b:e].unsqueeze(1)).view(e - b, 1, L, 1)
        k, v = k.masked_fill(~there, 0.0), v.masked_fill(~there, 0.0)
        q = s["q"][b * n:e * n].float().view(e - b, n, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(e - b, Hkv, -1, D)
        x = (q @ k.transpose(2, 3) * s["scale"]).view(e - b, H, n, L)
        lo = base[b:e].view(-1, 1, 1)
        node = (key - lo).clamp(0, n - 1).expand(-1, n, -1)
        drafted = see[b:e].gather(2, node) & (key >= lo) & (key < lo + n)
        cached = key < lo
        if s["window"]:
            cached = cached & (key > lo + place[b:e].unsqueeze(2) - s["window"])
        x = x.masked_fill(~(drafted | cached).unsqueeze(1), float("-inf"))
        w = torch.exp(x - x.max(3, keepdim=True).values)
        w = w / w.sum(3, keepdim=True)
        o = w.view(e - b, Hkv, -1, L) @ v
        outs.append(o.view(e - b, H, n, D).permute(0, 2, 1, 3).reshape((e - b) * n, H * D))
    return torch.cat(outs).to(s["q"].dtype)


def _plain_constrain(s):
    """Counts of every token for every row, then each edit over all the rows."""
    x, owner = s["logits"], s["owner"].long()
    R, V = x.shape
    start, tokens = s["history"]
    lo, hi = start[owner].long(), start[owner + 1].long()
    window = s["windows"][owner].long()
    room = torch.where(window > 0, window, 2 ** 30)
    counts = torch.zeros((R, V), device=DEV)
    if s["drafts"] is not None:
        q_start, drafted, seen = s["drafts"]
        n = R // s["windows"].numel()
        on = _bits(seen, n)
        rank = on.flip(1).cumsum(1).flip(1)                                 # 1 for the last token of the path
        on = on & (rank <= room.unsqueeze(1))
        at = q_start[owner].long().unsqueeze(1) + torch.arange(n, device=DEV)
        counts.scatter_add_(1, drafted[at].long(), on.float())
        room = room - on.sum(1)
    at = (hi - 1).unsqueeze(1) - torch.arange(s["longest"], device=DEV)    # the last tokens first
    on = (at >= lo.unsqueeze(1)) & (at >= (hi - room).unsqueeze(1))
    counts.scatter_add_(1, tokens[at.clamp(min=0)].long(), on.float())
    if s["bias"] is not None:
        first, ids, values = s["bias"]
        m = ids.numel() // s["windows"].numel()
        at = first[owner].long().unsqueeze(1) + torch.arange(m, device=DEV)
        x = x.scatter_add(1, ids[at].long(), values[at])
    rep, presence, frequency = s["penalties"][owner].unbind(1)
    edited = torch.where(x > 0, x / rep.unsqueeze(1), x * rep.unsqueeze(1))
    edited = edited - (presence.unsqueeze(1) + frequency.unsqueeze(1) * counts)
    x = torch.where(counts > 0, edited, x)
    if s["allowed"] is not None:
        words = s["allowed"][s["allowed_rows"].long()]
        ok = ((words.unsqueeze(2) >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1).view(R, -1)[:, :V] != 0
        x = torch.where(ok, x, float("-inf"))
    return x


def _plain_accept(s):
    """All requests a level at a time."""
    n = s["nodes"]
    tokens, parents, chosen = (s[k].view(-1, n).long() for k in ("tokens", "parents", "chosen"))
    B = tokens.shape[0]
    node = torch.arange(n, device=DEV)
    # the node that each node goes on to (n: none)
    goes = (parents.unsqueeze(1) == node.view(1, n, 1)) & (tokens.unsqueeze(1) == chosen.unsqueeze(2)) & (node > 0)
    to = torch.where(goes, node, n).min(2).values
    to = torch.cat([to, torch.full((B, 1), n, device=DEV)], 1)
    path = torch.zeros((B, n), dtype=torch.int64, device=DEV)
    for j in range(1, n):
        path[:, j] = to.gather(1, path[:, j - 1:j]).squeeze(1)
    counts = (path < n).sum(1)
    last = path.gather(1, (counts - 1).unsqueeze(1))
    following = chosen.gather(1, last).squeeze(1)
    path = torch.where(path < n, path, -1)
    return path.flatten().to(torch.int32), counts.to(torch.int32), following.to(torch.int32)


def _plain_keep(s):
    t, n = s["rows"], s["nodes"]
    path = s["path"].view(-1, n).long()
    slots = s["slots"].view(-1, n).long()
    kept = path >= 0
    source = slots.gather(1, path.clamp(min=0))[kept]
    goal = slots[kept]
    view = t.permute(2, 4, 0, 1, 3, 5)                                       # [pages, places, layers, planes, heads, dim]
    view[goal // PAGE, goal % PAGE] = view[source // PAGE, source % PAGE]
    return t


# ---------------------------------------------------------------------------- definitions


def work(case):
    """What a call cannot do without: each input it needs once, each output once."""
    T = case["requests"] * case["nodes"]
    if case["op"] == "attention":
        e = 4 if case["dtype"] == "float32" else 2
        H, Hkv, D, n, w = case["heads"], case["kv_heads"], case["dim"], case["nodes"], case["window"]
        keys = sum((min(c, w - 1) if w else c) + n for c in _contexts(case))
        seen = sum(n * (min(c, w - 1) if w else c) for c in _contexts(case)) + T
        return {"bytes": 2 * keys * Hkv * D * e + 2 * T * H * D * e + 4 * sum(-(-(c + n) // PAGE) for c in _contexts(case)) + 12 * T,
                "flops": 4.0 * H * D * seen}
    if case["op"] == "constrain":
        V, B = case["vocab"], case["requests"]
        history = sum(max(1, round(case["history"] * (1.0 - 0.6 * i / B))) for i in range(B))
        return {"bytes": 8 * T * V + (T * ((V + 31) // 32) * 4 if case["masked"] else 0) + 4 * history + 8 * B * case["bias"] + 20 * T,
                "flops": 2.0 * T * V}
    if case["op"] == "accept":
        return {"bytes": 16 * T + 12 * case["requests"], "flops": 4.0 * T}
    moved = case["requests"] * (case["most"] / 2.0)                          # of 2 to `most` accepted nodes, without the first
    e = 4 if case["dtype"] == "float32" else 2
    return {"bytes": int(2 * moved * case["layers"] * 2 * case["kv_heads"] * case["dim"] * e) + 8 * T, "flops": 0}


def exact(case, seed):
    """The operators in 64 bits from the same inputs, a request, a row or a node at a time."""
    s = prepare(case, seed)
    n, B = case["nodes"], case["requests"]
    if s["op"] == "attention":
        H, Hkv, D, lens = s["heads"], s["kv_heads"], s["dim"], s["lens"].tolist()
        out = torch.zeros((B * n, H, D), dtype=torch.float64, device=DEV)
        for b in range(B):
            base, pages = lens[b] - n, s["tables"][b, :-(-lens[b] // PAGE)].long()
            bits = [w & (1 << 64) - 1 for w in s["seen"][b * n:(b + 1) * n].tolist()]
            sees = torch.zeros((n, lens[b]), dtype=torch.bool)
            for i, w in enumerate(bits):
                sees[i, max(0, base + w.bit_count() - s["window"]) if s["window"] else 0:base] = True
                for j in range(n):
                    sees[i, base + j] = bool(w >> j & 1)
            sees = sees.to(DEV)
            for h in range(H):
                k = s["k"][pages, h * Hkv // H].reshape(-1, D)[:lens[b]].double()
                v = s["v"][pages, h * Hkv // H].reshape(-1, D)[:lens[b]].double()
                q = s["q"][b * n:(b + 1) * n, h * D:(h + 1) * D].double()
                x = torch.where(sees, (q @ k.T) * s["scale"], -torch.inf)
                out[b * n:(b + 1) * n, h] = torch.softmax(x, 1) @ v
        return out.view(B * n, H * D)
    if s["op"] == "constrain":
        out = s["logits"].double()
        V, owner = case["vocab"], s["owner"].tolist()
        starts, tokens = s["history"][0].tolist(), s["history"][1].tolist()
        for r in range(B * n):
            b = owner[r]
            said = tokens[starts[b]:starts[b + 1]]
            if s["drafts"] is not None:
                w = int(s["drafts"][2][r])
                said = said + [int(t) for j, t in enumerate(s["drafts"][1][b * n:(b + 1) * n].tolist()) if w >> j & 1]
            if case["window"]:
                said = said[-case["window"]:]
            if s["bias"] is not None:
                m = case["bias"] if case["bias"] < V else V
                out[r].index_add_(0, s["bias"][1][b * m:(b + 1) * m].long(), s["bias"][2][b * m:(b + 1) * m].double())
            ids, times = torch.tensor(said, device=DEV).unique(return_counts=True)
            rep, presence, frequency = s["penalties"][b].double().tolist()
            x = out[r, ids]
            out[r, ids] = torch.where(x > 0, x / rep, x * rep) - presence - frequency * times
            if s["allowed"] is not None:
                words = s["allowed"][int(s["allowed_rows"][r])].long()
                token = torch.arange(V, device=DEV)
                out[r, words[token // 32] >> token % 32 & 1 == 0] = -torch.inf
        return out
    if s["op"] == "accept":
        tokens, parents, chosen = (s[k].tolist() for k in ("tokens", "parents", "chosen"))
        path, counts, following = [], [], []
        for b in range(B):
            at, one = 0, [0]
            while True:
                found = [j for j in range(1, n) if parents[b * n + j] == at and tokens[b * n + j] == chosen[b * n + at]]
                if not found:
                    break
                at = found[0]
                one.append(at)
            path += one + [-1] * (n - len(one))
            counts.append(len(one))
            following.append(chosen[b * n + at])
        return _ints(path), _ints(counts), _ints(following)
    t, slots = s["rows"], s["slots"].tolist()
    new = t.clone()
    for b, one in enumerate(_kept(case, seed)):
        for j, i in enumerate(one):
            to, fro = slots[b * n + j], slots[b * n + i]
            new[:, :, to // PAGE, :, to % PAGE] = t[:, :, fro // PAGE, :, fro % PAGE]
    return new
