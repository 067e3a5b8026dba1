"""The operators of drafted tokens, alone: attention of trees, constrained logits, the path that is accepted and its rows of
the cache, against statements in 64 bits at the sizes, masks and mixtures where they can go wrong."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
INF, NAN = float("inf"), float("nan")


def ops():
    from tgo_b200.kernels import ops as o
    return o


def ints(values, kind=torch.int32):
    return torch.tensor(values, dtype=kind, device=DEV)


def signed(bits):
    return [b - (1 << 64) if b >> 63 else b for b in bits]


def random_parents(rng, n):
    return [-1] + [rng.randrange(max(0, i - 5), i) for i in range(1, n)]


def paths_of(parents):
    bits = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << i)
    return bits


WAYS = ["chosen", "FMA units", "one tile whole", "one tile cut", "two tiles whole", "two tiles cut"]


@pytest.fixture(params=WAYS)
def way(request):
    """The attention goes the way that the framework chooses, and all the others where they take the call."""
    if request.param not in WAYS[:2] and request.node.callspec.params.get("dtype", torch.bfloat16) != torch.bfloat16:
        pytest.skip("these ways are bfloat16's")
    ops().attention_tree_force_way(WAYS.index(request.param))
    yield request.param
    ops().attention_tree_force_way(0)
    assert ops().attention_tree_error() == 0


# ------------------------------------------------------------------------------ attention


class Trees:
    """Requests with caches in pages in any order, NaN wherever no key is stored; q inside a wider matrix."""

    def __init__(self, dtype, heads, kv_heads, dim, lens, nodes, page=16, window=0, seed=0, spare=3, size=1.0, shape=None):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rng = random.Random(seed)
        self.dtype, self.H, self.Hkv, self.D, self.page, self.window = dtype, heads, kv_heads, dim, page, window
        self.lens, self.nodes = lens, nodes                   # lens: cached tokens before the step
        B, T = len(lens), sum(nodes)
        total = [c + n for c, n in zip(lens, nodes)]
        pages = [-(-x // page) for x in total]
        self.k, self.v = (torch.full((sum(pages) + 1, kv_heads, page, dim), NAN, dtype=dtype, device=DEV) for _ in range(2))
        self.tables = torch.zeros((B, max(pages + [1]) + 2), dtype=torch.int32, device=DEV)
        order, at = list(range(1, sum(pages) + 1)), 0
        rng.shuffle(order)
        for b, p in enumerate(pages):
            mine = order[at:at + p]
            at += p
            self.tables[b, :p] = ints(mine)
            for i, pg in enumerate(mine):
                there = min(page, total[b] - i * page)
                for t in (self.k, self.v):
                    t[pg, :, :there] = (torch.randn((kv_heads, there, dim), generator=g, device=DEV) * size).to(dtype)
        self.context = ints(total)
        starts = [sum(nodes[:b]) for b in range(B + 1)]
        self.q_start = ints(starts)
        self.bits = sum([paths_of(random_parents(rng, n)) if n else [] for n in nodes], [])
        wide = (heads + 2 * kv_heads) * dim
        self.qkv = (torch.randn((T + spare, wide), generator=g, device=DEV) * size).to(dtype)
        self.out = torch.full((T + spare, heads * dim + 8), 7.0, dtype=dtype, device=DEV)
        self.starts, self.T, self.scale = starts, T, dim ** -0.5

    def run(self, tables=None):
        q = self.qkv[:, :self.H * self.D]
        seen = ints(signed(self.bits) + [-1] * (q.shape[0] - self.T), torch.int64)
        ops().attention_tree(q, self.out, self.H, self.Hkv, self.D, self.k, self.v, self.page,
                             self.tables if tables is None else tables, self.context, self.q_start, seen, self.scale,
                             self.window, max(self.nodes + [0]), max([c + n for c, n in zip(self.lens, self.nodes)] + [0]))
        return self.out

    def plain(self):
        """(result in 64 bits [T, H, D], how far a result may be off).

        The bound. A score is a sum of D products in 32 bits: off by less than (D + 2) 2^-24 sum |q k| scale, and by as much
        again where parts of it are scaled or subtracted; its exponential within 2^-21 of itself (approximate ones
        2^-22, and the argument's rounding, at most 40 log2 e in size, 2^-18). Sums over n keys are off by n 2^-24 at most.
        Weights may be rounded to the storage type (2^-8 in bfloat16), and the result is. All of it weighs on
        sum p |v|, twice: in the sum and in the normaliser."""
        out = torch.zeros((self.T, self.H, self.D), dtype=torch.float64, device=DEV)
        off = torch.full_like(out, 1e-30)                     # a token that sees nothing: exactly zero
        G = self.H // self.Hkv
        half = 2.0 ** -8 if self.dtype == torch.bfloat16 else 2.0 ** -24
        for b, (c, n) in enumerate(zip(self.lens, self.nodes)):
            if not n:
                continue
            pg = self.tables[b, :-(-(c + n) // self.page)].long()
            k = self.k[pg].double().permute(1, 0, 2, 3).reshape(self.Hkv, -1, self.D)[:, :c + n]
            v = self.v[pg].double().permute(1, 0, 2, 3).reshape(self.Hkv, -1, self.D)[:, :c + n]
            for i in range(n):
                t = self.starts[b] + i
                w = self.bits[t]
                first = max(0, c + bin(w).count("1") - self.window) if self.window else 0
                keys = list(range(min(first, c), c)) + [c + j for j in range(n) if w >> j & 1]
                if not keys:
                    continue
                for h in range(self.H):
                    q = self.qkv[t, h * self.D:(h + 1) * self.D].double()
                    kk, vv = k[h // G][keys], v[h // G][keys]
                    x = kk @ q * self.scale
                    p = torch.softmax(x, 0)
                    out[t, h] = p @ vv
                    dx = float((kk.abs() @ q.abs()).max()) * self.scale * 2 * (self.D + 2) * 2.0 ** -24
                    rel = 2 * (dx + 2.0 ** -18 + 2.0 ** -21 + len(keys) * 2.0 ** -24) + half
                    off[t, h] = rel * (p @ vv.abs()) + half * out[t, h].abs() + 1e-30
        return out, off

    def check(self):
        got = self.run()
        want, off = self.plain()
        T, W = self.T, self.H * self.D
        mine = got[:T, :W].double().view(T, self.H, self.D)
        odd = ~torch.isfinite(want)
        assert torch.equal(torch.isnan(mine), torch.isnan(want))
        assert torch.equal(mine[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)])
        far = ((mine - want).abs() / off)[~odd]
        assert not far.numel() or float(far.max()) <= 1.0, float(far.max())
        assert bool((got[T:] == 7).all()) and bool((got[:, W:] == 7).all())     # nobody's rows, nobody's columns
        return got


F32, BF = torch.float32, torch.bfloat16
LAYOUTS = [(16, 4, 128), (32, 8, 128), (8, 2, 64), (5, 5, 64), (10, 2, 128), (16, 1, 128), (6, 2, 96), (4, 2, 72), (48, 2, 128),
           (4, 1, 256), (3, 1, 50)]


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
def test_layouts(way, dtype, heads, kv_heads, dim):
    Trees(dtype, heads, kv_heads, dim, [0, 37, 300, 128], [3, 13, 1, 64], seed=dim + heads).check()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 32, 64, 128, 256])
def test_page_sizes(way, dtype, page):
    Trees(dtype, 8, 2, 128, [page - 1, 2 * page, 127], [2, 7, 33], page=page, seed=page).check()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 15, 64, 129, 300])
def test_windows(way, dtype, dim, window):
    Trees(dtype, 8, 2, dim, [0, 5, 63, 64, 500], [9, 30, 1, 17, 64], window=window, seed=window).check()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("base", [0, 1, 62, 63, 64, 65, 126, 127, 128, 129, 255, 256])
def test_tile_edges(way, dtype, base):
    Trees(dtype, 4, 2, 128, [base], [5], seed=base).check()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_one_node_is_a_decode_step(way, dtype):
    """The same keys through the decode attention: a node alone sees its whole request."""
    c = Trees(dtype, 16, 4, 128, [700, 15, 0, 129], [1, 1, 1, 1], seed=4, spare=0)
    mine = c.check()[:, :16 * 128].float()
    other = torch.empty((4, 16 * 128), dtype=dtype, device=DEV)
    args = (c.qkv[:, :16 * 128], other, 16, 4, 128, c.k, c.v, 16, c.tables)
    position, seq = c.context - 1, torch.arange(4, dtype=torch.int32, device=DEV)
    if dtype == F32:
        ops().attention_generic(*args, seq, position, c.scale, 0)
    else:
        ops().attention_flash(*args, position, seq, None, None, c.scale, 0)
    # both within the bound of `plain`
    want, off = c.plain()
    assert float(((mine.double() - other.double()).abs() / (2 * off.view(4, -1))).max()) <= 1.0


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_requests_of_unlike_lengths(way, dtype, dim):
    """Requests without nodes and padded ones among them, items that several workers share."""
    rng = random.Random(dim)
    lens = [rng.choice([0, 1, 17, 130, 900, 2500]) for _ in range(41)]
    nodes = [rng.choice([0, 1, 1, 2, 8, 31]) for _ in range(41)]
    c = Trees(dtype, 8, 2, dim, lens, nodes, seed=dim)
    c.check()
    # a padded request: one token, no context: zeros
    pad = [b for b, n in enumerate(nodes) if n == 1][:3]
    for b in pad:
        c.context[b] = 0
    got = c.run()
    for b in pad:
        assert bool((got[c.starts[b], :8 * dim] == 0).all())
    again = got.clone()
    assert torch.equal(c.run().view(torch.int16 if dtype == BF else torch.int32), again.view(torch.int16 if dtype == BF else torch.int32))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_one_long_request(way, dtype):
    Trees(dtype, 4, 1, 128, [33000], [3], seed=9).check()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("dim", [64, 128])
def test_empty_rows_and_masks_that_are_no_tree(way, dtype, dim):
    c = Trees(dtype, 8, 2, dim, [0, 0, 40], [4, 64, 20], seed=1)
    rng = random.Random(5)
    c.bits = [0, 1 << 3, 0b1011, 0] + [rng.getrandbits(64) & rng.getrandbits(64) & rng.getrandbits(64) for _ in range(64)] + \
        [rng.getrandbits(64) for _ in range(20)]                  # bits past a request's nodes say nothing
    c.bits[5] = 0
    got = c.run().clone()
    c.bits = [b & (1 << n) - 1 for b, n in zip(c.bits, [4] * 4 + [64] * 64 + [20] * 20)]
    assert torch.equal(c.check(), got)
    assert bool((got[[0, 3, 5], :8 * dim] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("what", [INF, -INF, NAN])
@pytest.mark.parametrize("where", ["k", "v"])
def test_what_is_masked_does_not_show(way, dtype, dim, what, where):
    """A node whose key or value is no finite number is nothing to the nodes that do not see it; to those that do it is
    what the formula makes of it."""
    for base, window in ((0, 0), (100, 0), (120, 33), (127, 0)):
        c = Trees(dtype, 8, 2, dim, [base, 11], [12, 3], window=window, seed=base)
        full = paths_of([-1, 0, 0, 1, 1, 2, 2, 3, 4, 5, 6, 6])
        c.bits[:12] = full
        place = base + 2                                       # node 2: seen by 2, 5, 6, 9, 10, 11
        page = int(c.tables[0, place // 16])
        (c.k if where == "k" else c.v)[page, 1, place % 16, 5] = what
        if where == "k":                                       # a score of inf or NaN makes NaN, one of -inf nothing
            got = c.run()[:15, :8 * dim].double().view(15, 8, dim)
            sees = torch.tensor([bool(b >> 2 & 1) for b in full], device=DEV)
            assert torch.isfinite(got[:12][~sees]).all() and torch.isfinite(got[12:]).all() and torch.isfinite(got[:, :4]).all()
            q = c.qkv[:12, 4 * dim:8 * dim].view(12, 4, dim)[:, :, 5].double()
            hits = sees.unsqueeze(1) & ((q * what) != -INF)
            assert torch.equal(torch.isnan(got[:12, 4:]).all(2), hits)
        else:
            c.check()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_behind_the_window_do_not_show(way, dtype, dim):
    """Cached keys that the first nodes see and deeper ones no more."""
    c = Trees(dtype, 8, 2, dim, [200], [20], window=50, seed=3)
    c.bits = paths_of([i - 1 for i in range(20)])              # a chain: node i at 200 + i sees keys from 151 + i on
    for key in (152, 160, 165):
        c.v[int(c.tables[0, key // 16]), 0, key % 16, 7] = INF
        c.v[int(c.tables[0, key // 16]), 1, key % 16, 9] = NAN
    c.check()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_scores_of_any_size(way, dtype):
    """Scores up to a few hundred apart, and all alike."""
    Trees(dtype, 8, 2, 128, [500, 20], [16, 5], seed=2, size=5.0).check()
    c = Trees(dtype, 8, 2, 128, [500, 20], [16, 5], seed=2)
    c.qkv.zero_()
    c.check()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_pages_that_nobody_has(way, dtype):
    """Numbers outside the pages behind a request's end are not looked at; inside it they are no fault."""
    c = Trees(dtype, 8, 2, 128, [100, 33], [4, 4], seed=6)
    want = c.check().clone()
    bad = c.tables.clone()
    for b in range(2):
        bad[b, -(-int(c.context[b]) // 16):] = ints([2 ** 30, -7] * 20)[:bad.shape[1] - -(-int(c.context[b]) // 16)]
    assert torch.equal(c.run(bad), want)
    bad[1, 0] = 2 ** 28
    assert torch.equal(c.run(bad)[:4], want[:4])


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("lens", [[300, 40], [900, 7, 0, 131]])
def test_queries_off_every_boundary(way, dtype, lens):
    """Where the tensor cores do not take the rows, whatever a call of these sizes would have kept whole or cut."""
    c = Trees(dtype, 16, 4, 128, lens, [8] * len(lens), seed=15)
    wide = torch.zeros((c.qkv.shape[0], c.qkv.shape[1] + 1), dtype=dtype, device=DEV)
    wide[:, 1:] = c.qkv
    c.qkv = wide[:, 1:]
    c.check()


@pytest.mark.parametrize("dtype", [F32, BF])
def test_pages_far_into_a_cache(way, dtype):
    """Numbers of a cache beyond 2^31, bytes beyond 2^32; rows kept there move too."""
    c = Trees(dtype, 16, 8, 128, [300, 40], [9, 3], seed=14)
    far, own = 140000, c.k.shape[0]                            # 16384 numbers a page
    for name in ("k", "v"):
        big = torch.empty((far, 8, 16, 128), dtype=dtype, device=DEV)
        big[far - own:] = getattr(c, name)
        setattr(c, name, big)
    c.tables += far - own
    c.check()
    old, at = c.k[far - own:].clone(), (far - 2) * 16
    ops().tree_keep([c.k], ints([at, at + 1, at + 17]), ints([0, 3]), ints([0, 2, -1]), ints([2]))
    old[own - 2, :, 1] = old[own - 1, :, 1]
    assert torch.equal(torch.nan_to_num(c.k[far - own:]), torch.nan_to_num(old))


def test_attention_captured_beside_another_stream(way):
    """A captured call follows what its inputs hold; two graphs and an eager call on another stream share nothing."""
    cases = [Trees(BF, 16, 4, 128, [2000, 77], [16, 5], seed=s) for s in range(3)]
    want = [c.run().clone() for c in cases]
    graphs = []
    for c in cases[:2]:
        c.seen = ints(signed(c.bits) + [-1] * 3, torch.int64)
        args = (c.qkv[:, :2048], c.out, 16, 4, 128, c.k, c.v, 16, c.tables, c.context, c.q_start, c.seen, c.scale, 0, 16, 4096)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops().attention_tree(*args)
        graphs.append(g)
    for c in cases:
        c.out.fill_(0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            cases[2].run()
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c.out[:c.T, :2048], w[:c.T, :2048])
    # other lengths in the same graph
    c = cases[0]
    shorter = Trees(BF, 16, 4, 128, [300, 1500], [11, 10], seed=8)
    w = shorter.run()[:21, :2048]
    n = min(c.k.shape[0], shorter.k.shape[0])
    assert shorter.k.shape[0] <= c.k.shape[0]
    c.k[:n].copy_(shorter.k), c.v[:n].copy_(shorter.v), c.qkv[:21].copy_(shorter.qkv[:21])
    c.tables.zero_()
    c.tables[:, :shorter.tables.shape[1]].copy_(shorter.tables)
    c.context.copy_(shorter.context), c.q_start.copy_(shorter.q_start)
    c.seen[:21].copy_(ints(signed(shorter.bits), torch.int64))
    graphs[0].replay()
    torch.cuda.synchronize()
    far = (c.out[:21, :2048].float() - w.float()).abs().max()
    assert float(far) <= 2.0 ** -6 * float(w.float().abs().max())     # pieces may be cut elsewhere: two roundings each


def test_attention_refusals():
    c = Trees(F32, 8, 2, 64, [10], [4], seed=0)
    K = ops().KernelError
    ok = dict(q=c.qkv[:, :512], out=c.out, num_heads=8, num_kv_heads=2, head_dim=64, k_cache=c.k, v_cache=c.v, page_size=16,
              block_tables=c.tables, context_lens=c.context, q_start=c.q_start,
              seen=ints(c.bits + [0] * 3, torch.int64), scale=0.1, window=0, max_nodes=4, max_context=14)
    ops().attention_tree(**ok)
    for change, error in [(dict(max_nodes=65), K), (dict(window=-1), K), (dict(q=ok["q"].half()), K),
                          (dict(out=c.out.bfloat16()), AssertionError), (dict(seen=ok["seen"].int()), AssertionError),
                          (dict(seen=ok["seen"][:2]), AssertionError), (dict(k_cache=c.k[:, :, :8]), AssertionError),
                          (dict(q_start=c.q_start[:1]), AssertionError), (dict(q=ok["q"].cpu()), K),
                          (dict(block_tables=c.tables.long()), AssertionError), (dict(num_heads=7), (K, AssertionError)),
                          (dict(q=ok["q"][:, ::2]), AssertionError), (dict(v_cache=c.v[:-1]), AssertionError)]:
        with pytest.raises(error):
            ops().attention_tree(**{**ok, **change})
    ops().attention_tree(**{**ok, "q": ok["q"][:0], "out": c.out[:0], "seen": ok["seen"][:0], "q_start": c.q_start * 0})


# ----------------------------------------------------------------------- constrained logits


def plain_constrain(x, owner, bias, history, penalties, windows, drafts, allowed, allowed_rows):
    """Row by row in 64 bits."""
    x = x.double().cpu()
    R, V = x.shape
    for r in range(R):
        q = r if owner is None else int(owner[r])
        n_req = next((len(t[0]) - 1 for t in (bias, history, drafts) if t is not None), None)
        if n_req is None:
            n_req = len(penalties) if penalties is not None else R
        if 0 <= q < n_req:
            if bias is not None:
                for i in range(int(bias[0][q]), int(bias[0][q + 1])):
                    if 0 <= int(bias[1][i]) < V:
                        x[r, int(bias[1][i])] += float(bias[2][i])
            said = history[1][int(history[0][q]):int(history[0][q + 1])].tolist() if history is not None else []
            if drafts is not None:
                d0, d1 = int(drafts[0][q]), int(drafts[0][q + 1])
                said += [int(drafts[1][d0 + j]) for j in range(min(d1 - d0, 64)) if int(drafts[2][r]) >> j & 1]
            w = int(windows[q]) if windows is not None else 0
            if w > 0:
                said = said[-w:]
            if penalties is not None:
                rep, presence, frequency = (float(p) for p in penalties[q])
                for t in set(said):
                    if not 0 <= t < V:
                        continue
                    v = float(x[r, t])
                    if rep not in (0.0, 1.0):
                        v = v / rep if v > 0 else v * rep
                    x[r, t] = v - (presence + frequency * said.count(t))
        if allowed is not None:
            m = r if allowed_rows is None else int(allowed_rows[r])
            if 0 <= m < allowed.shape[0]:
                words = allowed[m].cpu().long()
                token = torch.arange(V)
                x[r, words[token // 32] >> token % 32 & 1 == 0] = -INF
    return x


def constrained(R, V, Q, seed=0, owner=True, bias=0, history=0, windows=None, nodes=0, allowed=0, rows_of=None, penalised=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    c = dict(owner=None, bias=None, history=None, penalties=None, windows=None, drafts=None, allowed=None, allowed_rows=None)
    if owner:
        c["owner"] = ints([rng.randrange(Q) for _ in range(R)])
    if bias:
        per = [rng.choice([0, bias, max(1, bias // 2)]) for _ in range(Q)]
        ids = sum([rng.sample(range(V), min(n, V)) for n in per], [])
        starts = [sum(min(n, V) for n in per[:i]) for i in range(Q + 1)]
        c["bias"] = (ints(starts), ints(ids), torch.randn(len(ids), generator=g, device=DEV) * 4)
    if history:
        per = [rng.choice([0, 1, history]) if i else history for i in range(Q)]
        tokens = [rng.choice([rng.randrange(V), rng.randrange(min(V, 7)), V - 1]) for _ in range(sum(per))]
        c["history"] = (ints([sum(per[:i]) for i in range(Q + 1)]), ints(tokens))
    if penalised:
        c["penalties"] = torch.tensor([[rng.choice([0.0, 1.0, 1.3]), rng.choice([0.0, 0.4]), rng.choice([0.0, 0.2])]
                                       for _ in range(Q)], device=DEV)
        c["penalties"][0] = torch.tensor([1.2, 0.3, 0.1])
    if windows is not None:
        c["windows"] = ints([rng.choice(windows) for _ in range(Q)])
    if nodes:
        drafted = [rng.randrange(min(V, 50)) for _ in range(Q * nodes)]
        c["drafts"] = (ints([nodes * i for i in range(Q + 1)]), ints(drafted),
                       ints(signed([rng.getrandbits(64) for _ in range(R)]), torch.int64))
    if allowed:
        c["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (allowed, (V + 31) // 32 + 1), generator=g, device=DEV).to(torch.int32)
        c["allowed_rows"] = ints([rng.randrange(-1, allowed + 1) for _ in range(R)])
    return torch.randn((R, V), generator=g, device=DEV) * 3, c


def check_constrain(x, c, strided=False):
    want = plain_constrain(x, **c).to(DEV)
    # five roundings of 32 bits at most (bias, product or quotient, the two penalties, their difference), each of a number
    # no larger than what goes in or what comes out
    size = x.abs().double() * 2 + 4 * 6 + 50
    R, V = x.shape
    for out in ("apart", "in place"):
        if strided:
            rows = torch.full((R, V + 5), 9.0, device=DEV)
            src = rows[:, 1:V + 1]
        else:
            rows = None
            src = torch.empty_like(x)
        src.copy_(x)
        dst = torch.full((R, V), 5.0, device=DEV) if out == "apart" else src
        ops().logits_constrain(src, out=dst if out == "apart" else None, **c)
        gone = want == -INF
        assert torch.equal(dst == -INF, gone)
        far = (dst.double() - want).abs()[~gone]
        assert not far.numel() or bool((far <= 5 * 2.0 ** -24 * size[~gone]).all()), float(far.max())
        if out == "apart":
            assert torch.equal(src, x)
            first = dst.clone()
        else:
            assert torch.equal(dst, first)                     # both ways the same bits
        if rows is not None:
            assert bool((rows[:, 0] == 9).all()) and bool((rows[:, V + 1:] == 9).all())


@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 8191, 8192, 8193, 20003, 151936])
def test_constrain_every_stage(V):
    x, c = constrained(7, V, 4, seed=V, bias=9, history=300, windows=[0, 1, 5, 40, 1000], nodes=9, allowed=5)
    check_constrain(x, c)
    check_constrain(x, c, strided=True)


@pytest.mark.parametrize("stage", ["bias", "history", "drafts", "allowed", "nothing", "no owner", "many biases"])
def test_constrain_single_stages(stage):
    x, c = constrained(6, 9001, 6, seed=3, owner=stage != "no owner", bias={"bias": 5, "no owner": 3, "many biases": 3000}.get(stage, 0),
                       history=77 if stage in ("history", "no owner") else 0, nodes=64 if stage == "drafts" else 0,
                       allowed=6 if stage in ("allowed", "no owner") else 0,
                       penalised=stage not in ("bias", "allowed", "nothing"))
    check_constrain(x, c)


@pytest.mark.parametrize("V", [1, 3, 6143, 6145, 12289, 30002])
@pytest.mark.parametrize("first,stride", [(0, 0), (1, 0), (2, 3), (3, 1), (0, 4)])
def test_constrain_rows_anywhere_to_boundaries(V, first, stride):
    """Rows that begin at any place of 16 bytes, in both matrices alike or not; nothing beside them is written."""
    x, c = constrained(5, V, 3, seed=V + first, bias=7, history=200, windows=[0, 9], nodes=5, allowed=4)
    want = plain_constrain(x, **c).to(DEV)
    size = x.abs().double() * 2 + 4 * 6 + 50
    for out_first in (first, (first + 1) % 4):
        src, dst = (torch.full((5 * (V + stride) + 8,), 9.0, device=DEV) for _ in range(2))
        rows = src[first:].as_strided((5, V), (V + stride, 1), first)
        rows.copy_(x)
        held = src.clone()
        to = dst.as_strided((5, V), (V + stride, 1), out_first)
        ops().logits_constrain(rows, out=to, **c)
        gone = want == -INF
        assert torch.equal(to == -INF, gone) and torch.equal(src, held)
        assert bool(((to.double() - want).abs()[~gone] <= 5 * 2.0 ** -24 * size[~gone]).all())
        to.fill_(9.0)
        assert bool((dst == 9).all())


def test_constrain_odd_values():
    """Infinities and NaN in the logits pass through; -inf stays; a token said a thousand times; ids outside."""
    x, c = constrained(3, 5000, 3, seed=5, history=3000, allowed=3)
    c["history"][1][:1000] = 17
    c["history"][1][1000:1010] = ints([-1, 5000, 2 ** 30, -2 ** 31, 6, 6, 6, 6, 6, 6])
    x[:, 3] = -INF
    x[0, 100] = INF
    want = plain_constrain(x, **c)
    got = x.clone()
    ops().logits_constrain(got, **c)
    assert torch.equal(got.cpu() == -INF, want == -INF) and torch.equal(got.cpu() == INF, want == INF)
    fine = torch.isfinite(want)
    assert float((got.cpu().double() - want)[fine].abs().max()) <= 5 * 2.0 ** -24 * 300
    y = torch.full((1, 64), NAN, device=DEV)
    words = ints([[0, -1]])
    ops().logits_constrain(y, allowed=words)
    assert bool((y[0, :32] == -INF).all()) and bool(torch.isnan(y[0, 32:]).all())
    ops().logits_constrain(y, allowed=words * 0)               # nothing is allowed
    assert bool((y == -INF).all())


@pytest.mark.parametrize("V,first", [(5000, 0), (20003, 1), (151936, 3)])
def test_constrain_long_histories(V, first):
    """More tokens than a block's threads keep, many of them alike, others none at all, at every boundary."""
    x, c = constrained(5, V, 3, seed=V, history=9001, windows=[0, 8000, 4500], nodes=12, bias=1400, allowed=3)
    tokens = c["history"][1]
    tokens[::7] = ints([-1, -V, V, 2 ** 31 - 1, -2 ** 31, 5, V - 1]).repeat(tokens.numel())[:tokens[::7].numel()]
    c["drafts"][1][::5] = -3
    want = plain_constrain(x, **c).to(DEV)
    rows = torch.full((5, V + 8), 9.0, device=DEV)
    src = rows[:, first:V + first]
    src.copy_(x)
    kept = torch.full((5, V + 8), 9.0, device=DEV)
    dst = kept[:, first:V + first]
    ops().logits_constrain(src, out=dst, **c)
    assert torch.equal(src, x) and torch.equal(dst == -INF, want == -INF)
    # 9012 times the frequency penalty's 0.2, and the roundings of `check_constrain`
    size = x.abs().double() * 2 + 4 * 6 + 1900
    fine = want != -INF
    assert bool(((dst.double() - want).abs()[fine] <= 5 * 2.0 ** -24 * size[fine]).all())
    assert bool((kept[:, :first] == 9).all()) and bool((kept[:, V + first:] == 9).all())
    ops().logits_constrain(src, **c)
    assert torch.equal(src, dst)
    c["allowed"] = c["allowed_rows"] = None                    # in place without masks: only what changes is written
    src.copy_(x)
    ops().logits_constrain(src, out=dst, **c)
    ops().logits_constrain(src, **c)
    assert torch.equal(src, dst) and bool((rows[:, :first] == 9).all()) and bool((rows[:, V + first:] == 9).all())


@pytest.mark.parametrize("masked", [True, False])
def test_constrain_rows_far_into_a_matrix(masked):
    """Numbers beyond 2^31; of all rows only the last has anything to edit."""
    R, V = 15000, 151936
    x, c = constrained(1, V, 1, seed=8, history=400, bias=20, allowed=1)
    c["allowed_rows"] = ints([0])
    if not masked:
        c["allowed"] = c["allowed_rows"] = None
    want = x.clone()
    ops().logits_constrain(want, **c)
    rows = torch.full((R, V), 2.5, device=DEV)
    rows[-1] = x[0]
    c["owner"] = ints([-1] * (R - 1) + [0])
    if masked:
        c["allowed_rows"] = ints([-1] * (R - 1) + [0])
    ops().logits_constrain(rows, **c)
    assert torch.equal(rows[-1:], want) and bool((rows[:-1] == 2.5).all())


def test_constrain_starts_outside_their_lists():
    x, c = constrained(3, 700, 3, seed=3, history=30, bias=8, nodes=5, owner=False)
    lists = {k: [t.clone() for t in c[k]] for k in ("history", "bias", "drafts")}
    for k in lists:
        n = c[k][1].numel()
        c[k][0].copy_(ints([-4, min(3, n), n + 9, 2 ** 31 - 1]))   # -4..: from 0 on; 3..n + 9: to the end; n + 9..: nothing
        lists[k][0].copy_(ints([0, min(3, n), n, n]))
    want = plain_constrain(x, **dict(c, **lists)).to(DEV)
    for out in (torch.empty_like(x), None):
        got = x.clone()
        ops().logits_constrain(got, out=out, **c)
        assert float(((got if out is None else out).double() - want).abs().max()) <= 5 * 2.0 ** -24 * 100


def test_constrain_owners_outside_are_left_alone():
    x, c = constrained(4, 777, 2, seed=8, bias=4, history=30)
    c["owner"] = ints([-1, 0, 2, 1])
    got = x.clone()
    ops().logits_constrain(got, **c)
    assert torch.equal(got[[0, 2]], x[[0, 2]]) and not torch.equal(got[1], x[1])
    check_constrain(x, c)


def test_constrain_is_the_sampler_of_single_rows():
    """Bit for bit what `logits_adjust` makes of each row."""
    from tgo_b200.sampling.sampler import penalty_counts
    x, c = constrained(5, 30011, 5, seed=2, owner=False, bias=40, history=500, windows=[0, 60])
    want = x.clone()
    for r in range(5):
        b0, b1 = c["bias"][0][r:r + 2].tolist()
        h0, h1 = c["history"][0][r:r + 2].tolist()
        ids, counts = penalty_counts(c["history"][1][h0:h1].tolist(), int(c["windows"][r]))
        ops().logits_adjust(want[r], c["bias"][1][b0:b1], c["bias"][2][b0:b1], ints(ids) if ids else None,
                            ints(counts) if ids else None, *c["penalties"][r].tolist())
    ops().logits_constrain(x, **c)
    assert torch.equal(x, want)


def test_constrain_refusals():
    x, c = constrained(4, 100, 4, seed=1, bias=2, history=5, allowed=2)
    K = ops().KernelError
    wide = torch.randn((4, 300), device=DEV)
    for change, error in [(dict(allowed=c["allowed"][:, :3].contiguous()), K), (dict(owner=c["owner"][:2]), AssertionError),
                          (dict(penalties=c["penalties"][:2]), AssertionError), (dict(out=x.bfloat16()), AssertionError),
                          (dict(history=(c["history"][0][:3], c["history"][1])), AssertionError),
                          (dict(allowed=c["allowed"].long()), AssertionError), (dict(owner=c["owner"].cpu()), K),
                          (dict(out=torch.empty((4, 99), device=DEV)), AssertionError)]:
        with pytest.raises(error):
            ops().logits_constrain(x, **{**c, **change})
    with pytest.raises(K):                                     # rows over each other
        ops().logits_constrain(wide[:, :100], out=wide[:, 50:150])
    with pytest.raises(K):
        ops().logits_constrain(x.cpu())
    ops().logits_constrain(x[:0], owner=c["owner"][:0])
    ops().logits_constrain(x[:, :0])


# --------------------------------------------------------------------- accepted paths


def plain_accept(tokens, parents, chosen, starts):
    path, counts, following = [-1] * len(tokens), [], []
    for a, e in zip(starts, starts[1:]):
        if a == e:
            counts.append(0), following.append(-1)
            continue
        at, j = 0, 0
        while at is not None:
            path[a + j], j, last = at, j + 1, at
            at = next((i for i in range(at + 1, e - a) if parents[a + i] == at and tokens[a + i] == chosen[a + at]), None)
        counts.append(j), following.append(chosen[a + last])
    return path, counts, following


def run_accept(tokens, parents, chosen, starts):
    T, B = len(tokens), len(starts) - 1
    path, counts, following = ints([7] * T), ints([7] * B), ints([7] * B)
    ops().tree_accept(ints(tokens), ints(parents), ints(chosen), ints(starts), path, counts, following)
    return path.tolist(), counts.tolist(), following.tolist()


@pytest.mark.parametrize("nodes", [[1], [64], [5, 0, 33, 32, 2, 64, 1, 0], [31] * 130])
@pytest.mark.parametrize("vocab", [1, 2, 40])
def test_accept(nodes, vocab):
    """Few tokens: long paths, siblings with one token."""
    rng = random.Random(vocab + len(nodes))
    starts = [sum(nodes[:i]) for i in range(len(nodes) + 1)]
    parents = sum([random_parents(rng, n) if n else [] for n in nodes], [])
    tokens = [rng.randrange(vocab) for _ in parents]
    chosen = [rng.randrange(vocab) for _ in parents]
    assert run_accept(tokens, parents, chosen, starts) == plain_accept(tokens, parents, chosen, starts)


def test_accept_a_chain_of_64_and_links_that_are_none():
    chain = list(range(-1, 63))
    assert run_accept(list(range(64)), chain, list(range(1, 65)), [0, 64]) == (list(range(64)), [64], [64])
    # parents that are no earlier node: nobody gets there, and nothing goes round
    parents = [1, 0, 5, 3, -9, 2, 900]
    assert run_accept([4] * 7, parents, [4] * 7, [0, 7]) == plain_accept([4] * 7, parents, [4] * 7, [0, 7]) == \
        ([0, 1, -1, -1, -1, -1, -1], [2], [4])
    path, counts, following = run_accept([1] * 3, [-1, 0, 1], [1] * 3, [0, 0, 3, 3])
    assert (path, counts, following) == ([0, 1, 2], [0, 3, 0], [-1, 1, -1])


def test_accept_starts_outside():
    assert run_accept([1] * 4, [-1, 0, 1, 2], [1] * 4, [-3, 2, 9, 12]) == ([0, 1, 0, -1], [2, 1, 0], [1, 1, -1])


def test_accept_refusals():
    t, s, c = ints([1, 2]), ints([0, 2]), ints([0])
    with pytest.raises(AssertionError):
        ops().tree_accept(t, t[:1], t, s, t.clone(), c, c.clone())
    with pytest.raises(AssertionError):
        ops().tree_accept(t, t, t.long(), s, t.clone(), c, c.clone())
    with pytest.raises(AssertionError):
        ops().tree_accept(t, t, t, s[:1], t.clone(), c, c.clone())
    with pytest.raises(ops().KernelError):
        ops().tree_accept(t.cpu(), t, t, s, t.clone(), c, c.clone())
    ops().tree_accept(t[:0], t[:0], t[:0], s[:1], t[:0], c[:0], c[:0])


# ------------------------------------------------------------------------- kept rows


@pytest.mark.parametrize("shape,axis", [((3, 2, 40, 4, 16, 128), 2), ((40, 2, 8, 64), 0), ((2, 40, 16, 33), 1), ((40, 4, 5), 0),
                                        ((1, 2, 40, 3, 16, 50), 2)])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_keep(shape, axis, dtype):
    """Any ascending paths: rows that others are moved to are moved on."""
    rng = random.Random(axis)
    g = torch.Generator(device=DEV).manual_seed(axis)
    pages, ps = shape[axis], shape[-2]
    tensors = [torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(2)]
    nodes = [9, 1, 0, min(64, pages * ps // 4), 5]
    starts = [sum(nodes[:i]) for i in range(6)]
    slots = rng.sample(range(pages * ps), starts[-1])
    path, counts = [-1] * starts[-1], []
    for a, n in zip(starts, nodes):
        c = rng.randint(min(n, 1), n)
        one = [0] + sorted(rng.sample(range(1, n), c - 1)) if n else []
        path[a:a + c] = one
        counts.append(c)
    path[starts[4]:starts[5]], counts[4] = [0, 2, 3, 4, -1], 4
    want = []
    for t in tensors:
        new = t.clone()
        lead = (slice(None),) * axis
        for a, c in zip(starts, counts):
            for j in range(c):
                to, fro = slots[a + j], slots[a + path[a + j]]
                place = (lambda p: lead + (p // ps,) + (slice(None),) * (len(shape) - axis - 3) + (p % ps,))
                new[place(to)] = t[place(fro)]
        want.append(new)
    ops().tree_keep(tensors, ints(slots), ints(starts), ints(path), ints(counts), axis=axis)
    assert all(torch.equal(t, w) for t, w in zip(tensors, want))


def test_keep_passes_over_what_is_outside():
    t = torch.arange(8 * 4 * 6, dtype=torch.float32, device=DEV).view(8, 4, 6)
    old = t.clone()
    # entries: a slot outside, one below zero, a path entry below its place, outside its request
    ops().tree_keep([t], ints([0, 9, 50, -1, 20, 21]), ints([0, 6]), ints([0, 2, 3, 2, 9, 5]), ints([6]))
    assert torch.equal(t, old)
    ops().tree_keep([t], ints([0, 9, 50, -1, 20, 21]), ints([0, 6]), ints([0, 4, 3, -1, -1, -1]), ints([99]))
    old[2, 1] = old[5, 0]
    assert torch.equal(t, old)
    ops().tree_keep([t[:0]], ints([0]), ints([0, 1]), ints([0]), ints([1]))
    ops().tree_keep([], ints([0]), ints([0, 1]), ints([0]), ints([1]))


def test_keep_starts_outside():
    t = torch.randn((8, 4, 6), device=DEV)
    want = t.clone()
    want[0, 1] = t[0, 2]
    ops().tree_keep([t], ints([0, 1, 2]), ints([-5, 3, 40, 2 ** 31 - 1]), ints([0, 2, -1]), ints([3, 3, 3]))
    assert torch.equal(t, want)


def test_keep_more_tensors_than_a_launch_takes():
    tensors = [torch.randn((6, 2, 8, 16), device=DEV) for _ in range(67)]
    want = [t.clone() for t in tensors]
    for w in want:
        w[1, :, 3] = w[2, :, 0]
    ops().tree_keep(tensors, ints([8, 11, 16]), ints([0, 3]), ints([0, 2, -1]), ints([2]))
    assert all(torch.equal(t, w) for t, w in zip(tensors, want))


def test_keep_refusals():
    s, K = ints([1]), ops().KernelError
    t = torch.zeros((4, 2, 8, 16), device=DEV)
    with pytest.raises(K):
        ops().tree_keep([t, torch.zeros((4, 2, 4, 16), device=DEV)], s, ints([0, 1]), s, s)
    with pytest.raises(AssertionError):
        ops().tree_keep([t[:, :, ::2]], s, ints([0, 1]), s, s)
    with pytest.raises(AssertionError):
        ops().tree_keep([t], s.long(), ints([0, 1]), s, s)
    with pytest.raises(K):
        ops().tree_keep([t.cpu()], s, ints([0, 1]), s, s)


def test_every_call_runs_on_the_device_of_the_current_stream():
    """On a stream other than the default one, in order with it."""
    s = torch.cuda.Stream()
    x, c = constrained(4, 5000, 4, seed=1, history=50)
    want = x.clone()
    ops().logits_constrain(want, **c)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        y = x.clone()
        ops().logits_constrain(y, **c)
    s.synchronize()
    assert torch.equal(y, want)


def test_sizes_are_those_the_kernels_state():
    assert ops().TREE_NODES == 64 and math.log2(ops().TREE_NODES) == 6


def test_no_wait_ran_out():
    x, c = constrained(40, 70001, 4, seed=2, history=50)
    ops().logits_constrain(x, out=torch.empty_like(x), **c)
    assert not {"logits_constrain", "attention_tree"} & set(ops().kernel_wait_errors())


def test_the_operators_of_a_step_captured_and_replayed():
    """Constrained rows, the path that their tokens confirm, its rows of a cache moved: one graph, new inputs."""
    n, V, rng = 9, 5000, random.Random(4)
    x, c = constrained(2 * n, V, 2, seed=6, history=200, nodes=n, allowed=2 * n)
    c["owner"] = ints([0] * n + [1] * n)
    starts, slots = ints([0, n, 2 * n]), ints(rng.sample(range(80), 2 * n))
    tokens, parents, picked = c["drafts"][1], ints([0] * 2 * n), ints([0] * 2 * n)
    path, counts, following = ints([0] * 2 * n), ints([0] * 2), ints([0] * 2)
    cache, out = torch.zeros((3, 5, 2, 16, 32), device=DEV), torch.empty_like(x)

    def step():
        ops().logits_constrain(x, out=out, **c)
        picked.copy_(out.argmax(1))
        ops().tree_accept(tokens, parents, picked, starts, path, counts, following)
        ops().tree_keep([cache], slots, starts, path, counts, axis=1)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device=DEV).manual_seed(turn), device=DEV))
        trees = [random_parents(rng, n) for _ in range(2)]
        parents.copy_(ints(sum(trees, [])))
        c["drafts"][2].copy_(ints(signed(paths_of(trees[0]) + paths_of(trees[1])), torch.int64))
        c["allowed"].copy_(torch.zeros_like(c["allowed"]))
        for r in range(2 * n):                                 # a token each, mostly one that was drafted there
            kids = [i for i, p in enumerate(trees[r // n]) if p == r % n]
            t = int(tokens[r // n * n + kids[0]]) if kids and turn else rng.randrange(V)
            c["allowed"][r, t // 32] = signed([1 << t % 32 | (0xffffffff00000000 if t % 32 == 31 else 0)])[0]
        c["allowed_rows"].copy_(ints(list(range(2 * n))))
        cache.normal_()
        old = cache.clone()
        graph.replay()
        got = [t.clone() for t in (out, picked, path, counts, following, cache)]
        assert torch.equal(got[0] == -INF, plain_constrain(x, **c).to(DEV) == -INF)
        assert tuple(t.tolist() for t in got[2:5]) == plain_accept(tokens.tolist(), parents.tolist(), got[1].tolist(), [0, n, 2 * n])
        cache.copy_(old)
        step()
        assert all(torch.equal(a, b) for a, b in zip(got, (out, picked, path, counts, following, cache)))
