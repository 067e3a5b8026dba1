"""The selection over beams and vocabulary and the reordering of rows, alone: against plain
restatements in 64 bits, at the sizes, masks and ties where they can go wrong."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
INF = float("inf")


def ops():
    from tgo_b200.kernels import ops as o
    return o


@pytest.fixture(params=["chosen", "two kernels", "clusters"], autouse=True)
def way(request):
    """Every test goes the way that the framework chooses, and both of them wherever they take its call."""
    ops().beam_force_way(["chosen", "two kernels", "clusters"].index(request.param))
    yield request.param
    ops().beam_force_way(0)


def plain_values(logits, scores):
    """[B, W, V] in 64 bits on the CPU; -inf where the pair is no candidate."""
    B, W = scores.shape
    x = logits.double().cpu().view(B, W, -1)
    c = scores.double().cpu()
    m = x.max(dim=2, keepdim=True).values
    fine = torch.isfinite(c).unsqueeze(2) & torch.isfinite(m) & ~torch.isnan(x).any(2, keepdim=True)
    s = torch.exp(x - m).sum(2, keepdim=True)
    v = (x - m) - torch.log(s) + c.unsqueeze(2)
    return torch.where(fine & (x > -INF), v, torch.full_like(v, -INF))


def select(logits, scores, K):
    B = scores.shape[0]
    picked = torch.full((B, K), 7.0, device=DEV)
    parents = torch.full((B, K), 7, dtype=torch.int32, device=DEV)
    tokens = torch.full((B, K), 7, dtype=torch.int32, device=DEV)
    ops().beam_select(logits, scores, picked, parents, tokens)
    return picked.cpu(), parents.cpu(), tokens.cpu()


def check(logits, scores, K):
    """Every place: the pick's own value is the one reported, and it is the plain k-th; where the plain
    values around a place are further apart than the bound, the pair itself is the plain one.

    The bound: a thread adds at most V / 256 + 4 rounded exponentials (each within 2^-22 and 2^-24 of
    its exponent's size, at most 150) one after the other, then 5 + 8 + 256 partial sums in a tree: the sum
    is off by less than (V / 256 + 300) 2^-24 + 2^-22 + 150 * 2^-23 of itself, its logarithm by as much;
    the result is rounded once."""
    v = plain_values(logits, scores)
    B, W, V = v.shape
    flat = v.view(B, W * V)
    picked, parents, tokens = select(logits, scores, K)
    off = (V / 256 + 300) * 2.0 ** -24 + 2.0 ** -22 + 150 * 2.0 ** -23
    for b in range(B):
        order = flat[b].argsort(descending=True, stable=True)[:K + 1]
        want = flat[b][order]
        for k in range(K):
            if k >= W * V or want[k] == -INF:
                assert picked[b, k] == -INF and parents[b, k] == -1 and tokens[b, k] == -1, (b, k)
                continue
            tol = off + abs(float(want[k])) * 2.0 ** -23
            at = int(parents[b, k]) * V + int(tokens[b, k])
            assert 0 <= at < W * V and 0 <= int(tokens[b, k]) < V
            assert abs(float(flat[b][at]) - float(picked[b, k])) <= tol, (b, k)
            assert abs(float(want[k]) - float(picked[b, k])) <= tol, (b, k)
            apart = (k == 0 or want[k - 1] - want[k] > 2 * tol) and \
                (k + 1 >= len(want) or want[k] - want[k + 1] > 2 * tol)
            if apart:
                assert at == int(order[k]), (b, k)
    return picked, parents, tokens


def rows(n, V, seed, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, V, generator=g) * scale).to(DEV)


def so_far(B, W, seed):
    g = torch.Generator().manual_seed(seed + 100)
    return (-10.0 - 20.0 * torch.rand(B, W, generator=g)).to(DEV)


@pytest.mark.parametrize("B,W,V,K", [
    (1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 7, 6), (1, 2, 4096, 4), (1, 4, 32768, 8), (3, 5, 4097, 10), (2, 2, 151936, 64),
    (1, 32, 1000, 64), (5, 8, 999, 16), (40, 4, 8191, 8), (1, 1, 300000, 33), (2, 7, 20011, 1), (130, 3, 2050, 6)])
def test_select(B, W, V, K):
    check(rows(B * W, V, seed=V + K), so_far(B, W, seed=V), K)


@pytest.mark.parametrize("first", [0, 1, 2, 3])
@pytest.mark.parametrize("V", [1, 3, 4, 1023, 4099, 9001])
def test_select_of_strided_rows_at_any_alignment(first, V):
    wide = rows(6, V + 7, seed=first)
    wide[:, :first] = 1e30                      # what lies beside the rows is not theirs
    wide[:, first + V:] = 1e30
    check(wide[:, first:first + V], so_far(2, 3, seed=V), 5)


@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_select_with_masked_tokens(V):
    x = rows(8, V, seed=V)
    g = torch.Generator().manual_seed(V)
    x[torch.rand(8, V, generator=g).to(DEV) < 0.9] = -INF
    x[1] = -INF                                 # nothing left of a beam
    x[2] = -INF
    x[2, V - 1] = 3.0                           # one token left
    x[5] = torch.finfo(torch.float32).min       # masked with the type's lowest value: all tokens alike
    x[6, 1:] = torch.finfo(torch.float32).min
    check(x, so_far(2, 4, seed=V), 8)


def test_beams_that_give_nothing():
    """Scores that are no numbers, rows with a NaN or +inf, beams that have ended: none of their tokens, and
    the others' as if they were not there."""
    x = rows(6, 5003, seed=3)
    c = so_far(1, 6, seed=3)
    c[0, 0], c[0, 1], c[0, 2] = -INF, float("nan"), INF
    x[3, 77] = float("nan")
    x[4, 4999] = INF
    picked, parents, _ = check(x, c, 12)
    assert (parents == 5).all()
    x[5] = -INF
    picked, parents, tokens = check(x, c, 12)
    assert (parents == -1).all() and (tokens == -1).all() and (picked == -INF).all()


@pytest.mark.parametrize("V", [3, 100, 4096, 20000, 151936])
def test_ties_go_to_the_lowest_place(V):
    """Constant rows, equal beams: the order is (beam, token)."""
    K = 16
    x = torch.full((4, V), 1.25, device=DEV)
    picked, parents, tokens = select(x, torch.full((1, 4), -2.0, device=DEV), K)
    n = min(K, 4 * V)
    want = torch.arange(n)
    assert torch.equal(parents[0, :n].long(), want // V) and torch.equal(tokens[0, :n].long(), want % V)
    assert torch.allclose(picked[0, :n], torch.full((n,), -2.0 - math.log(V)), rtol=0, atol=1e-4)
    # a few larger equal values, at both ends and in the middle, in each of two equal beams
    x = rows(1, V, seed=V).clamp(max=5.0).repeat(2, 1)
    top = sorted({0, V // 2, V - 1})
    x[:, top] = 9.0
    _, parents, tokens = select(x, torch.full((1, 2), -2.0, device=DEV), 2 * len(top))
    assert tokens[0].tolist() == top + top and parents[0].tolist() == [0] * len(top) + [1] * len(top)


def test_zeros_of_either_sign_are_equal():
    x = torch.full((1, 3000), -1.0, device=DEV)
    x[0, 10], x[0, 20], x[0, 2999] = 0.0, -0.0, 0.0
    x[0, 5] = -0.0
    _, _, tokens = select(x, torch.zeros(1, 1, device=DEV), 4)
    assert tokens[0].tolist() == [5, 10, 20, 2999]


@pytest.mark.parametrize("V", [4096, 40001, 151936])
@pytest.mark.parametrize("order", ["ascending", "descending", "one warp low"])
def test_select_of_ordered_rows(V, order):
    """Every value of a row beats those before it; none does; a warp's share of the first turn is far below
    the rest."""
    x = torch.linspace(-20.0, 10.0, V, device=DEV).repeat(2, 1)
    if order == "descending":
        x = x.flip(1).contiguous()
    elif order == "one warp low":
        x = rows(2, V, seed=1)
        x.view(2, -1)[:, : V // 128 * 128].view(2, -1, 128)[:, ::8] = -100.0
    check(x, so_far(1, 2, seed=V), 40)


def test_select_on_another_stream():
    x, c = rows(8, 50000, seed=9), so_far(2, 4, seed=9)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [select(x, c, 8) for _ in range(3)]
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, select(x, c, 8)))


def test_select_refuses():
    o = ops()
    x, c = rows(2, 50, seed=1), so_far(1, 2, seed=1)

    def outs(K):
        return (torch.empty(1, K, device=DEV), torch.empty(1, K, dtype=torch.int32, device=DEV),
                torch.empty(1, K, dtype=torch.int32, device=DEV))
    with pytest.raises(o.KernelError, match="65"):
        o.beam_select(x, c, *outs(65))
    with pytest.raises(o.KernelError):
        o.beam_select(rows(33, 50, seed=1), so_far(1, 33, seed=1), *outs(4))
    with pytest.raises(o.KernelError):
        o.beam_select(rows(2, 0, seed=1), c, *outs(4))
    with pytest.raises(o.KernelError, match="CUDA device"):
        o.beam_select(x.cpu(), c, *outs(4))
    with pytest.raises(AssertionError):
        o.beam_select(x.to(torch.bfloat16), c, *outs(4))
    with pytest.raises(AssertionError):
        o.beam_select(x, c.double(), *outs(4))
    o.beam_select(rows(0, 50, seed=1), so_far(0, 2, seed=1), *(t[:0] for t in outs(4)))


# ------------------------------------------------------------------------ reorder_rows


def plain_reorder(t, index, parents, axis):
    new = t.clone()
    R = t.shape[axis]
    for row, par in zip(index.tolist(), parents.tolist()):
        W = len(row)
        for w, p in enumerate(par):
            if p != w and 0 <= p < W and 0 <= row[w] < R and 0 <= row[p] < R:
                new.select(axis, row[w]).copy_(t.select(axis, row[p]))
    return new


def some_parents(G, W, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, W, (G, W), generator=g)
    p[0] = torch.arange(W).roll(1)                       # a ring
    if G > 1:
        p[1] = torch.arange(W)                           # nothing moves
    if G > 2:
        p[2] = W - 1 - torch.arange(W)                   # exchanges
    return p.to(torch.int32)


def run_reorder(tensors, index, parents, axis=0):
    want = [plain_reorder(t.cpu(), index, parents, axis) for t in tensors]
    ops().reorder_rows(tensors, index.to(DEV), parents.to(DEV), axis=axis)
    for t, w in zip(tensors, want):
        assert torch.equal(t.cpu().view(torch.uint8) if t.is_contiguous() else t.cpu(), w.view(torch.uint8)
                           if t.is_contiguous() else w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("W", [1, 2, 3, 4, 5, 8, 13, 16, 32])
@pytest.mark.parametrize("row", [1, 3, 8, 6000])
def test_reorder(dtype, W, row):
    G = 4
    g = torch.Generator().manual_seed(W + row)
    R = G * W + 5
    index = torch.randperm(R, generator=g)[:G * W].view(G, W).to(torch.int32)
    t = torch.randn(R, row, generator=g).to(dtype).to(DEV)
    t[0] = float("nan")                                  # bits are moved, whatever they mean
    run_reorder([t], index, some_parents(G, W, seed=row), 0)


@pytest.mark.parametrize("dtype,W,row", [(torch.float32, 4, 75004), (torch.float32, 3, 74001), (torch.bfloat16, 16, 4999),
                                         (torch.bfloat16, 4, 140002)])
def test_reorder_of_large_rows(dtype, W, row):
    """So many rows, and so large, that a block goes through several pieces of them."""
    g = torch.Generator().manual_seed(row)
    groups, outer = (64 if W == 16 else 16), 4
    t = torch.randn(outer, groups * W + 3, row, generator=g).to(dtype).to(DEV)
    index = torch.randperm(groups * W + 3, generator=g)[:groups * W].view(groups, W).to(torch.int32)
    run_reorder([t], index, some_parents(groups, W, row), axis=1)


def test_reorder_of_many_tensors_of_unlike_rows():
    g = torch.Generator().manual_seed(5)
    tensors = [torch.randn(9, 1 + 37 * i % 211, generator=g).to(torch.float32 if i % 3 else torch.bfloat16).to(DEV)
               for i in range(130)]
    tensors.append(torch.empty(9, 0, device=DEV))
    index = torch.tensor([[3, 1, 8, 6]], dtype=torch.int32)
    run_reorder(tensors, index, torch.tensor([[1, 2, 0, 0]], dtype=torch.int32), 0)


def test_reorder_inside_every_layer_and_plane():
    g = torch.Generator().manual_seed(6)
    t = torch.randn(3, 2, 11, 2, 4, 24, generator=g).to(torch.bfloat16).to(DEV)
    index = torch.tensor([[3, 1, 8], [10, 4, 2]], dtype=torch.int32)
    run_reorder([t], index, torch.tensor([[2, 2, 1], [1, 0, 2]], dtype=torch.int32), 2)


def test_reorder_of_strided_rows():
    wide = torch.randn(8, 50, device=DEV)
    keep = wide[:, 33:].clone()
    run_reorder([wide[:, :33]], torch.tensor([[7, 0, 5]], dtype=torch.int32), torch.tensor([[1, 2, 0]], dtype=torch.int32))
    assert torch.equal(wide[:, 33:], keep)


def test_rows_that_stay():
    """Parents and rows that name nothing leave what they belong to as it is."""
    t = torch.randn(6, 40, device=DEV)
    index = torch.tensor([[0, -1, 2, 6], [3, 4, 5, 1]], dtype=torch.int32)
    run_reorder([t], index, torch.tensor([[1, 0, 3, 0], [-1, 4, 0, 9]], dtype=torch.int32))


def test_reorder_beyond_31_bits_of_a_pool():
    """The last rows of a pool of more than 2^31 elements."""
    t = torch.empty(70000, 32768, dtype=torch.bfloat16, device=DEV)
    rows_ = [69999, 65536, 0]
    for i, r in enumerate(rows_):
        t[r] = i + 1.0
    ops().reorder_rows([t], torch.tensor([rows_], dtype=torch.int32, device=DEV),
                       torch.tensor([[1, 2, 0]], dtype=torch.int32, device=DEV))
    assert [float(t[r, 0]) for r in rows_] == [2.0, 3.0, 1.0] and [float(t[r, -1]) for r in rows_] == [2.0, 3.0, 1.0]


def test_reorder_refuses():
    o = ops()
    t = torch.randn(40, 8, device=DEV)

    def ints(*shape):
        return torch.zeros(shape, dtype=torch.int32, device=DEV)
    with pytest.raises(o.KernelError, match="33"):
        o.reorder_rows([t], ints(1, 33), ints(1, 33))
    with pytest.raises(AssertionError):
        o.reorder_rows([t], ints(1, 3), ints(1, 4))
    with pytest.raises(AssertionError):
        o.reorder_rows([t], ints(1, 3).long(), ints(1, 3))
    with pytest.raises(AssertionError):
        o.reorder_rows([t.t()], ints(1, 3), ints(1, 3))
    with pytest.raises(AssertionError):
        o.reorder_rows([t.to(torch.uint8)], ints(1, 3), ints(1, 3))
    with pytest.raises(o.KernelError, match="CUDA device"):
        o.reorder_rows([t.cpu()], ints(1, 3), ints(1, 3))
    o.reorder_rows([], ints(1, 3), ints(1, 3))
    o.reorder_rows([t], ints(0, 3), ints(0, 3))
