"""The low-rank product of every row's own adapter, alone: against the formula in 64 bits at widths, ranks,
strides and mixtures of adapters where it can go wrong."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF = torch.float32, torch.bfloat16


def ops():
    from tgo_b200.kernels import ops as o
    return o


@pytest.fixture(params=["chosen", "tiles"], autouse=True)
def way(request):
    """Every test goes the way that the framework chooses, and by tiles of 128 rows wherever they take its call."""
    ops().low_rank_force_way(2 if request.param == "tiles" else 0)
    yield request.param
    ops().low_rank_force_way(0)


def columns_of(widths, interleaved):
    if interleaved:
        return (torch.arange(sum(widths)) // 8) % 2
    return torch.repeat_interleave(torch.arange(len(widths)), torch.tensor(widths))


def plain(x, y, a, b, scale, ids, widths, interleaved):
    """(the formula in 64 bits, what a sum's terms come to in size), on the CPU."""
    x, y, a, b, scale = (t.double().cpu() for t in (x, y, a, b, scale))
    n, S, r, K = a.shape
    out, size = y.clone(), torch.zeros_like(y)
    col = columns_of(widths, interleaved)
    for i in range(n):
        rows = (ids.cpu() == i).nonzero().flatten()
        for s in range(S):
            at = (col == s).nonzero().flatten()
            u, m = x[rows] @ a[i, s].T, x[rows].abs() @ a[i, s].abs().T
            out[rows.unsqueeze(1), at] += scale[i] * (u @ b[i][at].T)
            size[rows.unsqueeze(1), at] = scale[i].abs() * (m @ b[i][at].abs().T)
    return out, size


def bound(out, size, K, r, x_type, y_type):
    """A sum of K products, times the scale, times b, summed over r: each of at most K + r + 8 roundings to
    24 bits is at most 2^-24 of what the terms come to in size; with bfloat16 rows u may be held in two
    bfloat16 parts, 2^-16 of it; the result is rounded once more, to its type."""
    e = (K + r + 8) * 2.0 ** -24 + (2.0 ** -16 if x_type == BF else 0.0)
    return size * e + out.abs() * (2.0 ** -8 if y_type == BF else 2.0 ** -23) + 1e-30


def inputs(T, K, widths, rank, adapters, x_type, y_type, seed, ids=None):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g)                 # noqa: E731
    N, S = sum(widths), len(widths)
    if ids is None:
        ids = torch.randint(-1, adapters, (T,), generator=g).to(torch.int32)
    return dict(x=normal(T, K).to(x_type).to(DEV), y=normal(T, N).to(y_type).to(DEV),
                a=(normal(adapters, S, rank, K) * K ** -0.5).to(x_type).to(DEV),
                b=(normal(adapters, N, rank) * 0.5 * rank ** -0.5).to(x_type).to(DEV),
                scale=(0.5 + torch.rand(adapters, generator=g)).to(DEV), ids=ids.to(DEV))


def check(p, widths, interleaved=False, in_place=False):
    x, y, a = p["x"], p["y"], p["a"]
    want, size = plain(x, y, a, p["b"], p["scale"], p["ids"], widths, interleaved)
    same = ((p["ids"] < 0) | (p["ids"] >= a.shape[0])).cpu()
    kept = y.clone()
    out = y if in_place else torch.full_like(y, float("nan"))
    ops().low_rank_add(x, y, a, p["b"], p["scale"], p["ids"], widths, interleaved, out=None if in_place else out)
    got = out.double().cpu()
    off = (got - want).abs()
    lim = bound(want, size, a.shape[3], a.shape[2], x.dtype, y.dtype)
    assert (off <= lim).all(), (float((off / lim).max()), (off > lim).nonzero()[:5].tolist())
    assert torch.equal(out[same.to(DEV)], kept[same.to(DEV)])       # rows without an adapter keep their bits
    if not in_place:
        assert torch.equal(y, kept)
    return out


TYPES = [(F32, F32), (BF, BF), (BF, F32)]


@pytest.mark.parametrize("x_type,y_type", TYPES)
@pytest.mark.parametrize("T,K,widths,rank,adapters", [
    (1, 2048, (2048,), 16, 4), (1, 64, (8,), 1, 1), (3, 100, (37,), 3, 2), (7, 257, (33, 5, 9), 5, 3),
    (17, 512, (256, 64, 64), 8, 5), (33, 520, (264, 72), 16, 40), (64, 1024, (1024,), 64, 9),
    (130, 2048, (512, 128, 128), 32, 3), (257, 1032, (200, 104, 56, 8), 24, 6), (40, 4096, (96,), 128, 3),
    (20, 384, (136, 40), 200, 2)])
def test_low_rank(x_type, y_type, T, K, widths, rank, adapters):
    check(inputs(T, K, widths, rank, adapters, x_type, y_type, seed=T + K), widths)


@pytest.mark.parametrize("x_type,y_type", TYPES)
@pytest.mark.parametrize("T,K,f,rank", [(1, 128, 8, 8), (5, 300, 40, 4), (70, 1024, 1536, 16), (200, 2048, 520, 64)])
def test_columns_in_eights(x_type, y_type, T, K, f, rank):
    check(inputs(T, K, (f, f), rank, 3, x_type, y_type, seed=f), (f, f), interleaved=True)


@pytest.mark.parametrize("y_type", [BF, F32])
@pytest.mark.parametrize("T,K,widths,rank,adapters,interleaved", [
    (300, 64, (64,), 8, 1, False), (301, 2048, (2048,), 16, 4, False), (513, 1032, (256, 64, 64), 24, 3, False),
    (1000, 512, (96, 32), 40, 7, False), (640, 4096, (512, 128, 128), 64, 2, False), (333, 768, (1056,), 128, 3, False),
    (700, 640, (512, 64, 32, 96), 128, 2, False), (310, 320, (64, 32, 96, 128), 72, 2, False), (400, 256, (512, 512), 16, 5, True), (777, 1000, (96, 96), 32, 3, True),
    (450, 512, (160, 160), 128, 2, True), (2500, 192, (64, 64), 8, 30, True)])
def test_many_rows(y_type, T, K, widths, rank, adapters, interleaved):
    """Mixed rows, and runs of unlike lengths as prompts of requests leave them."""
    p = inputs(T, K, widths, rank, adapters, BF, y_type, seed=T + rank)
    check(p, widths, interleaved)
    cuts = sorted(torch.randint(0, T, (5,), generator=torch.Generator().manual_seed(T)).tolist())
    runs = torch.zeros(T, dtype=torch.int32)
    for i, c in enumerate(cuts):
        runs[c:] = i % adapters if i % 3 else -1
    check({**p, "ids": runs.to(DEV)}, widths, interleaved)


@pytest.mark.parametrize("x_type,y_type", TYPES)
@pytest.mark.parametrize("T", [1, 6, 300])
def test_in_place(x_type, y_type, T):
    check(inputs(T, 768, (320, 64), 16, 4, x_type, y_type, seed=T), (320, 64), in_place=True)


@pytest.mark.parametrize("x_type,y_type", TYPES)
@pytest.mark.parametrize("T", [4, 150, 333])
def test_strided_rows(x_type, y_type, T):
    """x and y as columns of wider matrices, at an odd and at an even place."""
    for first in (1, 8):
        p = inputs(T, 640, (256,), 16, 3, x_type, y_type, seed=first)
        wide_x = torch.randn(T, 700, device=DEV).to(x_type)
        wide_y = torch.randn(T, 300, device=DEV).to(y_type)
        p["x"], p["y"] = wide_x[:, first:first + 640], wide_y[:, first:first + 256]
        beside = wide_y[:, first + 256:].clone()
        check(p, (256,), in_place=True)
        assert torch.equal(wide_y[:, first + 256:], beside)


@pytest.mark.parametrize("x_type", [F32, BF])
def test_rows_further_apart_than_31_bits(x_type):
    """Rows of x and y whose offsets pass 2^31 numbers."""
    T, apart = 300, 1 << 23
    p = inputs(T, 128, (64, 32), 16, 3, x_type, x_type, seed=9)
    for name in ("x", "y"):
        wide = torch.empty(T, apart, dtype=x_type, device=DEV)[:, :p[name].shape[1]]
        p[name] = wide.copy_(p[name])
    check(p, (64, 32), in_place=True)


@pytest.mark.parametrize("x_type", [F32, BF])
@pytest.mark.parametrize("T", [1, 40, 700])
def test_one_row_for_all(x_type, T):
    """x expanded from a single row."""
    p = inputs(T, 256, (128, 64), 16, 3, x_type, x_type, seed=T)
    p["x"] = p["x"][:1].expand(T, 256)
    check(p, (128, 64))


@pytest.mark.parametrize("x_type", [F32, BF])
@pytest.mark.parametrize("kind", ["none", "one", "all different", "runs", "outside"])
@pytest.mark.parametrize("T", [1, 9, 96, 700])
def test_mixtures_of_adapters(x_type, kind, T):
    n = 50 if kind == "all different" else 4
    ids = {"none": torch.full((T,), -1), "one": torch.full((T,), 2), "all different": torch.arange(T) % n,
           "runs": torch.arange(T) * 5 // max(T, 1) - 1, "outside": torch.tensor([n, -7, 1, 2 ** 31 - 1])[torch.arange(T) % 4]}
    check(inputs(T, 512, (256, 64, 64), 16, n, x_type, x_type, seed=T, ids=ids[kind].to(torch.int32)), (256, 64, 64))


def test_float32_rows_do_not_hang_on_their_batch():
    """Each row's bits are the same alone, in a short batch and in a long one."""
    widths = (256, 64, 64)
    p = inputs(300, 1000, widths, 12, 3, F32, F32, seed=4)
    whole = check(p, widths)
    for lo, hi in [(0, 1), (17, 18), (40, 49), (100, 229)]:
        part = torch.empty(hi - lo, 384, device=DEV)
        ops().low_rank_add(p["x"][lo:hi], p["y"][lo:hi], p["a"], p["b"], p["scale"], p["ids"][lo:hi].contiguous(),
                           widths, out=part)
        assert torch.equal(part, whole[lo:hi])


@pytest.mark.parametrize("x_type", [F32, BF])
def test_values_that_are_not_finite_stay_in_their_row(x_type):
    """A NaN or an infinity in a row of x, or in an adapter that no other row has, reaches that row alone."""
    for T in (6, 140, 500):
        p = inputs(T, 512, (256,), 16, 4, x_type, x_type, seed=T, ids=(torch.arange(T) % 3).to(torch.int32))
        out = check(p, (256,))
        p["x"][4, 100] = float("nan")
        p["x"][5, 7] = float("inf")
        p["b"][3] = float("nan")                 # an adapter that nobody uses
        bad = torch.empty_like(out)
        ops().low_rank_add(p["x"], p["y"], p["a"], p["b"], p["scale"], p["ids"], (256,), out=bad)
        rest = [t for t in range(T) if t not in (4, 5)]
        assert torch.equal(bad[rest], out[rest])
        assert torch.isnan(bad[4]).all() and not torch.isfinite(bad[5]).any()


@pytest.mark.parametrize("x_type", [F32, BF])
@pytest.mark.parametrize("T", [3, 140, 333])
def test_infinite_products(x_type, T):
    """An infinity in x gives infinities of B's signs, not NaN."""
    p = inputs(T, 64, (32,), 8, 1, x_type, x_type, seed=T, ids=torch.zeros(T, dtype=torch.int32))
    p["a"].fill_(1.0)
    p["x"][1] = 0.0
    p["x"][1, 7] = float("inf")
    out = torch.empty_like(p["y"])
    p["b"].copy_(p["b"].abs())
    p["b"][0, 3] *= -1.0
    ops().low_rank_add(p["x"], p["y"], p["a"], p["b"], p["scale"], p["ids"], (32,), out=out)
    want = torch.full((32,), float("inf"), device=DEV)
    want[3] = -float("inf")
    assert torch.equal(out[1].float(), want) and torch.isfinite(out[torch.arange(T) != 1]).all()


@pytest.mark.parametrize("x_type", [F32, BF])
@pytest.mark.parametrize("T", [255, 257, 511, 512, 513])
@pytest.mark.parametrize("adapters", [1, 255, 256])
def test_rows_found_and_planned(x_type, T, adapters):
    """Both sides of the numbers of rows and adapters up to which a call needs no plan."""
    ids = torch.randint(-2, adapters + 1, (T,), generator=torch.Generator().manual_seed(T + adapters)).to(torch.int32)
    check(inputs(T, 64, (32,), 8, adapters, x_type, x_type, seed=T, ids=ids), (32,))


@pytest.mark.parametrize("T,K,widths,rank", [(1210, 2048, (2048,), 64), (700, 1024, (1536, 512, 512), 72)])
def test_sizes_that_go_by_tiles(T, K, widths, rank):
    check(inputs(T, K, widths, rank, 3, BF, BF, seed=T), widths)


@pytest.mark.parametrize("T,widths,rank,interleaved", [
    (1, (64,), 16, False), (40, (96, 64), 32, False), (300, (64,), 8, False), (333, (128, 32), 16, False), (700, (256,), 64, False),
    (520, (96,), 128, False), (400, (64, 64), 16, True), (260, (160, 160), 64, True), (300, (64, 64), 128, True)])
def test_float32_rows_of_bfloat16_products(T, widths, rank, interleaved):
    """What is added to float32 rows is as exact as 32 bits make it: the errors of 64 + rank additions of random signs come to
    sqrt(64 + rank) 2^-24 of the sum, below 2^-20; two bfloat16 parts of u alone would be off by 2^-18."""
    p = inputs(T, 64, widths, rank, 3, BF, F32, seed=rank, ids=(torch.arange(T) // 50 % 3).to(torch.int32))
    p["y"].zero_()
    want, _ = plain(p["x"], p["y"], p["a"], p["b"], p["scale"], p["ids"], widths, interleaved)
    ops().low_rank_add(p["x"], p["y"], p["a"], p["b"], p["scale"], p["ids"], widths, interleaved)
    off = (p["y"].double().cpu() - want).norm() / want.norm()
    assert off < 2.0 ** -20, float(off) * 2 ** 20


def test_no_rows_and_other_streams():
    p = inputs(0, 64, (32,), 8, 2, BF, BF, seed=1)
    ops().low_rank_add(p["x"], p["y"], p["a"], p["b"], p["scale"], p["ids"], (32,))
    p = inputs(200, 512, (256,), 16, 4, BF, BF, seed=2)
    want = check(p, (256,))
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        out = torch.empty_like(want)
        ops().low_rank_add(p["x"], p["y"], p["a"], p["b"], p["scale"], p["ids"], (256,), out=out)
        assert torch.equal(out, want)


def test_refusals():
    o = ops()
    p = inputs(3, 64, (32, 16), 8, 2, BF, BF, seed=1)

    def call(widths=(32, 16), interleaved=False, **other):
        q = {**p, **other}
        o.low_rank_add(q["x"], q["y"], q["a"], q["b"], q["scale"], q["ids"], widths, interleaved)
    call()
    with pytest.raises(o.KernelError, match="48 columns"):
        call(widths=(32, 15))
    with pytest.raises(o.KernelError, match="eights"):
        call(interleaved=True)
    with pytest.raises(AssertionError):
        call(widths=(48,))
    for wrong in (dict(x=p["x"].float()), dict(ids=p["ids"].long()), dict(y=p["y"].to(torch.float16)),
                  dict(b=p["b"][:, :40]), dict(scale=p["scale"][:1]), dict(x=p["x"][:2])):
        with pytest.raises(AssertionError):
            call(**wrong)
    for widths in ((32, 16, 0), (64, -16)):
        with pytest.raises((o.KernelError, AssertionError)):
            call(widths=widths)
    with pytest.raises(AssertionError):
        call(y=torch.zeros(1, 48, dtype=BF, device=DEV).expand(3, 48))
    with pytest.raises(o.KernelError, match="CUDA device"):
        call(x=p["x"].cpu())
    with pytest.raises(o.KernelError):
        q = inputs(3, 64, (32,), 8, 2, torch.float16, torch.float16, seed=1)
        o.low_rank_add(q["x"], q["y"], q["a"], q["b"], q["scale"], q["ids"], (32,))
