"""The low-rank product of every row's own adapter at the ends of its ranges: numbers that round to infinity, more rows than a
plan or a grid holds, the widest product. Statement and bounds of test_adapters_gpu.py, each test by the ways it names."""
import pytest
import torch

from test_adapters_gpu import BF, DEV, F32, TYPES, bound, check, inputs, ops, plain

pytestmark = pytest.mark.gpu

CHOSEN, CLUSTERS, TILES = 0, 1, 2


@pytest.fixture()
def by():
    yield ops().low_rank_force_way
    ops().low_rank_force_way(CHOSEN)


@pytest.mark.parametrize("x_type,y_type", TYPES)
@pytest.mark.parametrize("way", [CLUSTERS, TILES])
def test_products_near_the_end_of_the_range(by, way, x_type, y_type):
    """x A^T above the largest bfloat16 number, which would round to infinity, and still a 32-bit number."""
    by(way)
    for T, K in ((3, 64), (333, 64), (5, 60)):              # 60: the general kernels
        p = inputs(T, K, (32,), 8, 1, x_type, y_type, seed=T, ids=torch.zeros(T, dtype=torch.int32))
        p["scale"].fill_(1.0)
        p["a"].zero_()
        p["a"][0, 0, :, :2] = 2.0 ** 64
        p["x"][1, :2] = torch.tensor([1.9921875 * 2.0 ** 63, 1.5 * 2.0 ** 55], device=DEV)      # u = 1.998046875 x 2^127
        p["x"][2, :2] = -p["x"][1, :2]
        p["b"].mul_(2.0 ** -100)
        check(p, (32,))


@pytest.mark.parametrize("way", [CHOSEN, TILES])
def test_more_rows_than_a_grid_has_tiles(by, way):
    """8.4 million rows, 65536 tiles of 128: more than a launch's second extent takes."""
    by(way)
    T, g = 65536 * 128, torch.Generator(device=DEV).manual_seed(6)
    p = inputs(1, 32, (32,), 8, 2, BF, BF, seed=6)
    p["x"], p["y"] = (torch.randn(T, 32, generator=g, device=DEV, dtype=BF) for _ in range(2))
    p["ids"] = (torch.arange(T, device=DEV) // 4999 % 3 - 1).to(torch.int32)
    out = torch.empty_like(p["y"])
    ops().low_rank_add(p["x"], p["y"], p["a"], p["b"], p["scale"], p["ids"], (32,), out=out)
    at = torch.cat([torch.arange(0, T, 4001), torch.arange(T - 300, T)]).to(DEV)
    x, y, ids = p["x"][at], p["y"][at], p["ids"][at]
    want, size = plain(x, y, p["a"], p["b"], p["scale"], ids, (32,), False)
    off = (out[at].double().cpu() - want).abs()
    assert (off <= bound(want, size, 32, 8, BF, BF)).all()


@pytest.mark.parametrize("T,adapters", [(8192, 3), (8193, 255), (20001, 3), (20001, 255), (20001, 300)])
@pytest.mark.parametrize("way,x_type", [(CLUSTERS, F32), (CLUSTERS, BF), (TILES, BF)])
def test_more_rows_than_the_plan_holds(by, way, x_type, T, adapters):
    """From 8193 rows on the plan reads some of their adapters a second time; from 256 adapters on it counts another way.
    Rows in any order, then in runs of one adapter."""
    by(way)
    ids = torch.randint(-1, adapters, (T,), generator=torch.Generator().manual_seed(T + adapters))
    p = inputs(T, 32, (32,), 8, adapters, x_type, x_type, seed=T, ids=ids.to(torch.int32))
    check(p, (32,))
    check({**p, "ids": ids.sort().values.roll(77).to(torch.int32).to(DEV)}, (32,))


@pytest.mark.parametrize("T", [1, 96, 1100])
@pytest.mark.parametrize("way,rank", [(CLUSTERS, 4), (CLUSTERS, 16), (TILES, 16)])
def test_the_widest_product(by, way, rank, T):
    """A feed-forward's last product, 12288 wide, into the float32 stream: one token, a batch of tokens, a prompt."""
    by(way)
    check(inputs(T, 12288, (256,), rank, 3, BF, F32, seed=T + rank), (256,), in_place=True)


@pytest.mark.parametrize("T,K,counts", [(1, 64, (1, 1, 3)), (300, 64, (1, 1, 3)), (600, 64, (2, 2, 3)), (1024, 64, (3, 2, 3)),
                                        (20, 60, (2, 2, 2)), (600, 60, (2, 2, 2))])
def test_launches_are_counted(by, T, K, counts):
    """One kernel where the clusters find their rows, two with a plan or by the general kernels, three by tiles."""
    o = ops()
    p = inputs(T, K, (32,), 8, 2, BF, BF, seed=T)
    for way in (CHOSEN, CLUSTERS, TILES):
        by(way)
        before = o.LAUNCHES[0]
        o.low_rank_add(p["x"], p["y"], p["a"], p["b"], p["scale"], p["ids"], (32,))
        assert o.LAUNCHES[0] - before == counts[way]


def test_rows_that_need_no_workspace():
    """The number of rows up to which a call is tried without a workspace is the library's own."""
    assert ops().LOW_RANK_SCANNED == ops().entry_points("adapters").tgo_low_rank_scanned_rows()
