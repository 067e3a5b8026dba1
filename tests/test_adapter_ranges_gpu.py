"""The low-rank product of every row's own adapter at the ends of its ranges: numbers that round to
infinity. Statement and bounds of test_adapters_gpu.py, each test by the ways it names."""
import pytest
import torch

from test_adapters_gpu import DEV, TYPES, check, inputs, ops

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
