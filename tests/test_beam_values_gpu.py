"""The selection over beams and vocabulary where the logits' values could lose it: masks of large finite numbers, rows far
from zero. Against the statement in 64 bits and with the bound of test_beams_gpu.py, by both ways."""
import pytest
import torch

from test_beams_gpu import DEV, check, ops, rows, so_far

pytestmark = pytest.mark.gpu


def both_ways(logits, scores, K):
    try:
        for way in (1, 2):
            ops().beam_force_way(way)
            check(logits, scores, K)
    finally:
        ops().beam_force_way(0)


@pytest.mark.parametrize("V", [4099, 40001])
@pytest.mark.parametrize("mask", [-1e4, -1e8, -1e9, -1e10, -1e12, -1e18, -1e20, -1e30, -1e36])
def test_tokens_masked_by_a_finite_number(V, mask):
    """A mask is a value like any other: its tokens weigh nothing beside others, and count where there are no others."""
    g = torch.Generator().manual_seed(V)
    x = rows(20, V, seed=V + 1)
    for i, share in enumerate([0.3, 0.9, 0.99]):
        x[i:16:8][torch.rand(2, V, generator=g).to(DEV) < share] = mask      # rows 0, 1, 2 and 8, 9, 10
    x[3], x[11] = mask, mask                    # a beam without another token
    for i in (12, 13, 14, 15):                  # so few others that masked ones are picked too
        x[i] = mask
        x[i, [7 * i, V - i]] = torch.tensor([1.0, 2.5], device=DEV)
    x[16:20] = mask                             # beams without another token alone
    both_ways(x, so_far(5, 4, seed=V), 12)


@pytest.mark.parametrize("offset", [-1e6, -3e4, -1e4, 1e4, 3e4, 1e6])
def test_rows_with_an_offset(offset):
    """Logits far from zero, whose differences are ordinary ones."""
    both_ways(rows(8, 20011, seed=5) + offset, so_far(2, 4, seed=5), 8)
