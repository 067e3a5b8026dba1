"""What policies ask of rows of logits, handed to the kernel as one batch; no GPU."""
import random

import pytest
import torch

from test_beam_search import cpu_model, tiny_model
from test_drafting import emulated                                # noqa: F401  (a fixture)
from tgo_b200.sampling.policy import Policy
from tgo_b200.sampling.sampler import constrain


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 40, 2 ** 70])
def test_windows_of_any_size(emulated, tmp_path, window):        # noqa: F811
    """A window longer than any history is the whole history."""
    d, cfg, run = tiny_model(tmp_path, "A")
    model = cpu_model(d, cfg)
    whole, wide = (Policy(max_tokens=8, repetition_penalty=1.5, frequency_penalty=0.4, penalty_window=w) for w in (0, window))
    wide.check(cfg["vocab_size"])
    assert model.generate([[1, 2, 3]], wide, page_size=8) == model.generate([[1, 2, 3]], whole, page_size=8)
    x = torch.randn(2, 50)
    y = x.clone()
    constrain(x, [wide, Policy()], [[3, 4, 3], ()])
    constrain(y, [whole, Policy()], [[3, 4, 3], ()])
    assert torch.equal(x, y)


def test_rows_that_lie_over_each_other():
    """By counting the numbers that two matrices have in common."""
    from tgo_b200.kernels.ops import _over_each_other
    rng = random.Random(0)
    seen = set()
    for _ in range(4000):
        rows, columns = rng.randint(1, 4), rng.randint(1, 6)
        stride = rng.randint(columns, 3 * columns)
        other = stride if rng.random() < 0.8 else rng.randint(columns, 3 * columns)
        a, b = rng.randint(0, 30), rng.randint(0, 30)
        mine = {a + r * stride + i for r in range(rows) for i in range(columns)}
        common = mine & {b + r * other + i for r in range(rows) for i in range(columns)}
        got = _over_each_other(rows, columns, 1024 + 4 * a, stride, 1024 + 4 * b, other)
        if a == b:
            assert got == (rows > 1 and stride != other)       # the same rows
        elif stride == other or rows == 1:
            assert got == bool(common)
        else:
            assert got or not common                           # where strides differ, ranges apart
        seen.add((got, bool(common)))
    assert len(seen) >= 3
