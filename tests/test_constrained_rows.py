"""What policies ask of rows of logits, handed to the kernel as one batch; no GPU."""
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
