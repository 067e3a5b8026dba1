"""Draws from rows of logits that a mask or a bias of -inf cut: whatever the rounding of the sums, a token without weight is
never drawn. Weights here are 1 (logit 0), next to nothing beside the sum before them, or none (-inf)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
INF = float("inf")
V, THREADS = 151936, 1024
RANGE = -(-V // THREADS)                     # ids that a thread sums, in order; the threads' sums come by 32


def draw(logits, draws, top_k=0, top_p=0.0, temperature=1.0, report=False):
    from tgo_b200.kernels import ops
    n = len(draws)
    rows = logits.expand(n, -1).contiguous()
    full = lambda v, t=torch.float32: torch.full((n,), v, dtype=t, device=DEV)         # noqa: E731
    out, lp = full(-7, torch.int32), full(7.0)
    more = (full(0, torch.int32), lp) if report else ()
    ops.sample(rows, full(temperature), full(top_k, torch.int32), full(top_p), torch.tensor(draws, dtype=torch.float32, device=DEV), out, *more)
    return (out.tolist(), lp.tolist()) if report else out.tolist()


def masked():
    return torch.full((V,), -INF, device=DEV)


def to_targets(targets, total):
    return [t / total for t in targets]


def test_a_range_whose_last_id_is_masked():
    """Thread 500's 148 weights of 0.0025 vanish one by one beside the 74500 before them (half a unit there is 0.0039), but not
    their sum: targets between the two fall through its whole range."""
    row, c0 = masked(), 500 * RANGE
    row[:c0] = 0
    row[c0:c0 + RANGE - 1] = -6
    u = to_targets([c0 + x for x in (0.05, 0.1, 0.2, 0.3, 0.34)], c0 + (RANGE - 1) * math.exp(-6))
    got, lp = draw(row, u, report=True)
    assert all(i == c0 + RANGE - 2 for i in got)
    want = -6 - math.log(c0 + (RANGE - 1) * math.exp(-6))
    assert all(abs(x - want) < 1e-4 for x in lp)


@pytest.mark.parametrize("behind", [False, True])
def test_a_range_without_weight(behind):
    """One weight of 0.0025 each for threads 480 to 510, none for 511, the last whose sum joins theirs: the sum of the 32 is
    more than they make one by one."""
    row, c0 = masked(), 480 * RANGE
    row[:c0] = 0
    last = [c0 + t * RANGE + 5 for t in range(31)]
    row[last] = -6
    total = c0 + 31 * math.exp(-6)
    if behind:
        row[600 * RANGE + 3] = 0
        total += 1
    got = draw(row, to_targets([c0 + x for x in (0.03, 0.04, 0.05, 0.06)], total))
    assert all(i == (600 * RANGE + 3 if behind else last[-1]) for i in got), got


def test_two_ranges_that_both_hold_the_target():
    """Weights of 0.0045 that round up to 0.0078 one by one, and do not in their sum: the first range of the two, always."""
    row, c0 = masked(), 480 * RANGE
    row[:c0] = 0
    ids = [c0 + t * RANGE + 5 for t in range(32)]
    row[ids] = math.log(0.0045)
    row[512 * RANGE] = 0
    total = c0 + 32 * 0.0045 + 1
    got = draw(row, to_targets([c0 + 0.2] * 64, total))
    # 2^-7 a step, 0.2 between two: the 26th is the first above (a draw's own rounding is 0.0045 here)
    assert len(set(got)) == 1 and got[0] in ids[24:28], got


@pytest.mark.parametrize("u", [0.99999994, 1.0, 0.5])
def test_fewer_tokens_with_weight_than_k(u):
    """Summed from the largest on 1 + 7e-8 + 7e-8 is two units above 1, in the order of the ids one: the last target is not
    reached, and what is kept behind has no weight."""
    row = masked()
    row[:2] = -16.5
    row[2] = 0
    for k in (3, 7, 128):
        got, lp = draw(row, [u], top_k=k, report=True)
        assert got == [2] and abs(lp[0]) < 1e-5
    assert draw(row, [u], top_p=0.999999) == [2]


@pytest.mark.parametrize("size", [5, 1000, 20003, V])
@pytest.mark.parametrize("share", [0.5, 0.002])
def test_masked_rows_at_any_draw(size, share):
    """Every draw gives a token that has weight, and one whose place in the running sum the draw falls on.

    Sums of 32 bits in runs of a thread's ids, 32 threads and 32 such sums: each addition is off by 2^-24 of the sum at most;
    a weight by the roundings of x / T - m (below 64 in size: 2^-24 of that, twice) and 4 units of the exponential."""
    g = torch.Generator(device=DEV).manual_seed(size)
    row = torch.randn(size, generator=g, device=DEV) * 3
    row[torch.rand(size, generator=g, device=DEV) > share] = -INF
    row[size // 2] = 1.0
    n = 300
    u = torch.rand(n, generator=g, device=DEV).tolist() + [0.0, 0.99999994]
    w = torch.exp((row / 0.7 - (row / 0.7).max()).double())
    upto = w.cumsum(0)
    off = float(upto[-1]) * 2.0 ** -24 * (-(-size // THREADS) + 64 + 1 + 2 * 64 + 4)
    got = torch.tensor(draw(row, u, temperature=0.7), device=DEV)
    assert bool((row[got] > -INF).all())
    target = torch.tensor(u, device=DEV).double() * upto[-1]
    assert bool((upto[got] >= target - 2 * off).all()) and bool((upto[got] - w[got] <= target + 2 * off).all())
    for kw in (dict(top_k=40), dict(top_p=0.9), dict(top_k=128, top_p=1.0)):
        assert bool((row[torch.tensor(draw(row, u, temperature=0.7, **kw), device=DEV)] > -INF).all())


def test_a_grammar_holds_whatever_is_drawn():
    """Through the sampler's own hook: rows with a mask, draws that fall between the sums."""
    import numpy as np

    from tgo_b200.sampling.policy import Policy
    from tgo_b200.sampling.sampler import sample_batch
    c0 = 500 * RANGE
    logits = torch.full((1, V), -20.0, device=DEV)
    logits[0, :c0] = 0
    logits[0, c0:c0 + RANGE - 1] = -6
    ok = [*range(c0 + RANGE - 1)]
    pol = Policy(temperature=1.0, allowed=lambda out: ok)
    mask = pol.allowed_words([], V)
    for x in np.linspace(0.02, 0.35, 12):
        u = float((c0 + x) / (c0 + (RANGE - 1) * math.exp(-6)))
        assert sample_batch(logits.clone(), [pol], [u], masks=[mask]).item() <= ok[-1]
