"""Rows of logits between other rows, single rows and very many of them, on the device."""
import pytest
import torch

from test_tree_ops_gpu import constrained, ops, plain_constrain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def close(got, want, x):
    """The roundings that `check_constrain` counts."""
    size = x.abs().double() * 2 + 4 * 6 + 50
    gone = want == -float("inf")
    assert torch.equal(got == -float("inf"), gone)
    assert bool(((got.double() - want).abs()[~gone] <= 5 * 2.0 ** -24 * size[~gone]).all())


@pytest.mark.parametrize("first,second", [(0, 150), (150, 0), (0, 100), (200, 99), (3, 103), (0, 200), (1, 200)])
def test_rows_between_each_other(first, second):
    """Two matrices whose rows alternate in one buffer."""
    x, c = constrained(4, 99, 4, seed=1, bias=2, history=5, allowed=2)
    wide = torch.full((4, 300), 7.0, device=DEV)
    src, dst = wide[:, first:first + 99], wide[:, second:second + 99]
    src.copy_(x)
    ops().logits_constrain(src, out=dst, **c)
    close(dst, plain_constrain(x, **c).to(DEV), x)
    assert torch.equal(src, x)
    left = torch.ones(300, dtype=torch.bool, device=DEV)
    left[first:first + 99] = left[second:second + 99] = False
    assert bool((wide[:, left] == 7).all())


def test_rows_over_each_other_are_refused():
    wide = torch.zeros((4, 300), device=DEV)
    flat = wide.view(-1)
    for src, dst in [(wide[:, :99], wide[:, 98:197]), (wide[:, 98:197], wide[:, :99]), (wide[:3, :99], flat.as_strided((3, 99), (300, 1), 202)),
                     (wide[:, 5:104], wide[:, 4:103]), (wide[:3, :99], wide[1:, :99]),
                     (flat.as_strided((4, 99), (200, 1), 0), wide[:, :99]), (wide[:1, :99], wide[:1, 50:149])]:
        with pytest.raises(ops().KernelError, match="over other rows"):
            ops().logits_constrain(src, out=dst)


def test_one_row_has_no_stride():
    """A row in place through two views of unlike strides."""
    x, c = constrained(1, 60, 1, seed=2, bias=4, history=9)
    flat = torch.zeros(400, device=DEV)
    a, b = flat.as_strided((1, 60), (100, 1), 3), flat.as_strided((1, 60), (7, 1), 3)
    a.copy_(x)
    ops().logits_constrain(a, out=b, **c)
    close(a, plain_constrain(x, **c).to(DEV), x)


@pytest.mark.parametrize("form", ["in place", "apart", "apart, at another boundary", "masked", "no owners"])
def test_more_rows_than_a_grids_second_extent(form):
    R, V = 65535 + 700, 37
    many = lambda t: t.repeat(-(-R // 300), *[1] * (t.dim() - 1))[:R].contiguous()       # noqa: E731
    x, c = constrained(300, V, 300 if form == "no owners" else 5, seed=3, owner=form != "no owners", bias=3,
                       history=4 if form == "no owners" else 30, allowed=4 if form == "masked" else 0)
    rows = many(x)
    for name in ("owner", "allowed_rows"):
        if c[name] is not None:
            c[name] = many(c[name])
    if form == "no owners":                                    # as many requests as rows
        c["penalties"] = many(c["penalties"])
        for name in ("bias", "history"):
            first, *lists = c[name]
            ends = many(first.diff()).cumsum(0).to(torch.int32)
            c[name] = (torch.cat([first[:1], ends]), *[t.repeat(-(-R // 300)).contiguous() for t in lists])
    small = slice(R - 300, R)
    want = rows[small].clone()
    part = dict(c, owner=torch.arange(R - 300, R, dtype=torch.int32, device=DEV) if c["owner"] is None else c["owner"][small].contiguous(),
                allowed_rows=None if c["allowed_rows"] is None else c["allowed_rows"][small].contiguous())
    ops().logits_constrain(want, **part)
    out = None
    if form.startswith("apart"):
        shift = 1 if "another" in form else 0
        out = torch.full((R * V + 4,), 5.0, device=DEV)[shift:shift + R * V].view(R, V)
    start = rows.clone()
    n = ops().LAUNCHES[0]
    ops().logits_constrain(rows, out=out, **c)
    got = rows if out is None else out
    assert torch.equal(got[small], want)
    first = slice(0, 300)
    head = start[first].clone()
    ops().logits_constrain(head, **dict(c, owner=torch.arange(300, dtype=torch.int32, device=DEV) if c["owner"] is None else c["owner"][first].contiguous(),
                                        allowed_rows=None if c["allowed_rows"] is None else c["allowed_rows"][first].contiguous()))
    assert torch.equal(got[first], head)
    # (each of the other two counted one)
    assert ops().LAUNCHES[0] - n == 1 + (2 if form in ("in place", "no owners", "apart, at another boundary") else 1)
