"""What wrappers ask of their tensors: the extension and the plain Python form say the same, and a refusal says why."""
import pytest
import torch

from tgo_b200.kernels import build, ops


def samples(device):
    t = torch.arange(24, dtype=torch.int32, device=device)
    return [t, t[3:], t[:0], t[::2], t.view(4, 6), t.view(4, 6)[:, 1:4], t.view(4, 6).t(), t.long(), t.float(), t.bfloat16(), t.half(),
            t.float().view(2, 3, 4), torch.zeros((0, 5), device=device), torch.zeros((), device=device),
            torch.zeros((2, 3, 4, 5, 6), device=device), torch.zeros((2, 0, 4, 5, 6), device=device).half(), t.view(2, 3, 4).transpose(1, 2)]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_both_forms_agree(device):
    reader = build.tensor_reader()
    if reader is None:
        pytest.skip("no extension here")
    for t in samples(device):
        for kind in "ilfb":
            got = reader.look(kind, t)
            assert got == ops._look_plain(kind, t)
            assert (got is not None) == (t.is_cuda and t.dtype is ops._KINDS[kind] and t.is_contiguous())
        assert reader.rows(t) == ops._rows_plain(t)
        for axis in range(-1, 4):
            assert reader.pages(t, axis) == ops._pages_plain(t, axis)
    a, b = torch.zeros(3, dtype=torch.int32, device=device), torch.zeros(2, device=device)
    for kinds, tensors in (("if", (a, b)), ("iff", (a, None, b)), ("fi", (a, b)), ("", ()), ("l", (None,))):
        assert reader.look(kinds, *tensors) == ops._look_plain(kinds, *tensors)
    assert reader.look("lf", None, None) == [0, 0, 0, 0]


def test_calls_that_are_wrong():
    reader = build.tensor_reader()
    if reader is None:
        pytest.skip("no extension here")
    for args in ((), ("i",), ("ii", None), (3, None), ("", None)):
        with pytest.raises(TypeError):
            reader.look(*args)
    for args in ((), (None,), (None, "x")):
        with pytest.raises(TypeError):
            reader.pages(*args)
    assert reader.pages(None, 0) is None
    assert reader.look("i", [1, 2]) is None and reader.look("i", 7) is None and reader.rows("x") is None


def test_without_the_extension(monkeypatch):
    first = ops._look, ops._rows, ops._pages
    monkeypatch.setattr(ops, "tensor_reader", lambda: None)
    try:
        ops._find_reader()
        assert (ops._look, ops._rows, ops._pages) == (ops._look_plain, ops._rows_plain, ops._pages_plain)
    finally:
        ops._look, ops._rows, ops._pages = first


def test_an_extension_that_does_not_build(monkeypatch, capfd):
    def fails(name, **kw):
        raise build.KernelBuildError(f"the compiler failed on {name}")
    monkeypatch.setattr(build, "compile_library", fails)
    assert build.tensor_reader() is None and "read from Python" in capfd.readouterr().err


def test_a_refusal_says_why():
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="cpu"):
        ops._refuse("i", i)


@pytest.mark.gpu
def test_a_refusal_names_the_type_and_the_layout():
    i = torch.zeros(4, dtype=torch.int32, device="cuda:0")
    with pytest.raises(AssertionError, match="int32 for one of torch.int64"):
        ops._refuse("il", i, i)
    with pytest.raises(AssertionError, match="contiguous"):
        ops._refuse("ii", i, i[::2])
    with pytest.raises(AssertionError, match="no matrix"):
        ops._refuse("i", i)
