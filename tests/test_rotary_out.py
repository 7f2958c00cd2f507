"""Which results `Rotary.rotate` takes, and which it refuses because rows would be written on
others or read after they were written: what it says of two layouts of a buffer against the
values that they name, one by one (CPU only)."""

import itertools

import pytest

torch = pytest.importorskip("torch")

from graftrepository_b200.rotary import Rotary


def rotary(layout="half"):
    r = Rotary.__new__(Rotary)
    r.layout, r._index, r.device = layout, -1, "cpu"
    return r


BUFFER = torch.arange(4096, dtype=torch.float32)


def view(shape, strides, offset=0):
    return BUFFER.as_strided(shape, (*strides, 1), offset)


def answer(x, out):
    try:
        rotary()._check_out(x, out)
    except ValueError as e:
        return str(e)


SHAPES = [(1, 1, 8), (4, 1, 8), (1, 3, 8), (4, 2, 8), (3, 4, 8)]
STRIDES = [0, 4, 8, 12, 16, 24, 32, 48, 64, 96]


def test_rows_of_out_on_one_another():
    for shape, strides in itertools.product(SHAPES, itertools.product(STRIDES, STRIDES)):
        out = view(shape, strides)
        x = torch.zeros(shape)
        twice = out.reshape(-1).unique().numel() < out.numel()
        got = answer(x, out)
        if twice:
            assert got and "rows of out overlap" in got, (shape, strides)
        # what has its rows one after another in either dimension is taken
        a, b = sorted(s for s, n in zip(strides, shape) if n > 1)[-2:] if min(shape) > 1 else (0, 0)
        inner = shape[1] if strides[1] < strides[0] else shape[0]
        if not twice and (min(shape) == 1 or b >= (inner - 1) * a + 8):
            assert got is None, (shape, strides, got)


@pytest.mark.parametrize("shape,strides", [((4, 2, 64), (64, 64)), ((2, 8, 128), (128, 128)),
                                           ((5, 3, 8), (16, 8)), ((5, 3, 8), (8, 32))])
def test_two_strides_that_each_hold_a_head(shape, strides):
    x = view(shape, strides)
    for out in (x, view(shape, strides, 2048)):
        assert "rows of out overlap" in answer(x, out)
    assert answer(torch.zeros(shape), torch.zeros(shape)) is None
