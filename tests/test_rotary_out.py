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


def test_results_over_rows():
    """Against the values that both name: what shares one is refused, and what shares none
    taken, where both lie the same way."""
    for shape, strides in itertools.product(SHAPES, itertools.product(STRIDES, STRIDES)):
        x = view(shape, strides, 512)
        if answer(torch.zeros(shape), x) is not None:
            continue
        names = set(x.reshape(-1).tolist())
        for offset in range(1, 1024, 7):
            out = view(shape, strides, offset)
            got = answer(x, out)
            if out.data_ptr() == x.data_ptr():
                assert got is None
            elif names.intersection(out.reshape(-1).tolist()):
                assert got == "out overlaps x", (shape, strides, offset)
            else:
                assert got is None, (shape, strides, offset, got)


def test_heads_before_tokens_side_by_side():
    both = torch.zeros((6, 2, 10, 32))  # heads, kind, tokens, values
    x, out = both[:, 0].transpose(0, 1), both[:, 1].transpose(0, 1)
    assert answer(x, out) is None and answer(out, x) is None
    assert answer(x, both[:, 0].transpose(0, 1)) is None  # in place


def test_one_token_or_head_lies_any_way():
    x = view((1, 4, 8), (96, 16))
    assert answer(x, view((1, 4, 8), (640, 16), 8)) is None
    assert answer(x, view((1, 4, 8), (640, 16), 4)) == "out overlaps x"


def test_the_same_memory_by_another_tensor():
    """A tensor that shares memory without sharing torch's storage."""
    import ctypes

    raw = (ctypes.c_float * 256)()
    x = torch.frombuffer(raw, dtype=torch.float32).view(4, 2, 32)
    other = torch.frombuffer(raw, dtype=torch.float32, count=192, offset=64).view(3, 2, 32)
    assert x.untyped_storage().data_ptr() != other.untyped_storage().data_ptr()
    assert answer(x[:3], other) == "out overlaps x"
    assert answer(x[:1], other[1:2]) is None
