"""Rotary frequencies and refusals that need no GPU."""

import ctypes
import math

import pytest

from graftrepository_b200 import _lib
from graftrepository_b200.rotary import Rotary, _RotaryC, rotary_frequencies
from test_paged_protocol import PLACE, answer, arena_c, plan_c


def test_frequencies():
    f, a = rotary_frequencies(8, 10000.0)
    assert f == pytest.approx([1.0, 0.1, 0.01, 0.001]) and a == 1.0
    f, a = rotary_frequencies(8, scaling=dict(kind="linear", factor=4.0))
    assert f == pytest.approx([0.25, 0.025, 0.0025, 0.00025]) and a == 1.0
    f, a = rotary_frequencies(8, scaling=dict(kind="ntk", factor=4.0))
    assert f[0] == 1.0 and f[3] == pytest.approx(0.001 / 4.0) and a == 1.0
    f, a = rotary_frequencies(4, scaling=dict(kind="factors", factors=[2.0, 5.0], amplitude=1.5))
    assert f == pytest.approx([0.5, 0.002]) and a == 1.5


def test_yarn():
    """Pairs that turn more than 32 times over the original context keep their
    frequency, those that turn less than once are divided, and it never rises."""
    dim, original, factor = 128, 4096, 16.0
    f, a = rotary_frequencies(dim, scaling=dict(kind="yarn", factor=factor, original=original))
    plain, _ = rotary_frequencies(dim)
    assert a == pytest.approx(0.1 * math.log(factor) + 1.0)
    for x, y in zip(f, plain):
        turns = y * original / (2 * math.pi)
        if turns > 32 * 10000.0 ** (2 / dim):  # a pair past the ramp's rounding
            assert x == y
        if turns < 10000.0 ** (-2 / dim):
            assert x == pytest.approx(y / factor)
        assert y / factor * (1 - 1e-12) <= x <= y
    assert f == sorted(f, reverse=True)
    assert rotary_frequencies(dim, scaling=dict(kind="yarn", factor=2.0, original=100,
                                                amplitude=1.0))[1] == 1.0


@pytest.mark.parametrize("dim,base,scaling", [
    (7, 1e4, None), (0, 1e4, None), (5000, 1e4, None), (8, 0.0, None), (8, math.inf, None),
    (8, 1e4, dict(kind="other")), (8, 1e4, dict(kind="linear")),
    (8, 1e4, dict(kind="linear", factor=0.0)), (8, 1e4, dict(kind="linear", factor=2.0, base=3)),
    (2, 1e4, dict(kind="ntk", factor=2.0)), (8, 1e4, dict(kind="factors", factors=[1.0] * 3)),
    (8, 1e4, dict(kind="factors", factors=[1.0, 1.0, 1.0, 0.0])),
    (8, 1e4, dict(kind="factors", factors=[1.0] * 4, amplitude=-1.0)),
    (8, 1e4, dict(kind="yarn", factor=2.0)), (8, 1e4, dict(kind="yarn", factor=2.0, original=0)),
    (8, 1e4, dict(kind="yarn", factor=2.0, original=9, beta_fast=1.0)),
    (8, 0.5, dict(kind="yarn", factor=2.0, original=9))])
def test_refused_frequencies(dim, base, scaling):
    with pytest.raises(ValueError):
        rotary_frequencies(dim, base, scaling)


def test_refused_rotaries():
    with pytest.raises(ValueError, match="layout"):
        Rotary(8, layout="other")
    with pytest.raises(ValueError, match="offset"):
        Rotary(8, offset=-1)
    with pytest.raises(ValueError, match="CUDA device"):
        Rotary(8, device="cpu")


def rotary_c(**change):
    return _RotaryC(**(dict(turns=PLACE, dim=32, offset=0, layout=0, amplitude=1.0) | change))


@pytest.mark.parametrize("change", [
    dict(turns=None), dict(dim=0), dict(dim=33), dict(dim=4098), dict(offset=-8), dict(layout=3),
    dict(layout=-1), dict(amplitude=0.0), dict(amplitude=math.nan), dict(amplitude=math.inf)])
def test_the_rotary_of_a_call(change):
    lib, r = _lib.load(), rotary_c(**change)
    answer(lib.grm_b200_rotate(ctypes.byref(r), PLACE, 0, 4, 2, 64, 128, 64, PLACE, 0, PLACE, 128,
                               64, None), "a rotary needs")
    plan, arena = plan_c(), arena_c()
    answer(lib.grm_b200_paged_append_rotary(ctypes.byref(plan), ctypes.byref(arena),
                                            ctypes.byref(r), PLACE, PLACE, _lib.GRM_B200_F16, 128,
                                            64, 128, 64, None), "a rotary needs")


def test_rotate_arguments():
    lib = _lib.load()
    good = [ctypes.byref(rotary_c()), PLACE, 0, 4, 2, 64, 128, 64, PLACE, 0, 2 * PLACE, 128, 64,
            None]
    for at, bad, text in ((0, None, "a rotary needs"), (1, None, "rows"), (2, 7, "rows"),
                          (3, -1, "rows"), (4, 0, "rows"), (4, 1 << 17, "rows"), (5, 16, "rows"),
                          (5, 1 << 17, "rows"), (6, -8, "rows"), (7, -8, "rows"), (8, None, "rows"),
                          (10, None, "rows"), (11, -8, "rows"), (12, -8, "rows"),
                          (1, PLACE + 2, "rows")):
        answer(lib.grm_b200_rotate(*(good[:at] + [bad] + good[at + 1:])), text)
    same = good[:10] + [PLACE, 256, 64, None]
    answer(lib.grm_b200_rotate(*same), "in place")
    swap = [ctypes.byref(rotary_c(layout=2))] + good[1:10] + [PLACE, 128, 64, None]
    answer(lib.grm_b200_rotate(*swap), "in place")
    assert lib.grm_b200_rotate(*(good[:3] + [0] + good[4:])) == 0  # no rows, nothing to do


@pytest.mark.parametrize("change", [dict(layout=2), dict(dim=24), dict(offset=8),
                                    dict(dim=64, offset=16), dict(dim=128)])
def test_append_arguments(change):
    lib, r, plan, arena = _lib.load(), rotary_c(**change), plan_c(), arena_c()
    rc = lib.grm_b200_paged_append_rotary(ctypes.byref(plan), ctypes.byref(arena), ctypes.byref(r),
                                          PLACE, PLACE, _lib.GRM_B200_F16, 128, 64, 128, 64, None)
    answer(rc, "rotates dims")
