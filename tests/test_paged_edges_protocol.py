"""Refusals of the 8-bit paged arena's commit that need no GPU (CPU only)."""

import ctypes

import pytest

from graftrepository_b200 import _lib
from test_paged_protocol import EINVAL, PLACE, answer, plan_c


@pytest.mark.parametrize("change,lens,cursor", [
    (dict(grow=0), PLACE, 3 * PLACE), ({}, 20 * PLACE, 3 * PLACE), ({}, PLACE, 20 * PLACE),
    ({}, None, 3 * PLACE), ({}, PLACE, None)])
def test_commit_takes_the_plan_s_own_lengths(change, lens, cursor):
    plan = plan_c(**change)
    rc = _lib.load().grm_b200_paged_commit(ctypes.byref(plan), lens, cursor, None)
    answer(rc, "paged commit")


def test_commit_checks_the_plan():
    answer(_lib.load().grm_b200_paged_commit(None, PLACE, PLACE, None), "null plan")
    plan = plan_c(status=None)
    assert _lib.load().grm_b200_paged_commit(ctypes.byref(plan), PLACE, 3 * PLACE, None) == EINVAL
