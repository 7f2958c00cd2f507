"""Refusals of the 8-bit paged arena that need no GPU: commit's, and plans and arenas
of different devices (CPU only)."""

import ctypes

import pytest

from graftrepository_b200 import _lib
from graftrepository_b200 import paged_arena as PA
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


def test_a_plan_of_another_device():
    """Nothing is launched: the arena has no buffers here, the plan no tables."""
    torch = pytest.importorskip("torch")
    arena, plan = PA.PagedArena.__new__(PA.PagedArena), PA.PagePlan.__new__(PA.PagePlan)
    arena.layers, arena._index, arena.device = 1, 0, torch.device("cuda", 0)
    plan.planned, plan.grow, plan._turn = True, True, None
    plan._index, plan.device = 1, torch.device("cuda", 1)
    plan.kv_shape = plan.query_shape = torch.Size((2, 1, 64))
    rows = torch.zeros((2, 1, 64), dtype=torch.float16)
    for call in (lambda: arena.append(plan, rows, rows), lambda: arena.attend(plan, rows)):
        with pytest.raises(ValueError, match="plan is on cuda:1, the arena on cuda:0"):
            call()
