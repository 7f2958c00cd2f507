"""Refusals of the 8-bit paged arena that need no GPU: what the C entries answer
to missing buffers, sizes out of range and descriptions that do not match, and
what the Python layer raises before it touches a device (CPU only)."""

import ctypes

import pytest

from graftrepository_b200 import _lib
from graftrepository_b200 import paged_arena as PA

EINVAL = -1
PLACE = 1 << 20  # stands for a 256-byte aligned device address; nothing reads it


def plan_c(**change):
    sizes = dict(requests=2, tokens=4, max_fresh=4, table_width=4, pages=8, page_tokens=16,
                 kv_heads=2, query_heads=4, head_dim=64, grow=1)
    buffers = ("cached ring cursor_in table lens starts positions rows slots cursor status "
               "scratch").split()
    fields = sizes | {name: PLACE * (i + 1) for i, name in enumerate(buffers)}
    fields["scratch_bytes"] = 1 << 30
    return PA._PlanC(**(fields | change))


def arena_c(**change):
    fields = dict(k_codes=PLACE, v_codes=2 * PLACE, k_scales=3 * PLACE, v_scales=4 * PLACE,
                  pages=8, kv_heads=2, page_tokens=16, head_dim=64)
    return PA._ArenaC(**(fields | change))


def answer(rc, text):
    assert rc == EINVAL
    assert text in _lib.thread_error(), _lib.thread_error()


@pytest.mark.parametrize("change,text", [
    (dict(requests=0), "sizes"), (dict(requests=(1 << 20) + 1), "sizes"), (dict(tokens=0), "sizes"),
    (dict(tokens=1 << 31), "sizes"), (dict(max_fresh=0), "sizes"), (dict(table_width=0), "sizes"),
    (dict(table_width=(1 << 28) + 1), "sizes"), (dict(pages=0), "sizes"),
    (dict(pages=1 << 31), "sizes"), (dict(page_tokens=48), "page_tokens"),
    (dict(head_dim=96), "head_dim"), (dict(kv_heads=0), "query_heads"),
    (dict(kv_heads=1025, query_heads=1025), "query_heads"), (dict(query_heads=5), "query_heads"),
    (dict(query_heads=1), "query_heads"), (dict(query_heads=258), "query_heads")])
def test_plan_sizes(change, text):
    lib, need = _lib.load(), ctypes.c_int64(0)
    plan = plan_c(**change)
    answer(lib.grm_b200_paged_scratch_bytes(ctypes.byref(plan), ctypes.byref(need)), text)
    answer(lib.grm_b200_paged_plan_step(ctypes.byref(plan), PLACE, None), text)


def test_plan_buffers():
    lib = _lib.load()
    answer(lib.grm_b200_paged_scratch_bytes(None, None), "null plan")
    plan = plan_c()
    answer(lib.grm_b200_paged_scratch_bytes(ctypes.byref(plan), None), "null out_bytes")
    for name in ("cached", "ring", "cursor_in", "table", "lens", "starts", "positions", "rows",
                 "slots", "cursor", "status", "scratch"):
        plan = plan_c(**{name: None})
        answer(lib.grm_b200_paged_plan_step(ctypes.byref(plan), PLACE, None), "missing")
    for change in (dict(cursor=3 * PLACE), dict(lens=PLACE)):
        plan = plan_c(**change)
        answer(lib.grm_b200_paged_plan_step(ctypes.byref(plan), PLACE, None), "made from")
    plan = plan_c(scratch=12 * PLACE + 128)
    answer(lib.grm_b200_paged_plan_step(ctypes.byref(plan), PLACE, None), "aligned")


@pytest.mark.parametrize("change,text", [
    (dict(k_codes=None), "missing"), (dict(v_codes=None), "missing"),
    (dict(k_scales=None), "missing"), (dict(v_scales=None), "missing"), (dict(pages=0), "pages"),
    (dict(pages=1 << 30), "pages"), (dict(kv_heads=0), "kv_heads"),
    (dict(page_tokens=8), "page_tokens"), (dict(head_dim=32), "head_dim"),
    (dict(k_codes=PLACE + 8), "aligned"), (dict(v_codes=PLACE + 4), "aligned")])
def test_arena(change, text):
    arena = arena_c(**change)
    answer(_lib.load().grm_b200_paged_read(ctypes.byref(arena), PLACE, 4, _lib.GRM_B200_F32, PLACE,
                                           PLACE, None), text)


def test_read():
    lib, arena = _lib.load(), arena_c()
    ref = ctypes.byref(arena)
    for slots, count, k, v in ((None, 4, PLACE, PLACE), (PLACE, -1, PLACE, PLACE),
                               (PLACE, 4, None, PLACE), (PLACE, 4, PLACE, None),
                               (PLACE, 4, PLACE + 4, PLACE), (PLACE, 1 << 62, PLACE, PLACE)):
        answer(lib.grm_b200_paged_read(ref, slots, count, _lib.GRM_B200_F32, k, v, None), "read")
    answer(lib.grm_b200_paged_read(ref, PLACE, 4, 77, PLACE, PLACE, None), "element type")
    assert lib.grm_b200_paged_read(ref, None, 0, _lib.GRM_B200_F32, None, None, None) == 0


def test_release():
    lib = _lib.load()
    good = [PLACE, 2, 2, 4, 8, 16, PLACE, PLACE, PLACE, PLACE, None]
    for i, bad in ((0, None), (1, -1), (2, 0), (3, 0), (4, 0), (5, 24), (6, None), (7, None),
                   (8, None), (9, None)):
        args = good[:i] + [bad] + good[i + 1:]
        assert lib.grm_b200_paged_release(*args) == EINVAL, i
        assert "release" in _lib.thread_error()


def test_python_layer():
    for args in ((0, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError, match="positive"):
            PA.PageTables(*args)
    with pytest.raises(ValueError, match="page_tokens"):
        PA.PageTables(1, 1, 1, page_tokens=24)
    with pytest.raises(ValueError, match="CUDA device"):
        PA.PageTables(1, 1, 1, device="cpu")
    for args in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64)):
        with pytest.raises(ValueError, match="positive"):
            PA.PagedArena(*args)
    with pytest.raises(ValueError, match="head_dim"):
        PA.PagedArena(1, 1, 1, 80)
    with pytest.raises(ValueError, match="CUDA device"):
        PA.PagedArena(1, 1, 1, 64, device="cpu")
