"""Refusals of the pages of latent rows that need no GPU: what the C entries answer
and what the Python layer raises before it touches a device (CPU only)."""

import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

from graftrepository_b200 import _lib
from graftrepository_b200 import latent_arena as LA
from graftrepository_b200 import paged_arena as PA
from test_paged_protocol import PLACE, answer, plan_c
from test_rotary import rotary_c


def latent_plan(step=None, **change):
    sizes = dict(heads=4, latent=256, rope=32, nope=64, value=64, expand_tokens=128, work=PLACE,
                 work_bytes=1 << 40)
    one = dict(kv_heads=1, query_heads=1) | (step or {})
    return LA._LatentPlanC(step=plan_c(**one), **(sizes | change))


def latent_arena(**change):
    fields = dict(rows=PLACE, pages=8, page_tokens=16, latent=256, rope=32,
                  dtype=_lib.GRM_B200_BF16)
    return LA._LatentArenaC(**(fields | change))


def append(plan, arena, rotary=None, c=PLACE, c_row=288, r=PLACE, r_row=288):
    ref = [None if x is None else ctypes.byref(x) for x in (plan, arena, rotary)]
    return _lib.load().grm_b200_latent_append(*ref, c, c_row, r, r_row, None)


def attend(plan, arena, q=PLACE, strides=(1024, 256), r=PLACE, r_strides=(128, 32), scale=0.1,
           causal=1, out=PLACE):
    ref = [None if x is None else ctypes.byref(x) for x in (plan, arena)]
    return _lib.load().grm_b200_latent_attend(*ref, q, *strides, r, *r_strides, scale, causal, out,
                                              None, None)


def expanded(plan, arena, q=PLACE, strides=(384, 96), w=PLACE, w_strides=(1 << 15, 256),
             scale=0.1, causal=1, out=PLACE):
    ref = [None if x is None else ctypes.byref(x) for x in (plan, arena)]
    return _lib.load().grm_b200_latent_attend_expanded(*ref, q, *strides, w, *w_strides, scale,
                                                       causal, out, None, None)


@pytest.mark.parametrize("change,text", [
    (dict(latent=64), "latent 64"), (dict(latent=288), "latent 288"), (dict(rope=16), "rope 16"),
    (dict(heads=0), "heads"), (dict(heads=1025), "heads"), (dict(nope=32, value=32), "nope"),
    (dict(nope=64, value=128), "nope"), (dict(nope=0, value=0), "nope"),
    (dict(expand_tokens=0), "nope"), (dict(expand_tokens=(1 << 28) + 1), "nope")])
def test_plan_sizes(change, text):
    lib, plan, arena = _lib.load(), latent_plan(**change), latent_arena()
    need = ctypes.c_int64(0)
    answer(lib.grm_b200_latent_work_bytes(ctypes.byref(plan), ctypes.byref(need)), text)
    answer(lib.grm_b200_latent_plan_step(ctypes.byref(plan), PLACE, None), text)
    for call in (append, attend, expanded):
        answer(call(plan, arena), text)


def test_missing_plans_and_work():
    lib = _lib.load()
    answer(lib.grm_b200_latent_work_bytes(None, None), "null plan")
    answer(lib.grm_b200_latent_work_bytes(ctypes.byref(latent_plan()), None), "null out_bytes")
    answer(lib.grm_b200_latent_plan_step(None, PLACE, None), "null plan")
    for work in (None, PLACE + 128):
        plan = latent_plan(work=work)
        answer(lib.grm_b200_latent_plan_step(ctypes.byref(plan), PLACE, None), "aligned")
        for call in (append, attend, expanded):
            answer(call(plan, latent_arena()), "aligned")
    for call in (append, attend, expanded):
        answer(call(None, latent_arena()), "null plan")
        answer(call(latent_plan(), None), "latent arena")
        answer(call(latent_plan(dict(scratch=None)), latent_arena()), "missing")
        answer(call(latent_plan(dict(requests=0)), latent_arena()), "sizes")


@pytest.mark.parametrize("change,text", [
    (dict(rows=None), "rows"), (dict(rows=PLACE + 8), "rows"), (dict(pages=0), "pages"),
    (dict(pages=1 << 24), "pages"), (dict(page_tokens=8), "page_tokens"),
    (dict(latent=64), "latent"), (dict(rope=48), "rope"), (dict(dtype=_lib.GRM_B200_F32), "fp16"),
    (dict(pages=9), "differ"), (dict(page_tokens=32), "differ"), (dict(latent=512), "differ"),
    (dict(rope=64), "differ")])
def test_arena(change, text):
    for call in (append, attend, expanded):
        answer(call(latent_plan(), latent_arena(**change)), text)


def test_append():
    plan, arena = latent_plan(), latent_arena()
    for bad in (dict(c=None), dict(c=PLACE + 2), dict(c_row=283), dict(r=None), dict(r_row=-8)):
        answer(append(plan, arena, **bad), "rows must be")
    for rotary in (rotary_c(dim=64), rotary_c(dim=32, offset=32)):
        answer(append(plan, arena, rotary), "the rotary's dim")
    answer(append(plan, arena, rotary_c(amplitude=-1.0)), "a rotary needs")
    answer(append(latent_plan(dict(grow=0)), arena), "do not join")


def test_attend():
    plan, arena = latent_plan(), latent_arena()
    for bad in (dict(q=None), dict(q=PLACE + 4), dict(strides=(1024, 250)), dict(r=None),
                dict(r_strides=(127, 32)), dict(r_strides=(128, -32))):
        answer(attend(plan, arena, **bad), "rows must be")
    for bad in (dict(w=None), dict(w_strides=(1 << 15, 255)), dict(q=PLACE + 2)):
        answer(expanded(plan, arena, **bad), "rows must be")
    for call in (attend, expanded):
        for scale in (0.0, -1.0, math.inf, math.nan):
            answer(call(plan, arena, scale=scale), "softmax_scale")
        for out in (None, PLACE + 8):
            answer(call(plan, arena, out=out), "out must")
        answer(call(latent_plan(dict(grow=0)), arena), "no position")
    answer(expanded(latent_plan(nope=0, value=0, expand_tokens=0), arena), "expand_tokens")


def test_python_layer():
    for args in ((0, 1, 256, 32), (1, 0, 256, 32)):
        with pytest.raises(ValueError, match="positive"):
            LA.LatentArena(*args)
    for args in ((1, 1, 64, 32), (1, 1, 256, 48)):
        with pytest.raises(ValueError, match="latent must be"):
            LA.LatentArena(*args)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        LA.LatentArena(1, 1, 256, 32, dtype=torch.float32)
    with pytest.raises(ValueError, match="page_tokens"):
        LA.LatentArena(1, 1, 256, 32, page_tokens=24)
    with pytest.raises(ValueError, match="CUDA device"):
        LA.LatentArena(1, 1, 256, 32, device="cpu")


def test_a_plan_for_latent_rows_is_not_the_8_bit_arena_s():
    arena, plan = PA.PagedArena.__new__(PA.PagedArena), LA.LatentPlan.__new__(LA.LatentPlan)
    plan.planned, plan.latent = True, 256
    with pytest.raises(ValueError, match="latent rows"):
        arena._ready(plan, 0)
    arena, plan = LA.LatentArena.__new__(LA.LatentArena), PA.PagePlan.__new__(PA.PagePlan)
    arena.latent = 256
    with pytest.raises(ValueError, match="such rows"):
        arena._ready(plan, 0)


@pytest.mark.parametrize("strides", [(1 << 15, 248), (1 << 15, 0), (248, 256), (8, 256)])
def test_rows_of_weights_that_overlap(strides):
    answer(expanded(latent_plan(), latent_arena(), w_strides=strides), "overlap")


def test_room_for_more_rows_of_keys_than_there_are_numbers_for():
    lib, need = _lib.load(), ctypes.c_int64(0)
    for heads, tokens, refused in ((8, 1 << 28, True), (1024, 1 << 21, True),
                                   (1024, (1 << 21) - 1, False)):
        rc = lib.grm_b200_latent_work_bytes(
            ctypes.byref(latent_plan(heads=heads, expand_tokens=tokens)), ctypes.byref(need))
        if refused:
            answer(rc, "2^31")
        else:  # the next thing it looks at is the device
            assert rc != -1
