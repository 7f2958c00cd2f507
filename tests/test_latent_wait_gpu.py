"""The path of latent attention on which a bounded wait gives up.

A child process with GRM_B200_WAIT_LIMIT=0 has waits give up before their first probe,
or after one, and nothing is copied, so no wait hangs (the drain at the end of a block has
a limit of its own).  The step's status says so, its rows are NaN rather than what the
memory held, those included that parts of several blocks are joined for, rows that wait
for nothing are what they always are, and the context stays usable."""

import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]

CHILD = r"""
import math, sys
import torch
sys.path.insert(0, sys.argv[1])
from graftrepository_b200 import _lib, latent_arena as LA, paged_arena as PA

D = "cuda:0"
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=D)

def lost(plan, out, lse, n):
    torch.cuda.synchronize()
    assert plan.status.item() == PA.PLAN_WAIT, plan.status.item()
    try:
        plan.check()
    except _lib.GrmB200Error as e:
        assert "gave up" in str(e)
    else:
        raise AssertionError("check")
    assert bool(out[:n].isnan().all()) and bool(lse[:n].isnan().all())
    assert not out[n:].any() and bool((lse[n:] == -math.inf).all())

def step(latent, rope, heads, cached, fresh, max_fresh=None, nope=0):
    room = sum(-(-(c + n) // 64) * 64 for c, n in zip(cached, fresh))
    expand = dict(nope=nope, value=nope, expand_tokens=room) if nope else {}
    for kind in (torch.bfloat16, torch.float16):
        tables = PA.PageTables(len(cached), 600, 400, page_tokens=64, device=D)
        arena = LA.LatentArena(1, 600, latent, rope, page_tokens=64, dtype=kind, device=D)
        first = arena.make_plan(tables, sum(cached) or 1, heads=1)
        tables.plan(first, i32(cached))
        tables.commit(first)
        T, n = sum(fresh) + 3, sum(fresh)
        plan = arena.make_plan(tables, T, heads=heads, max_fresh=max_fresh, **expand)
        q = torch.randn((T, heads, latent + rope), device=D).to(kind)
        wide = nope or latent
        out = torch.full((T, heads, wide), 3.0, dtype=kind, device=D)
        lse = torch.full((T, heads), 3.0, device=D)
        tables.plan(plan, i32(fresh))
        arena.append(plan, q[:, 0, :latent], q[:, 0, latent:])
        plan.check()
        if nope:
            w = torch.randn((heads, 2 * nope, latent), device=D).to(kind)
            arena.attend_expanded(plan, q[:, :, :nope + rope].contiguous(), w, scale=0.1, out=out,
                                  lse=lse)
        else:
            arena.attend(plan, q[:, :, :latent], q[:, :, latent:], scale=0.1, out=out, lse=lse)
        lost(plan, out, lse, n)
        # rows of a request that holds nothing wait for nothing
        tables.lens.zero_()
        tables.plan(plan, i32([1] + [0] * (len(cached) - 1)), grow=False)
        if nope:
            arena.attend_expanded(plan, q[:, :, :nope + rope].contiguous(), w, scale=0.1, out=out,
                                  lse=lse, causal=False)
        else:
            arena.attend(plan, q[:, :, :latent], q[:, :, latent:], scale=0.1, out=out, lse=lse,
                         causal=False)
        plan.check()
        assert not out.any() and bool((lse == -math.inf).all())

for latent, rope, heads in ((128, 32, 9), (256, 32, 40), (512, 64, 16)):
    step(latent, rope, heads, [7000, 90, 3000], [1, 1, 1], 1)  # parts of several blocks
    step(latent, rope, heads, [100, 20, 50], [3, 0, 2])        # and tiles of one
    step(latent, rope, heads, [5000, 0], [40, 300])
step(256, 32, 200, [3000], [2])                                # more heads than a tile's rows
for latent, rope, nope in ((256, 32, 64), (512, 64, 128), (128, 32, 64)):
    step(latent, rope, 5, [5000, 10], [40, 300], nope=nope)
    step(latent, rope, 40, [0, 700], [2600, 513], nope=nope)   # tiles that go out whole
x = torch.arange(1024, device=D, dtype=torch.float32)
torch.cuda.synchronize()
print("CTX", float(x.sum().item()))
"""


def test_a_wait_that_gives_up_leaves_no_numbers():
    env = dict(os.environ, GRM_B200_WAIT_LIMIT="0")
    out = subprocess.run([sys.executable, "-c", CHILD, str(ROOT)], env=env, capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    assert out.stdout.split() == ["CTX", str(1023 * 1024 / 2)]
