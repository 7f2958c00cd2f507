"""The path of attention over the 8-bit paged arena on which a bounded wait gives up.

A child process with GRM_B200_WAIT_LIMIT=0 has waits give up before their first probe,
or after one where another warp has given up, so no wait hangs and every copy that was
issued ends as ever (the drain at the end of a block has a limit of its own).  The step's status says so, its rows are NaN
rather than what the memory held, parts of a prompt tile that others join included,
rows that wait for nothing are what they always are, and the context stays usable."""

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
from graftrepository_b200 import _lib, paged_arena as PA

D = "cuda:0"
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=D)

def step(dim, cached, fresh, max_fresh, heads=2):
    tables = PA.PageTables(len(cached), 400, 100, page_tokens=64, device=D)
    arena = PA.PagedArena(1, 400, heads, dim, page_tokens=64, device=D)
    tables.lens.copy_(i32(cached))
    held = sum(-(-n // 64) for n in cached)
    table, at = tables.table.cpu(), 0
    for r, n in enumerate(cached):
        k = -(-n // 64)
        table[r, :k] = torch.arange(at, at + k, dtype=torch.int32)
        at += k
    tables.table.copy_(table)
    tables.cursor[0] = held
    plan = tables.make_plan(sum(fresh) + 3, kv_heads=heads, query_heads=4 * heads, head_dim=dim,
                            max_fresh=max_fresh)
    rows = torch.randn((plan.tokens, 6 * heads, dim), device=D).to(torch.bfloat16)
    tables.plan(plan, i32(fresh))
    arena.append(plan, rows[:, :heads], rows[:, heads:2 * heads])
    plan.check()
    for kind in (torch.bfloat16, torch.float16):
        # what a call before this one left in the results
        out = torch.full((plan.tokens, 4 * heads, dim), 3.0, dtype=kind, device=D)
        lse = torch.full((plan.tokens, 4 * heads), 3.0, device=D)
        tables.plan(plan, i32(fresh))
        arena.attend(plan, rows[:, 2 * heads:].to(kind), out=out, lse=lse)
        torch.cuda.synchronize()
        n = sum(fresh)
        assert plan.status.item() == PA.PLAN_WAIT, plan.status.item()
        try:
            plan.check()
        except _lib.GrmB200Error as e:
            assert "gave up" in str(e)
        else:
            raise AssertionError("check")
        assert bool(out[:n].isnan().all()) and bool(lse[:n].isnan().all())
        assert not out[n:].any() and bool((lse[n:] == -math.inf).all())
    # rows of a request that holds nothing wait for nothing
    read = tables.make_plan(2, kv_heads=heads, query_heads=4 * heads, head_dim=dim)
    tables.lens.zero_()
    tables.plan(read, i32([2] + [0] * (len(cached) - 1)), grow=False)
    out, lse = arena.attend(read, rows[:2, 2 * heads:], causal=False)
    read.check()
    assert not out.any() and bool((lse == -math.inf).all())

for dim in (64, 128, 256):
    step(dim, [700, 90, 3000], [1, 1, 1], 1)            # shares of several workers
    step(dim, [100, 20, 50], [3, 0, 2], 4)              # whole segments, two blocks of rows
    step(dim, [5000], [40], 40)                         # prompt tiles in parts
    step(dim, [1000, 0, 300], [500, 1, 130], 500)       # prompts and single tokens
    step(dim, [0] * 30, [100] * 30, 100, heads=8)       # prompt tiles that are whole
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
