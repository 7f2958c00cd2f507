"""The 8-bit paged arena on the GPU: the step plan, append and read, attention.

The plan is compared with a simulation request by request; codes and scales
with the law in fp32 (bit for bit) and the values with the rows in 64 bits;
attention with the formula in 64 bits over the dequantised arena.

Tolerances of attention, for a row with weights w_t (sum 1) over n tokens:
* weights: a score is D exact products summed in fp32 on the tensor cores, at
  most D/16 + 2 roundings of 2^-22 of the sum of magnitudes, below 2^-17 of it
  for D <= 256; base-2 exponent and its argument add 2^-20.  So the exponent is
  off by at most e = 2^-17 sum|q_d k_d| scale + 2^-20, a weight by 2e relative.
* a weight is rounded to fp16: 2^-11 relative, or 2^-25 of the largest (with
  the value scale u in it) where it is subnormal: n 2^-25 127 u_max in all.
* the result is rounded once: 2^-8 (bf16) or 2^-11 (fp16) relative, and 2^-25
  absolute for fp16's smallest.
* the log-sum-exp is off by e, n 2^-24 from the sum, and 2^-22 of itself.
"""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_b200 import _lib  # noqa: E402
from graftrepository_b200 import paged_arena as PA  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def ceil(a, b):
    return -(-a // b)


class Sim:
    """PageTables, one page at a time."""

    def __init__(self, requests, pages, width, page):
        self.page, self.width, self.pages = page, width, pages
        self.table = np.full((requests, width), -1, np.int64)
        self.lens = [0] * requests
        self.ring = list(range(pages))
        self.cursor = [0, pages]

    def plan(self, fresh, grow=True):
        cur, table, lens = list(self.cursor), self.table.copy(), []
        starts, pos, rows, slots = [0], [], [], []
        for r, n in enumerate(fresh):
            have, after = ceil(self.lens[r], self.page), self.lens[r] + (n if grow else 0)
            for j in range(have, ceil(after, self.page)):
                table[r, j] = self.ring[cur[0] % self.pages]
                cur[0] += 1
            lens.append(after)
            for i in range(n):
                p = self.lens[r] + i
                pos.append(p)
                rows.append(r)
                slots.append(table[r, p // self.page] * self.page + p % self.page if grow else -1)
            starts.append(len(pos))
        return table, lens, starts, pos, rows, slots, cur

    def commit(self, got):
        self.table, self.lens, self.cursor = got[0], got[1], got[6]

    def release(self, rows):
        for r in rows:
            for j in range(ceil(self.lens[r], self.page)):
                self.ring[self.cursor[1] % self.pages] = int(self.table[r, j])
                self.cursor[1] += 1
            self.lens[r] = 0


def check_plan(plan, tables, want, tokens):
    table, lens, starts, pos, rows, slots, cursor = want
    pad = [-1] * (tokens - len(pos))
    assert plan.status.item() == 0
    held = tables.table.cpu().numpy()
    for r, n in enumerate(lens):
        k = ceil(n, tables.page_tokens)
        assert np.array_equal(held[r, :k], table[r, :k]), r
    assert plan.lens.tolist() == lens
    assert plan.starts.tolist() == starts
    assert plan.positions.tolist() == pos + pad
    assert plan.rows.tolist() == rows + pad
    assert plan.slots.tolist() == slots + pad
    assert plan.cursor.tolist() == cursor


# ----------------------------------------------------------------------- plan

@pytest.mark.parametrize("requests,page", [(1, 16), (3, 64), (257, 32), (1024, 16), (2500, 128)])
def test_plan_steps_follow_the_simulation(requests, page):
    rng = np.random.default_rng(requests)
    most = 40 if requests > 100 else 700
    width = ceil(3 * most, page) + 1
    pages = requests * width
    sim = Sim(requests, pages, width, page)
    tables = PA.PageTables(requests, pages, width, page_tokens=page, device=DEV)
    tokens = requests * most
    plan = tables.make_plan(tokens, kv_heads=2, query_heads=6, head_dim=64)
    for step in range(4):
        fresh = rng.integers(0, most + 1, requests)
        fresh[rng.random(requests) < 0.3] = 0
        if step == 2:
            fresh[:] = 1
        grow = step != 1
        for r in range(requests):  # keep within the table
            if sim.lens[r] + fresh[r] > width * page:
                fresh[r] = 0
        want = sim.plan(fresh.tolist(), grow)
        tables.plan(plan, i32(fresh.tolist()), grow=grow)
        check_plan(plan, tables, want, tokens)
        tables.plan(plan, i32(fresh.tolist()), grow=grow)  # planning again is the same step
        check_plan(plan, tables, want, tokens)
        tables.commit(plan)
        if grow:
            sim.commit(want)
        gone = rng.permutation(requests)[: requests // 3].tolist()
        tables.release(i32(gone))
        sim.release(gone)
        assert tables.lens.tolist() == sim.lens
        assert tables.cursor.tolist() == sim.cursor
        c = sim.cursor
        at = np.arange(c[0], c[1]) % pages
        assert np.array_equal(tables.ring.cpu().numpy()[at], np.array(sim.ring)[at])


def test_ring_turns_and_no_page_has_two_owners():
    tables = PA.PageTables(4, 9, 9, page_tokens=16, device=DEV)
    plan = tables.make_plan(64, kv_heads=1, query_heads=1, head_dim=64)
    for step in range(20):
        tables.plan(plan, i32([16 + step % 5, 0, 17, 3]))
        plan.check()
        tables.commit(plan)
        held, lens = tables.table.tolist(), tables.lens.tolist()
        own = [p for r in range(4) for p in held[r][: ceil(lens[r], 16)]]
        assert len(own) == len(set(own)) and all(0 <= p < 9 for p in own)
        tables.release(i32([0, 1, 2, 3, 3, 0, -1, 4]))  # twice and out of range: no harm
        assert tables.lens.tolist() == [0] * 4
        taken, returned = tables.cursor.tolist()
        assert returned - taken == 9


def test_a_step_that_cannot_be_planned_takes_nothing():
    tables = PA.PageTables(3, 8, 4, page_tokens=16, device=DEV)
    arena = PA.PagedArena(1, 8, 1, 64, page_tokens=16, device=DEV)
    plan = tables.make_plan(100, kv_heads=1, query_heads=2, head_dim=64, max_fresh=70)
    tables.plan(plan, i32([20, 5, 0]))
    plan.check()
    tables.commit(plan)
    lens, cursor = tables.lens.tolist(), tables.cursor.tolist()
    kv = torch.ones((100, 1, 64), dtype=torch.float16, device=DEV)
    q = torch.ones((100, 2, 64), dtype=torch.float16, device=DEV)
    for fresh, bit in (([1, -1, 0], PA.PLAN_BAD_LENGTH), ([60, 41, 0], PA.PLAN_ROWS),
                       ([0, 71, 0], PA.PLAN_ROWS), ([50, 0, 0], PA.PLAN_TABLE),
                       ([44, 59, 0], PA.PLAN_ROWS), ([40, 0, 60], PA.PLAN_PAGES),
                       ([2 ** 31 - 1, 0, 0], PA.PLAN_BAD_LENGTH)):
        tables.plan(plan, i32(fresh))
        assert plan.status.item() & bit, fresh
        with pytest.raises(_lib.GrmB200Error):
            plan.check()
        assert plan.lens.tolist() == lens and plan.cursor.tolist() == cursor
        assert plan.starts.tolist() == [0] * 4
        assert set(plan.slots.tolist()) == {-1} and set(plan.rows.tolist()) == {-1}
        before = arena.k_codes.clone()
        arena.append(plan, kv, kv)
        assert torch.equal(before, arena.k_codes)
        out, lse = arena.attend(plan, q)
        assert not out.any() and bool((lse == -math.inf).all())


# --------------------------------------------------------------- append, read

def quant_law(held, x, s_old, off):
    """The law in fp32: codes of the older tokens and of rows x [m, D], scale."""
    s = np.float32(np.abs(x.astype(np.float32)).max()) / np.float32(127)
    if off:
        s = max(np.float32(s_old), s)
    if s == 0:
        return held[:off] * 0, np.zeros(x.shape, np.int8), s
    old = np.rint(held[:off].astype(np.float32) * np.float32(s_old) / s).astype(np.int8)
    return old, np.rint(x.astype(np.float32) / s).astype(np.int8), s


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,heads,max_fresh", [(16, 3, 1), (64, 8, 1), (64, 2, 90), (32, 5, 200),
                                                  (128, 1, 300), (16, 2, 6)])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_append_writes_the_law(dim, page, heads, max_fresh, kind):
    rng = np.random.default_rng(dim + page + max_fresh)
    requests, steps = 5, 7 if max_fresh < 10 else 4
    width = ceil(steps * max_fresh, page) + 1
    pages = requests * width
    tables = PA.PageTables(requests, pages, width, page_tokens=page, device=DEV)
    arena = PA.PagedArena(2, pages, heads, dim, page_tokens=page, device=DEV)
    arena.k_codes.fill_(77)  # what an earlier owner left
    arena.v_scales.fill_(1e9)
    tokens = requests * max_fresh + 3
    plan = tables.make_plan(tokens, kv_heads=heads, query_heads=heads, head_dim=dim,
                            max_fresh=max_fresh)
    sim = Sim(requests, pages, width, page)
    codes = [arena.k_codes[1].cpu().numpy(), arena.v_codes[1].cpu().numpy()]
    scales = [arena.k_scales[1].cpu().numpy(), arena.v_scales[1].cpu().numpy()]
    for step in range(steps):
        fresh = rng.integers(0, max_fresh + 1, requests)
        fresh[0] = max_fresh
        want = sim.plan(fresh.tolist())
        tables.plan(plan, i32(fresh.tolist()))
        plan.check()
        # a fused projection's rows: k and v are strided views; sizes that make
        # scales grow and stay, one head of zeros
        kv = torch.from_numpy(rng.standard_normal((tokens, 2, heads, dim)).astype(np.float32))
        kv *= float(10.0 ** rng.integers(-3, 3))
        kv[:, :, heads // 2] *= 0 if step == 1 else 1
        kv = kv.to(kind).to(DEV)
        arena.append(plan, kv[:, 0], kv[:, 1], layer=1)
        arena.append(plan, kv[:, 0], kv[:, 1], layer=1)  # twice is once
        rows = kv.float().cpu().numpy()
        for side in range(2):
            at = 0
            for r, n in enumerate(fresh.tolist()):
                pos = sim.lens[r]
                while pos < sim.lens[r] + n:
                    p, off = int(want[0][r, pos // page]), pos % page
                    m = min(page - off, sim.lens[r] + n - pos)
                    for h in range(heads):
                        x = rows[at:at + m, side, h]
                        old, new, s = quant_law(codes[side][p, h], x, scales[side][p, h], off)
                        codes[side][p, h, :off], codes[side][p, h, off:off + m] = old, new
                        scales[side][p, h] = s
                        err = np.abs(new.astype(np.float64) * float(s) - x.astype(np.float64))
                        assert err.max() <= 0.5 * float(s) * (1 + 2.0 ** -15)
                    pos += m
                    at += m
        assert np.array_equal(arena.k_codes[1].cpu().numpy(), codes[0]), step
        assert np.array_equal(arena.v_codes[1].cpu().numpy(), codes[1]), step
        assert np.array_equal(arena.k_scales[1].cpu().numpy(), scales[0])
        assert np.array_equal(arena.v_scales[1].cpu().numpy(), scales[1])
        assert bool((arena.k_codes[0] == 77).all())  # the other layer
        tables.commit(plan)
        sim.commit(want)


@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,heads,page", [(64, 3, 16), (128, 8, 64), (256, 1, 128)])
def test_read_gives_code_times_scale(kind, dim, heads, page):
    gen = torch.Generator(device=DEV).manual_seed(dim)
    arena = PA.PagedArena(1, 11, heads, dim, page_tokens=page, device=DEV)
    for t in (arena.k_codes, arena.v_codes):
        t.copy_(torch.randint(-127, 128, t.shape, device=DEV, generator=gen, dtype=torch.int8))
    for t in (arena.k_scales, arena.v_scales):
        t.copy_(torch.rand(t.shape, device=DEV, generator=gen))
    slots = torch.randint(0, 11 * page, (77,), device=DEV, generator=gen)
    slots[5], slots[20], slots[30] = -1, 11 * page, 11 * page - 1
    for codes, scales, got in zip((arena.k_codes, arena.v_codes), (arena.k_scales, arena.v_scales),
                                  arena.read(slots, dtype=kind)):
        ok = (slots >= 0) & (slots < 11 * page)
        s = torch.where(ok, slots, 0)
        want = codes[0, s // page, :, s % page].float() * scales[0, s // page][:, :, None]
        want = torch.where(ok[:, None, None], want, 0.0).to(kind)
        assert torch.equal(got, want)
    k, v = arena.read(slots[:0])
    assert k.shape == (0, heads, dim) and k.dtype == torch.bfloat16


def test_a_number_that_is_none_marks_its_page_and_head_only():
    tables = PA.PageTables(1, 3, 3, page_tokens=16, device=DEV)
    arena = PA.PagedArena(1, 3, 2, 64, page_tokens=16, device=DEV)
    plan = tables.make_plan(40, kv_heads=2, query_heads=2, head_dim=64)
    kv = torch.ones((40, 2, 64), dtype=torch.bfloat16, device=DEV)
    k = kv.clone()
    k[20, 1, 3] = math.nan
    k[3, 0, 9] = math.inf
    tables.plan(plan, i32([40]))
    arena.append(plan, k, kv)
    got, v = arena.read(plan.slots, dtype=torch.float32)
    bad = torch.zeros((40, 2), dtype=torch.bool, device=DEV)
    bad[16:32, 1] = True
    bad[:16, 0] = True
    assert torch.equal(got.isnan().all(2), bad) and torch.equal(got.isnan().any(2), bad)
    assert torch.equal(v, torch.ones_like(v))
    tables.commit(plan)
    tables.release(i32([0]))  # a page that starts anew holds numbers again
    tables.plan(plan, i32([40]))
    arena.append(plan, kv, kv)
    assert not arena.read(plan.slots)[0].isnan().any()


# ------------------------------------------------------------------ attention

def make_arena(lens, fresh, *, heads, group, dim, page, seed, spread=0.5, tokens=None, layers=1,
               grow=True, max_fresh=None):
    """Tables and an arena whose requests hold lens tokens (the fresh ones
    included when they join) with random codes and scales, and the step's plan."""
    rng = np.random.default_rng(seed)
    requests = len(lens)
    before = [a - n if grow else a for a, n in zip(lens, fresh)]
    width = max(1, max(ceil(a, page) for a in lens)) + 2
    pages = sum(ceil(a, page) for a in lens) + 3
    tables = PA.PageTables(requests, pages, width, page_tokens=page, device=DEV)
    tables.ring.copy_(torch.from_numpy(rng.permutation(pages).astype(np.int32)))
    if sum(before):
        fill = tables.make_plan(sum(before), kv_heads=heads, query_heads=heads, head_dim=dim)
        tables.plan(fill, i32(before))
        fill.check()
        tables.commit(fill)
    arena = PA.PagedArena(layers, pages, heads, dim, page_tokens=page, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    for t in (arena.k_codes, arena.v_codes):
        t.copy_(torch.randint(-127, 128, t.shape, device=DEV, generator=gen, dtype=torch.int8))
    for t in (arena.k_scales, arena.v_scales):
        t.copy_(0.02 * torch.exp(spread * torch.randn(t.shape, device=DEV, generator=gen)))
    plan = tables.make_plan(tokens or max(1, sum(fresh)), kv_heads=heads,
                            query_heads=heads * group, head_dim=dim,
                            max_fresh=max_fresh or max(1, max(fresh)))
    tables.plan(plan, i32(fresh), grow=grow)
    plan.check()
    return tables, arena, plan


def reference(tables, arena, plan, q, causal, scale=None, layer=0):
    """(out, lse, weighted |v|, largest sum of |q k| scale, n) in 64 bits."""
    H, D, page = arena.kv_heads, arena.head_dim, arena.page_tokens
    T, heads, G = q.shape[0], q.shape[1], q.shape[1] // H
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    mag = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    size = torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    seen = torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    lens, starts = plan.lens.tolist(), plan.starts.tolist()
    for r, L in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        if a == b or L == 0:
            continue
        pages = tables.table[r, : ceil(L, page)].long()

        def side(codes, scales):
            x = codes[layer, pages].double() * scales[layer, pages].double()[:, :, None, None]
            return x.transpose(1, 2).reshape(-1, H, D)[:L].repeat_interleave(G, 1)

        k, v = side(arena.k_codes, arena.k_scales), side(arena.v_codes, arena.v_scales)
        x = q[a:b].double()
        z = torch.einsum("ihd,thd->iht", x, k) * scale
        zs = torch.einsum("ihd,thd->iht", x.abs(), k.abs()) * scale
        n = torch.full((b - a,), L, device=DEV)
        if causal:
            n = L - (b - a) + 1 + torch.arange(b - a, device=DEV)
        hide = torch.arange(L, device=DEV)[None, :] >= n[:, None]
        z = z.masked_fill(hide[:, None, :], -math.inf)
        zs = zs.masked_fill(hide[:, None, :], 0.0)
        lse[a:b] = torch.logsumexp(z, 2)
        w = torch.exp(z - lse[a:b, :, None])
        zero = torch.where(w == 0, 0.0, 1.0)  # a NaN in a hidden place counts for nothing
        v_seen = torch.where(zero.amax((0, 1)).bool()[:, None, None], v, 0.0)
        out[a:b] = torch.einsum("iht,thd->ihd", w, v_seen)
        mag[a:b] = torch.einsum("iht,thd->ihd", w, v_seen.abs())
        size[a:b] = zs.amax(2)
        seen[a:b] = n[:, None].double()
    return out, lse, mag, size, seen


def check_attention(got, lse, ref, u_max):
    out, want_lse, mag, size, n = ref
    e = 2.0 ** -17 * size + 2.0 ** -20
    unit = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -11
    tol = unit * out.abs() + (2.0 ** -11 + 2 * e)[:, :, None] * mag * (1 + unit) + \
        (n * 2.0 ** -25 * 127 * u_max)[:, :, None] + 2.0 ** -25
    err = (got.double() - out).abs()
    # a result past the type's range is that infinity
    top = torch.finfo(got.dtype).max
    past = (got.double() == torch.sign(out) * math.inf) & (out.abs() + tol > top)
    err = torch.where(past, 0.0, err)
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.2f} of the tolerance"
    empty = want_lse == -math.inf
    assert bool((lse[empty] == -math.inf).all()) and not got[empty].any()
    tol = e + n * 2.0 ** -24 + 2.0 ** -22 * torch.where(empty, 0.0, want_lse.abs())
    err = torch.where(empty, 0.0, (lse.double() - torch.where(empty, 0.0, want_lse)).abs())
    assert bool((err[~empty] <= tol[~empty]).all()), float((err / tol)[~empty].max())


def run_attention(lens, fresh, *, heads, group, dim, page, kind=torch.bfloat16, causal=True,
                  grow=True, seed=0, scale=None, spread=0.5, q_scale=1.0, max_fresh=None):
    tables, arena, plan = make_arena(lens, fresh, heads=heads, group=group, dim=dim, page=page,
                                     seed=seed, spread=spread, grow=grow, max_fresh=max_fresh)
    gen = torch.Generator(device=DEV).manual_seed(seed + 1)
    q = (q_scale * torch.randn((plan.tokens, heads * group, dim), device=DEV,
                               generator=gen)).to(kind)
    got, lse = arena.attend(plan, q, causal=causal, scale=scale)
    assert got.dtype == kind
    check_attention(got, lse, reference(tables, arena, plan, q, causal, scale),
                    float(arena.v_scales.max()))
    again, lse2 = arena.attend(plan, q, causal=causal, scale=scale)
    assert torch.equal(got, again) and torch.equal(lse, lse2)
    return tables, arena, plan, q, got, lse


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_decode_at_lengths_around_pages_and_tiles(dim, page, kind):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 517, 1023]
    run_attention(lens, [1] * len(lens), heads=2, group=4, dim=dim, page=page, kind=kind, seed=page)


@pytest.mark.parametrize("heads,group", [(1, 1), (8, 1), (5, 3), (2, 5), (4, 8), (1, 12), (2, 16),
                                         (3, 7), (1, 64), (1, 128)])
def test_decode_head_layouts(heads, group):
    run_attention([700, 1, 90], [1, 1, 1], heads=heads, group=group, dim=128, page=64, seed=group)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 3, 4, 8])
@pytest.mark.parametrize("causal", [True, False])
def test_several_rows_a_request(dim, group, causal):
    run_attention([5, 300, 64, 1000, 77], [5, 3, 1, 4, 2], heads=2, group=group, dim=dim, page=32,
                  causal=causal, seed=dim + group)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group,page", [(1, 16), (4, 64), (5, 32), (8, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(dim, group, page, causal):
    run_attention([300, 129, 1, 700, 64], [300, 100, 1, 257, 33], heads=2, group=group, dim=dim,
                  page=page, causal=causal, seed=dim + group, kind=torch.bfloat16)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,group,page", [(64, 1, 16), (64, 5, 128), (128, 1, 32), (128, 3, 64),
                                            (256, 1, 64), (256, 4, 16), (128, 40, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_on_many_heads(dim, group, page, kind, causal):
    """Enough tiles to fill the GPU, so that short prompts are prompts too."""
    run_attention([190, 45, 500, 64, 1, 130], [190, 40, 130, 64, 1, 33], heads=40, group=group,
                  dim=dim, page=page, causal=causal, seed=dim + group, kind=kind)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lens,fresh", [([5000], [40]), ([9001, 130, 700], [33, 129, 70]),
                                        ([3000, 90, 2000], [300, 64, 1])])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_in_parts(lens, fresh, dim, kind, causal):
    """Few prompt tiles over long contexts, which several blocks share."""
    run_attention(lens, fresh, heads=2, group=4, dim=dim, page=64, kind=kind, causal=causal, seed=41)


def test_prompts_in_parts_on_one_head():
    """All of the GPU on one tile, some parts past what a causal row sees."""
    run_attention([40000], [20], heads=1, group=8, dim=128, page=128, seed=42)
    run_attention([300], [260], heads=1, group=1, dim=128, page=16, seed=43)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_prompts_and_single_tokens_in_one_step(kind):
    run_attention([2000, 700, 350, 1, 900, 1500], [1, 600, 0, 1, 1, 130], heads=2, group=4, dim=128,
                  page=64, kind=kind, seed=3)


def test_long_requests_are_joined():
    run_attention([70001, 3, 40000], [1, 1, 1], heads=2, group=4, dim=128, page=64, seed=1)
    run_attention([50000], [1], heads=1, group=2, dim=64, page=16, seed=2, kind=torch.float16)
    run_attention([30000], [4], heads=1, group=4, dim=256, page=128, seed=3)


def test_many_requests_share_a_worker():
    rng = np.random.default_rng(5)
    lens = rng.integers(1, 80, 600).tolist()
    run_attention(lens, [1] * 600, heads=2, group=2, dim=64, page=16, seed=4)


def test_rows_that_do_not_join_and_empty_requests():
    _, _, plan, _, out, lse = run_attention([0, 50, 0, 0, 700, 0], [2, 3, 0, 1, 1, 4], heads=3,
                                            group=2, dim=64, page=16, causal=False, grow=False,
                                            seed=6)
    starts = plan.starts.tolist()
    for r in (0, 3, 5):
        assert not out[starts[r]:starts[r + 1]].any()
        assert bool((lse[starts[r]:starts[r + 1]] == -math.inf).all())
    run_attention([0, 0], [1, 300], heads=1, group=4, dim=128, page=64, causal=False, grow=False)


def test_rows_past_the_step_are_empty():
    tables, arena, plan = make_arena([100, 5], [1, 2], heads=2, group=2, dim=64, page=16, seed=0,
                                     tokens=50)
    q = torch.randn((50, 4, 64), device=DEV).to(torch.float16)
    q[3:] = math.nan
    out = torch.full_like(q, math.nan)
    lse = torch.full((50, 4), math.nan, device=DEV)
    got, got_lse = arena.attend(plan, q, out=out, lse=lse)
    assert got is out and got_lse is lse
    assert not out[3:].any() and bool((lse[3:] == -math.inf).all())
    ref = reference(tables, arena, plan, q[:3], True)
    check_attention(out[:3], lse[:3], ref, float(arena.v_scales.max()))


@pytest.mark.parametrize("rows", [1, 300])
def test_value_scales_far_apart(rows):
    # pages whose scales lie e^(4 x normal) apart, and pages of zeros
    tables, arena, plan = make_arena([900], [rows], heads=2, group=4, dim=128, page=32, seed=8,
                                     spread=0.3)
    gen = torch.Generator(device=DEV).manual_seed(9)
    arena.v_scales.copy_(torch.exp(4 * torch.randn(arena.v_scales.shape, device=DEV,
                                                   generator=gen)))
    zero = tables.table[0, 3].long()
    arena.v_codes[0, zero] = 0
    arena.v_scales[0, zero] = 0
    q = torch.randn((rows, 8, 128), device=DEV, generator=gen).to(torch.float16)
    got, lse = arena.attend(plan, q)
    check_attention(got, lse, reference(tables, arena, plan, q, True),
                    float(arena.v_scales.max()))


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("q_scale", [1e-30, 1e-3, 30.0, 1e4])
def test_query_sizes_fp16_cannot_hold(q_scale, rows):
    run_attention([400], [rows], heads=1, group=4, dim=128, page=64, q_scale=q_scale,
                  scale=min(1.0, 3.0 / q_scale), seed=10)


@pytest.mark.parametrize("rows", [2, 200])
def test_hidden_and_stale_places_do_not_count(rows):
    """Pages beyond a request's tokens and the end of its last page hold what
    an earlier owner left; a page without numbers hides behind the causal mask."""
    run = dict(heads=2, group=2, dim=64, page=16)
    tables, arena, plan = make_arena([rows + 14], [rows], seed=11, **run)
    q = torch.randn((rows, 4, 64), device=DEV).to(torch.bfloat16)
    want, want_lse = arena.attend(plan, q)
    L = rows + 14
    last = int(tables.table[0, (L - 1) // 16])
    if L % 16:
        arena.k_codes[0, last, :, L % 16:] = -128
        arena.v_codes[0, last, :, L % 16:] = 127
    free = [p for p in range(arena.pages) if p not in tables.table[0, : ceil(L, 16)].tolist()]
    arena.k_scales[0, free] = math.nan
    arena.v_scales[0, free] = math.inf
    got, lse = arena.attend(plan, q)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    # the last page without numbers: only rows that see into it lose theirs
    arena.v_scales[0, last] = math.nan
    arena.k_scales[0, last] = math.nan
    got, lse = arena.attend(plan, q)
    clear = (L - 1) // 16 * 16 - 14  # rows whose positions lie before that page
    assert torch.equal(got[:clear], want[:clear]) and torch.equal(lse[:clear], want_lse[:clear])
    assert bool(got[clear:].isnan().all()) and bool(lse[clear:].isnan().all())


@pytest.mark.parametrize("rows", [1, 150])
def test_a_query_without_numbers_loses_its_own_row_only(rows):
    tables, arena, plan = make_arena([500], [rows], heads=1, group=8, dim=128, page=64, seed=12)
    q = torch.randn((rows, 8, 128), device=DEV).to(torch.bfloat16)
    want, want_lse = arena.attend(plan, q)
    q[rows // 2, 3, 77] = math.nan
    got, lse = arena.attend(plan, q)
    hit = torch.zeros((rows, 8), dtype=torch.bool, device=DEV)
    hit[rows // 2, 3] = True
    assert bool(got[hit].isnan().all()) and bool(lse[hit].isnan().all())
    assert torch.equal(got[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])


@pytest.mark.parametrize("rows", [1, 140])
def test_strided_queries_and_streams(rows):
    tables, arena, plan = make_arena([333, 20], [rows, 1], heads=2, group=2, dim=64, page=32,
                                     seed=13)
    wide = torch.randn((plan.tokens, 3, 4, 72), device=DEV).to(torch.float16)
    q = wide[:, 1, :, 8:]  # rows 864 elements apart, heads 72
    want, want_lse = arena.attend(plan, q.contiguous())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got, lse = arena.attend(plan, q, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(lse, want_lse)


def test_a_step_in_a_cuda_graph():
    tables, arena, plan = make_arena([300, 40, 7], [1, 1, 1], heads=2, group=4, dim=128, page=64,
                                     seed=14)
    fresh = i32([1, 1, 1])
    kv = torch.randn((3, 2, 2, 128), device=DEV).to(torch.bfloat16)
    q = torch.randn((3, 8, 128), device=DEV).to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty((3, 8), device=DEV)

    def step():
        tables.plan(plan, fresh)
        arena.append(plan, kv[:, 0], kv[:, 1])
        arena.attend(plan, q, out=out, lse=lse)
        tables.commit(plan)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    lens = tables.lens.tolist()
    graph.replay()
    torch.cuda.synchronize()
    assert tables.lens.tolist() == [n + 1 for n in lens]
    check_attention(out, lse, reference(tables, arena, plan, q, True), float(arena.v_scales.max()))


def test_slots_past_32_bits():
    # 2^32 codes a side and more: the last pages lie past every 32-bit offset
    page, heads, dim, pages = 128, 8, 256, 16500
    tables = PA.PageTables(1, pages, 8, page_tokens=page, device=DEV)
    arena = PA.PagedArena(1, pages, heads, dim, page_tokens=page, device=DEV)
    tables.ring.copy_(torch.arange(pages - 1, -1, -1, dtype=torch.int32))
    plan = tables.make_plan(300, kv_heads=heads, query_heads=heads, head_dim=dim)
    gen = torch.Generator(device=DEV).manual_seed(1)
    kv = torch.randn((300, 2, heads, dim), device=DEV, generator=gen).to(torch.bfloat16)
    tables.plan(plan, i32([300]))
    arena.append(plan, kv[:, 0], kv[:, 1])
    assert int(plan.slots[0]) * heads * dim > 2 ** 32
    k, v = arena.read(plan.slots, dtype=torch.float32)
    for side, got in enumerate((k, v)):
        step = got.abs().amax(2) / 127
        assert bool(((got - kv[:, side].float()).abs().amax(2) <= kv.float().abs().max() / 127).all())
        assert bool((step > 0).all())
    q = torch.randn((300, heads, dim), device=DEV, generator=gen).to(torch.bfloat16)
    out, lse = arena.attend(plan, q)
    check_attention(out, lse, reference(tables, arena, plan, q, True), float(arena.v_scales.max()))


# ------------------------------------------------------------------- refusals

def test_refusals():
    with pytest.raises(ValueError):
        PA.PageTables(0, 1, 1, device=DEV)
    with pytest.raises(ValueError):
        PA.PageTables(1, 1, 1, page_tokens=48, device=DEV)
    with pytest.raises(ValueError):
        PA.PagedArena(1, 4, 2, 96, device=DEV)
    with pytest.raises(ValueError):
        PA.PagedArena(1, 4, 2, 64, device="cpu")
    tables = PA.PageTables(2, 8, 4, page_tokens=16, device=DEV)
    arena = PA.PagedArena(1, 8, 2, 64, page_tokens=16, device=DEV)
    for bad in (dict(kv_heads=2, query_heads=3, head_dim=64), dict(kv_heads=2, query_heads=4,
                head_dim=80), dict(kv_heads=0, query_heads=4, head_dim=64)):
        with pytest.raises(ValueError):
            tables.make_plan(4, **bad)
    with pytest.raises(ValueError):
        tables.make_plan(0, kv_heads=2, query_heads=4, head_dim=64)
    with pytest.raises(_lib.GrmB200Error):
        tables.make_plan(4, kv_heads=1, query_heads=129, head_dim=64)
    plan = tables.make_plan(4, kv_heads=2, query_heads=4, head_dim=64)
    half = dict(dtype=torch.float16, device=DEV)
    kv, q = torch.zeros((4, 2, 64), **half), torch.zeros((4, 4, 64), **half)
    with pytest.raises(ValueError, match="planned"):
        arena.append(plan, kv, kv)
    for fresh in (torch.zeros(2, dtype=torch.int64, device=DEV), i32([1]),
                  torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="fresh"):
            tables.plan(plan, fresh)
    tables.plan(plan, i32([2, 2]))
    with pytest.raises(ValueError, match="float16"):
        arena.append(plan, kv.float(), kv.float())
    with pytest.raises(ValueError, match="differ"):
        arena.append(plan, kv, kv.bfloat16())
    with pytest.raises(ValueError, match="must be"):
        arena.append(plan, kv[:3], kv)
    with pytest.raises(ValueError, match="contiguous"):
        arena.attend(plan, torch.zeros((4, 4, 128), **half)[:, :, ::2])
    with pytest.raises(ValueError, match="aligned"):
        arena.attend(plan, torch.zeros((4, 4, 65), **half)[:, :, 1:])
    with pytest.raises(ValueError, match="out"):
        arena.attend(plan, q, out=torch.zeros((4, 4, 64), dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="lse"):
        arena.attend(plan, q, lse=torch.zeros((4, 4), **half))
    with pytest.raises(ValueError, match="layer"):
        arena.attend(plan, q, layer=1)
    with pytest.raises(ValueError, match="slots"):
        arena.read(plan.slots.int())
    with pytest.raises(ValueError, match="read gives"):
        arena.read(plan.slots, dtype=torch.float64)
    with pytest.raises(_lib.GrmB200Error, match="softmax_scale"):
        arena.attend(plan, q, scale=0.0)
    other = PA.PagedArena(1, 9, 2, 64, page_tokens=16, device=DEV)
    with pytest.raises(_lib.GrmB200Error, match="differ"):
        other.append(plan, kv, kv)
    tables.plan(plan, i32([2, 2]), grow=False)
    with pytest.raises(ValueError, match="causal"):
        arena.attend(plan, q)
    with pytest.raises(ValueError, match="grow"):
        arena.append(plan, kv, kv)
    with pytest.raises(ValueError):
        PA.PageTables(2, 8, 4, page_tokens=16, device=DEV).plan(plan, i32([0, 0]))


@pytest.mark.parametrize("lens,fresh", [([400, 33, 5000], [1, 1, 1]), ([700, 5000], [300, 40])])
def test_scratch_may_hold_anything(lens, fresh):
    """A plan's scratch need not be cleared: what a step reads there, its plan wrote."""
    tables, arena, plan = make_arena(lens, fresh, heads=2, group=4, dim=128, page=64, seed=51)
    gen = torch.Generator(device=DEV).manual_seed(52)
    q = torch.randn((plan.tokens, 8, 128), device=DEV, generator=gen).to(torch.bfloat16)
    want = arena.attend(plan, q)
    for byte in (0, 255, 17):
        plan.scratch.fill_(byte)
        tables.plan(plan, i32(fresh))
        got = arena.attend(plan, q)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("lens,fresh", [([700, 5000, 90], [300, 40, 1]), ([3000] * 40, [70, 1] * 20)])
def test_a_mixed_step_in_a_cuda_graph(lens, fresh):
    """Prompts and single tokens of one step, two kernels after one another, replayed on
    other queries and in a row."""
    tables, arena, plan = make_arena(lens, fresh, heads=2, group=4, dim=128, page=64, seed=61)
    gen = torch.Generator(device=DEV).manual_seed(62)
    q = torch.randn((plan.tokens, 8, 128), device=DEV, generator=gen).to(torch.bfloat16)
    want = arena.attend(plan, q)
    check_attention(*want, reference(tables, arena, plan, q, True), float(arena.v_scales.max()))
    held = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = arena.attend(plan, held)
        second = arena.attend(plan, first[0])
    held.copy_(q)
    for _ in range(3):
        graph.replay()
    assert torch.equal(first[0], want[0]) and torch.equal(first[1], want[1])
    again = arena.attend(plan, want[0])
    assert torch.equal(second[0], again[0]) and torch.equal(second[1], again[1])
