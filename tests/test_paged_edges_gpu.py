"""Edges of the 8-bit paged arena: the ends of the prompt kernel's rings, weights
far below a row's largest, streams other than the current one, steps that are
overtaken, waits that give up.

The 64-bit reference, the makers of arenas and the tolerances of attention are
those of test_paged_gpu.py, where they are derived."""

import math

import pytest

torch = pytest.importorskip("torch")

from graftrepository_b200 import _lib  # noqa: E402
from graftrepository_b200 import paged_arena as PA  # noqa: E402
from test_paged_gpu import DEV, ceil, i32, run_attention  # noqa: E402

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ ends of the rings

@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("tokens", [959, 1024, 1025, 1088, 2112])
def test_wide_heads_past_the_end_of_the_ring_of_scales(tokens, page):
    """At head_dim 256 a block holds the scales of 16 key tiles of 64 tokens: the
    last place, the first one again, and twice around."""
    run_attention([tokens] * 19, [40] * 19, heads=4, group=4, dim=256, page=page, seed=tokens)


# ------------------------------------------------- weights far below the largest

def two_kinds(requests, tokens, rows, far, gap, kind, *, heads, group, dim, page):
    """Requests whose tokens in `far` score `gap` above the others and have value 0,
    the others 1: (kernel's result, its lse, the formula's result, its lse)."""
    tables = PA.PageTables(requests, requests * ceil(tokens, page), ceil(tokens, page),
                           page_tokens=page, device=DEV)
    plan = tables.make_plan(requests * rows, kv_heads=heads, query_heads=heads * group,
                            head_dim=dim, max_fresh=rows)
    if tokens > rows:
        fill = tables.make_plan(requests * (tokens - rows), kv_heads=heads, query_heads=heads,
                                head_dim=dim)
        tables.plan(fill, i32([tokens - rows] * requests))
        tables.commit(fill)
    tables.plan(plan, i32([rows] * requests))
    plan.check()
    arena = PA.PagedArena(1, tables.pages, heads, dim, page_tokens=page, device=DEV)
    arena.k_scales.fill_(abs(gap) / (127 * dim ** 0.5))
    arena.v_scales.fill_(1 / 127)
    arena.v_codes.fill_(127)
    at = torch.tensor(far, device=DEV)
    pages, places = tables.table.long()[:, at // page].reshape(-1), (at % page).repeat(requests)
    arena.k_codes[0, pages, :, places] = 127 if gap > 0 else -127
    arena.v_codes[0, pages, :, places] = 0
    q = torch.ones((plan.tokens, heads * group, dim), dtype=kind, device=DEV)
    got, lse = arena.attend(plan, q)
    plan.check()
    g = 127 * dim ** 0.5 * float(arena.k_scales[0, 0, 0]) * math.copysign(1, gap)
    v = 127 * float(arena.v_scales[0, 0, 0])
    n = tokens - rows + 1 + torch.arange(rows, device=DEV, dtype=torch.float64)  # a row sees
    k = (at[None] < n[:, None]).sum(1).double()
    total = k * math.exp(g) + n - k
    want, want_lse = (n - k) * v / total, total.log()
    return (got.double().view(requests, rows, -1), lse.double().view(requests, rows, -1),
            want[:, None], want_lse[:, None], abs(g), n[:, None])


def check_two_kinds(got, lse, want, want_lse, size, n):
    """As in test_paged_gpu.py, but for weights that fp16 holds as subnormals: one of
    the largest weight's 2^-32, since the largest is held as 2^7 at least."""
    e = 2.0 ** -17 * size + 2.0 ** -20
    tol = 2.0 ** -11 * want + (2.0 ** -11 + 2 * e) * want * (1 + 2.0 ** -11) + n * 2.0 ** -32 + \
        2.0 ** -25
    err = (got - want).abs()
    assert bool((err <= tol).all()), f"worst {float((err / tol).max()):.2f} of the tolerance"
    tol = e + n * 2.0 ** -24 + 2.0 ** -22 * want_lse.abs()
    assert bool(((lse - want_lse).abs() <= tol).all())


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 128)])
@pytest.mark.parametrize("requests,rows", [(56, 1), (28, 4), (1, 300), (20, 65)])
@pytest.mark.parametrize("gap", [12.0, 16.0, 17.6, 19.0])
def test_a_token_that_takes_nearly_all_of_the_weight(gap, requests, rows, dim, page):
    """Its value is 0, so the result is what the many others add up to."""
    check_two_kinds(*two_kinds(requests, 16384, rows, [0], gap, torch.float16, heads=8, group=2,
                               dim=dim, page=page))


@pytest.mark.parametrize("rows", [1, 300])
def test_the_same_over_a_long_context(rows):
    for far in ([0], [5, 130000, 249000]):
        check_two_kinds(*two_kinds(1, 250007, rows, far, 17.6, torch.float16, heads=1, group=2,
                                   dim=64, page=128))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 4, 300])
def test_scores_that_stay_just_below_a_new_reference(rows, dim):
    """Every later weight is almost 2^8 of the first ones': the largest that fp16 has
    to hold.  The first 512 tokens are all that any warp's first tile reads."""
    check_two_kinds(*two_kinds(4, 9000, rows, list(range(512)), -5.5, torch.float16, heads=2,
                               group=2, dim=dim, page=64))


# ---------------------------------------------------------------------- streams

SLEEP = 40_000_000  # clocks, some 20 ms


def small_step(stream, before=None):
    """Tables, an arena and a plan made and used at once; (slots, out, lse, k, v)."""
    if before:
        before()
    tables = PA.PageTables(3, 40, 20, page_tokens=16, device=DEV)
    arena = PA.PagedArena(1, 40, 2, 64, page_tokens=16, device=DEV)
    plan = tables.make_plan(120, kv_heads=2, query_heads=4, head_dim=64)
    tables.plan(plan, FRESH, stream=stream)
    arena.append(plan, KV[:, 0], KV[:, 1], stream=stream)
    out, lse = arena.attend(plan, Q, stream=stream)
    tables.commit(plan, stream=stream)
    k, v = arena.read(plan.slots, stream=stream)
    return (plan.slots, out, lse, k, v, tables.lens, tables.cursor), (tables, arena, plan)


@pytest.fixture
def inputs():
    global FRESH, KV, Q
    gen = torch.Generator(device=DEV).manual_seed(71)
    FRESH = i32([70, 1, 40])
    KV = torch.randn((120, 2, 2, 64), device=DEV, generator=gen).to(torch.float16)
    Q = torch.randn((120, 4, 64), device=DEV, generator=gen).to(torch.float16)
    torch.cuda.synchronize()


@pytest.mark.parametrize("explicit", [True, False])
def test_a_stream_waits_for_the_one_that_buffers_were_made_on(inputs, explicit):
    want, _ = small_step(None)
    want = [t.clone() for t in want]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    if explicit:  # the buffers are made behind a long kernel and used at once elsewhere
        got, _ = small_step(side, before=lambda: torch.cuda._sleep(SLEEP))
    else:
        torch.cuda._sleep(SLEEP)
        tables = PA.PageTables(3, 40, 20, page_tokens=16, device=DEV)
        plan = tables.make_plan(120, kv_heads=2, query_heads=4, head_dim=64)
        with torch.cuda.stream(side):
            tables.plan(plan, FRESH)
        got, want = (plan.slots,), want[:1]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_a_plan_made_on_another_stream_than_its_tables(inputs):
    want, _ = small_step(None)
    want = [t.clone() for t in want[:3]]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    torch.cuda._sleep(SLEEP)
    tables = PA.PageTables(3, 40, 20, page_tokens=16, device=DEV)
    arena = PA.PagedArena(1, 40, 2, 64, page_tokens=16, device=DEV)
    with torch.cuda.stream(side):
        plan = tables.make_plan(120, kv_heads=2, query_heads=4, head_dim=64)
        tables.plan(plan, FRESH)
        arena.append(plan, KV[:, 0], KV[:, 1])
        out, lse = arena.attend(plan, Q)
        got = [t.clone() for t in (plan.slots, out, lse)]
    places = {tables.table.data_ptr(), arena.k_codes.data_ptr()}
    with torch.cuda.stream(side):
        torch.cuda._sleep(SLEEP)
        arena.attend(plan, Q, out=out, lse=lse)
    del tables, arena, plan
    new = [torch.empty(n, dtype=torch.uint8, device=DEV) for n in (240, 240, 81920, 81920)]
    assert not places & {t.data_ptr() for t in new}
    torch.cuda.synchronize()
    for a, b in zip(got + [out, lse], want + want[1:]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("explicit", [True, False])
def test_a_dropped_plan_keeps_its_memory_until_its_step_has_run(inputs, explicit):
    (_, want, want_lse, *_), held = small_step(None)
    tables, arena, _ = held
    tables.release(i32([0, 1, 2]))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    plan = tables.make_plan(120, kv_heads=2, query_heads=4, head_dim=64)
    out, lse = torch.empty_like(Q), torch.empty((120, 4), device=DEV)
    places = {t.data_ptr(): t.numel() * t.element_size() for t in (plan.scratch, plan.slots)}
    if explicit:
        places |= {t.data_ptr(): t.numel() * t.element_size() for t in (out, lse)}
    with torch.cuda.stream(side):
        torch.cuda._sleep(SLEEP)
    if explicit:
        tables.plan(plan, FRESH, stream=side)
        arena.append(plan, KV[:, 0], KV[:, 1], stream=side)
        arena.attend(plan, Q, out=out, lse=lse, stream=side)
        with torch.cuda.stream(side):
            result = [out.clone(), lse.clone()]
        del out, lse
    else:
        with torch.cuda.stream(side):
            tables.plan(plan, FRESH)
            arena.append(plan, KV[:, 0], KV[:, 1])
            result = arena.attend(plan, Q, out=out, lse=lse)
    del plan
    # memory of the same sizes on the current stream, filled while the step waits
    new = [torch.full((n,), 255, dtype=torch.uint8, device=DEV) for n in places.values()
           for _ in range(3)]
    assert not {t.data_ptr() for t in new} & set(places)
    torch.cuda.synchronize()
    assert torch.equal(result[0], want) and torch.equal(result[1], want_lse)


@pytest.mark.parametrize("explicit", [True, False])
def test_check_waits_for_the_stream_of_the_step(inputs, explicit):
    tables = PA.PageTables(3, 4, 20, page_tokens=16, device=DEV)
    plan = tables.make_plan(120, kv_heads=2, query_heads=4, head_dim=64)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(SLEEP)
        if not explicit:
            tables.plan(plan, FRESH)  # 8 pages of 4
    if explicit:
        tables.plan(plan, FRESH, stream=side.cuda_stream)
    with pytest.raises(_lib.GrmB200Error, match="not enough free pages"):
        plan.check()
    tables.plan(plan, i32([1, 0, 0]))
    plan.check()
    torch.cuda._sleep(SLEEP)
    tables.plan(plan, FRESH)  # and the other way round
    with torch.cuda.stream(side), pytest.raises(_lib.GrmB200Error, match="free pages"):
        plan.check()


@pytest.mark.parametrize("handle", [0, None])
def test_a_raw_handle_is_that_stream(inputs, handle):
    """0 is the default stream: what was queued there before comes first."""
    side = torch.cuda.Stream()
    stream = torch.cuda.default_stream() if handle == 0 else side
    tables = PA.PageTables(3, 40, 20, page_tokens=16, device=DEV)
    arena = PA.PagedArena(1, 40, 2, 64, page_tokens=16, device=DEV)
    plan = tables.make_plan(120, kv_heads=2, query_heads=4, head_dim=64)
    fresh = i32([1, 2, 3])
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(SLEEP)
        fresh.copy_(FRESH)
    with torch.cuda.stream(side if handle == 0 else torch.cuda.default_stream()):
        raw = stream.cuda_stream
        assert (raw == 0) == (handle == 0)
        tables.plan(plan, fresh, stream=raw)
        arena.append(plan, KV[:, 0], KV[:, 1], stream=raw)
        out, lse = arena.attend(plan, Q, stream=raw)
        k, v = arena.read(plan.slots, stream=raw)
        tables.commit(plan, stream=raw)
        tables.release(FRESH[1:2], stream=raw)  # request 1
        plan.check()
    torch.cuda.synchronize()
    (_, want, want_lse, want_k, want_v, *_), _ = small_step(None)
    for a, b in zip((out, lse, k, v), (want, want_lse, want_k, want_v)):
        assert torch.equal(a, b)
    assert tables.lens.tolist() == [70, 0, 40]


def test_check_after_the_replay_of_a_graph(inputs):
    tables = PA.PageTables(3, 4, 20, page_tokens=16, device=DEV)
    plan = tables.make_plan(120, kv_heads=2, query_heads=4, head_dim=64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tables.plan(plan, FRESH)
    torch.cuda._sleep(SLEEP)
    graph.replay()
    with pytest.raises(_lib.GrmB200Error, match="not enough free pages"):
        plan.check()


def test_a_graph_of_a_step_whose_plan_no_stream_has_used(inputs):
    """Captured at once, without a step before on the capturing stream."""
    want, _ = small_step(None)
    want = [t.clone() for t in want[:3]]
    tables = PA.PageTables(3, 40, 20, page_tokens=16, device=DEV)
    arena = PA.PagedArena(1, 40, 2, 64, page_tokens=16, device=DEV)
    plan = tables.make_plan(120, kv_heads=2, query_heads=4, head_dim=64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tables.plan(plan, FRESH)
        arena.append(plan, KV[:, 0], KV[:, 1])
        out, lse = arena.attend(plan, Q)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((plan.slots, out, lse), want))


# ----------------------------------------------------- steps that are overtaken

def two_requests():
    """Requests 0 and 1 of three hold 20 and 40 tokens in pages of 16."""
    tables = PA.PageTables(3, 12, 6, page_tokens=16, device=DEV)
    plans = [tables.make_plan(60, kv_heads=1, query_heads=1, head_dim=64) for _ in range(2)]
    tables.plan(plans[0], i32([20, 40, 0]))
    tables.commit(plans[0])
    plans[0].check()
    assert tables.lens.tolist() == [20, 40, 0] and tables.cursor.tolist() == [5, 12]
    return tables, *plans


def free_pages(tables):
    a, b = tables.cursor.tolist()
    ring = tables.ring.tolist()
    return [ring[i % tables.pages] for i in range(a, b)]


def held_pages(tables):
    return [p for row, n in zip(tables.table.tolist(), tables.lens.tolist())
            for p in row[: ceil(n, tables.page_tokens)]]


def test_a_release_between_plan_and_commit():
    tables, plan, _ = two_requests()
    tables.plan(plan, i32([30, 0, 5]))  # 50 tokens and 5: three pages more
    tables.release(i32([1]))            # has no row in the step
    tables.commit(plan)
    plan.check()
    assert tables.lens.tolist() == [50, 0, 5]
    assert sorted(free_pages(tables) + held_pages(tables)) == list(range(12))


@pytest.mark.parametrize("fresh", [[30, 0, 5], [2, 0, 0]])
def test_a_release_of_a_request_with_rows_in_the_step(fresh):
    tables, plan, _ = two_requests()
    tables.plan(plan, i32(fresh))
    tables.release(i32([0]))
    tables.commit(plan)
    with pytest.raises(_lib.GrmB200Error, match="not committed"):
        plan.check()
    assert tables.lens.tolist() == [0, 40, 0]
    assert sorted(free_pages(tables) + held_pages(tables)) == list(range(12))
    tables.plan(plan, i32(fresh))  # planned again it is a step like any other
    tables.commit(plan)
    plan.check()
    assert tables.lens.tolist() == [fresh[0], 40, fresh[2]]
    assert sorted(free_pages(tables) + held_pages(tables)) == list(range(12))


def test_a_commit_given_twice_and_one_that_is_late():
    tables, plan, other = two_requests()
    tables.plan(plan, i32([1, 0, 17]))
    tables.commit(plan)
    tables.commit(plan)
    plan.check()
    state = tables.lens.tolist(), tables.cursor.tolist()
    assert state == ([21, 40, 17], [7, 12])
    tables.plan(other, i32([0, 20, 0]))
    tables.commit(other)
    tables.commit(plan)  # its requests hold what it gave them: still nothing to do
    plan.check()
    assert tables.lens.tolist() == [21, 60, 17] and tables.cursor.tolist() == [8, 12]
    tables.release(i32([2]))
    tables.commit(plan)  # and now they do not
    with pytest.raises(_lib.GrmB200Error, match="not committed"):
        plan.check()
    assert tables.lens.tolist() == [21, 60, 0] and tables.cursor.tolist() == [8, 14]
    assert sorted(free_pages(tables) + held_pages(tables)) == list(range(12))


def test_two_steps_side_by_side():
    tables, plan, other = two_requests()
    arena = PA.PagedArena(1, 12, 1, 64, page_tokens=16, device=DEV)
    rows = torch.ones((60, 1, 64), dtype=torch.float16, device=DEV)
    tables.plan(plan, i32([30, 0, 0]))
    tables.plan(other, i32([0, 0, 33]))  # takes the pages that `plan` would
    for call in (lambda: arena.append(plan, rows, rows), lambda: arena.attend(plan, rows),
                 lambda: tables.commit(plan)):
        with pytest.raises(ValueError, match="planned since"):
            call()
    arena.append(other, rows, rows)
    arena.attend(other, rows)
    tables.commit(other)
    tables.plan(plan, i32([30, 0, 0]))
    arena.append(plan, rows, rows)
    tables.commit(plan)
    arena.attend(other, rows)  # committed steps stay good
    plan.check()
    other.check()
    assert tables.lens.tolist() == [50, 40, 33]
    assert sorted(free_pages(tables) + held_pages(tables)) == list(range(12))
    # rows that only read are no such step, and a step that is left behind harms none
    reader = tables.make_plan(4, kv_heads=1, query_heads=1, head_dim=64)
    tables.plan(plan, i32([1, 0, 0]))
    tables.plan(reader, i32([2, 1, 1]), grow=False)
    arena.attend(reader, rows[:4], causal=False)
    arena.append(plan, rows, rows)
    tables.commit(plan)
    assert tables.lens.tolist() == [51, 40, 33]


def test_a_graph_that_plans_is_committed_outside():
    """The host does not see a replay's plan, and refuses nothing for it."""
    tables, plan, other = two_requests()
    fresh = i32([1, 1, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tables.plan(plan, fresh)
    for step in range(3):
        tables.plan(other, i32([0, 0, 7]))
        tables.commit(other)
        graph.replay()
        tables.commit(plan)
        plan.check()
        assert tables.lens.tolist() == [21 + step, 41 + step, 7 + 7 * step]
    assert sorted(free_pages(tables) + held_pages(tables)) == list(range(12))


@pytest.mark.parametrize("requests", [1, 33, 1024, 5000])
def test_commit_of_many_requests(requests):
    gen = torch.Generator().manual_seed(requests)
    tables = PA.PageTables(requests, 3 * requests, 3, page_tokens=16, device=DEV)
    plan = tables.make_plan(20 * requests, kv_heads=1, query_heads=1, head_dim=64, max_fresh=20)
    lens = torch.zeros(requests, dtype=torch.int32)
    for _ in range(2):
        fresh = torch.randint(0, 21, (requests,), generator=gen, dtype=torch.int32)
        tables.plan(plan, fresh.to(DEV))
        tables.commit(plan, stream=torch.cuda.current_stream())
        plan.check()
        lens += fresh
        assert torch.equal(tables.lens.cpu(), lens)
        assert tables.cursor.tolist() == [int(((lens + 15) // 16).sum()), 3 * requests]


# ------------------------------------------------------------- the longest requests

MOST = 2 ** 31 - 1024


@pytest.mark.parametrize("grow", [True, False])
@pytest.mark.parametrize("fresh", [1, 40, 1000])
def test_lengths_up_to_the_last_that_is_planned(fresh, grow):
    """Lengths that tiles and pages round up past 31 bits, for single tokens and for
    prompts; the tokens themselves all lie in one page here."""
    width = ceil(MOST, 128)
    tables = PA.PageTables(2, 8, width, page_tokens=128, device=DEV)
    tables.table.zero_()
    plan = tables.make_plan(fresh + 5, kv_heads=1, query_heads=4, head_dim=64)
    for over, bits in ((0, 0), (1, PA.PLAN_BAD_LENGTH), (1023, PA.PLAN_BAD_LENGTH)):
        tables.lens.copy_(i32([MOST - fresh + over, 3]))
        tables.plan(plan, i32([fresh, 2]), grow=grow)
        assert plan.status.item() == bits
        if not bits:
            assert plan.lens.tolist() == ([MOST, 5] if grow else [MOST - fresh, 3])
            assert plan.positions[[0, fresh - 1]].tolist() == [MOST - fresh, MOST - 1]
            taken = ceil(MOST, 128) - ceil(MOST - fresh, 128)  # pages 0, 1, ... of the ring
            last = 128 * max(taken - 1, 0) + 127
            assert plan.slots[fresh - 1].item() == (last if grow else -1)
    tables.lens.copy_(i32([2 ** 31 - 1, 3]))
    tables.plan(plan, i32([0, 2]), grow=grow)
    assert plan.status.item() == PA.PLAN_BAD_LENGTH


def test_a_row_over_the_longest_request():
    """2^31 - 1024 tokens of one page: equal weights, values 1."""
    tables = PA.PageTables(1, 8, ceil(MOST, 128), page_tokens=128, device=DEV)
    arena = PA.PagedArena(1, 8, 1, 64, page_tokens=128, device=DEV)
    arena.k_scales.fill_(1.0)
    arena.v_scales.fill_(1.0)
    arena.v_codes.fill_(1)
    tables.table.zero_()
    tables.lens.fill_(MOST - 1)
    plan = tables.make_plan(1, kv_heads=1, query_heads=4, head_dim=64)
    q = torch.ones((1, 4, 64), dtype=torch.float16, device=DEV)
    for grow in (True, False):
        tables.plan(plan, i32([1]), grow=grow)
        out, lse = arena.attend(plan, q, causal=grow)
        plan.check()
        assert bool((out == 1).all())
        # sums of equal powers of two: one rounding of 2^-24 for each of the joins of a
        # share's warps, of the shares, and of the logarithm
        assert bool(((lse.double() - math.log(MOST - 1 + grow)).abs() < 2.0 ** -12).all())


# ----------------------------------------------------------------------- strides

def test_a_dimension_of_one_entry_may_have_any_stride():
    """One row cut out of a wide projection, and one head."""
    tables = PA.PageTables(1, 4, 4, page_tokens=16, device=DEV)
    for tokens, heads in ((1, 3), (5, 1), (1, 1)):
        arena = PA.PagedArena(1, 4, heads, 64, page_tokens=16, device=DEV)
        plan = tables.make_plan(tokens, kv_heads=heads, query_heads=heads, head_dim=64)
        tables.plan(plan, i32([tokens]))
        x = torch.randn(4096, device=DEV).to(torch.float16)
        rows, head = 77 if tokens == 1 else 72, 13 if heads == 1 else 64
        view = torch.as_strided(x, (tokens, heads, 64), (rows, head, 1))
        arena.append(plan, view.contiguous(), view.contiguous())
        want, want_lse = arena.attend(plan, view.contiguous())
        codes, scales = arena.k_codes.clone(), arena.k_scales.clone()
        arena.k_codes.zero_()
        arena.k_scales.zero_()
        arena.append(plan, view, view)
        out, lse = arena.attend(plan, view)
        assert torch.equal(arena.k_codes, codes) and torch.equal(arena.k_scales, scales)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    with pytest.raises(ValueError, match="multiples of 8"):
        plan = tables.make_plan(2, kv_heads=1, query_heads=1, head_dim=64)
        tables.plan(plan, i32([2]))
        arena.attend(plan, torch.as_strided(x, (2, 1, 64), (77, 13, 1)))


# ------------------------------------------------------------------ many requests

@pytest.mark.parametrize("requests", [20_000, 70_001, 2 ** 20])
def test_as_many_requests_as_a_plan_takes(requests):
    """Two steps of 0 to 3 rows each; a first row sees itself alone."""
    gen = torch.Generator(device=DEV).manual_seed(requests)
    tables = PA.PageTables(requests, requests + 5, 1, page_tokens=16, device=DEV)
    arena = PA.PagedArena(1, requests + 5, 1, 64, page_tokens=16, device=DEV)
    tables.ring.copy_(torch.randperm(requests + 5, device=DEV, generator=gen).int())
    plan = tables.make_plan(3 * requests, kv_heads=1, query_heads=2, head_dim=64, max_fresh=3)
    cached = torch.zeros(requests, dtype=torch.int32, device=DEV)
    for step in range(2):
        fresh = torch.randint(0, 4, (requests,), device=DEV, generator=gen, dtype=torch.int32)
        tables.plan(plan, fresh)
        plan.check()
        total = int(fresh.sum())
        rows = torch.repeat_interleave(torch.arange(requests, device=DEV), fresh.long())
        starts = torch.zeros(requests + 1, dtype=torch.int64, device=DEV)
        starts[1:] = fresh.cumsum(0)
        pos = cached[rows] + torch.arange(total, device=DEV) - starts[rows]
        assert torch.equal(plan.starts.long(), starts)
        assert torch.equal(plan.rows[:total].long(), rows)
        assert torch.equal(plan.positions[:total].long(), pos)
        assert torch.equal(plan.slots[:total], tables.table[rows, 0].long() * 16 + pos)
        assert bool((plan.slots[total:] == -1).all())
        kv = torch.randn((3 * requests, 4, 64), device=DEV, generator=gen).to(torch.float16)
        arena.append(plan, kv[:, :1], kv[:, 1:2])
        out, lse = arena.attend(plan, kv[:, 2:])
        v = arena.read(plan.slots[:total], dtype=torch.float32)[1]
        alone = pos == 0
        assert bool(alone.any())
        # weight 1 exactly, codes exact, one rounding of the scale's factors and one to fp16
        err = (out[:total][alone] - v[alone]).abs()
        assert bool((err <= 2.0 ** -10 * v[alone].abs() + 2.0 ** -24).all())
        assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse[:total]).all())
        tables.commit(plan)
        cached += fresh
        assert torch.equal(tables.lens, cached)
        held = tables.table[cached > 0, 0].long()
        assert held.unique().numel() == held.numel()
        assert tables.cursor.tolist() == [held.numel(), requests + 5]
    tables.release(torch.arange(requests, dtype=torch.int32, device=DEV))
    assert not tables.lens.any() and tables.ring.unique().numel() == requests + 5


# ------------------------------------------------------- sums of few, small scores

@pytest.mark.parametrize("dim,heads,group,kind,rows,seed", [
    (64, 3, 8, torch.float16, 1, 2617), (64, 16, 16, torch.float16, 1, 1),
    (128, 16, 16, torch.bfloat16, 1, 2), (256, 8, 32, torch.bfloat16, 1, 3),
    (64, 4, 16, torch.bfloat16, 40, 4), (128, 4, 4, torch.float16, 40, 5),
    (256, 4, 16, torch.float16, 40, 6)])
def test_the_sum_where_scores_are_small_and_scales_far_apart(dim, heads, group, kind, rows, seed):
    """There the log-sum-exp has little but its own roundings to be off by."""
    n = 1 if seed == 2617 else 200 // rows
    run_attention([rows] * n, [rows] * n, heads=heads, group=group, dim=dim, page=16, kind=kind,
                  causal=False, grow=False, seed=seed, spread=2.0, max_fresh=501)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("requests,heads,group", [(6000, 16, 1), (1500, 16, 48)])
def test_one_token_has_a_sum_of_one_and_its_weight_is_not_rounded(requests, heads, group, dim):
    """Whatever the scale of its values: a query of zeros over one token, for which the
    kernels take the logarithm of that scale, powers of it and a logarithm again.  Two
    powers are off by 2^-22 each, the last logarithm by a unit in the last place of a
    number below 16.  The result is rounded to fp16, 2^-11; its weight lies within 2^-15
    of a power of two (in the exponent), and fp16 makes it that; the scale's logarithm,
    two units off, and the power are 2^-19 each."""
    gen = torch.Generator(device=DEV).manual_seed(dim + group)
    tables = PA.PageTables(requests, requests, 1, page_tokens=16, device=DEV)
    arena = PA.PagedArena(1, requests, heads, dim, page_tokens=16, device=DEV)
    arena.v_scales.copy_(torch.exp2(22 * torch.rand(arena.v_scales.shape, device=DEV,
                                                    generator=gen) - 14.9))
    arena.v_codes.fill_(127)
    plan = tables.make_plan(requests, kv_heads=heads, query_heads=heads * group, head_dim=dim,
                            max_fresh=1)
    tables.plan(plan, i32([1] * requests))
    plan.check()
    q = torch.zeros((requests, heads * group, dim), dtype=torch.float16, device=DEV)
    out, lse = arena.attend(plan, q)
    assert float(lse.abs().max()) <= 2 * 2.0 ** -22 + math.log(2) * 2.0 ** -20
    want = 127 * arena.v_scales[0][tables.table[:, 0].long()].repeat_interleave(group, 1).double()
    err = (out.double() / want[:, :, None] - 1).abs().amax()
    assert float(err) <= 2.0 ** -11 + math.log(2) * 2.0 ** -15 + 2 * 2.0 ** -19
