"""Latent attention where sizes, strides and tables are out of the ordinary: more
requests than one pass of the plan, rows past 2^32 elements, weights that heads share or
that lie another way, tables that name no page, plans that captured graphs share.
Tolerances as in test_latent_gpu."""

import pytest

torch = pytest.importorskip("torch")

from graftrepository_b200 import _lib  # noqa: E402
from graftrepository_b200 import latent_arena as LA  # noqa: E402
from graftrepository_b200 import paged_arena as PA  # noqa: E402
from test_latent_gpu import BF, DEV, HF, Turn, close, gen_of, i32, normal  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("latent,rope", [(256, 32), (512, 64)])
def test_more_requests_than_a_pass(latent, rope):
    cached = [(7 * r) % 90 for r in range(1500)]
    fresh = [0 if r % 5 == 3 else 1 + (r % 7 == 0) for r in range(1500)]
    turn = Turn(cached, fresh, 2, latent, rope, 32, BF, nope=64)
    close(turn.attend(), turn.want(True))
    close(turn.expanded(), turn.want(True, True))


def test_rows_past_32_bits():
    """Pages at the end of an arena of 4.4 * 10^9 values; the same step in a small one
    gives the same bits."""
    got = []
    for pages in (12, 120_000):
        gen = gen_of(5)
        tables = PA.PageTables(2, pages, 6, page_tokens=128, device=DEV)
        tables.ring.copy_(torch.arange(pages - 1, -1, -1, device=DEV).int())
        arena = LA.LatentArena(1, pages, 256, 32, page_tokens=128, device=DEV)
        rows = normal((700, 288), gen, BF)
        plan = arena.make_plan(tables, 700, heads=4, nope=64, value=64, expand_tokens=1024)
        tables.plan(plan, i32([650, 50]))
        arena.append(plan, rows[:, :256], rows[:, 256:])
        q = normal((700, 4, 288), gen, BF, 0.3)
        w = normal((4, 128, 256), gen, BF, 0.06)
        got.append([*arena.attend(plan, q[:, :, :256], q[:, :, 256:], scale=0.1),
                    *arena.attend_expanded(plan, q[:, :, :96], w, scale=0.1)])
        plan.check()
        assert pages < 100 or int(plan.slots[0]) * 288 > 1 << 32
        del arena
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("latent,rope,nope", [(256, 32, 64), (512, 64, 128)])
def test_weights_that_heads_share_or_that_lie_another_way(latent, rope, nope):
    turn = Turn([200, 0], [30, 5], 6, latent, rope, 64, HF, nope=nope)
    first = turn.expanded()
    # rows before heads
    turn.weights = turn.weights.transpose(0, 1).contiguous().transpose(0, 1)
    assert all(torch.equal(a, b) for a, b in zip(first, turn.expanded()))
    # the same rows for every head
    turn.weights = turn.weights[2:3].expand(6, 2 * nope, latent)
    close(turn.expanded(), turn.want(True, True))
    # rows on top of each other, and heads that begin inside one
    row = torch.zeros((2 * nope + 6) * latent, dtype=HF, device=DEV)
    for strides in ((8, 8), (0, 8), (8, latent), (latent - 8, latent)):
        w = row.as_strided((6, 2 * nope, latent), (*strides, 1))
        with pytest.raises(_lib.GrmB200Error, match="overlap"):
            turn.arena.attend_expanded(turn.plan, turn.q, w, scale=0.1)


def test_one_head_and_the_most():
    for heads in (1, 1024):
        turn = Turn([70, 3], [1, 2], heads, 128, 32, 16, BF, nope=64)
        close(turn.attend(), turn.want(True))
        close(turn.expanded(), turn.want(True, True))


def test_tables_that_name_no_page():
    """Entries out of range are read as the nearest page; requests with good ones do not
    notice."""
    for latent, rope, heads in ((256, 32, 40), (512, 64, 16)):
        for max_fresh in (1, 4):
            turn = Turn([300, 900], [1, 1], heads, latent, rope, 32, BF, nope=64,
                        max_fresh=max_fresh, tokens=2)
            a, b = turn.attend(), turn.expanded()
            turn.tables.table[0, 1:4] = i32([1 << 30, -7, 2 ** 31 - 1])
            for want, got in ((a, turn.attend()), (b, turn.expanded())):
                assert all(torch.equal(x[1], y[1]) for x, y in zip(want, got))
            torch.cuda.synchronize()


def test_two_graphs_of_one_plan_and_of_two():
    """Replayed in turn on one stream; a plan's work area is written anew by each."""
    turn = Turn([2500, 40], [1, 1], 40, 256, 32, nope=64)
    other = turn.arena.make_plan(turn.tables, 2, heads=40)
    fresh = i32([1, 1])
    rows = normal((2, 288), turn.gen, BF)
    turn.held = [torch.cat([h[:c], rows[i:i + 1]]) for i, (h, c) in
                 enumerate(zip(turn.held, turn.cached))]

    def absorbed(plan):
        turn.tables.plan(plan, fresh)
        turn.arena.append(plan, rows[:, :256], rows[:, 256:])
        return turn.arena.attend(plan, turn.q_latent, turn.q_rope, scale=turn.scale)

    def expanded(plan):
        turn.tables.plan(plan, fresh)
        turn.arena.append(plan, rows[:, :256], rows[:, 256:])
        return turn.arena.attend_expanded(plan, turn.q, turn.weights, scale=turn.scale)

    for call, plan in ((absorbed, turn.plan), (expanded, turn.plan), (absorbed, other)):
        call(plan)
    torch.cuda.synchronize()
    made = []
    for call, plan in ((absorbed, turn.plan), (expanded, turn.plan), (absorbed, other)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made.append((graph, call(plan)))
    for _ in range(3):
        for out, lse in (r for _, r in made):
            out.fill_(3.0)
            lse.fill_(3.0)
        for graph, _ in made:
            graph.replay()
        torch.cuda.synchronize()
        close(made[0][1], turn.want(True))
        close(made[1][1], turn.want(True, True))
        assert all(torch.equal(a, b) for a, b in zip(made[0][1], made[2][1]))


def test_results_over_the_queries_are_refused():
    turn = Turn([700], [2], 16, 256, 32, nope=64)
    with pytest.raises(ValueError, match="overlaps"):
        turn.attend(out=turn.q_latent)
    both = torch.zeros((3, 16, 256), dtype=BF, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        turn.arena.attend(turn.plan, both[:2], turn.q_rope, scale=0.1, out=both[1:])
    turn.q = torch.zeros(2 * 16 * 96 + 64, dtype=BF, device=DEV)
    over = turn.q[1024:1024 + 2 * 16 * 64].view(2, 16, 64)
    turn.q = turn.q[:2 * 16 * 96].view(2, 16, 96)
    with pytest.raises(ValueError, match="overlaps"):
        turn.expanded(out=over)
