"""Pages of latent rows on the GPU: append, the absorbed and the expanded form of
latent attention, against the formulas in 64 bits over the rows that the arena holds.

Tolerances, for a row with weights w_t (sum 1) over n tokens, u half a step of the
arena's type (2^-8 bf16, 2^-11 fp16):
* a score is up to 576 exact products summed in fp32, at most 576/16 + 2 roundings of
  2^-22 of the sum of magnitudes, below 2^-16 of it; base-2 exponent and argument
  add 2^-20.  So the exponent is off by at most e = 2^-16 sum|q_d k_d| scale + 2^-20, a
  weight by 2e relative.
* a weight is rounded to the type: u relative, and in fp16 2^-25 of the largest where
  it is subnormal (n 2^-25 |v|max in all); results are divided by the sum of the
  rounded ones, so twice that at most.
* the result is rounded once: u relative, and 2^-25 for fp16's smallest.
* the log-sum-exp is off by e, n 2^-24 from the sum, and 2^-22 of itself.
* expanded keys and values are sums of up to 512 products (2^-16 of their magnitudes).
  Keys are held as two numbers of the type, off by u^2 |k| (and fp16's 2^-25), which
  goes into e; values as one, off by u |v|, which goes into the result.
"""

import math

import pytest

torch = pytest.importorskip("torch")

from graftrepository_b200 import _lib  # noqa: E402
from graftrepository_b200 import latent_arena as LA  # noqa: E402
from graftrepository_b200 import paged_arena as PA  # noqa: E402
from graftrepository_b200.rotary import Rotary  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, HF = torch.bfloat16, torch.float16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def ceil(a, b):
    return -(-a // b)


def gen_of(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(shape, gen, kind, spread=1.0):
    return (torch.randn(shape, device=DEV, generator=gen) * spread).to(kind)


class Turn:
    """Tables and an arena whose requests hold `cached` tokens, with a step of `fresh`
    rows planned on them.  Pages are shuffled, and what no request holds is NaN."""

    def __init__(self, cached, fresh, heads, latent, rope, page=64, kind=BF, grow=True, seed=1,
                 nope=0, room=None, tokens=None, max_fresh=None, spread=1.0):
        self.cached, self.fresh, self.heads, self.page = cached, fresh, heads, page
        self.latent, self.rope, self.kind, self.grow, self.nope = latent, rope, kind, grow, nope
        self.gen = gen_of(seed)
        self.after = [c + (n if grow else 0) for c, n in zip(cached, fresh)]
        need = [ceil(a, page) for a in self.after]
        pages, width = sum(need) + 3, max(max(need), 1) + 1
        self.tables = PA.PageTables(len(cached), pages, width, page_tokens=page, device=DEV)
        self.tables.ring.copy_(torch.randperm(pages, device=DEV, generator=self.gen).int())
        self.arena = LA.LatentArena(1, pages, latent, rope, page_tokens=page, dtype=kind,
                                    device=DEV)
        self.arena.rows.fill_(math.nan)
        rows = normal((sum(self.after), latent + rope), self.gen, kind, spread)
        held, at = [], 0
        for a in self.after:
            held.append(rows[at:at + a])
            at += a
        self.held = held
        if sum(cached):
            plan = self.arena.make_plan(self.tables, sum(cached), heads=1)
            self.tables.plan(plan, i32(cached))
            old = torch.cat([h[:c] for h, c in zip(held, cached)])
            self.arena.append(plan, old[:, :latent], old[:, latent:])
            self.tables.commit(plan)
            plan.check()
        T = self.T = max(sum(fresh), 1) if tokens is None else tokens
        expand = {}
        if nope:
            need = sum(ceil(a, 64) * 64 for a, n in zip(self.after, fresh) if n)
            expand = dict(nope=nope, value=nope, expand_tokens=max(need, 1) if room is None
                          else room)
        self.plan = self.arena.make_plan(self.tables, T, heads=heads, max_fresh=max_fresh,
                                         **expand)
        self.tables.plan(self.plan, i32(fresh), grow=grow)
        if grow:
            new = torch.zeros((T, latent + rope), device=DEV, dtype=kind)
            got = torch.cat([h[c:] for h, c in zip(held, cached)])
            new[:got.shape[0]] = got
            self.arena.append(self.plan, new[:, :latent], new[:, latent:])
        q = 8 / math.sqrt(latent)
        self.q_latent = normal((T, heads, latent), self.gen, kind, q)
        self.q_rope = normal((T, heads, rope), self.gen, kind)
        if nope:
            self.q = normal((T, heads, nope + rope), self.gen, kind)
            self.weights = normal((heads, 2 * nope, latent), self.gen, kind, latent ** -0.5)
        self.scale = (64 + rope) ** -0.5

    def want(self, causal, expanded=False):
        """(out, lse, tolerances of both) in 64 bits."""
        C, H = self.latent, self.heads
        u = torch.finfo(self.kind).eps / 2
        tiny = 2.0 ** -25 if self.kind is HF else 0.0
        wide = self.nope if expanded else C
        shape = (self.T, H, wide)
        out, tol = (torch.zeros(shape, dtype=torch.float64, device=DEV) for _ in range(2))
        lse = torch.full(shape[:2], -math.inf, dtype=torch.float64, device=DEV)
        lse_tol = torch.zeros_like(lse)
        a = 0
        for c, n, L, rows in zip(self.cached, self.fresh, self.after, self.held):
            rows = rows.double()
            t = torch.arange(L, device=DEV)
            for h in range(H if n and L else 0):
                if expanded:
                    w = self.weights[h].double()
                    kv = rows[:, :C] @ w.T
                    dkv = 2.0 ** -16 * (rows[:, :C].abs() @ w.abs().T) + tiny
                    dkv[:, :self.nope] += u * u * kv[:, :self.nope].abs()
                    dkv[:, self.nope:] += u * kv[:, self.nope:].abs()
                    k = torch.cat([kv[:, :self.nope], rows[:, C:]], 1)
                    dk = torch.cat([dkv[:, :self.nope], torch.zeros_like(rows[:, C:])], 1)
                    v, dv = kv[:, self.nope:], dkv[:, self.nope:]
                    q = self.q[a:a + n, h].double()
                else:
                    k, v = rows, rows[:, :C]
                    dk, dv = None, torch.zeros_like(v)
                    q = torch.cat([self.q_latent[a:a + n, h], self.q_rope[a:a + n, h]],
                                  1).double()
                s = q @ k.T * self.scale
                e = 2.0 ** -16 * self.scale * (q.abs() @ k.abs().T) + 2.0 ** -20
                if dk is not None:
                    e = e + self.scale * (q.abs() @ dk.T)
                if causal:
                    hide = t[None] > c + torch.arange(n, device=DEV)[:, None]
                    s = s.masked_fill(hide, -math.inf)
                    e = e.masked_fill(hide, 0.0)
                z = torch.logsumexp(s, 1, keepdim=True)
                w_t = torch.exp(s - z)
                y, mag = w_t @ v, w_t @ v.abs()
                e = e.amax(1, keepdim=True)
                out[a:a + n, h] = y
                tol[a:a + n, h] = (u * y.abs() + (2 * u + 2 * e) * mag * (1 + u) + (w_t @ dv) *
                                   (1 + 4 * u) + (2 * L * 2.0 ** -25 * float(v.abs().max()) + tiny
                                                  if tiny else 0.0))
                lse[a:a + n, h] = z[:, 0]
                lse_tol[a:a + n, h] = e[:, 0] + L * 2.0 ** -24 + 2.0 ** -22 * z[:, 0].abs()
            a += n
        return out, lse, tol, lse_tol

    def attend(self, causal=True, **more):
        return self.arena.attend(self.plan, self.q_latent, self.q_rope, scale=self.scale,
                                 causal=causal, **more)

    def expanded(self, causal=True, **more):
        return self.arena.attend_expanded(self.plan, self.q, self.weights, scale=self.scale,
                                          causal=causal, **more)


def close(got, want):
    (out, lse), (y, z, tol, lse_tol) = got, want
    off = (out.double() - y).abs() - tol
    assert bool((off <= 0).all()), (float(off.max()), torch.nonzero(~(off <= 0))[:3].tolist())
    empty = z == -math.inf
    assert bool((lse[empty] == -math.inf).all())
    off = ((lse.double() - z).abs() - lse_tol)[~empty]
    assert off.numel() == 0 or bool((off <= 0).all()), float(off.max())


# --------------------------------------------------------------------- append

@pytest.mark.parametrize("latent,rope", [(128, 64), (256, 32), (512, 64)])
@pytest.mark.parametrize("layout", [None, "half", "interleaved", "pair_swap"])
@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("page", [16, 128])
def test_append(latent, rope, layout, kind, page):
    gen = gen_of(latent + page)
    tables = PA.PageTables(4, 40, 10, page_tokens=page, device=DEV)
    arena = LA.LatentArena(2, 40, latent, rope, page_tokens=page, dtype=kind, device=DEV)
    arena.rows.fill_(7.0)
    plan = arena.make_plan(tables, 260, heads=3)
    rotary = None if layout is None else Rotary(rope, layout=layout, device=DEV)
    held = [[] for _ in range(4)]
    for fresh in ([100, 0, 1, 37], [1, 1, 1, 0], [17, 150, 0, 60]):
        # rows of a projection that also holds something else
        x = normal((260, latent + rope + 8), gen, kind)
        c, r = x[:, :latent], x[:, latent:latent + rope]
        tables.plan(plan, i32(fresh))
        arena.append(plan, c, r, layer=1, rotary=rotary)
        want = r if rotary is None else \
            rotary.rotate(r[:, None].contiguous(), plan.positions)[:, 0]
        starts = plan.starts.tolist()
        for i in range(4):
            a, b = starts[i], starts[i + 1]
            held[i].append(torch.cat([c[a:b], want[a:b]], 1))
        tables.commit(plan)
        plan.check()
    table, used = tables.table.tolist(), set()
    for i in range(4):
        rows = torch.cat(held[i])
        n = rows.shape[0]
        assert tables.lens[i].item() == n
        pages = table[i][:ceil(n, page)]
        used |= set(pages)
        got = arena.rows[1][pages].reshape(-1, latent + rope)
        assert torch.equal(got[:n], rows)
        assert bool((got[n:] == 7.0).all())  # what is past the last token stays
    rest = [p for p in range(40) if p not in used]
    assert bool((arena.rows[1][rest] == 7.0).all()) and bool((arena.rows[0] == 7.0).all())


# ------------------------------------------------------------------- absorbed

SIZES = [(256, 32), (128, 32), (128, 64), (256, 64), (512, 32), (512, 64)]


@pytest.mark.parametrize("latent,rope", SIZES)
@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("heads,page,cached,fresh", [
    (1, 16, [0], [1]), (40, 64, [332], [1]), (16, 32, [63, 64, 65, 0, 200], [1, 1, 1, 1, 0]),
    (40, 16, [100, 0, 1000], [5, 5, 5]), (5, 128, [0, 127, 700], [130, 1, 60]),
    (128, 64, [500, 30], [1, 3]), (200, 64, [70], [2]), (3, 64, [0, 0, 300], [0, 0, 0])])
def test_absorbed(latent, rope, kind, heads, page, cached, fresh):
    turn = Turn(cached, fresh, heads, latent, rope, page, kind, seed=heads + page)
    close(turn.attend(), turn.want(True))
    close(turn.attend(causal=False), turn.want(False))


@pytest.mark.parametrize("latent,rope,heads", [(256, 32, 40), (512, 64, 16), (128, 32, 9)])
def test_absorbed_long(latent, rope, heads):
    """Long contexts, one and several requests: parts of several blocks are joined."""
    for cached, fresh in (([30011], [1]), ([9000, 17, 20000, 3], [1, 4, 2, 3]),
                          ([1500] * 9, [1] * 9), ([2500], [300])):
        turn = Turn(cached, fresh, heads, latent, rope, 64, BF)
        close(turn.attend(), turn.want(True))


@pytest.mark.parametrize("latent,rope", [(256, 32), (512, 64)])
def test_absorbed_memory(latent, rope):
    """Rows that do not join: some requests hold nothing, the plan has more room."""
    turn = Turn([700, 0, 64, 1], [3, 2, 0, 4], 40, latent, rope, 16, grow=False, tokens=40)
    close(turn.attend(causal=False), turn.want(False))
    with pytest.raises(ValueError, match="no position"):
        turn.attend()


@pytest.mark.parametrize("expanded", [False, True])
def test_rows_that_see_one_token(expanded):
    turn = Turn([0, 0], [1, 3], 16, 256, 32, 64, HF, nope=64)
    out, lse = turn.expanded() if expanded else turn.attend()
    close((out, lse), turn.want(True, expanded))
    if not expanded:  # the only weight is 1
        assert torch.equal(out[0], turn.held[0][:, :256].expand(16, 256))


@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("form", ["absorbed", "expanded"])
def test_far_apart_scores(kind, form):
    """One token takes nearly all of a row's weight; all scores far below and far above 0."""
    for spread in (1e-3, 8.0, 30.0):
        turn = Turn([900, 40], [2, 30], 16, 256, 32, 64, kind, nope=64, spread=spread)
        got = turn.attend() if form == "absorbed" else turn.expanded()
        close(got, turn.want(True, form == "expanded"))
    turn.scale = 1e-6
    got = turn.attend() if form == "absorbed" else turn.expanded()
    close(got, turn.want(True, form == "expanded"))


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("latent,nope", [(256, 64), (512, 128), (128, 64)])
def test_tokens_without_a_number_reach_only_rows_that_see_them(form, bad, latent, nope):
    """A row of the cache that holds no number: rows before it, other requests and
    what shares a tile with it are as without it, rows that see it are not."""
    turn = Turn([90, 20, 300], [70, 9, 0], 8, latent, 32, 16, nope=nope)
    expanded = form == "expanded"
    call = turn.expanded if expanded else turn.attend
    want = turn.want(True, expanded)
    close(call(), want)
    at = 90 + 33  # a position within request 0's step
    page = turn.tables.table[0, at // 16].item()
    turn.arena.rows[0, page, at % 16, 5] = bad
    out, lse = call()
    rows = torch.arange(79, device=DEV)
    sees = (rows >= 33) & (rows < 70)
    keep = [t[~sees] for t in (out, lse)]
    close(keep, [t[~sees] for t in want])
    assert bool((~torch.isfinite(out[sees])).any())
    if bad != bad:
        assert bool(torch.isnan(out[sees]).all())


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
def test_queries_without_a_number_lose_only_their_rows(form):
    turn = Turn([100, 50], [40, 3], 8, 256, 32, 64, nope=64)
    expanded = form == "expanded"
    call = turn.expanded if expanded else turn.attend
    want = turn.want(True, expanded)
    (turn.q if expanded else turn.q_latent)[7, 3, 11] = math.nan
    out, lse = call()
    bad = torch.zeros((43, 8), dtype=torch.bool, device=DEV)
    bad[7, 3] = True
    assert torch.equal(torch.isnan(out).all(2), bad) and torch.equal(torch.isnan(lse), bad)
    close((out[~bad], lse[~bad]), [t[~bad] for t in want])


def test_strides_and_given_results():
    turn = Turn([130, 5], [4, 9], 12, 256, 32, nope=64)
    out, lse = turn.attend()
    # heads before tokens, as a product over heads leaves them; parts of a wider row
    q = turn.q_latent.transpose(0, 1).contiguous().transpose(0, 1)
    both = torch.cat([turn.q_rope, turn.q_rope], 2)[:, :, 32:]
    to, sums = torch.empty_like(out), torch.empty_like(lse)
    got = turn.arena.attend(turn.plan, q, both, scale=turn.scale, out=to, lse=sums)
    assert got[0] is to and got[1] is sums
    assert torch.equal(to, out) and torch.equal(sums, lse)
    y, z = turn.expanded()
    w = torch.cat([turn.weights, turn.weights], 2)[:, :, 256:]
    q = turn.q.transpose(0, 1).contiguous().transpose(0, 1)
    got = turn.arena.attend_expanded(turn.plan, q, w, scale=turn.scale)
    assert torch.equal(got[0], y) and torch.equal(got[1], z)
    # one query for all heads
    one = turn.q_latent[:, :1].expand(13, 12, 256)
    assert torch.equal(turn.arena.attend(turn.plan, one, turn.q_rope, scale=turn.scale)[0][:, 0],
                       out[:, 0])


# ------------------------------------------------------------------- expanded

@pytest.mark.parametrize("latent,rope,nope", [(256, 32, 64), (512, 64, 128), (128, 64, 64),
                                              (256, 64, 128), (128, 32, 128), (512, 32, 64)])
@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("heads,page,cached,fresh", [
    (1, 16, [0], [1]), (5, 64, [300], [1]), (4, 32, [0, 63, 64, 0], [130, 65, 1, 0]),
    (3, 128, [0, 700], [600, 300]), (16, 16, [5, 5, 5], [7, 250, 257]), (2, 64, [9, 0], [0, 0])])
def test_expanded(latent, rope, nope, kind, heads, page, cached, fresh):
    turn = Turn(cached, fresh, heads, latent, rope, page, kind, nope=nope, seed=heads)
    close(turn.expanded(), turn.want(True, True))
    close(turn.expanded(causal=False), turn.want(False, True))


@pytest.mark.parametrize("latent,rope,nope,heads", [(256, 32, 64, 5), (512, 64, 128, 3)])
def test_expanded_long(latent, rope, nope, heads):
    for cached, fresh in (([12000], [100]), ([3000, 0, 6000], [1100, 900, 30]), ([0], [4000])):
        turn = Turn(cached, fresh, heads, latent, rope, 64, BF, nope=nope)
        close(turn.expanded(), turn.want(True, True))


@pytest.mark.parametrize("latent,rope,nope", [(128, 32, 64), (128, 64, 128)])
def test_expanded_of_more_tiles_than_blocks(latent, rope, nope):
    """Tiles that go out whole, in the order of heads, before the rest is shared."""
    turn = Turn([0, 300, 5], [2600, 0, 1900], 40, latent, rope, 64, BF, nope=nope)
    close(turn.expanded(), turn.want(True, True))
    turn = Turn([700] * 9, [300, 1, 256, 257, 0, 40, 512, 300, 300], 40, latent, rope, 16, HF,
                nope=nope)
    close(turn.expanded(), turn.want(True, True))
    close(turn.expanded(causal=False), turn.want(False, True))


def test_expanded_memory_and_the_absorbed_form_agree():
    """Rows that do not join; and the two forms of the same attention: queries taken
    into the latent space by the keys' weights, latent results out of it by the
    values'."""
    turn = Turn([700, 0, 64], [30, 2, 40], 6, 256, 32, 16, grow=False, nope=64, tokens=90)
    got = turn.expanded(causal=False)
    close(got, turn.want(False, True))
    w = turn.weights.double()
    q = torch.einsum("thn,hnc->thc", turn.q[:, :, :64].double(), w[:, :64])
    turn.q_latent, turn.q_rope = q.to(BF), turn.q[:, :, 64:]
    latent, lse = turn.attend(causal=False)
    out = torch.einsum("thc,hvc->thv", latent.double(), w[:, 64:])
    # queries, rows' keys and values and latent results are rounded to bf16 on one way
    # or the other: scores differ by up to 2^-8 |q| |k| scale on either side
    k = torch.cat([turn.held[0], turn.held[2]]).double().abs()
    e = 2 * 2.0 ** -8 * turn.scale * float(q.abs().sum(2).max()) * float(k.max())
    assert float((lse - got[1])[:72].nan_to_num().abs().max()) <= e
    far = (out - got[0].double()).abs()
    assert float(far.mean()) <= 2.0 ** -6 * float(out.abs().mean()) + 2.0 ** -8


def test_no_room_to_expand():
    turn = Turn([100, 30], [3, 4], 4, 256, 32, nope=64, room=64 * 3)
    turn.plan.check()
    close(turn.expanded(), turn.want(True, True))
    turn = Turn([100, 30], [3, 4], 4, 256, 32, nope=64, room=64 * 3 - 1, tokens=9)
    with pytest.raises(_lib.GrmB200Error, match="expand"):
        turn.plan.check()
    out, lse = turn.expanded()
    assert bool(torch.isnan(out[:7]).all()) and bool(torch.isnan(lse[:7]).all())
    assert not out[7:].any() and bool((lse[7:] == -math.inf).all())
    close(turn.attend(), turn.want(True))  # the absorbed form needs none


# ------------------------------------------------------------ how it is called

def test_steps_that_cannot_be_planned_answer_empty_rows():
    turn = Turn([50, 20], [2, 3], 4, 256, 32, nope=64, tokens=8)
    turn.tables.plan(turn.plan, i32([9, 9]))
    with pytest.raises(_lib.GrmB200Error):
        turn.plan.check()
    before = turn.arena.rows.clone().view(torch.int16)
    turn.arena.append(turn.plan, turn.q_latent[:, 0], turn.q_rope[:, 0])
    assert torch.equal(before, turn.arena.rows.view(torch.int16))
    for out, lse in (turn.attend(), turn.expanded()):
        assert not out.any() and bool((lse == -math.inf).all())


def test_the_same_call_gives_the_same_bits():
    turn = Turn([5000, 17, 900], [1, 40, 3], 40, 256, 32, nope=64)
    for call in (turn.attend, turn.expanded):
        first = call()
        for _ in range(3):
            again = call()
            assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_a_step_in_a_graph():
    """Plan, append and attention captured once, replayed with other rows and counts."""
    turn = Turn([200, 70, 5], [1, 1, 1], 16, 256, 32, nope=64, room=1024, tokens=12, max_fresh=8)
    fresh = i32([1, 1, 1])
    rows = torch.zeros((12, 288), dtype=BF, device=DEV)
    results = [torch.empty_like(t) for f in (turn.attend, turn.expanded) for t in f()]

    def step():
        turn.tables.plan(turn.plan, fresh)
        turn.arena.append(turn.plan, rows[:, :256], rows[:, 256:])
        turn.attend(out=results[0], lse=results[1])
        turn.expanded(out=results[2], lse=results[3])

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for counts in ([1, 1, 1], [3, 0, 8], [0, 5, 2]):
        fresh.copy_(i32(counts))
        rows.copy_(normal((12, 288), turn.gen, BF))
        turn.q_latent.copy_(normal(turn.q_latent.shape, turn.gen, BF, 0.5))
        graph.replay()
        turn.plan.check()
        turn.fresh = counts
        turn.after = [c + n for c, n in zip(turn.cached, counts)]
        new, at = [], 0
        for h, c, n in zip(turn.held, turn.cached, counts):
            new.append(torch.cat([h[:c], rows[at:at + n]]))
            at += n
        turn.held = new
        close(results[:2], turn.want(True))
        close(results[2:], turn.want(True, True))
        assert not results[0][sum(counts):].any() and not results[2][sum(counts):].any()


def test_another_stream_and_a_plan_dropped_after_its_step():
    turn = Turn([300, 800], [4, 1], 16, 256, 32, nope=64)
    want, more = turn.want(True), turn.want(True, True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got, also = turn.attend(stream=side), turn.expanded(stream=side)
    turn.plan = None
    side.synchronize()
    close(got, want)
    close(also, more)


def test_two_plans_on_two_streams():
    turn = Turn([3000, 800], [1, 1], 16, 256, 32)
    other = turn.arena.make_plan(turn.tables, 2, heads=16)
    torch.cuda.synchronize()
    turn.tables.plan(other, i32([1, 1]), grow=False)
    want = turn.arena.attend(other, turn.q_latent, turn.q_rope, scale=turn.scale, causal=False)
    first = turn.attend()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        a = turn.attend(stream=one)
        b = turn.arena.attend(other, turn.q_latent, turn.q_rope, scale=turn.scale, causal=False,
                              stream=two)
        torch.cuda.synchronize()
        assert torch.equal(a[0], first[0]) and torch.equal(b[0], want[0])


def test_refusals():
    turn = Turn([30], [2], 4, 256, 32, nope=64)
    arena, plan, q, r = turn.arena, turn.plan, turn.q_latent, turn.q_rope
    for a, b, text in ((q.half(), r, "bfloat16"), (q[:1], r, "must be"), (q, r[:, :3], "must be"),
                       (q.cpu(), r, "is on"), (q.transpose(1, 2).contiguous().transpose(1, 2), r,
                                               "contiguous"), (q, q[:, :, 3:35], "16-byte")):
        with pytest.raises(ValueError, match=text):
            arena.attend(plan, a, b, scale=0.1)
    with pytest.raises(ValueError, match="layer"):
        turn.attend(layer=1)
    for out in (q.half(), q[:1], q.transpose(0, 1).contiguous().transpose(0, 1)):
        with pytest.raises(ValueError, match="out must"):
            turn.attend(out=out)
    with pytest.raises(_lib.GrmB200Error, match="softmax_scale"):
        arena.attend(plan, q, r, scale=-1.0)
    with pytest.raises(ValueError, match="weights"):
        arena.attend_expanded(plan, turn.q, turn.weights[:, 1:], scale=0.1)
    bare = arena.make_plan(turn.tables, 2, heads=4)
    with pytest.raises(ValueError, match="not been planned"):
        arena.attend(bare, q, r, scale=0.1)
    turn.tables.plan(bare, i32([2]))
    with pytest.raises(ValueError, match="expanded form"):
        arena.attend_expanded(bare, turn.q, turn.weights, scale=0.1)
    with pytest.raises(ValueError, match="another step"):
        arena.attend(plan, q, r, scale=0.1)  # planned before `bare`
    eight = PA.PagedArena(1, turn.tables.pages, 1, 64, device=DEV)
    k = torch.zeros((2, 1, 64), dtype=BF, device=DEV)
    with pytest.raises(ValueError, match="latent rows"):
        eight.append(bare, k, k)
    wide = LA.LatentArena(1, turn.tables.pages, 512, 32, device=DEV)
    with pytest.raises(ValueError, match="such rows"):
        wide.attend(bare, q, r, scale=0.1)
    with pytest.raises(ValueError, match="tables have"):
        LA.LatentArena(1, 99, 256, 32, device=DEV).make_plan(turn.tables, 1, heads=1)
    for sizes in (dict(heads=0), dict(heads=4, nope=64), dict(heads=4, nope=64, value=128,
                                                             expand_tokens=64),
                  dict(heads=4, nope=64, value=64)):
        with pytest.raises(ValueError):
            arena.make_plan(turn.tables, 2, **sizes)
    rotary = Rotary(64, device=DEV)
    with pytest.raises(ValueError, match="rotary"):
        arena.append(bare, q[:, 0], r[:, 0], rotary=rotary)
