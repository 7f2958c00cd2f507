"""Latent attention where a visible token's score or value is no finite number, against the
formula in 64 bits, row by row: with s = scale q . k, w = softmax(s) and out = sum w v over
the tokens that the row sees,
* a score of NaN or +inf makes the row NaN;
* one of -inf weighs nothing, whatever part of the row's tokens it is in, but where the
  token's value is no number either, 0 times it makes the result's NaN;
* all of them -inf: the row is NaN and its log-sum -inf (a row that sees nothing is 0);
* what a row does not see does not reach it.
Rows that the formula leaves finite keep test_latent_gpu's tolerances."""

import math

import pytest

torch = pytest.importorskip("torch")

from test_latent_gpu import BF, DEV, HF, Turn  # noqa: E402

pytestmark = pytest.mark.gpu
F64 = torch.float64


def formula(turn, causal, expanded):
    """(out, lse, tolerances of both) in 64 bits, rows one after another."""
    C, H = turn.latent, turn.heads
    u = torch.finfo(turn.kind).eps / 2
    tiny = 2.0 ** -25 if turn.kind is HF else 0.0
    wide = turn.nope if expanded else C
    out, tol = (torch.zeros((turn.T, H, wide), dtype=F64, device=DEV) for _ in range(2))
    lse = torch.full((turn.T, H), -math.inf, dtype=F64, device=DEV)
    lse_tol = torch.zeros_like(lse)
    a = 0
    for c, n, L, rows in zip(turn.cached, turn.fresh, turn.after, turn.held):
        rows = rows.double()
        if expanded:
            W = turn.weights.double()
            kv = torch.einsum("tc,hnc->htn", rows[:, :C], W)
            mag = torch.einsum("tc,hnc->htn", rows[:, :C].abs(), W.abs()) * 2.0 ** -16
            k = torch.cat([kv[:, :, :wide], rows[None, :, C:].expand(H, -1, -1)], 2)
            v = kv[:, :, wide:]
            dv = mag[:, :, wide:] + u * v.abs() + tiny
            dk = torch.cat([mag[:, :, :wide] + u * u * kv[:, :, :wide].abs() + tiny,
                            torch.zeros_like(k[:, :, wide:])], 2)
        else:
            k, v = rows[None].expand(H, -1, -1), rows[None, :, :C].expand(H, -1, -1)
            dv, dk = torch.zeros_like(v), torch.zeros_like(k)
        for i in range(n):
            see = min(L, c + i + 1) if causal else L
            if see == 0:
                continue
            q = (turn.q[a + i] if expanded else
                 torch.cat([turn.q_latent[a + i], turn.q_rope[a + i]], 1)).double()
            x, y = k[:, :see], v[:, :see]
            s = torch.einsum("hd,htd->ht", q, x) * turn.scale
            z = torch.logsumexp(s, 1, keepdim=True)
            w = torch.softmax(s, 1)
            out[a + i] = torch.einsum("ht,htv->hv", w, y)
            e = turn.scale * torch.einsum("hd,htd->ht", q.abs(), 2.0 ** -16 * x.abs() +
                                          dk[:, :see])
            e = torch.where(torch.isfinite(s), e, 0.0).amax(1, keepdim=True) + 2.0 ** -20
            m = torch.einsum("ht,htv->hv", w, y.abs())
            tol[a + i] = (u * out[a + i].abs() + (2 * u + 2 * e) * m * (1 + u) +
                          torch.einsum("ht,htv->hv", w, dv[:, :see]) * (1 + 4 * u))
            if tiny:
                tol[a + i] += 2 * L * 2.0 ** -25 * y.abs().nan_to_num(0, 0, 0).amax((1, 2))[:, None]
                tol[a + i] += tiny
            lse[a + i] = z[:, 0]
            lse_tol[a + i] = e[:, 0] + L * 2.0 ** -24 + 2.0 ** -22 * z[:, 0].abs()
        a += n
    return out, lse, tol, lse_tol


def same(got, want):
    """Rows without a number are the formula's, the others as near as they have to be."""
    (out, lse), (y, z, tol, lse_tol) = got, want
    good = torch.isfinite(y).all(2)
    bad = torch.isfinite(out).all(2) != good
    assert not bool(bad.any()), ("rows", torch.nonzero(bad)[:5].tolist(), int(bad.sum()))
    off = ((out.double() - y).abs() - tol)[good]
    assert off.numel() == 0 or bool((off <= 0).all()), float(off.max())
    none = z == -math.inf
    assert torch.equal(lse == -math.inf, none)
    good = torch.isfinite(z)
    bad = torch.isfinite(lse) != good
    assert not bool(bad.any()), ("log-sums", torch.nonzero(bad)[:5].tolist(), int(bad.sum()))
    off = ((lse.double() - z).abs() - lse_tol)[good]
    assert off.numel() == 0 or bool((off <= 0).all()), float(off.max())


def put(turn, r, tokens, column, value):
    """Tokens of request r get `value` in one column of their rows."""
    page = turn.page
    for t in tokens:
        at = turn.tables.table[r, t // page].item()
        turn.arena.rows[0, at, t % page, column] = value
        turn.held[r][t, column] = value


# One row a request and several, kernels for few rows and for many, one part a tile and many
TURNS = [
    dict(cached=[400, 3000, 0], fresh=[3, 1, 2], heads=8, latent=512, rope=64, page=32,
         max_fresh=4, tokens=8),
    dict(cached=[9000, 300], fresh=[1, 1], heads=16, latent=512, rope=32, page=64, max_fresh=1),
    dict(cached=[400, 3000, 0], fresh=[9, 1, 2], heads=8, latent=512, rope=64, page=32),
    dict(cached=[9000, 300], fresh=[1, 1], heads=40, latent=256, rope=32, page=64),
    dict(cached=[300, 90], fresh=[70, 9], heads=5, latent=128, rope=64, page=16),
]


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
@pytest.mark.parametrize("kind", [BF, HF])
@pytest.mark.parametrize("sizes", TURNS)
@pytest.mark.parametrize("which", ["all", "first half", "second half", "one"])
def test_scores_without_a_number(form, kind, sizes, which):
    """An infinite positional value, whose score is -inf for some heads and +inf for others."""
    if form == "expanded" and sizes.get("max_fresh"):
        pytest.skip("the form does not go by the most rows")
    turn = Turn(**sizes, kind=kind, nope=64 if sizes["latent"] < 512 else 128)
    expanded = form == "expanded"
    turn.q[:, :, -1].abs_()
    turn.q_rope[:, :, -1].abs_()
    turn.q[:, 1, -1] *= -1
    turn.q_rope[:, 1, -1] *= -1
    L = turn.after[0]
    tokens = {"all": range(L), "first half": range(L // 2), "second half": range(L // 2, L),
              "one": [L // 3]}[which]
    put(turn, 0, tokens, turn.latent + turn.rope - 1, -math.inf)
    for causal in (True, False):
        got = turn.expanded(causal) if expanded else turn.attend(causal)
        same(got, formula(turn, causal, expanded))
    turn.plan.check()


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("column", [5, -70])
@pytest.mark.parametrize("sizes", TURNS)
def test_values_without_a_number(form, bad, column, sizes):
    """In tokens that some rows of a tile see and others do not, of request 0 alone: those that
    do have no number even where the score is -inf, those that do not do not notice."""
    if form == "expanded" and sizes.get("max_fresh"):
        pytest.skip("the form does not go by the most rows")
    turn = Turn(**sizes, nope=64 if sizes["latent"] < 512 else 128)
    expanded = form == "expanded"
    c, n = turn.cached[0], turn.fresh[0]
    put(turn, 0, {c + n // 3, c + n // 2, c + n - 1}, column, bad)
    for causal in (True, False):
        got = turn.expanded(causal) if expanded else turn.attend(causal)
        same(got, formula(turn, causal, expanded))
    turn.plan.check()
