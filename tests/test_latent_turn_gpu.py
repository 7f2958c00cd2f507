"""The example that runs mount, plan, append, positions, both forms of latent
attention, harvest and release together: its attention against the formulas in 64
bits over the rows that the arena holds, its rows against the rotation in 64 bits,
and a harvested graft against the rows that it was taken from."""

import importlib.util
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import oracle as O  # noqa: E402
from test_latent_gpu import BF, Turn, close  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -8  # half a step of bf16


def load_example():
    path = Path(__file__).resolve().parent.parent / "examples" / "latent_turn.py"
    spec = importlib.util.spec_from_file_location("latent_turn", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def turned(x, positions, rotary, sign=1):
    """Rows [n, dim] of layout half, rotated in 64 bits (amplitude 1)."""
    f = torch.tensor(rotary.frequencies, dtype=torch.float64, device=x.device)
    a = positions.double()[:, None] * f
    x1, x2 = x.double().chunk(2, 1)
    return torch.cat([x1 * a.cos() - sign * x2 * a.sin(), x2 * a.cos() + sign * x1 * a.sin()], 1)


@pytest.mark.parametrize("heads,latent,rope,nope,page", [(40, 256, 32, 64, 64),
                                                         (16, 512, 64, 128, 16)])
def test_a_turn(heads, latent, rope, nope, page):
    example = load_example()
    checked = []

    class Checked(example.LatentTurn):
        def formula(self, plan, layer):
            """What Turn.want goes by, of this step and layer."""
            t = Turn.__new__(Turn)
            lens, starts = plan.lens.tolist(), plan.starts.tolist()
            t.fresh = [b - a for a, b in zip(starts, starts[1:])]
            t.after = lens
            t.cached = [a - n for a, n in zip(lens, t.fresh)]
            t.held = [self.arena.rows[layer].flatten(0, 1)[self.slots(r, 0, n)]
                      for r, n in enumerate(lens)]
            t.T, t.heads, t.kind, t.scale = plan.tokens, heads, BF, self.scale
            t.latent, t.rope, t.nope = latent, rope, nope
            t.weights = self.wkv[layer]
            checked.extend(t.fresh)
            return t

        def attend(self, plan, q_latent, q_rope, layer):
            out, lse = self.arena.attend(plan, q_latent, q_rope, scale=self.scale, layer=layer)
            t = self.formula(plan, layer)
            t.q_latent, t.q_rope = q_latent, q_rope
            close((out, lse), t.want(True))
            return out

        def expanded(self, plan, q, layer):
            out, lse = self.arena.attend_expanded(plan, q, self.wkv[layer], scale=self.scale,
                                                  layer=layer)
            t = self.formula(plan, layer)
            t.q = q
            close((out, lse), t.want(True, True))
            return out

    turn = Checked(heads=heads, latent=latent, rope=rope, nope=nope, page_tokens=page, limit=512)
    append = turn.arena.append

    def appended(plan, c, r, *, layer, rotary=None):
        append(plan, c, r, layer=layer, rotary=rotary)
        n = int(plan.starts[-1])
        rows = turn.arena.rows[layer].flatten(0, 1)[plan.slots[:n]]
        assert torch.equal(rows[:, :latent], c[:n])
        if rotary is None:
            assert torch.equal(rows[:, latent:], r[:n])
        else:  # angles are good to 2^-22, products and their sum to 2^-23, one rounding
            want = turned(r[:n], plan.positions[:n], rotary)
            size = r[:n].double().abs().amax(1, keepdim=True)
            off = (rows[:, latent:].double() - want).abs()
            assert bool((off <= U * want.abs() + 2.0 ** -20 * size).all())

    turn.arena.append = appended
    x = example.run(turn, question=(5, 40, 1, 17), answer=3)
    assert x.shape == (4, turn.width) and bool(torch.isfinite(x).all())
    assert checked.count(40) == 2 and len(checked) == 2 * 4 * 4  # layers x steps x requests
    assert turn.tables.lens.tolist() == [256 + n + 3 for n in (5, 40, 1, 17)]

    # The positions come off to within a rounding to bf16, and the codes are within half
    # a step (a group's largest over 7, itself rounded to fp16) of that.
    (codes, scales), n = turn.harvest(1, 249, 50)
    assert n == 50 and codes.shape == (1, 2, 50 * (latent + rope) // 2)
    got = O.dequant_packed(codes.reshape(-1), scales.view(np.uint16).reshape(-1), 4)
    got = torch.from_numpy(got.astype(np.int32) << 16).view(torch.float32).reshape(2, 50, -1)
    at = torch.arange(249, 299, device=turn.device)
    for layer in range(2):
        rows = turn.arena.rows[layer].flatten(0, 1)[turn.slots(1, 249, 50)]
        want = torch.cat([rows[:, :latent].double(),
                          turned(rows[:, latent:], at, turn.rows, -1)], 1).cpu()
        size = float(rows.double().abs().max()) * 2 ** 0.5  # of a pair, turned
        assert float((got[layer].double() - want).abs().max()) <= size * (0.51 / 7 + 2 * U)

    free = lambda: int(turn.tables.cursor[1] - turn.tables.cursor[0])  # noqa: E731
    before = free()
    turn.release([1])
    assert free() == before + -(-(256 + 43) // page) and turn.tables.lens[1].item() == 0
    turn.admit(1, ((codes, scales), n))
    assert turn.tables.lens[1].item() == 50


def test_the_example_runs(capsys):
    load_example().main()
    text = capsys.readouterr().out
    assert "finite: True" in text and "[277, 56, 273, 289]" in text
