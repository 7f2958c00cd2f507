"""The example that runs mount, plan, append, attend, read and release together:
its attention against the formula in 64 bits over the rows that the arena gives
back, and the mounted grafts against what was packed."""

import importlib.util
import math
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import oracle as O  # noqa: E402

pytestmark = pytest.mark.gpu


def load_example():
    path = Path(__file__).resolve().parent.parent / "examples" / "paged_turn.py"
    spec = importlib.util.spec_from_file_location("paged_turn", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def slots_of(turn, request, n):
    page = turn.tables.page_tokens
    at = torch.arange(n, device=turn.device)
    return turn.tables.table[request].long()[at // page] * page + at % page


@pytest.mark.parametrize("head_dim,group,page", [(128, 4, 64), (64, 5, 16)])
def test_a_turn(head_dim, group, page):
    example = load_example()
    checked = []

    class Checked(example.PagedTurn):
        def attend(self, plan, q, layer):
            out = super().attend(plan, q, layer)
            lens, starts = plan.lens.tolist(), plan.starts.tolist()
            for r, n in enumerate(lens):
                a, b = starts[r], starts[r + 1]
                k, v = (t.double().repeat_interleave(group, 1) for t in self.arena.read(
                    slots_of(self, r, n), layer=layer, dtype=torch.float32))
                z = torch.einsum("ihd,thd->iht", q[a:b].double(), k) * head_dim ** -0.5
                seen = n - (b - a) + 1 + torch.arange(b - a, device=self.device)
                hide = torch.arange(n, device=self.device)[None] >= seen[:, None]
                w = torch.softmax(z.masked_fill(hide[:, None], -math.inf), 2)
                want = torch.einsum("iht,thd->ihd", w, v)
                mag = torch.einsum("iht,thd->ihd", w, v.abs())
                # the exponent is off by at most 2^-17 sum |q k| scale + 2^-20, a weight
                # by twice that and fp16's 2^-11, the result by bf16's 2^-8; a weight
                # below fp16's normal range by 2^-25 of the largest
                size = torch.einsum("ihd,thd->iht", q[a:b].double().abs(), k.abs()).amax(2)
                e = (2.0 ** -17 * size * head_dim ** -0.5 + 2.0 ** -20)[:, :, None]
                tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2 * e) * mag * (1 + 2.0 ** -8) + \
                    n * 2.0 ** -25 * float(v.abs().max()) + 2.0 ** -25
                assert bool(((out[a:b].double() - want).abs() <= tol).all()), (layer, r)
                checked.append(b - a)
            return out

    turn = Checked(kv_heads=4, group=group, head_dim=head_dim, page_tokens=page)
    x = example.run(turn, question=(5, 40, 1, 17), answer=3)
    assert x.shape == (4, turn.width) and bool(torch.isfinite(x).all())
    assert checked.count(40) == 2 and len(checked) == 2 * 4 * 4  # layers x steps x requests
    assert turn.tables.lens.tolist() == [256 + n + 3 for n in (5, 40, 1, 17)]

    # the grafts' values, 4 bits and then 8: within half a step of the page's scale
    # and one rounding to bf16
    _, (codes, scales), _ = example.random_grafts(turn, 2, 128, seed=2)
    want = O.dequant_packed(codes.reshape(-1), scales.view(np.uint16).reshape(-1), 4)
    want = torch.from_numpy(want.astype(np.int32) << 16).view(torch.float32)
    want = want.reshape(2, 2, 4, 128, head_dim).permute(1, 0, 3, 2, 4).reshape(2, 256, 4, head_dim)
    for layer in range(2):
        _, v = turn.arena.read(slots_of(turn, 2, 256), layer=layer, dtype=torch.float32)
        step = float(turn.arena.v_scales[layer].max())
        assert float((v.cpu() - want[layer]).abs().max()) <= 0.5 * step * (1 + 2.0 ** -7)

    # harvest and release
    (codes, scales), _ = turn.harvest(1, 256, 43)
    assert codes.shape == (1, 2 * 4, 43 * head_dim // 2)
    free = lambda: int(turn.tables.cursor[1] - turn.tables.cursor[0])  # noqa: E731
    before = free()
    turn.release([1])
    assert free() == before + -(-(256 + 43) // page) and turn.tables.lens[1].item() == 0
    turn.admit(1, example.random_grafts(turn, 1, 128, seed=9))
    assert turn.tables.lens[1].item() == 128


def test_the_example_runs(capsys):
    load_example().main()
    text = capsys.readouterr().out
    assert "finite: True" in text and "[277, 128, 273, 289]" in text
