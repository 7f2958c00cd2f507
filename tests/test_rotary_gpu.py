"""Rotary positions on the GPU: rotation put on and taken off, and appends into the
8-bit arena that rotate on the way, against the formula in 64 bits.

Tolerances: an angle within an eighth of a turn is rounded three times in fp32
(2^-24 of it each, so 3 x 2^-24 x pi / 4) after an exact reduction, its sine and
cosine a few times more: below 2^-22 in all.  With the amplitude, two products and a
sum a value is off by less than 2^-21 a (|x1| + |x2|), and by half a step of its
type (fp16: 2^-25 where it is subnormal).  A code is off by half a step of the scale
and by what the value is off."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from graftrepository_b200 import paged_arena as PA  # noqa: E402
from graftrepository_b200.rotary import Rotary, rotary_frequencies  # noqa: E402

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SCALINGS = {
    "none": None,
    "linear": dict(kind="linear", factor=3.0),
    "ntk": dict(kind="ntk", factor=8.0),
    "yarn": dict(kind="yarn", factor=16.0, original=512),
    "factors": dict(kind="factors", factors=None, amplitude=1.19),
}
SMALL = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def scaling(name, dim):
    s = SCALINGS[name]
    if name == "factors":
        s = dict(s, factors=[1.0 + 0.3 * i for i in range(dim // 2)])
    return s


def members(x, layout):
    if layout == "half":
        return x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
    return x[..., 0::2], x[..., 1::2]


def joined(a, b, layout):
    return torch.cat([a, b], -1) if layout == "half" else torch.stack([a, b], -1).flatten(-2)


def turned(x, positions, dim, offset, layout, scale, inverse=False):
    """(y, |x1| + |x2| times the gain, at both places) in 64 bits, on the CPU."""
    f, a = rotary_frequencies(dim, scaling=scale)
    x = x.double().cpu()
    t = positions.double().cpu()[:, None] * torch.tensor(f, dtype=torch.float64)
    c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
    if inverse:
        s, a = -s, 1 / a
    takes, puts = layout, layout
    if layout == "pair_swap":
        takes, puts = ("half", "interleaved") if inverse else ("interleaved", "half")
    part = x[:, :, offset:offset + dim]
    x1, x2 = members(part, takes)
    y, mag = x.clone(), torch.zeros_like(x)
    y[:, :, offset:offset + dim] = joined((x1 * c - x2 * s) * a, (x2 * c + x1 * s) * a, puts)
    m = (x1.abs() + x2.abs()) * a
    mag[:, :, offset:offset + dim] = joined(m, m, puts)
    return y, mag


def close(got, want, mag):
    half = torch.finfo(got.dtype).eps / 2
    tol = half * want.abs() + 2.0 ** -21 * (1 + half) * mag + SMALL[got.dtype]
    off = (got.double().cpu() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("layout", ["half", "interleaved", "pair_swap"])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,head_dim,offset,dim,scale", [
    (1, 1, 2, 0, 2, "none"), (3, 5, 96, 64, 32, "factors"), (61, 40, 96, 64, 32, "yarn"),
    (700, 7, 128, 0, 128, "ntk"), (1111, 3, 80, 16, 64, "linear"), (5, 2, 37, 3, 18, "none"),
    (2, 1, 4100, 2, 4096, "none"), (40, 300, 64, 0, 64, "factors")])
def test_rotate(layout, kind, tokens, heads, head_dim, offset, dim, scale):
    gen = torch.Generator(device=DEV).manual_seed(tokens + dim)
    x = torch.randn((tokens, heads, head_dim), device=DEV, generator=gen).to(kind)
    positions = torch.randint(0, 1 << 20, (tokens,), device=DEV, generator=gen, dtype=torch.int32)
    positions[0] = 2 ** 31 - 1 if tokens > 1 else 0
    rotary = Rotary(dim, offset=offset, layout=layout, scaling=scaling(scale, dim), device=DEV)
    # the last pairs of 4,096 turn 10^-4 radians a position: products in 64 bits hold
    # 2^31 of them to 2^-22
    y = rotary.rotate(x, positions)
    close(y, *turned(x, positions, dim, offset, layout, scaling(scale, dim)))
    z = rotary.rotate(y, positions, inverse=True)
    close(z, *turned(y, positions, dim, offset, layout, scaling(scale, dim), inverse=True))
    if layout != "pair_swap":
        held = x.clone()
        assert rotary.rotate(held, positions, out=held) is held
        assert torch.equal(held, y)


def test_angles_of_far_positions():
    """Position by position against exact arithmetic on the frequency's own bits."""
    from fractions import Fraction
    rotary = Rotary(64, device=DEV)
    where = [0, 1, 2, 1000, 2 ** 20 + 1, 2 ** 24 - 1, 2 ** 30 + 7, 2 ** 31 - 1]
    x = torch.zeros((len(where), 1, 64), device=DEV)
    x[:, :, :32] = 1.0
    got = rotary.rotate(x, torch.tensor(where, dtype=torch.int32, device=DEV)).double().cpu()
    two_pi = 2 * Fraction("3.14159265358979323846264338327950288419716939937511")
    for i, p in enumerate(where):
        for j, f in enumerate(rotary.frequencies):
            t = float((Fraction(f) * p / two_pi) % 1) * 2 * math.pi
            assert abs(float(got[i, 0, j]) - math.cos(t)) < 2.0 ** -21
            assert abs(float(got[i, 0, 32 + j]) - math.sin(t)) < 2.0 ** -21


def test_rows_without_a_position_and_other_strides():
    gen = torch.Generator(device=DEV).manual_seed(3)
    rotary = Rotary(64, offset=16, device=DEV)
    wide = torch.randn((9, 3, 4, 104), device=DEV, generator=gen).to(torch.bfloat16)
    x, to = wide[:, 0], wide[:, 1]  # side by side in one buffer
    positions = torch.tensor([5, -1, 0, 7, -1, 9, 3, -7, -1], dtype=torch.int32, device=DEV)
    before = wide.clone()
    got = rotary.rotate(x, positions, out=to)
    assert got is to and torch.equal(wide[:, 0], before[:, 0])
    assert torch.equal(wide[:, 2], before[:, 2])
    want, mag = turned(x, positions.clamp(min=0), 64, 16, "half", None)
    none = (positions < 0).cpu()
    want[none], mag[none] = x.double().cpu()[none], 0.0
    close(to, want, mag)
    assert torch.equal(to[none], x[none])
    # heads before tokens, a broadcast head, an odd offset
    flipped = wide[:, 0].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(rotary.rotate(flipped, positions), to)
    one = wide[:, 0, :1].expand(9, 4, 104)
    assert torch.equal(rotary.rotate(one, positions)[:, 2], to[:, 0])
    odd = torch.empty(9 * 4 * 104 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(9, 4, 104)
    odd.copy_(x)
    assert torch.equal(rotary.rotate(odd, positions), to)
    held = before[:, 0].clone()
    rotary.rotate(held, positions, out=held)
    assert torch.equal(held, to)
    assert rotary.rotate(wide[:0, 0], positions[:0]).shape == (0, 4, 104)


def test_rotate_refuses():
    rotary = Rotary(32, offset=8, device=DEV)
    x = torch.zeros((4, 2, 64), device=DEV)
    at = torch.zeros(4, dtype=torch.int32, device=DEV)
    for bad, where, text in (
            (x.double(), at, "float32"), (x[0], at, "tokens, heads"), (x[:, :, :32], at, "rotated"),
            (x.cpu(), at, "x is on"), (x, at.long(), "positions"), (x, at[:3], "positions"),
            (x, at.cpu(), "positions"), (x.transpose(1, 2), at, "rotated"),
            (x[:, :, ::1].transpose(0, 2).contiguous().transpose(0, 2), at, "contiguous")):
        with pytest.raises(ValueError, match=text):
            rotary.rotate(bad, where)
    for out, text in ((x[:, :1], "out must"), (x.half(), "out must"), (x.cpu(), "out must"),
                      (torch.zeros((4, 1, 64), device=DEV).expand(4, 2, 64), "overlap")):
        with pytest.raises(ValueError, match=text):
            rotary.rotate(x, at, out=out)
    flat = torch.zeros(4 * 2 * 64 + 64, device=DEV)
    with pytest.raises(ValueError, match="overlaps"):
        rotary.rotate(flat[:512].view(4, 2, 64), at, out=flat[32:544].view(4, 2, 64))
    with pytest.raises(ValueError, match="in place"):
        Rotary(32, layout="pair_swap", device=DEV).rotate(x, at, out=x)


def test_rotate_on_another_stream_and_in_a_graph():
    gen = torch.Generator(device=DEV).manual_seed(8)
    x = torch.randn((33, 4, 64), device=DEV, generator=gen)
    at = torch.arange(33, dtype=torch.int32, device=DEV)
    rotary = Rotary(64, layout="interleaved", device=DEV)
    want = rotary.rotate(x, at)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = rotary.rotate(x, at, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotary.rotate(x, at, out=out)
    x.mul_(2.0)
    graph.replay()
    assert torch.equal(out, 2.0 * want)  # powers of two round alike


# -------------------------------------------------- append into the 8-bit arena

def ceil(a, b):
    return -(-a // b)


@pytest.mark.parametrize("head_dim,offset,dim,layout", [
    (64, 0, 64, "half"), (64, 0, 32, "interleaved"), (64, 32, 16, "half"),
    (128, 0, 128, "interleaved"), (128, 0, 96, "half"), (128, 64, 64, "half"),
    (256, 0, 256, "half"), (256, 16, 64, "interleaved")])
@pytest.mark.parametrize("page,heads,steps", [(16, 3, (1, 1, 1)), (64, 8, (90, 1, 37)),
                                              (128, 1, (300, 2)), (32, 5, (5, 6, 7))])
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
def test_append_rotates(head_dim, offset, dim, layout, page, heads, steps, kind):
    rng = np.random.default_rng(head_dim + dim + page)
    requests, most = 4, max(steps)
    width = ceil(sum(steps), page) + 1
    tables = PA.PageTables(requests, requests * width, width, page_tokens=page, device=DEV)
    arena = PA.PagedArena(1, requests * width, heads, head_dim, page_tokens=page, device=DEV)
    plain = PA.PagedArena(1, requests * width, heads, head_dim, page_tokens=page, device=DEV)
    rotary = Rotary(dim, offset=offset, layout=layout, scaling=SCALINGS["yarn"], device=DEV)
    tokens = requests * most
    plan = tables.make_plan(tokens, kv_heads=heads, query_heads=heads, head_dim=head_dim,
                            max_fresh=most)
    held = [torch.zeros((0, heads, head_dim), dtype=torch.float64) for _ in range(requests)]
    mags = [torch.zeros((0, heads, head_dim), dtype=torch.float64) for _ in range(requests)]
    last = None
    for step in steps:
        fresh = [step, max(step - 1, 0), rng.integers(0, step + 1).item(), step]
        kv = torch.from_numpy(rng.standard_normal((tokens, 2, heads, head_dim))).to(DEV)
        kv = (kv * float(rng.uniform(0.5, 2))).to(kind)
        k, v = kv[:, 0], kv[:, 1]
        tables.plan(plan, torch.tensor(fresh, dtype=torch.int32, device=DEV))
        arena.append(plan, k, v, rotary=rotary)
        first = [t.clone() for t in (arena.k_codes, arena.k_scales, arena.v_codes)]
        arena.append(plan, k, v, rotary=rotary)  # a step twice is the same step
        assert all(torch.equal(a, b) for a, b in
                   zip(first, (arena.k_codes, arena.k_scales, arena.v_codes)))
        plain.append(plan, k, v)
        tables.commit(plan)
        plan.check()
        want, mag = turned(k, plan.positions.clamp(min=0), dim, offset, layout, SCALINGS["yarn"])
        starts = plan.starts.tolist()
        for r in range(requests):
            held[r] = torch.cat([held[r], want[starts[r]:starts[r + 1]]])
            mags[r] = torch.cat([mags[r], mag[starts[r]:starts[r + 1]]])
        last = plan
    last.check()
    # values are not rotated: the plain append's codes and scales
    assert torch.equal(arena.v_codes, plain.v_codes)
    assert torch.equal(arena.v_scales, plain.v_scales)
    lens, table = tables.lens.tolist(), tables.table.tolist()
    for r in range(requests):
        assert lens[r] == held[r].shape[0]
        for j in range(ceil(lens[r], page)):
            rows = held[r][j * page:(j + 1) * page].transpose(0, 1)      # [heads, n, head_dim]
            off = 2.0 ** -21 * mags[r][j * page:(j + 1) * page].transpose(0, 1)
            codes = arena.k_codes[0, table[r][j], :, :rows.shape[1]].double().cpu()
            scale = arena.k_scales[0, table[r][j]].double().cpu()
            top = rows.abs().amax((1, 2)) / 127
            assert bool(((scale - top).abs() <= off.amax((1, 2)) / 127 + 2.0 ** -23 * top).all())
            # half a step for each time that the page was written, once for every
            # step that reached into it
            times = 1 + sum(1 for _ in steps)
            err = (codes * scale[:, None, None] - rows).abs()
            assert bool((err <= scale[:, None, None] * (0.5 * times + 2.0 ** -15) + off).all())


def test_an_append_that_turns_nothing_is_the_plain_one():
    tables = PA.PageTables(2, 8, 4, page_tokens=64, device=DEV)
    plan = tables.make_plan(150, kv_heads=2, query_heads=2, head_dim=128)
    still = Rotary(128, scaling=dict(kind="linear", factor=1e30), device=DEV)
    one, two = (PA.PagedArena(1, 8, 2, 128, device=DEV) for _ in range(2))
    gen = torch.Generator(device=DEV).manual_seed(5)
    for fresh in ([100, 50], [3, 0], [1, 1]):
        kv = torch.randn((2, 150, 2, 128), device=DEV, generator=gen).to(torch.float16)
        tables.plan(plan, torch.tensor(fresh, dtype=torch.int32, device=DEV))
        one.append(plan, kv[0], kv[1], rotary=still)
        two.append(plan, kv[0], kv[1])
        tables.commit(plan)
        for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
            assert torch.equal(getattr(one, name), getattr(two, name)), name


def test_a_row_without_a_number_takes_its_page_with_it():
    tables = PA.PageTables(1, 4, 4, page_tokens=16, device=DEV)
    plan = tables.make_plan(40, kv_heads=2, query_heads=2, head_dim=64)
    arena = PA.PagedArena(1, 4, 2, 64, page_tokens=16, device=DEV)
    k = torch.ones((40, 2, 64), dtype=torch.bfloat16, device=DEV)
    k[20, 1, 5] = math.inf
    tables.plan(plan, torch.tensor([40], dtype=torch.int32, device=DEV))
    arena.append(plan, k, torch.ones_like(k), rotary=Rotary(64, device=DEV))
    got, v = arena.read(plan.slots, dtype=torch.float32)
    bad = torch.zeros((40, 2), dtype=torch.bool, device=DEV)
    bad[16:32, 1] = True
    assert torch.equal(torch.isnan(got).any(2), bad) and torch.equal(torch.isnan(got).all(2), bad)
    assert bool(torch.isfinite(v).all())


def test_append_refuses():
    tables = PA.PageTables(1, 4, 4, page_tokens=16, device=DEV)
    plan = tables.make_plan(4, kv_heads=2, query_heads=2, head_dim=64)
    arena = PA.PagedArena(1, 4, 2, 64, page_tokens=16, device=DEV)
    k = torch.ones((4, 2, 64), dtype=torch.bfloat16, device=DEV)
    tables.plan(plan, torch.tensor([4], dtype=torch.int32, device=DEV))
    for rotary in (Rotary(32, layout="pair_swap", device=DEV), Rotary(40, device=DEV),
                   Rotary(32, offset=8, device=DEV), Rotary(64, offset=16, device=DEV)):
        with pytest.raises(ValueError, match="multiples of 16"):
            arena.append(plan, k, k, rotary=rotary)
