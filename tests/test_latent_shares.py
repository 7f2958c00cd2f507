"""How a step over latent rows is cut into shares, on the CPU: the code that the plan's kernel
cuts them with, compiled for the host (latent_shares.cu).  Every tile's tokens are in one
part each, and what the join reads has been left by somebody, once."""

import random
import shutil
import subprocess
from pathlib import Path

import pytest

from graftrepository_b200 import build

HERE = Path(__file__).resolve().parent
SMS = 148


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not (shutil.which("nvcc") or Path("/usr/local/cuda/bin/nvcc").exists()):
        pytest.skip("no nvcc")
    exe = tmp_path_factory.mktemp("shares") / "shares"
    subprocess.run([build.nvcc(), *build.ARCH_FLAGS, "-std=c++17", "-O2", "-w",
                    "--expt-relaxed-constexpr", f"-I{build.INCLUDE}", "-o", str(exe),
                    str(HERE / "latent_shares.cu")], check=True)
    return exe


def shares(program, steps):
    """[(workers, whole tiles of each)] of steps (form, grow, heads, latent, [(rows, tokens)]);
    holds what must hold of each."""
    lines = []
    for form, grow, heads, latent, requests in steps:
        fresh, lens = zip(*requests)
        lines.append(" ".join(map(str, (form, grow, heads, latent, max(*fresh, 1), SMS, len(fresh),
                                        *fresh, *lens))))
    got = subprocess.run([str(program)], input="\n".join(lines), text=True, check=True,
                         capture_output=True).stdout.split("\n")[:-1]
    assert len(got) == len(steps)
    for line, step in zip(got, lines):
        workers, waves, *faults = map(int, line.split())
        assert not any(faults), (f"empty shares, steps, parts not left, left twice, not read: "
                                 f"{faults} of {workers} workers; step {step[:200]}")
    return [tuple(map(int, x.split()[:2])) for x in got]


SKEWED = [
    [(1, 300), (1, 1_000_000)] + [(1, 300)] * 3,
    [(256, 262_144)] * 3 + [(1, 100 + 6 * i) for i in range(9)],
    [(1, 400)] * 2 + [(256, 400_000)] + [(1, 400)] * 2,
    [(1, 2_000_000)] + [(1, 110 + i % 40) for i in range(700)],
    [(1, 110 + i % 40) for i in range(700)] + [(257, 3_000_000)],
]


@pytest.mark.parametrize("heads", [1, 3, 16, 40, 64, 128])
def test_whole_tiles_that_cost_very_different_amounts(program, heads):
    steps = [(1, 1, heads, 256, r) for r in SKEWED] + [(1, 0, heads, 256, r) for r in SKEWED]
    got = shares(program, steps)
    assert heads < 64 or all(waves > 0 for _, waves in got)


def test_the_plan_that_read_results_which_nobody_had_left(program):
    assert shares(program, [(1, 1, 64, 256, SKEWED[0])]) == [(SMS, 1)]


@pytest.mark.parametrize("form", [0, 1])
def test_random_steps(program, form):
    rng = random.Random(form)
    steps = []
    for _ in range(1500):
        requests = []
        for _ in range(rng.randrange(1, 40)):
            fresh = rng.choice([0, 1, 1, 2, rng.randrange(1, 300), rng.randrange(1, 2000)])
            held = int(2 ** rng.uniform(0, 16)) * rng.choice([1, 1, 1, 1, 1, 1, 20, 100])
            requests.append((fresh, fresh + held))
        grow = rng.randrange(4) > 0
        if not grow and rng.randrange(2):  # requests that hold nothing, asked all the same
            requests = [(n, 0 if rng.randrange(3) == 0 else t) for n, t in requests]
        if rng.randrange(3) == 0:
            requests = [(min(n, 4), t) for n, t in requests]
        steps.append((form, int(grow), rng.choice([1, 2, 5, 8, 16, 32, 40, 64, 128, 200]),
                      rng.choice([128, 256, 512]), requests))
    workers = {w for w, _ in shares(program, steps)}
    assert max(workers) == SMS or form == 0
