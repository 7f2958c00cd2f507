"""Steps whose whole tiles cost the workers very different amounts, on the GPU: what the join
reads has been written by this step.  Tolerances as in test_latent_gpu."""

import pytest

torch = pytest.importorskip("torch")

from test_latent_gpu import Turn, close, i32  # noqa: E402
from test_latent_shares import SKEWED  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests", [SKEWED[0], SKEWED[2]])
def test_every_part_that_is_joined_has_been_left(requests):
    cached, fresh = [t - n for n, t in requests], [n for n, _ in requests]
    turn = Turn(cached, fresh, 64, 128, 32, 128, nope=64)
    want = turn.want(True, True)
    turn.plan.work.fill_(255)  # NaN wherever nobody writes
    turn.tables.plan(turn.plan, i32(fresh))
    got = turn.expanded()
    turn.plan.check()
    close(got, want)
    assert all(torch.equal(a, b) for a, b in zip(got, turn.expanded()))
