"""Ragged questions in the example of a turn: as many rows as requests, but not one
each, requests that ask nothing, and a step that is refused."""

import pytest

torch = pytest.importorskip("torch")

from graftrepository_b200 import _lib  # noqa: E402
from test_paged_turn_gpu import load_example  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("question", [(2, 0, 1, 1), (1, 1, 1, 1), (0, 0, 1, 0), (0, 9, 0, 2)])
def test_as_many_tokens_join_as_were_given(question):
    example = load_example()
    turn = example.PagedTurn(kv_heads=2, group=2, head_dim=64, limit=512)
    x = example.run(turn, question=question, answer=3)
    assert x.shape == (sum(n > 0 for n in question), turn.width)
    assert turn.tables.lens.tolist() == [256 + n + (3 if n else 0) for n in question]


def test_a_step_that_is_refused_says_so():
    example = load_example()
    turn = example.PagedTurn(kv_heads=2, group=2, head_dim=64, limit=512)
    x = torch.zeros((600, turn.width), dtype=torch.bfloat16, device=turn.device)
    with pytest.raises(_lib.GrmB200Error, match="room"):
        turn.step(x[:512], [600, 0, 0, 0])
