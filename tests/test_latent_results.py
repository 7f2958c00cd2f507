"""Results that are given to latent attention: not over what the call reads, and not over
each other."""

import pytest

torch = pytest.importorskip("torch")

from graftrepository_b200 import latent_arena as LA


def test_results_over_what_is_read_and_over_each_other():
    arena = LA.LatentArena.__new__(LA.LatentArena)
    memory = torch.zeros(4096)
    a, b, c = memory[:1024], memory[1024:2048], memory[2048:]
    arena._apart(a, b, q=c)
    arena._apart(a, b, q=c[:512], rows=c[512:])
    for out, lse, read, text in (
            (a, b, dict(q=memory[1000:1100]), "out overlaps q"),
            (a, b, dict(q=c, rows=memory[2047:2050]), "lse overlaps rows"),
            (a, b, dict(q=c, weights=memory[:1]), "out overlaps weights"),
            (a, memory[1023:1030], dict(q=c), "out overlaps lse"),
            (a, a, dict(q=c), "out overlaps lse")):
        with pytest.raises(ValueError, match=text):
            arena._apart(out, lse, **read)


@pytest.mark.gpu
@pytest.mark.parametrize("expanded", [False, True])
def test_calls_with_results_that_overlap(expanded):
    from test_latent_gpu import Turn, close

    turn = Turn([70, 300], [2, 1], 16, 256, 32, nope=64)
    call = turn.expanded if expanded else turn.attend
    close(call(), turn.want(True, expanded))
    wide, T = 64 if expanded else 256, turn.T
    one = torch.zeros(2 * T * 16 * wide, dtype=turn.kind, device=turn.arena.device)
    out = one[:T * 16 * wide].view(T, 16, wide)
    over = one[T * 16 * wide - 64:].view(torch.float32)[:T * 16].view(T, 16)
    beside = one[T * 16 * wide:].view(torch.float32)[:T * 16].view(T, 16)
    with pytest.raises(ValueError, match="out overlaps lse"):
        call(out=out, lse=over)
    rows = turn.arena.rows.view(-1)
    with pytest.raises(ValueError, match="out overlaps rows"):
        call(out=rows[:T * 16 * wide].view(T, 16, wide))
    with pytest.raises(ValueError, match="lse overlaps rows"):
        call(lse=rows.view(torch.float32)[:T * 16].view(T, 16))
    if expanded:
        w = turn.weights.view(-1)
        with pytest.raises(ValueError, match="out overlaps weights"):
            call(out=w[:T * 16 * wide].view(T, 16, wide))
    got = call(out=out, lse=beside)
    assert got[0] is out and got[1] is beside
    close(got, turn.want(True, expanded))
