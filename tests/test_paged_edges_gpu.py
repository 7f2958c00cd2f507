"""Edges of the 8-bit paged arena: the ends of the prompt kernel's rings, weights
far below a row's largest, streams other than the current one, steps that are
overtaken, waits that give up.

The 64-bit reference, the makers of arenas and the tolerances of attention are
those of test_paged_gpu.py, where they are derived."""

import pytest

torch = pytest.importorskip("torch")

from test_paged_gpu import run_attention  # noqa: E402

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ ends of the rings

@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("tokens", [959, 1024, 1025, 1088, 2112])
def test_wide_heads_past_the_end_of_the_ring_of_scales(tokens, page):
    """At head_dim 256 a block holds the scales of 16 key tiles of 64 tokens: the
    last place, the first one again, and twice around."""
    run_attention([tokens] * 19, [40] * 19, heads=4, group=4, dim=256, page=page, seed=tokens)
