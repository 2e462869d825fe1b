"""The test of drafted tokens where its definition or its threads can go apart: what the threads of a block decide by."""
import numpy as np
import pytest

from test_gpu_sampling import logits
from test_gpu_verify import agree, device, drafter, engine      # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [3000, 20011, 120001])
def test_rows_whose_token_is_decided_in_front_of_where_top_p_ends(engine, width):
    """The first block's threads go by the place of top-p's end, and a token far in front of it is decided from that place on: all of them have to have read the place, in every run."""
    rng = np.random.default_rng(width)
    rows = 64
    x = logits(rng, rows, width)
    drafts, candidates = drafter(rng, x, width, 8, 0.3)
    u = np.stack([np.where(np.arange(rows) % 2 == 0, 0.01, 0.999), rng.random(rows)], 1).astype(np.float32)
    first, _, _ = agree(engine, x, width, [rows], drafts, candidates, (1.0, None, 0.9, None), u)
    assert (first < 0).any() and (first >= 0).any()
    for _ in range(40):
        again, _, _ = device(engine, x, width, [rows], drafts, candidates, (1.0, None, 0.9, None), u)
        assert np.array_equal(again, first)
