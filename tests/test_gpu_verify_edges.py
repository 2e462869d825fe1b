"""The test of drafted tokens where its definition or its threads can go apart: what the threads of a block decide by, and uniform numbers and probabilities at their ends."""
import numpy as np
import pytest

from test_gpu_sampling import logits
from test_gpu_verify import agree, device, drafter, engine, expected      # noqa: F401  (the fixture)

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


BELOW = np.float32(1.0 - 2.0 ** -24)


@pytest.mark.parametrize("settings", [(None, None, None, None), (1.0, 20, None, None), (0.9, 30, 0.95, 0.01), (1.0, None, 0.9, None), (1.0, None, 0.98, 0.001), (1.0, None, None, 0.02), (1.0, 2500, None, None),
                                      (1.0, 2500, 0.9, None), (1e4, None, None, None), (1e4, None, 0.9, None), (np.inf, 2000, None, None)])
@pytest.mark.parametrize("width", [3000, 40000])
def test_a_second_number_of_zero_takes_the_first_token_with_something_left(engine, width, settings):
    """The drafter is surer of the best tokens than the target: all of their weight is taken off, and 0 answers as the smallest number above it."""
    rng = np.random.default_rng(width)
    rows = 12
    x = rng.normal(0, 1.0, (rows, width)).astype(np.float32)
    x[9:] = np.float32(0.5)                                          # ties: the candidates are the first of the order
    order = np.argsort(-x, axis=1, kind="stable")
    ids = order[:, :6].copy()
    p = np.repeat(np.float32([[0.5, 0.25, 0.125, 0.0625, 0.03125, 0.03125]]), rows, 0)
    drafts = ids[np.arange(rows), np.arange(rows) % 3].copy()
    drafts[8] = -1
    zero, tiny = np.full((rows, 2), BELOW, np.float32), np.full((rows, 2), BELOW, np.float32)
    zero[:, 1], tiny[:, 1] = 0.0, 1e-30
    for candidates in ((ids, p), (ids[:, :1], np.full((rows, 1), 0.96875, np.float32)), None):
        want, _, _ = expected(x, width, [rows], drafts, candidates, settings, tiny)
        assert (want != drafts).any() and (want[:3] != order[:3, 0]).any()
        for u in (tiny, zero):
            got, _, _ = device(engine, x, width, [rows], drafts, candidates, settings, u)
            assert np.array_equal(got, want), (got.tolist(), want.tolist())


def test_the_largest_value_alone_beside_probabilities_above_one(engine):
    """Temperature 0: a token stays while its number times its drafter's probability is below one, in exact arithmetic. (A drafter's rounded probabilities may pass one by a step.)"""
    x = np.zeros((4, 50), np.float32)
    x[:, 17] = 1.0
    drafts = np.full(4, 17)
    step = np.float32(2.0 ** -23)
    p = np.array([[1 + step], [1 + step], [1.0], [1 + 2 * step]], np.float32)
    u = np.array([[1 - step, 0.5], [BELOW, 0.5], [BELOW, 0.5], [1 - 2 * step, 0.5]], np.float32)      # 1 - 2^-46, above 1, below 1, 1 - 2^-44
    got, accepted, following = device(engine, x, 50, [1, 1, 1, 1], drafts, (np.full((4, 1), 17), p), (0.0, None, None, None), u)
    assert got.tolist() == [-1, 17, -1, -1] and accepted.tolist() == [1, 0, 1, 1] and following.tolist() == [-1, 17, -1, -1]
