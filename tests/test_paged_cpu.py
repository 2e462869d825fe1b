"""The paged cache's host arithmetic without a GPU: which configurations and batches are taken, and how a batch's attention is dealt to blocks."""
import numpy as np
import pytest

import splosh_b200 as S
from splosh_b200.paged import debug_paged_plan, paged_check

CONFIG = dict(heads=4, kv_heads=2, head_dim=128, pages=8, page_tokens=32, max_sequences=2, max_rows=4, max_context=128)


def case_of(**more):
    with pytest.raises(S.EngineError) as caught:
        paged_check(**more)
    return caught.value.case


def test_configurations():
    for good in (dict(), dict(head_dim=64), dict(head_dim=256, heads=128, kv_heads=2), dict(page_tokens=256), dict(layout="token"), dict(rotary_dim=2), dict(rotary_dim=128), dict(window=1),
                 dict(strides=(3 * 2 * 32 * 192, 32 * 192, 192)), dict(max_context=1 << 30, page_tokens=256, max_sequences=1), dict(dtype="fp16", causal=False)):
        assert paged_check(**{**CONFIG, **good}) is False
    for bad in (dict(head_dim=96), dict(head_dim=0), dict(heads=5), dict(heads=0), dict(kv_heads=0), dict(heads=130), dict(heads=2048, kv_heads=64), dict(page_tokens=48), dict(page_tokens=512), dict(page_tokens=0), dict(pages=0),
                dict(rotary_dim=130), dict(rotary_dim=3), dict(rotary_dim=-2), dict(window=-1), dict(dtype="f32"), dict(max_rows=0), dict(max_rows=1 << 21), dict(max_sequences=0), dict(max_sequences=1 << 17),
                dict(max_context=0), dict(max_context=1 << 30, max_sequences=1 << 10), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(rotary_dim=64, rope_theta=0.0),
                dict(rotary_dim=64, rope_theta=float("inf")), dict(strides=(8192, 4096, 64)), dict(strides=(8192, 4100, 128)), dict(strides=(4096, 4096, 128)), dict(strides=(-8192, 4096, 128)), dict(strides=(1 << 40, 4096, 128)),
                dict(layout="channel"), dict(dtype="int8")):
        assert case_of(**{**CONFIG, **bad}) == "invalidArgument", bad


def test_batches():
    table = np.array([[0, 1, 9], [2, 3, 9]], np.int32)             # entries past a sequence's pages are not looked at
    assert paged_check([1, 1], [33, 20], table, **CONFIG) is False
    assert paged_check([0, 4], [0, 4], table, **CONFIG) is False
    assert paged_check([1, 1], [33, 20], np.array([[0, 1], [1, 3]], np.int32), **CONFIG) is True       # page 1 is written by both
    assert paged_check([1, 1], [33, 20], np.array([[2, 1], [2, 3]], np.int32), **CONFIG) is False      # page 2: written by the second alone, read by the first
    assert paged_check([1, 1], [33, 50], np.array([[2, 1], [2, 3]], np.int32), **CONFIG) is False      # a shared prefix that nobody writes to
    assert paged_check([3, 0], [33, 0], np.array([[1, 1], [2, 3]], np.int32), **CONFIG) is True        # one page twice among a sequence's own
    for case, rows, lengths, t in (("invalidRows", [2, 1], [1, 20], table), ("invalidRows", [-1, 1], [33, 20], table), ("contextExceeded", [1, 1], [129, 20], np.zeros((2, 5), np.int32)),
                                   ("invalidRows", [1, 1], [33, 20], np.array([[0, 8], [2, 3]], np.int32)), ("invalidRows", [1, 1], [33, 20], np.array([[0, -1], [2, 3]], np.int32)),
                                   ("invalidRows", [1, 1], [33, 20], np.array([[0], [2]], np.int32)), ("invalidRows", [0, 0], [33, 20], table), ("invalidRows", [3, 2], [33, 20], table),
                                   ("invalidRows", [1, 1, 1], [1, 1, 1], np.array([[0], [1], [2]], np.int32)), ("invalidRows", [1, -2147483648], [33, -2147483648], table)):
        assert case_of(rows=rows, lengths=lengths, page_table=t, **CONFIG) == case, (rows, lengths)
    for rows, lengths, t in (([1, 1], [33], table), ([1, 1], [33, 20], table[0]), ([1, 1], [33, 20], table[:1])):
        assert case_of(rows=rows, lengths=lengths, page_table=t, **CONFIG) == "invalidArgument"


def random_batch(rng):
    heads_of_kv, kv_heads = int(rng.choice([1, 3, 4, 6, 8, 64])), int(rng.choice([1, 2, 4, 8]))
    n = int(rng.integers(1, 12))
    rows = [int(x) for x in rng.choice([0, 1, 1, 1, 8, 16, 40, 300, 2048], n)]
    lengths = [r + int(rng.choice([0, 1, 127, 128, 1000, 9000, 40000])) for r in rows]
    return heads_of_kv * kv_heads, kv_heads, rows, lengths, int(rng.choice([0, 0, 1, 100, 128, 2048])), bool(rng.random() < 0.7)


@pytest.mark.parametrize("seed", range(60))
def test_every_visible_tile_is_done_once(seed):
    """Each (sequence, kv head, packed query row) meets every tile that holds a token it sees exactly once; a block's pieces are a stretch; pieces of shared rows have slots of their own, which
    one merge joins in order; no block carries much more than its share."""
    rng = np.random.default_rng(seed)
    heads, kv_heads, rows, lengths, window, causal = random_batch(rng)
    if not any(rows):
        rows[0], lengths[0] = 1, max(lengths[0], 1)
    blocks, group = int(rng.choice([1, 3, 132, 148])), heads // kv_heads
    begin, items, merges = debug_paged_plan(rows, lengths, blocks=blocks, heads=heads, kv_heads=kv_heads, head_dim=128, pages=1, page_tokens=256, window=window, causal=causal,
                                            max_sequences=len(rows), max_rows=max(sum(rows), 1), max_context=1 << 20)
    assert begin[0] == 0 and begin[-1] == len(items) and (np.diff(begin) >= 0).all()
    starts = np.concatenate([[0], np.cumsum(rows)])
    done = {}
    for s, row0, h, q0, count, t0, t1, slot in items.tolist():
        assert row0 == starts[s] and 0 <= h < kv_heads and q0 % 128 == 0 and 1 <= count <= 128 and q0 + count <= rows[s] * group and (count == 128 or q0 + count == rows[s] * group)
        assert 0 <= t0 < t1 <= -(-lengths[s] // 128)
        done.setdefault((s, h, q0, count), []).append((t0, t1, slot))
    expected = {(s, h, q0, min(128, rows[s] * group - q0)) for s in range(len(rows)) for h in range(kv_heads) for q0 in range(0, rows[s] * group, 128)}
    assert set(done) == expected
    joined = {}
    for row0, h, q0, count, slot, slots, *_ in merges.tolist():
        joined[(row0, h, q0, count)] = list(range(slot, slot + slots))
    used = []
    for (s, h, q0, count), pieces in done.items():
        base = lengths[s] - rows[s]
        first, last = base + q0 // group, base + (q0 + count - 1) // group
        low = max(0, first + 1 - window) if window else 0
        high = last + 1 if causal else lengths[s]
        assert pieces[0][0] == low // 128 and pieces[-1][1] == -(-high // 128)
        assert all(a[1] == b[0] for a, b in zip(pieces, pieces[1:]))
        slots = [p[2] for p in pieces]
        if len(pieces) == 1:
            assert slots == [-1] and (starts[s], h, q0, count) not in joined
        else:
            assert slots == joined.pop((starts[s], h, q0, count))
            used += slots
    assert not joined and sorted(used) == list(range(len(used))) and len(used) <= 2 * blocks and len(merges) <= blocks
    # A block's load: its tiles, two more a piece and the joining; no block carries much more than its share, or than the least that is not cut.
    def cost(item):
        rows_there = 0 if item[7] < 0 or item[4] <= 16 else 1 if item[4] <= 64 else 2
        return int(item[6] - item[5]) + 2 + rows_there
    load = [sum(cost(i) for i in items[a:b]) for a, b in zip(begin, begin[1:])]
    share = (sum(int(i[6] - i[5]) for i in items) + 4 * (len(expected) + blocks)) / blocks
    assert max(load) <= 2 * share + 14
    for (s, h, q0, count), pieces in done.items():
        if len(pieces) > 1:
            assert min(t1 - t0 for t0, t1, _ in pieces) >= (1 if count <= 16 else 3 if count <= 64 else 5)


def test_a_single_sequence_is_spread_over_the_blocks():
    """One decoding session: pieces of a tile or two on as many blocks; one long prompt: every block within two percent of its share."""
    begin, items, _ = debug_paged_plan([1], [1024], heads=8, kv_heads=2, head_dim=128, pages=1, max_sequences=1, max_rows=1, max_context=1024)
    assert len(items) == 16 and (np.diff(begin) <= 1).all()
    begin, items, _ = debug_paged_plan([2048], [26624], heads=24, kv_heads=4, head_dim=256, pages=1, max_sequences=1, max_rows=2048, max_context=1 << 16)
    tiles = np.array([sum(int(i[6] - i[5]) for i in items[a:b]) for a, b in zip(begin, begin[1:])])
    assert tiles.max() <= 1.02 * tiles.mean()
