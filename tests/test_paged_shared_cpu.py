"""Batches whose sequences begin with the same pages, and caches of e4m3, without a GPU: what is taken, and how the attention is dealt to blocks and joined."""
import numpy as np
import pytest

import splosh_b200 as S
from splosh_b200.paged import debug_paged_plan, debug_paged_plan_shared, paged_check

CONFIG = dict(heads=4, kv_heads=2, head_dim=128, pages=16, page_tokens=32, max_sequences=4, max_rows=8, max_context=256)


def case_of(**more):
    with pytest.raises(S.EngineError) as caught:
        paged_check(**more)
    return caught.value.case


def test_configurations_of_e4m3():
    for good in (dict(), dict(head_dim=64), dict(head_dim=256, heads=128, kv_heads=2), dict(layout="token"), dict(window=1), dict(strides=(3 * 2 * 32 * 192, 32 * 192, 192)), dict(strides=(2 * 32 * 144, 32 * 144, 144))):
        assert paged_check(**{**CONFIG, "dtype": "e4m3", **good}) is False
    for bad in (dict(head_dim=96), dict(strides=(2 * 32 * 136, 32 * 136, 136)), dict(strides=(2 * 32 * 128 + 8, 32 * 128, 128))):      # 16 bytes are sixteen codes
        assert case_of(**{**CONFIG, "dtype": "e4m3", **bad}) == "invalidArgument", bad


def test_groups():
    table = np.array([[0, 1, 2, 9], [0, 1, 3, 9], [4, 5, 6, 9], [4, 7, 8, 9]], np.int32)
    rows, lengths = [1, 2, 0, 1], [80, 90, 70, 96]
    for good in ((), [(2, 64)], [(2, 32), (2, 32)], [(1, 64), (1, 64), (2, 32)], [(2, 0), (2, 32)], [(4, 0)], [(2, 64), (1, 64)]):
        assert paged_check(rows, lengths, table, groups=good, **CONFIG) is False, good
    for bad in ([(0, 32)], [(-1, 32)], [(5, 0)], [(2, 64), (3, 0)], [(2, 48)], [(2, -32)], [(2, 96)], [(2, 64), (2, 64)], [(4, 32)], [(1, 32), (2, 32)], [(2147483647, 0)], [(2, 2147483616)], [(3, 64)]):
        assert case_of(rows=rows, lengths=lengths, page_table=table, groups=bad, **CONFIG) == "invalidRows", bad
    # The shared tokens lie in front of the new rows.
    assert paged_check([1, 1], [65, 66], table[:2], groups=[(2, 64)], **CONFIG) is False
    assert case_of(rows=[2, 1], lengths=[65, 66], page_table=table[:2], groups=[(2, 64)], **CONFIG) == "invalidRows"


def random_batch(rng):
    group, kv_heads = int(rng.choice([1, 3, 4, 6, 8, 64])), int(rng.choice([1, 2, 4, 8]))
    rows, lengths, groups = [], [], []
    for _ in range(int(rng.integers(1, 4))):
        n, shared = int(rng.choice([1, 2, 7, 12, 40, 130])), 256 * int(rng.choice([0, 1, 8, 40, 160]))
        rows += [int(x) for x in rng.choice([0, 1, 1, 1, 2, 8, 16, 40, 300], n)] if rng.random() < 0.5 else [int(rng.choice([1, 1, 4]))] * n
        lengths += [shared + r + int(rng.choice([0, 1, 127, 128, 1000])) for r in rows[len(lengths):]]
        groups.append((n, shared))
    for _ in range(int(rng.choice([0, 3]))):
        rows.append(int(rng.choice([0, 1, 20]))); lengths.append(rows[-1] + int(rng.choice([0, 5, 4000])))
    return group * kv_heads, kv_heads, rows, lengths, groups, int(rng.choice([0, 0, 0, 200])), bool(rng.random() < 0.7)


@pytest.mark.parametrize("dtype", ["bf16", "e4m3"])
@pytest.mark.parametrize("seed", range(80))
def test_every_row_meets_every_tile_once_and_is_joined_from_all_its_pieces(seed, dtype):
    rng = np.random.default_rng(seed)
    heads, kv_heads, rows, lengths, groups, window, causal = random_batch(rng)
    if not any(rows):
        rows[0] = 1; lengths[0] += 1
    blocks, group = int(rng.choice([1, 3, 148])), heads // kv_heads
    config = dict(heads=heads, kv_heads=kv_heads, head_dim=128, dtype=dtype, pages=1, page_tokens=256, window=window, causal=causal, max_sequences=len(rows), max_rows=max(sum(rows), 1), max_context=1 << 20)
    begin, items, records, partial_rows, joint = debug_paged_plan_shared(rows, lengths, groups, blocks=blocks, **config)
    assert begin[0] == 0 and begin[-1] == len(items) and (np.diff(begin) >= 0).all()
    starts = np.concatenate([[0], np.cumsum(rows)])
    total = int(starts[-1])
    owner = np.repeat(np.arange(len(rows)), rows)
    # The tiles that each (row, head) meets, by the place its sums are left at (-1: it is answered by its piece alone).
    met = {}
    places = np.zeros(partial_rows, np.int32)
    for s, row0, h, q0, count, t0, t1, slot in items.tolist():
        assert 0 <= t0 < t1 and 1 <= count <= 128
        if slot >= 0:
            places[slot:slot + count] += 1
        for i in range(count):
            row, head = row0 + (q0 + i) // group, h * group + (q0 + i) % group
            met.setdefault((row, head), []).append((t0, t1, slot + i if slot >= 0 else -1))
            assert row < total
    assert (places == 1).all()
    joined = {}
    for row0, q0, h, count, *sides in records.tolist():
        for i in range(count):
            key = (row0 + (q0 + i) // group, h * group + (q0 + i) % group)
            assert key not in joined
            joined[key] = sorted(first + n * step + i for first, step, pieces in (sides[:3], sides[3:]) for n in range(pieces))
    assert len(met) == total * heads
    for (row, head), pieces in met.items():
        s = owner[row]
        unit = (row - starts[s]) * group + head % group                       # the tiles go by the row's unit of 128 packed rows
        q0 = unit // 128 * 128
        count, base = min(128, rows[s] * group - q0), lengths[s] - rows[s]
        first, last = base + q0 // group, base + (q0 + count - 1) // group
        low, high = (max(0, first + 1 - window) if window else 0) // 128, -(-(last + 1 if causal else lengths[s]) // 128)
        tiles = sorted(pieces)
        assert tiles[0][0] == low and tiles[-1][1] == high and all(a[1] == b[0] for a, b in zip(tiles, tiles[1:]))
        left = sorted(p[2] for p in pieces)
        assert joined.pop((row, head), [-1]) == left
    assert not joined
    if window or not any(n > 1 and t >= 128 for n, t in groups):
        assert not joint
    if not joint and dtype == "e4m3" and 8 < max(rows) * group <= 128:
        assert partial_rows <= 2 * blocks * min(128, sum(rows) * group)       # what is set aside for batches without groups
    elif not joint:
        plain = debug_paged_plan(rows, lengths, blocks=blocks, **config)[1]
        assert (plain[:, :7] == items[:, :7]).all()


def test_a_prefix_is_read_once_for_128_packed_rows():
    """Forty-eight decoding sequences of 8,192 shared tokens: 288 packed rows a kv head meet them in three blocks of rows, not 48."""
    begin, items, records, _, joint = debug_paged_plan_shared([1] * 48, [8192 + 300] * 48, [(48, 8192)], heads=24, kv_heads=4, head_dim=256, pages=1, max_sequences=48, max_rows=48, max_context=1 << 16)
    assert joint
    tiles = sum(int(i[6] - i[5]) for i in items)
    assert tiles == 4 * (3 * 64 + 48 * 3)
    load = [sum(int(i[6] - i[5]) for i in items[a:b]) for a, b in zip(begin, begin[1:])]
    assert max(load) <= 2 * tiles / 148 + 4
    # Two sequences that share too little to be worth it.
    assert not debug_paged_plan_shared([1] * 2, [300] * 2, [(2, 256)], heads=24, kv_heads=4, head_dim=256, pages=1, max_sequences=2, max_rows=2, max_context=1 << 16)[4]


def test_over_a_cache_of_e4m3_few_rows_meet_a_prefix_48_at_a_time():
    """Two verify blocks of four rows, six heads a kv head, over 20,480 shared tokens: their 48 packed rows are one block's. With a sequence of nine rows (54 packed) beside them the batch's form has 128."""
    config = dict(heads=24, kv_heads=4, head_dim=256, dtype="e4m3", pages=1, max_sequences=16, max_rows=128, max_context=1 << 16)
    for rows, width in (([4] * 6, 48), ([4] * 6 + [9], 128), ([1] * 16, 48)):
        begin, items, records, _, joint = debug_paged_plan_shared(rows, [20480 + 300] * len(rows), [(len(rows), 20480)], **config)
        assert joint
        packed = 6 * sum(rows)
        over = [(int(i[3]), int(i[4])) for i in items if i[6] <= 160]
        assert set(over) <= {(q, min(width, packed - q)) for q in range(0, packed, width)}
        assert sum(int(i[6] - i[5]) for i in items if i[6] <= 160) == 4 * 160 * -(-packed // width)
        joined = np.zeros((sum(rows) * 6, 4), int)
        for row0, q0, h, count, *_ in records.tolist():
            joined[6 * row0 + q0:6 * row0 + q0 + count, h] += 1
        assert (joined == 1).all()
