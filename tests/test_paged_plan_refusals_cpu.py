"""What the plan of a batch with groups is not made for: it would read behind the caller's arrays."""
import pytest

import splosh_b200 as S
from splosh_b200.paged import debug_paged_plan_shared

CONFIG = dict(heads=4, kv_heads=2, head_dim=128, pages=16, page_tokens=32, max_sequences=4, max_rows=8, max_context=256)


def test_batches_and_groups_that_are_refused():
    assert debug_paged_plan_shared([1, 1], [40, 40], [(2, 32)], **CONFIG)[0][-1] > 0
    for rows, lengths, groups in (([1, 1], [40, 40], [(3, 0)]), ([1, 1], [40, 40], [(1, 32), (2, 0)]), ([1, 1], [40, 40], [(2147483647, 0)]), ([1, 1], [40, 40], [(0, 32)]), ([1, 1], [40, 40], [(-1, 32)]),
                                  ([1, 1], [40, 40], [(2, -32)]), ([1, 1], [40, 40], [(2, 64)]), ([1, 9], [40, 40], [(2, 32)]), ([-1, 1], [40, 40], []), ([1, 41], [40, 40], [])):
        with pytest.raises(S.EngineError) as caught:
            debug_paged_plan_shared(rows, lengths, groups, **CONFIG)
        assert caught.value.case == "invalidRows", (rows, lengths, groups)
