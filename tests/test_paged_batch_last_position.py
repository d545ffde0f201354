"""The token at position 2^31 - 1.  Lengths stop at 2^31 - 1, so it is behind the last one that is counted and has a block only if it shares that of the token in front
of it; it must never get one that another request took."""
from __future__ import annotations

import pytest
import torch

import flaggems_vllm as fg
from test_paged_batch import DEV, INT_MAX, extended, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [False, True])
def test_a_page_that_nobody_took_gives_no_slot(in_place):
    """Blocks of 2^31 - 1 tokens: position 2^31 - 1 is alone on page 1, which the lengths do not reach.  Request 1 takes the only block."""
    context, table, num_free = i32([INT_MAX, 0]).to(DEV), i32([[4, -7], [-7, -7]]).to(DEV), i32([1]).to(DEV)
    new, free = i32([1, 2]).to(DEV), i32([9]).to(DEV)
    out = None
    if in_place:
        out = [torch.zeros(3, dtype=torch.int32, device=DEV), context, *(torch.zeros(3, dtype=torch.int64, device=DEV) for _ in range(2)),
               torch.zeros(3, dtype=torch.int32, device=DEV), num_free, torch.zeros(1, dtype=torch.int32, device=DEV)]
    got = fg.extend_block_tables(context, new, table, free, num_free, INT_MAX, 3, out)
    assert got.slot_mapping.tolist() == [-1, 9 * INT_MAX, 9 * INT_MAX + 1] and got.position_ids.tolist() == [INT_MAX, 0, 1]
    assert got.seq_lens.tolist() == [INT_MAX, 2] and got.num_free.tolist() == [0] and got.num_missing.tolist() == [0] and table.tolist() == [[4, -7], [9, -7]]


@pytest.mark.parametrize("bs", [1 << 30, (1 << 30) + 1, INT_MAX - 1])
def test_a_page_that_the_lengths_reach_gives_its_own(bs):
    """Elsewhere positions 2^31 - 2 and 2^31 - 1 share a page, held or taken by this call."""
    context, new, rows = [INT_MAX, INT_MAX - 1, bs - 1], [1, 2, 2], [[4, 5], [6, 7], [8, -7]]
    table = i32(rows).to(DEV)
    got = fg.extend_block_tables(i32(context).to(DEV), i32(new).to(DEV), table, i32([11, 12]).to(DEV), i32([2]).to(DEV), bs, 5)
    want, rows = extended(context, new, rows, [11, 12], 2, bs, 5)
    assert [t.tolist() for t in got] == list(want) and table.tolist() == rows
    assert got.slot_mapping[0].item() == 5 * bs + INT_MAX - bs and min(want[3]) > 0
