"""How far a value of the cache in 4 bits is from what was written, for groups of every magnitude.

In units of the group's scale the largest value is at most 6, and e2m1 values are 1/2 apart up to 2, 1 apart up to 4, 2 apart up to 6: an error of 1/4, 1/2 or 1 happens beside
values of at least 1/4, 5/2 and 5.  Above the floor of the scale, 2^-126, the largest is more than 3, so every error is at most a fifth of it (1/2 where it is below 5: a sixth).
At the floor it can be any: errors of 1/2 and 1 are a fifth of 5/2 and of 5 still, and that of 1/4 is 2^-128."""
from __future__ import annotations

import pytest
import torch

from test_mxfp4_cache import E2M1, Insertion, mx_rows, quantised

gpu = pytest.mark.gpu
FLOOR = 2.0 ** -128
# groups of one largest value and its parts, 31 of them on and beside the borders between e2m1 values
PARTS = torch.tensor([1.0] + [i / 32 for i in range(1, 32)])


def every_group():
    top = torch.arange(1, 0x7F80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    groups = (top.double()[:, None] * PARTS).to(torch.bfloat16)
    tiny = torch.arange(1, 257, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).view(-1, 32)  # every subnormal value, in groups of neighbours
    groups = torch.cat([groups, tiny])
    return torch.cat([groups, groups[: -len(groups) % 14]]).view(-1, 448)


def check(rows, x):
    rows, x = rows.reshape(-1, 32), x.double().reshape(-1, 32)
    top = x.abs().amax(-1, keepdim=True)
    bound = torch.where(top < 1.25 * 2.0 ** -126, torch.full_like(top, FLOOR), top / 5)
    assert ((rows - x).abs() <= bound).all()
    small = ((rows - x).abs() > top / 5).any(-1)
    assert small.any() and (top[small] < 1.25 * 2.0 ** -126).all()  # where a fifth is not kept
    limit = 3.5 * 2.0 ** 126
    assert ((rows.to(torch.bfloat16).isinf()) == (x.abs() >= limit)).all() and (x == limit).any()  # 3.5 is a tie, which goes to 4


def test_definition():
    x = every_group()
    data, codes = quantised(x)
    rows = torch.stack([E2M1[(data & 15).long()], E2M1[(data >> 4).long()]], -1).view(-1, 448)
    check(rows * torch.exp2(codes.double() - 127).repeat_interleave(32, -1), x)


@gpu
@pytest.mark.parametrize("odd", [0, 1])
def test_writer(odd):
    x = every_group()
    i = Insertion(len(x), 0, skip=0.0)
    i.kv = torch.cat([x, i.kv[:, 448:]], 1)
    _, storage = i.run(odd=odd)
    check(mx_rows(i.cache_of(storage, 368), i.bs, i.slots.tolist())[:, :448], x)
