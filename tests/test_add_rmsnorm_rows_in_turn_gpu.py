"""The residual norm where a CTA takes several rows in turn, the next one on its way to shared memory while one is worked on: against the definition of
test_fused_add_rmsnorm_quant_fp8.py, bit for bit.  Three to ten rows a CTA, for every number of pieces a thread, rows that divide evenly and that do
not, and rows of which no two fit (16384 columns)."""
from __future__ import annotations

import pytest
import torch

import flaggems_vllm as fg
from test_fused_add_rmsnorm_quant_fp8 import DEV, EPS, definition, rows, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,cols,group", [(4097, 7168, 128), (4099, 4096, 4096), (2500, 2048, 128), (5001, 512, 64), (3700, 320, 32), (700, 10240, 256), (3001, 2304, 128),
                                               (2900, 1544, 1544), (700, 16384, 128), (650, 16640, 16640)])
@pytest.mark.parametrize("dtype,weight_type,pow2,gap", [(torch.bfloat16, torch.bfloat16, True, 0), (torch.bfloat16, torch.float32, False, 24), (torch.float16, torch.float16, False, 8)])
def test_many_rows_a_cta(tokens, cols, group, dtype, weight_type, pow2, gap):
    g = torch.Generator().manual_seed(tokens + cols + group)
    x, xc = rows(tokens, cols, dtype, cols + gap, g)
    res, resc = rows(tokens, cols, dtype, cols + 2 * gap, g, 3.0)
    whole, before = res._base if gap else res, (res._base if gap else res).clone()
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(weight_type)
    want = definition(xc, resc, w, group, pow2)
    x_q, scales = fg.fused_add_rmsnorm_quant_fp8(x, res, w.to(DEV), EPS, group, gap != 0, pow2)
    assert same(res, want[0]) and same(scales, want[2]) and same(x_q, want[1]) and same(x, xc)
    assert not gap or torch.equal(whole[:, cols:], before[:, cols:])


@pytest.mark.parametrize("tokens,cols", [(4097, 7168), (5001, 512), (700, 16384)])
def test_many_rows_without_a_residual(tokens, cols):
    g = torch.Generator().manual_seed(tokens)
    x, xc = rows(tokens, cols, torch.bfloat16, cols, g)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(torch.bfloat16)
    want = definition(xc, None, w, 128, True)
    x_q, scales = fg.fused_add_rmsnorm_quant_fp8(x, None, w.to(DEV), EPS, 128, False, True)
    assert same(scales, want[2]) and same(x_q, want[1]) and same(x, xc)
