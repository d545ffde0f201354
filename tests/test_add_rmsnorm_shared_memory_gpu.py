"""The residual norm's launches and the shared memory they ask for.  From 48 KiB on, with what the kernel has of its own, a launch needs the function's consent, which
lasts for the process: the widths that lie on that line are tried in a process of their own, and widths of one kernel by two threads at once."""
from __future__ import annotations

import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import flaggems_vllm as fg
from test_fused_add_rmsnorm_quant_fp8 import DEV, EPS, definition, rows, same

pytestmark = pytest.mark.gpu

WIDTHS = """
import sys
sys.path[:0] = {paths!r}
import torch
import flaggems_vllm as fg
from test_fused_add_rmsnorm_quant_fp8 import DEV, EPS, definition, rows, same
for tokens, widths in ((3, (5888, 5896, 6016, 6144, 6152)), (149, (5120, 5128, 5632, 6144, 6152))):
    for cols in widths:
        for dtype, weight_type in ((torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32)):
            g = torch.Generator().manual_seed(cols)
            x, xc = rows(tokens, cols, dtype, cols, g)
            res, resc = rows(tokens, cols, dtype, cols, g, 3.0)
            w = (1 + 0.3 * torch.randn(cols, generator=g)).to(weight_type)
            want = definition(xc, resc, w, cols, False)
            x_q, scales = fg.fused_add_rmsnorm_quant_fp8(x, res, w.to(DEV), EPS, cols)
            assert same(res, want[0]) and same(scales, want[2]) and same(x_q, want[1]), (tokens, cols, dtype)
"""


def test_widths_that_take_just_48_kib():
    here = Path(__file__).resolve().parent
    code = WIDTHS.format(paths=[str(here), str(here.parent / "flaggems-vllm_b200")])
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("widths", [(6656, 8192), (8320, 16384)])
def test_two_threads_with_rows_of_different_width(widths):
    cases, errors = [], []
    for cols in widths:
        g = torch.Generator().manual_seed(cols)
        x, xc = rows(150, cols, torch.bfloat16, cols, g)
        w = torch.ones(cols, dtype=torch.bfloat16)
        cases.append((x, w.to(DEV), definition(xc, None, w, 128, True)))
    torch.cuda.synchronize()

    def work(x, w, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(1500):
                    x_q, scales = fg.fused_add_rmsnorm_quant_fp8(x, None, w, EPS, 128, False, True)
                assert same(scales, want[2]) and same(x_q, want[1])
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=c) for c in cases]
    [t.start() for t in threads], [t.join() for t in threads]
    assert not errors, errors
