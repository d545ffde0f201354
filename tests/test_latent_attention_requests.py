"""Requests and scales at the edge of what the latent attention takes, against the definition of test_latent_attention.py (and its tolerances)."""
from __future__ import annotations

import pytest
import torch

from test_attention_operator_checks import OPS, accepts
from test_latent_attention import Batch, check, key_rows

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("heads,window", [(16, None), (64, 20)])
def test_requests_that_end_behind_the_rows_of_q(heads, window):
    """Of the last request q has only the first tokens, or none: they keep their positions."""
    b = Batch([300, 900, 40], [9, 30, 7], heads, 64, seed=26)
    want = b.want(window, 3)
    for tokens in (39, 38, 12, 9, 4):
        b.tokens, b.q = tokens, b.q[:tokens]
        out, lse = b.run(window, 3)
        check(out, lse, want[:tokens])


@pytest.mark.skipif(torch.cuda.is_available(), reason="accepted calls would launch on addresses that are not memory")
@pytest.mark.parametrize("name", ["paged", "sparse"])
def test_scales_that_are_no_number_once_divided_by_ln_2(name, monkeypatch):
    """The exponentials are powers of two: from 2 ** 128 * ln 2 = 2.3586e38 on every score would be infinite or NaN."""
    monkeypatch.setattr(torch.cuda, "_lazy_init", lambda: None)
    op, args, at = OPS[name]
    index = next(i for i, a in enumerate(args) if isinstance(a, float))
    for scale, fine in ((1e-45, True), (1.0, True), (2.35e38, True), (2.3585e38, True), (2.3587e38, False), (3e38, False), (3.402e38, False), (3.4e39, False), (1e-46, False)):
        changed = args[:index] + (scale,) + args[index + 1 :]
        for native in (True, False):
            assert accepts(op, changed, at, native, monkeypatch)[0] == fine, (scale, native)


@gpu
@pytest.mark.parametrize("scale", [2.0 ** -140, 1e-30])
def test_scores_that_are_all_but_equal(scale):
    b = Batch([70], [3], 8, 64, seed=27)
    out, lse = b.run(scale=scale)
    check(out, lse, b.want(scale=scale))


@gpu
def test_the_largest_scale():
    """Scores of 0 for one key and of -2.3e38 for the others, exact in 32 bits: the row is that key, with an lse of 0."""
    b = Batch([70], [3], 8, 64, seed=27)
    b.q[:] = 0
    b.q[:, :, 511] = 1.0
    raw = b.cache.view(-1)
    for j in range(70):
        at = b.slot(0, j) // 64 * b.cache.shape[1] + b.slot(0, j) % 64 * 576
        raw[at + 574 : at + 576] = torch.tensor([0.0 if j == 11 else -1.0], dtype=torch.bfloat16).view(torch.uint8)
    out, lse = b.run(scale=2.3e38, sink=False)
    assert torch.equal(out.double(), key_rows(b.cache, 64, [b.slot(0, 11)]).expand(3, 8, 512)) and (lse == 0).all()
