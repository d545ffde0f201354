"""Requests and scales at the edge of what the latent attention takes, against the definition of test_latent_attention.py (and its tolerances)."""
from __future__ import annotations

import pytest

from test_latent_attention import Batch, check

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
