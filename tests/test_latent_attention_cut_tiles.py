"""Tiles of the latent attention that are cut into pieces and joined: lists of more than 15 blocks of 48 keys, in every form a tile can have.  Against
the definition of test_latent_attention.py (and its tolerances, which know nothing of pieces: the join adds sums in 32 bits, as a tile does)."""
from __future__ import annotations

import math

import pytest
import torch

from flaggems_vllm import _native
from test_latent_attention import DEV, SCALE, Batch, check, definition, key_rows

pytestmark = pytest.mark.gpu


def run(b, *args, **kwargs):
    """The batch's call, which must have been two launches: the pieces, and their join."""
    before = _native.launch_count()
    results = b.run(*args, **kwargs)
    assert _native.launch_count() == before + 2
    return results


@pytest.mark.parametrize("heads", [1, 8, 16, 24, 32, 65, 96, 128])
@pytest.mark.parametrize("window,first", [(None, 0), (1500, 40), (800, 1000)])
def test_several_tokens_a_tile(heads, window, first):
    """Tiles of 64, 8, 4 and 2 tokens and of one, of two requests; masks that start and end inside pieces."""
    b = Batch([2500, 900], [37, 5], heads, 64, seed=30 + heads)
    out, lse = run(b, window, first)
    check(out, lse, b.want(window, first))


@pytest.mark.parametrize("sink", [False, True])
def test_strided_results(sink):
    """Heads cut out of a wider tensor, tokens and heads exchanged, lse transposed; nothing between the rows is written."""
    b = Batch([1900, 40], [6, 3], 24, 64, seed=40)
    q = torch.full((9, 40, 1024), 3.0, dtype=torch.bfloat16, device=DEV)[:, 8:32, 256:768]
    q.copy_(b.q)
    holder, lses = torch.full((24, 9, 520), 7.0, dtype=torch.bfloat16, device=DEV), torch.full((24, 18), 7.0, device=DEV)
    out, lse = run(b, q=q, out=holder.transpose(0, 1)[..., :512], lse=lses[:, ::2].t(), sink=sink)
    check(out, lse, b.want(sink=sink))
    assert (holder[..., 512:] == 7).all() and (lses[:, 1::2] == 7).all()


@pytest.mark.parametrize("scale", [SCALE, 0.7])
@pytest.mark.parametrize("heads", [16, 128])
def test_maxima_that_move_from_piece_to_piece(scale, heads):
    """Scores that rise along one request's keys and fall along the other's."""
    b = Batch([3000, 2900], [6, 6], heads, 64, seed=41)
    for r, n in enumerate(b.seq_lens):
        for j in range(n):
            step = j / n if r == 0 else 1 - j / n
            raw, at = b.cache[b.slot(r, j) // 64], b.slot(r, j) % 64
            raw[at * 576 + 448 : at * 576 + 576] = torch.full((64,), 4 * step).to(torch.bfloat16).view(torch.uint8)
    b.q[:, :, 448:] = b.q[:, :, 448:].abs() * 4
    out, lse = run(b, scale=scale)
    check(out, lse, b.want(scale=scale))


@pytest.mark.parametrize("heads", [8, 16, 128])
@pytest.mark.parametrize("poison", [0xFF, 0x7F])
def test_a_key_that_is_no_number_in_one_piece(heads, poison):
    """Seen by all rows of the request (in its first, a middle and its last piece), or by the later tokens of a tile alone: only rows that see it are NaN."""
    b = Batch([2000, 1000], [11, 4], heads, 64, seed=42)
    want, clean = b.want(), b.cache.clone()
    for j in (5, 700, 1500, 1984, 1988, 1991, 1994, 1999):
        slot = b.slot(0, j)
        b.cache[slot // 64, slot % 64 * 576 : slot % 64 * 576 + 576] = poison
        b.cache[slot // 64, 64 * 576 + slot % 64 * 8 : 64 * 576 + slot % 64 * 8 + 8] = poison
        out, lse = run(b)
        seeing = [i for i in range(11) if 1989 + i >= j]
        assert torch.isnan(out[seeing]).all() and torch.isnan(lse[seeing]).all()
        rest = [i for i in range(15) if i not in seeing]
        check(out[rest], lse[rest], [want[i] for i in rest])
        b.cache.copy_(clean)


@pytest.mark.parametrize("heads", [16, 128])
def test_an_infinite_value_in_one_piece(heads):
    """Scores of +inf and -inf, one key of many: NaN in all of the row, or at least where the value is."""
    b = Batch([2000, 1000], [11, 4], heads, 64, seed=43)
    want = b.want()
    slot = b.slot(0, 800)
    raw = b.cache[slot // 64]
    raw[slot % 64 * 576 + 448 : slot % 64 * 576 + 450] = torch.tensor([math.inf], dtype=torch.bfloat16).view(torch.uint8)
    out, lse = run(b)
    assert torch.isnan(out[:11, :, 448]).all()
    below = b.q[:11, :, 448] < 0  # a score of -inf: the other dimensions are those of the other keys
    assert below.any() and (~below).any() and torch.isnan(out[:11][~below]).all() and torch.isfinite(lse[:11][below]).all()
    check(out[11:], lse[11:], want[11:])


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_queries_that_are_no_numbers_stay_in_their_row(value):
    b = Batch([1800], [9], 8, 64, seed=44)
    want = b.want()
    b.q[4, 3, 100] = value
    out, lse = run(b)
    rows = [(i, h) for i in range(9) for h in range(8) if (i, h) != (4, 3)]
    check(torch.stack([out[i, h] for i, h in rows])[:, None], torch.stack([lse[i, h] for i, h in rows])[:, None],
          [tuple(t[h : h + 1] for t in want[i]) for i, h in rows])
    assert torch.isnan(out[4, 3]).all()


@pytest.mark.parametrize("heads", [16, 64, 128])
def test_pieces_without_any_key(heads):
    """Pages outside the cache leave whole pieces empty: at the start, in the middle and at the end of a tile, and all of another."""
    b = Batch([3000, 1500], [7, 3], heads, 64, seed=45)
    keys = [key_rows(b.cache, 64, [b.slot(r, j) for j in range(n)]) for r, n in enumerate(b.seq_lens)]
    pages = {*range(0, 8), *range(17, 33), *range(42, 47)}
    for p in pages:
        b.table[0, p] = -1 if p % 2 else b.cache.shape[0]
    b.table[1] = -1
    out, lse = run(b)
    want = [definition(b.q[i], keys[0][[j for j in range(2994 + i) if j // 64 not in pages]], SCALE, b.sink) for i in range(7)]
    want += [definition(b.q[7 + i], keys[1][:0], SCALE, b.sink) for i in range(3)]
    check(out, lse, want)
    assert (out[7:] == 0).all() and (lse[7:] == -math.inf).all()


@pytest.mark.parametrize("heads,lens,new", [(16, [5000, 800, 0, 760, 70], [9, 5, 0, 4, 2]), (8, [900] * 30, [3] * 30), (128, [770, 721, 720, 1200], [2, 1, 3, 5])])
def test_many_tiles_some_of_which_are_cut(heads, lens, new):
    """Pieces of several tiles on a CTA: ends, whole tiles and heads; rows in front of the first request and behind the last stay."""
    b = Batch(lens, new, heads, 64, seed=46, extra_rows=6)
    want, n = b.want(), sum(new)
    b.q, b.starts = b.q.roll(2, 0), b.starts + 2
    out, lse = run(b)
    check(out[2 : n + 2], lse[2 : n + 2], want)
    for rows in (slice(0, 2), slice(n + 2, None)):
        assert (out[rows] == 7).all() and (lse[rows] == 7).all()


def test_the_same_call_gives_the_same_bits():
    """Pieces are joined in a fixed order."""
    b = Batch([2500, 900], [37, 5], 16, 64, seed=47)
    first = run(b, 1500, 40)
    for _ in range(5):
        again = run(b, 1500, 40)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
