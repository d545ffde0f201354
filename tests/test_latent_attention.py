"""Attention over the paged latent cache against its definition in 64 bits.

Tolerances.  With the weights p_j (sum over the seen keys at most 1) and A = sum_j p_j |k_j| per dimension, the kernel may round each
unnormalised weight to bf16 (half a step: 2^-8 of it) before the second product, and rounds the result once: |error| <= 2^-8 A + 2^-8 |out|.
A score is a sum of 512 exact products in 32 bits, off by at most d = 512 * 2^-23 * scale * sum |q| |k| (steps rounded or cut, in any order); it
changes a weight by the factor e^(+-2d).  What 32-bit sums of n weights and products add, and the exponential's 2^-21, is below
(n + 8) * 2^-23 A.  An lse is off by d + (n + 8) * 2^-23 + 2^-22 |lse|."""
from __future__ import annotations

import math

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native

gpu = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 512 ** -0.5


def make_cache(blocks, block_size, g, pitch=None, extremes=False):
    """Random cache bytes on the CPU: finite values, scale codes around 1 (or over the whole range that keeps bf16 finite)."""
    pitch = pitch or block_size * 584
    cache = torch.full((blocks, pitch), 0xFF, dtype=torch.uint8)
    data = cache[:, : block_size * 576].view(blocks, block_size, 576)
    nope = torch.randint(0, 256, (blocks, block_size, 448), generator=g, dtype=torch.uint8)
    data[..., :448] = torch.where((nope & 0x7F) == 0x7F, nope ^ 1, nope)
    data[..., 448:] = torch.randn(blocks, block_size, 64, generator=g).to(torch.bfloat16).view(torch.uint8)
    codes = cache[:, block_size * 576 : block_size * 584].view(blocks, block_size, 8)
    low, high = (0, 128) if extremes else (116, 121)
    codes[...] = torch.randint(low, high, (blocks, block_size, 8), generator=g, dtype=torch.uint8)
    return cache


E4M3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def key_rows(cache, block_size, slots):
    """[n, 512] in 64 bits, values as the cache's reader gives them (bf16)."""
    out = torch.empty(len(slots), 512, dtype=torch.float64)
    for i, slot in enumerate(slots):
        raw, at = cache[slot // block_size], slot % block_size
        data = raw[at * 576 : at * 576 + 576]
        codes = raw[block_size * 576 + at * 8 : block_size * 576 + at * 8 + 7].double()
        out[i, :448] = E4M3[data[:448].long()] * torch.exp2(codes - 127).repeat_interleave(64)
        out[i, 448:] = data[448:].clone().view(torch.bfloat16).double()
    return out


def definition(q, keys, scale, sink):
    """q [heads, 512], keys [n, 512] -> out, lse, and the error bounds of both."""
    heads, n = q.shape[0], keys.shape[0]
    if n == 0:
        return torch.zeros(heads, 512).double(), torch.full((heads,), -math.inf).double(), torch.zeros(heads, 512).double(), torch.zeros(heads).double()
    q = q.double()
    s = q @ keys.t() * scale
    lse = torch.logsumexp(s, -1)
    total = lse if sink is None else torch.logaddexp(lse, sink.double())
    p = torch.exp(s - total[:, None])
    out, a = p @ keys, p @ keys.abs()
    d = (q.abs() @ keys.abs().t()).amax(-1, keepdim=True) * scale * 512 * 2.0 ** -23
    bound = (2.0 ** -8 + torch.expm1(2 * d) + (n + 8) * 2.0 ** -23) * a + 2.0 ** -8 * out.abs() + 2.0 ** -130
    return out, lse, bound, d[:, 0] + (n + 8) * 2.0 ** -23 + 2.0 ** -22 * lse.abs() + 2.0 ** -22


def check(got, got_lse, want):
    out, lse, bound, lse_bound = (torch.stack(t) for t in zip(*want))
    worst = ((got.double() - out).abs() / bound.clamp(min=1e-300)).max().item() if got.numel() else 0.0
    assert not torch.isnan(got).any() and (got.double() - out).abs().le(bound).all(), f"{worst} of the bound"
    finite = torch.isfinite(lse)
    assert torch.equal(finite, torch.isfinite(got_lse)) and (got_lse[~finite] == -math.inf).all()
    assert (got_lse.double() - lse).abs()[finite].le(lse_bound[finite]).all()


class Batch:
    """Requests with ragged contexts and chunks over a shuffled cache."""

    def __init__(self, seq_lens, new, heads, block_size, seed=0, extra_rows=0, pitch=None, extremes=False, extra_pages=1):
        g = torch.Generator().manual_seed(seed)
        self.seq_lens, self.new, self.heads, self.bs = seq_lens, new, heads, block_size
        pages = [-(-max(n, 0) // block_size) for n in seq_lens]
        self.cache = make_cache(sum(pages) + 2, block_size, g, pitch, extremes)
        order = torch.randperm(sum(pages) + 2, generator=g).to(torch.int32)
        self.table = torch.full((len(seq_lens), max(pages + [0]) + extra_pages), 1 << 30, dtype=torch.int32)  # pages behind the end are never read
        at = 0
        for r, n in enumerate(pages):
            self.table[r, :n] = order[at : at + n]
            at += n
        self.starts = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)
        self.tokens = sum(new) + extra_rows
        self.q = torch.randn(self.tokens, heads, 512, generator=g).to(torch.bfloat16)
        self.sink = torch.randn(heads, generator=g)

    def slot(self, r, j):
        return int(self.table[r, j // self.bs]) * self.bs + j % self.bs

    def seen(self, r, p, window, first):
        return [j for j in range(p + 1) if window is None or j > p - window or j < first]

    def want(self, window=None, first=0, sink=True, scale=SCALE):
        rows = []
        for r, n in enumerate(self.new):
            keys = key_rows(self.cache, self.bs, [self.slot(r, j) for j in range(max(self.seq_lens[r], 0))])
            for i in range(n):
                seen = self.seen(r, self.seq_lens[r] - n + i, window, first)
                rows.append(definition(self.q[int(self.starts[r]) + i], keys[seen], scale, self.sink if sink else None))
        return rows

    def run(self, window=None, first=0, sink=True, scale=SCALE, out=None, lse=None, q=None):
        lse = torch.full((self.tokens, self.heads), 7.0, device=DEV) if lse is None else lse
        out = torch.full((self.tokens, self.heads, 512), 7.0, dtype=torch.bfloat16, device=DEV) if out is None else out
        q = self.q.to(DEV) if q is None else q
        got = fg.paged_latent_attention(q, self.cache.to(DEV), self.table.to(DEV), torch.tensor(self.seq_lens, dtype=torch.int32, device=DEV),
                                        self.starts.to(DEV), self.bs, scale, window, first, self.sink.to(DEV) if sink else None, out, lse)
        torch.cuda.synchronize()
        assert got.data_ptr() == out.data_ptr() and _native.device_error() == 0
        return out.cpu(), lse.cpu()


@gpu
@pytest.mark.parametrize("heads", [1, 8, 24, 64, 65, 96, 128, 200])
@pytest.mark.parametrize("lengths,new", [([1], [1]), ([63, 64, 65], [1, 1, 1]), ([300, 5, 129], [1, 1, 1]), ([130, 70, 9], [70, 3, 9])])
def test_causal(heads, lengths, new):
    b = Batch(lengths, new, heads, 64, seed=heads)
    out, lse = b.run()
    check(out, lse, b.want())


@gpu
@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (7, 0), (64, 4), (100, 70), (128, 4), (1000, 3), (3, 1000), (1 << 40, 1 << 40)])
@pytest.mark.parametrize("heads", [16, 128])
def test_window_and_first_tokens(window, first, heads):
    b = Batch([330, 3, 130, 200], [40, 3, 1, 9], heads, 64, seed=1)
    out, lse = b.run(window, first)
    check(out, lse, b.want(window, first))


@gpu
@pytest.mark.parametrize("block_size,pitch", [(1, 592), (16, None), (16, 16 * 584 + 48), (50, None), (64, None), (256, None)])
def test_block_sizes(block_size, pitch):
    b = Batch([150, 70], [5, 2], 32, block_size, seed=2, pitch=pitch)
    out, lse = b.run(64, 2)
    check(out, lse, b.want(64, 2))


@gpu
def test_requests_without_tokens_or_keys_and_rows_behind_the_last():
    """A request that brings no tokens, one whose tokens lie before its sequence (no keys for some rows), rows behind the last request."""
    b = Batch([70, 0, 90, 2, -3], [2, 0, 0, 4, 2], 16, 64, seed=3, extra_rows=5)
    out, lse = b.run()
    check(out[:8], lse[:8], b.want())
    assert (out[2:4] == 0).all() and (lse[2:4] == -math.inf).all() and (out[6:8] == 0).all()
    assert (out[8:] == 7).all() and (lse[8:] == 7).all()


@gpu
@pytest.mark.parametrize("heads,new", [(64, [150, 40]), (128, [70, 4]), (128, [71, 4]), (16, [139, 5]), (16, [146, 5])])
def test_short_lists_with_and_without_a_cta_for_each(heads, new):
    """No tile is long enough to be cut: fewer or as many tokens (times groups of heads) as CTAs, or more."""
    b = Batch([200, 60], new, heads, 64, seed=14)
    out, lse = b.run(16, 2)
    check(out, lse, b.want(16, 2))


@gpu
@pytest.mark.parametrize("window", [16, None])
def test_rows_in_front_of_the_first_request(window):
    """Rows that belong to no request lie in front of the first one and behind the last, and stay as they are."""
    b = Batch([80, 30], [3, 6], 16, 64, seed=15, extra_rows=6)
    want = b.want(window)
    b.q = b.q.roll(4, 0)
    b.starts += 4
    out, lse = b.run(window)
    check(out[4:13], lse[4:13], want)
    for rows in (slice(0, 4), slice(13, None)):
        assert (out[rows] == 7).all() and (lse[rows] == 7).all()


@gpu
@pytest.mark.parametrize("heads", [16, 64, 128])
def test_long_contexts(heads):
    """Work split over the keys of few rows; ragged."""
    b = Batch([9000, 77, 3001], [1, 1, 1], heads, 64, seed=4)
    out, lse = b.run()
    check(out, lse, b.want())


@gpu
@pytest.mark.parametrize("scale", [SCALE, 0.7, 1e-4])
def test_scores_that_rise_and_fall(scale):
    """The maximum moves often, far, and backwards: keys along the queries' common direction, ascending and descending."""
    b = Batch([700, 700], [3, 3], 64, 64, seed=5)
    for r in range(2):
        for j in range(700):
            step = j if r == 0 else 700 - j
            raw, at = b.cache[b.slot(r, j) // 64], b.slot(r, j) % 64
            raw[at * 576 + 448 : at * 576 + 576] = (torch.ones(64) * (step / 700) * 4).to(torch.bfloat16).view(torch.uint8)
    b.q[:, :, 448:] = b.q[:, :, 448:].abs() * 4
    out, lse = b.run(scale=scale)
    check(out, lse, b.want(scale=scale))


@gpu
def test_sinks():
    """Sinks far above and below the scores, infinite ones, none."""
    b = Batch([80, 3], [5, 3], 12, 64, seed=6)
    b.sink = torch.tensor([0.0, 50.0, -50.0, 200.0, -200.0, float("-inf"), 3.0, 1.0, 0.5, -1.0, 80.0, float("inf")])
    out, lse = b.run()
    want = b.want()
    check(out[:, :11], lse[:, :11], [tuple(t[:11] for t in row) for row in want])
    assert (out[:, 11] == 0).all()
    out, lse = b.run(sink=False)
    check(out, lse, b.want(sink=False))


@gpu
def test_extreme_scale_codes():
    """Powers of two from 2^-127 on: values that are subnormal in bf16, zero scores, wide ranges within a key."""
    b = Batch([100, 64], [2, 64], 16, 64, seed=7, extremes=True)
    out, lse = b.run(scale=0.001)
    # keys are what the cache's reader gives: below bf16's normal range its half step is 2^-134, inside the absolute part of the bound
    check(out, lse, b.want(scale=0.001))


@gpu
@pytest.mark.parametrize("heads", [8, 64, 128])
def test_bytes_that_are_not_seen_do_not_matter(heads):
    """Everything a row does not see is NaN or infinite: other slots, pages behind the end, tokens out of the window, later tokens of the
    chunk, which share a tile with rows that do see them."""
    b = Batch([130, 70], [6, 5], heads, 64, seed=8)
    window, first = 20, 3
    seen = {b.slot(r, j) for r, n in enumerate(b.new) for i in range(n - 1) for j in b.seen(r, b.seq_lens[r] - n + i, window, first)}
    want = b.want(window, first)
    for poison in (0xFF, 0x7F, None):
        clean = b.cache.clone()
        for slot in range(b.cache.shape[0] * 64):
            if slot not in seen:
                raw, at = b.cache[slot // 64], slot % 64
                if poison is None:  # infinite rotary values only
                    raw[at * 576 + 448 : at * 576 + 576] = torch.full((64,), float("inf"), dtype=torch.bfloat16).view(torch.uint8)
                else:
                    raw[at * 576 : at * 576 + 576] = poison
                    raw[64 * 576 + at * 8 : 64 * 576 + at * 8 + 8] = poison
        out, lse = b.run(window, first)
        last = [int(s) - 1 for s in b.starts[1:]]  # the last token of each request sees its own, poisoned key
        assert torch.isnan(out[last]).all()
        rows = [i for i in range(11) if i not in last]
        check(out[rows], lse[rows], [want[i] for i in rows])
        b.cache = clean


@gpu
def test_pages_and_slots_outside_the_cache_are_seen_by_nobody():
    b = Batch([300], [3], 64, 64, seed=9)
    keys = key_rows(b.cache, 64, [b.slot(0, j) for j in range(300)])
    bad = {1: -1, 3: int(b.cache.shape[0])}
    for page, value in bad.items():
        b.table[0, page] = value
    out, lse = b.run()
    want = [definition(b.q[i], keys[[j for j in range(298 + i) if j // 64 not in bad]], SCALE, b.sink) for i in range(3)]
    check(out, lse, want)
    # sequences that are longer than their row of the table: positions without a page are not seen
    b.table, b.seq_lens = b.table[:, :2].contiguous(), [2 ** 31 - 1]
    out, lse = b.run()
    check(out, lse, [definition(b.q[i], keys[:64], SCALE, b.sink) for i in range(3)])


@gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_queries_that_are_not_finite_stay_in_their_row(value):
    b = Batch([70], [9], 8, 64, seed=10)
    want = b.want()
    b.q[4, 3, 100] = value
    out, lse = b.run()
    rows = [(i, h) for i in range(9) for h in range(8) if (i, h) != (4, 3)]
    check(torch.stack([out[i, h] for i, h in rows])[:, None], torch.stack([lse[i, h] for i, h in rows])[:, None],
          [tuple(t[h : h + 1] for t in want[i]) for i, h in rows])
    assert torch.isnan(out[4, 3]).all()


@gpu
def test_strided_queries_and_results():
    """Heads cut out of a wider tensor, tokens and heads exchanged, lse transposed."""
    b = Batch([150, 20], [4, 2], 24, 64, seed=11)
    want = b.want()
    wide = torch.full((6, 40, 1024), 3.0, dtype=torch.bfloat16, device=DEV)
    q = wide[:, 8:32, 256:768]
    q.copy_(b.q)
    holder = torch.full((24, 6, 520), 7.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.zeros(24, 6, device=DEV).t()
    out, lse = b.run(q=q, out=holder.transpose(0, 1)[..., :512], lse=lse)
    check(out, lse, want)
    assert (holder[..., 512:] == 7).all()


@gpu
def test_results_are_allocated_and_lse_is_optional():
    b = Batch([150, 20], [4, 2], 24, 64, seed=12)
    out = fg.paged_latent_attention(b.q.to(DEV), b.cache.to(DEV), b.table.to(DEV), torch.tensor(b.seq_lens, dtype=torch.int32, device=DEV), b.starts.to(DEV), 64, SCALE)
    want = b.want(sink=False)
    check(out.cpu(), torch.stack([w[1] for w in want]).float(), want)


def sparse_case(tokens, heads, topk, seed, block_size=64):
    g = torch.Generator().manual_seed(seed)
    cache = make_cache(40, block_size, g)
    indices = torch.randint(0, 40 * block_size, (tokens, topk), generator=g, dtype=torch.int32)
    lens = torch.randint(0, topk + 1, (tokens,), generator=g, dtype=torch.int32)
    lens[0] = topk
    q = torch.randn(tokens, heads, 512, generator=g).to(torch.bfloat16)
    return cache, indices, lens, q, torch.randn(heads, generator=g)


def run_sparse(cache, indices, lens, q, sink, block_size=64):
    lse = torch.zeros(q.shape[:2], device=DEV)
    out = fg.sparse_latent_attention(q.to(DEV), cache.to(DEV), indices.to(DEV), lens.to(DEV), block_size, SCALE, sink.to(DEV), None, lse)
    torch.cuda.synchronize()
    assert _native.device_error() == 0
    return out.cpu(), lse.cpu()


@gpu
@pytest.mark.parametrize("tokens,heads,topk", [(1, 64, 1), (1, 128, 512), (5, 8, 63), (3, 64, 65), (7, 96, 200), (2, 130, 1000), (40, 16, 130)])
def test_sparse(tokens, heads, topk):
    case = sparse_case(tokens, heads, topk, seed=topk)
    cache, indices, lens, q, sink = case
    lens[-1] = 0 if tokens > 2 else lens[-1]
    if topk > 5:
        indices[:, 2] = indices[:, 4]  # the same slot twice
        indices[0, 3], indices[0, 1] = -1, 40 * 64  # skipped: negative, outside the cache
    for t in range(tokens):
        indices[t, lens[t] :] = 2 ** 31 - 1 if t % 2 else -7  # never read
    out, lse = run_sparse(*case)
    want = [definition(q[t], key_rows(cache, 64, [int(i) for i in indices[t, : lens[t]] if 0 <= i < 40 * 64]), SCALE, sink) for t in range(tokens)]
    check(out, lse, want)


@gpu
@pytest.mark.parametrize("tokens,topk", [(74, 1100), (75, 1100), (74, 1200), (3, 700), (3, 800), (150, 700)])
def test_sparse_lists_that_may_be_cut_or_not(tokens, topk):
    """Both sides of the rules on when a CTA takes a whole tile and when tiles may be cut; a few long lists among short ones."""
    cache, indices, lens, q, sink = sparse_case(tokens, 128, topk, seed=topk)
    lens[1:] = lens[1:] % 50
    lens[tokens // 2] = topk - 1
    out, lse = run_sparse(cache, indices, lens, q, sink)
    check(out, lse, [definition(q[t], key_rows(cache, 64, indices[t, : lens[t]].tolist()), SCALE, sink) for t in range(tokens)])


@gpu
def test_sparse_lengths_outside_the_list():
    case = sparse_case(4, 16, 70, seed=20)
    cache, indices, lens, q, sink = case
    lens[:] = torch.tensor([100, -5, 2 ** 31 - 1, -(2 ** 31)], dtype=torch.int32)
    out, lse = run_sparse(*case)
    want = [definition(q[t], key_rows(cache, 64, indices[t].tolist() if t % 2 == 0 else []), SCALE, sink) for t in range(4)]
    check(out, lse, want)


@gpu
def test_lists_and_tables_of_no_entries():
    """Nobody sees a key: rows of zeros."""
    cache, _, _, q, sink = sparse_case(5, 16, 4, seed=21)
    for lens in (0, 3):
        out, lse = run_sparse(cache, torch.empty(5, 0, dtype=torch.int32), torch.full((5,), lens, dtype=torch.int32), q, sink)
        assert (out == 0).all() and (lse == -math.inf).all()
    b = Batch([70, 9], [4, 3], 16, 64, seed=22)
    b.table = b.table[:, :0].contiguous()
    out, lse = b.run()
    assert (out == 0).all() and (lse == -math.inf).all()
    b.cache = b.cache[:0]
    b.table = torch.zeros(2, 2, dtype=torch.int32)
    out, lse = b.run()
    assert (out == 0).all() and (lse == -math.inf).all()


def table_of_rows(cache, block_size):
    """All rows of a small cache at once, in 64 bits."""
    return key_rows(cache, block_size, range(cache.shape[0] * block_size))


@gpu
@pytest.mark.parametrize("tokens", [57000, 70000])
def test_sparse_of_very_many_tokens(tokens):
    """More lengths than shared memory holds while the shares are worked out, and just as many as it does; rows of one head."""
    g = torch.Generator().manual_seed(tokens)
    cache = make_cache(4, 16, g)
    indices = torch.randint(0, 64, (tokens, 3), generator=g, dtype=torch.int32)
    lens = torch.randint(0, 4, (tokens,), generator=g, dtype=torch.int32)
    q = torch.randn(tokens, 1, 512, generator=g).to(torch.bfloat16)
    out, lse = run_sparse(cache, indices, lens, q, torch.zeros(1), 16)
    rows = table_of_rows(cache, 16)
    for t in torch.cat([torch.arange(0, tokens, 997), torch.arange(tokens - 5, tokens)]).tolist():
        check(out[t : t + 1], lse[t : t + 1], [definition(q[t], rows[indices[t, : lens[t]].long()], SCALE, torch.zeros(1))])
    # the rest against sums over all rows at once, in 32 bits: the module's bound, with scores that are off by d on both sides
    live = torch.arange(3)[None] < lens[:, None]
    s = (q[:, 0].float() @ rows.float().t() * SCALE).gather(1, indices.long()).masked_fill(~live, -math.inf)
    d = (q[:, 0].float().abs() @ rows.float().abs().t()).amax(1) * SCALE * 512 * 2.0 ** -23
    weights = torch.exp(s) / (1 + torch.exp(s).sum(1, keepdim=True))
    for start in range(0, tokens, 10000):
        part = slice(start, start + 10000)
        keys = rows.float()[indices[part].long()]
        want, a = (weights[part, :, None] * keys).sum(1), (weights[part, :, None] * keys.abs()).sum(1)
        bound = (2.0 ** -8 + torch.expm1(4 * d[part])[:, None] + 22 * 2.0 ** -23) * a + 2.0 ** -8 * want.abs() + 2.0 ** -100
        assert (out[part, 0].float() - want).abs().le(bound).all()


@gpu
def test_very_many_requests():
    """Starts and lengths of 30000 requests do not fit in shared memory; some bring no token."""
    g = torch.Generator().manual_seed(30)
    n, heads = 30000, 2
    cache = make_cache(4, 16, g)
    new = torch.randint(0, 3, (n,), generator=g)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).to(torch.int32)
    tokens, seq = int(starts[-1]), (new + torch.randint(0, 12, (n,), generator=g)).to(torch.int32)
    table = torch.randint(0, 4, (n, 1), generator=g, dtype=torch.int32)
    q = torch.randn(tokens, heads, 512, generator=g).to(torch.bfloat16)
    lse = torch.zeros(tokens, heads, device=DEV)
    out = fg.paged_latent_attention(q.to(DEV), cache.to(DEV), table.to(DEV), seq.to(DEV), starts.to(DEV), 16, SCALE, None, 0, None, None, lse).cpu()
    assert _native.device_error() == 0
    rows = table_of_rows(cache, 16)
    lse = lse.cpu()
    for r in [*range(0, n, 101), n - 2, n - 1]:
        for i in range(int(new[r])):
            t, p = int(starts[r]) + i, int(seq[r]) - int(new[r]) + i
            page = int(table[r, 0]) * 16
            check(out[t : t + 1], lse[t : t + 1], [definition(q[t], rows[page : page + p + 1], SCALE, None)])


@gpu
def test_a_replayed_graph_follows_lengths_and_tables():
    """What a captured call was given by its shapes holds for every replay; lengths, starts and pages may change between replays."""
    b = Batch([900, 40, 300], [1, 1, 1], 64, 64, seed=23)
    dev = [t.to(DEV) for t in (b.q, b.cache, b.table, torch.tensor(b.seq_lens, dtype=torch.int32), b.starts)]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        fg.paged_latent_attention(*dev, 64, SCALE)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = fg.paged_latent_attention(*dev, 64, SCALE)
    torch.cuda.synchronize()
    for lens in ([900, 40, 300], [1, 64, 65], [512, 0, 299], [7, 40, 1]):
        dev[3].copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        b.seq_lens = lens
        want = b.want(sink=False)
        check(out.cpu(), torch.stack([w[1] for w in want]).float(), want)


@gpu
def test_sparse_equals_paged():
    """The list of a token's positions gives what the block table gives."""
    b = Batch([500, 90], [1, 1], 64, 64, seed=13)
    out, lse = b.run()
    indices = torch.full((2, 500), -1, dtype=torch.int32)
    for r in range(2):
        indices[r, : b.seq_lens[r]] = torch.tensor([b.slot(r, j) for j in range(b.seq_lens[r])], dtype=torch.int32)
    got, got_lse = run_sparse(b.cache, indices, torch.tensor(b.seq_lens, dtype=torch.int32), b.q, b.sink)
    want = b.want()
    check(out, lse, want)
    check(got, got_lse, want)


@gpu
def test_offsets_beyond_32_bits():
    """A cache of more than 4 GiB whose first and last blocks are used; a list of slots in it too."""
    blocks = (5 << 30) // (64 * 584)
    g = torch.Generator().manual_seed(14)
    small = make_cache(4, 64, g)
    cache = torch.empty(blocks, 64 * 584, dtype=torch.uint8, device=DEV)
    where = [0, blocks - 1, blocks // 2, blocks - 2]
    for i, at in enumerate(where):
        cache[at] = small[i].to(DEV)
    q, sink = torch.randn(2, 64, 512, generator=g).to(torch.bfloat16), torch.randn(64, generator=g)
    keys = key_rows(small, 64, range(256))
    table = torch.tensor([where], dtype=torch.int32, device=DEV)
    lse = torch.zeros(2, 64, device=DEV)
    out = fg.paged_latent_attention(q.to(DEV), cache, table, torch.tensor([256], dtype=torch.int32, device=DEV), torch.tensor([0, 2], dtype=torch.int32, device=DEV),
                                    64, SCALE, None, 0, sink.to(DEV), None, lse)
    check(out.cpu(), lse.cpu(), [definition(q[i], keys[: 255 + i], SCALE, sink) for i in range(2)])
    indices = torch.tensor([[w * 64 + 5 for w in where]] * 2, dtype=torch.int32, device=DEV)
    out = fg.sparse_latent_attention(q.to(DEV), cache, indices, torch.tensor([4, 2], dtype=torch.int32, device=DEV), 64, SCALE, sink.to(DEV), None, lse)
    check(out.cpu(), lse.cpu(), [definition(q[i], keys[[5, 69, 133, 197][: 4 - 2 * i]], SCALE, sink) for i in range(2)])


@gpu
def test_two_graphs_and_two_streams_at_once():
    """Calls on two streams, and replays of two captured graphs, share no workspace: both give what a call alone gives, bit for bit."""
    batches = [Batch([4000, 100], [1, 1], 64, 64, seed=15), Batch([100, 5000, 900], [1, 1, 1], 64, 64, seed=16)]
    inputs, want = [], []
    for b in batches:
        inputs.append((b.q.to(DEV), b.cache.to(DEV), b.table.to(DEV), torch.tensor(b.seq_lens, dtype=torch.int32, device=DEV), b.starts.to(DEV), 64, SCALE))
        want.append(fg.paged_latent_attention(*inputs[-1]).clone())
    streams = [torch.cuda.Stream() for _ in range(2)]
    graphs, captured = [], []
    torch.cuda.synchronize()
    for s, i in zip(streams, inputs):
        with torch.cuda.stream(s):
            fg.paged_latent_attention(*i)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                captured.append(fg.paged_latent_attention(*i))
            graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(10):
        eager = []
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
                eager.append(fg.paged_latent_attention(*inputs[1 - k]))
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(captured[k], want[k]) and torch.equal(eager[k], want[1 - k])


@gpu
@pytest.mark.parametrize("what", ["q", "out", "cache", "pitch"])
def test_unaligned_arguments_are_refused(what):
    b = Batch([20], [2], 4, 16, seed=17, pitch=16 * 584 + (8 if what == "pitch" else 0))
    shifted = lambda t: torch.empty(t.numel() + 8, dtype=t.dtype, device=DEV)[1 : 1 + t.numel()].view(t.shape).copy_(t)
    q, cache = b.q.to(DEV), b.cache.to(DEV)
    with pytest.raises(_native.Dsv4Error):
        fg.paged_latent_attention(shifted(q) if what == "q" else q, shifted(cache) if what == "cache" else cache, b.table.to(DEV),
                                  torch.tensor([20], dtype=torch.int32, device=DEV), b.starts.to(DEV), 16, SCALE, None, 0, None,
                                  shifted(torch.zeros_like(q)) if what == "out" else None)


@gpu
@pytest.mark.parametrize("tokens,heads", [(1, 12), (5, 1), (1, 1)])
def test_strides_of_single_tokens_and_heads_are_not_used(tokens, heads):
    b = Batch([50], [tokens], heads, 64, seed=24)
    strides = (3 if tokens == 1 else heads * 512, 5 if heads == 1 else 512, 1)
    q, out = (torch.empty(tokens * heads * 512, dtype=torch.bfloat16, device=DEV).as_strided((tokens, heads, 512), strides) for _ in range(2))
    q.copy_(b.q)
    out, lse = b.run(q=q, out=out)
    check(out, lse, b.want())


@gpu
def test_queries_shared_by_tokens_and_heads():
    """A broadcast q is read, not written."""
    b = Batch([90, 40], [3, 2], 20, 64, seed=25)
    b.q[:] = b.q[:1, :1]
    out, lse = b.run(q=b.q[0, 0].to(DEV).expand(5, 20, 512))
    check(out, lse, b.want())


@gpu
def test_overlapping_results_are_refused():
    b = Batch([20], [2], 4, 64, seed=18)
    q = b.q.to(DEV)
    args = (b.cache.to(DEV), b.table.to(DEV), torch.tensor([20], dtype=torch.int32, device=DEV), b.starts.to(DEV), 64, SCALE, None, 0, None)
    for out, lse in ((q, None), (q[:1].expand(2, 4, 512), None), (torch.zeros(1, 4, 512, dtype=torch.bfloat16, device=DEV).expand(2, 4, 512), None),
                     (None, torch.zeros(1, 4, device=DEV).expand(2, 4))):
        with pytest.raises(AssertionError, match="overlap"):
            fg.paged_latent_attention(q, *args, out, lse)
