"""The latent cache in 4 bits: its writer byte for byte against the definition in 64 bits, and the attention over it against the definition with the
bounds that test_latent_attention.py derives (the cached values, e2m1 times a power of two, are exact in bf16, as there).

What the writer leaves is whole numbers but for the rotated values, which are compared with those of the e4m3 writer: the same products and sums in the
same order.  So are q's."""
from __future__ import annotations

import math

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native
from flaggems_vllm.testing.workloads import cos_sin_table
from test_latent_attention import Batch, check, definition

gpu = pytest.mark.gpu
DEV = "cuda:0"
SCALE = 512 ** -0.5
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0] + [-0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]).double()
insert = fg.fused_deepseek_v4_qnorm_rope_kv_rope_mxfp4_insert


def quantised(nope):
    """Bytes of e2m1 pairs and scale codes of [n, 448] values, in 64 bits."""
    x = nope.double().view(-1, 14, 32)
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], torch.zeros_like(x), x)
    code = torch.ceil(torch.log2(x.abs().amax(-1).clamp(min=6 * 2.0 ** -126) / 6)) + 127
    y = x / torch.exp2(code - 127)[..., None]
    distance = (y.abs()[..., None] - E2M1[:8]).abs()
    nearest = distance == distance.amin(-1, keepdim=True)
    pick = (nearest.int() * torch.tensor([2, 1] * 4)).argmax(-1)  # of two, the even code
    pick = torch.where(bad[..., None], 0, pick + 8 * torch.signbit(y)).view(-1, 224, 2).to(torch.uint8)
    return pick[..., 0] + 16 * pick[..., 1], torch.where(bad, 255, code).to(torch.uint8)


def make_mx_cache(blocks, block_size, g, pitch=None, extremes=False):
    """Random bytes, finite: codes around 1, or all that keep 6 * 2^(code - 127) finite in bf16."""
    cache = torch.full((blocks, pitch or block_size * 368), 0xFF, dtype=torch.uint8)
    data = cache[:, : block_size * 352].view(blocks, block_size, 352)
    data[..., :224] = torch.randint(0, 256, (blocks, block_size, 224), generator=g, dtype=torch.uint8)
    data[..., 224:] = torch.randn(blocks, block_size, 64, generator=g).to(torch.bfloat16).view(torch.uint8)
    codes = cache[:, block_size * 352 : block_size * 368].view(blocks, block_size, 16)
    codes[...] = torch.randint(*((0, 126) if extremes else (124, 128)), (blocks, block_size, 16), generator=g, dtype=torch.uint8)
    return cache


def mx_rows(cache, block_size, slots):
    """[n, 512] in 64 bits."""
    out = torch.empty(len(slots), 512, dtype=torch.float64)
    for i, slot in enumerate(slots):
        raw, at = cache[slot // block_size], slot % block_size
        data = raw[at * 352 : at * 352 + 352]
        codes = raw[block_size * 352 + at * 16 :][:14].double()
        scale = torch.where(codes == 255, math.nan, torch.exp2(codes - 127))
        out[i, 0:448:2], out[i, 1:448:2] = E2M1[(data[:224] & 15).long()], E2M1[(data[:224] >> 4).long()]
        out[i, :448] *= scale.repeat_interleave(32)
        out[i, 448:] = data[224:].clone().view(torch.bfloat16).double()
    return out


class MxBatch(Batch):
    def __init__(self, *args, pitch=None, extremes=False, seed=0, **kw):
        super().__init__(*args, seed=seed, **kw)
        self.cache = make_mx_cache(self.cache.shape[0], self.bs, torch.Generator().manual_seed(seed + 1000), pitch, extremes)

    def want(self, window=None, first=0, sink=True, scale=SCALE):
        rows = []
        for r, n in enumerate(self.new):
            keys = mx_rows(self.cache, self.bs, [self.slot(r, j) for j in range(max(self.seq_lens[r], 0))])
            for i in range(n):
                seen = self.seen(r, self.seq_lens[r] - n + i, window, first)
                rows.append(definition(self.q[int(self.starts[r]) + i], keys[seen], scale, self.sink if sink else None))
        return rows

    def run(self, window=None, first=0, sink=True, scale=SCALE, out=None, lse=None, q=None):
        lse = torch.full((self.tokens, self.heads), 7.0, device=DEV) if lse is None else lse
        out = torch.full((self.tokens, self.heads, 512), 7.0, dtype=torch.bfloat16, device=DEV) if out is None else out
        q = self.q.to(DEV) if q is None else q
        got = fg.paged_latent_attention_mxfp4(q, self.cache.to(DEV), self.table.to(DEV), torch.tensor(self.seq_lens, dtype=torch.int32, device=DEV),
                                              self.starts.to(DEV), self.bs, scale, window, first, self.sink.to(DEV) if sink else None, out, lse)
        torch.cuda.synchronize()
        assert got.data_ptr() == out.data_ptr() and _native.device_error() == 0
        return out.cpu(), lse.cpu()


# ---- the writer -----------------------------------------------------------------------------------------------------------------


class Insertion:
    def __init__(self, tokens, heads, block_size=64, blocks=None, pitch=None, seed=0, base=0, inserted=None, skip=0.2):
        g = torch.Generator().manual_seed(seed)
        self.bs, self.blocks = block_size, blocks or 2 * -(-tokens // block_size) + 3
        pitch = pitch or block_size * 368
        self.q = torch.randn(tokens, heads, 512, generator=g).to(torch.bfloat16)
        self.kv = (torch.randn(tokens, 512, generator=g) * torch.exp2(torch.randint(-20, 20, (tokens, 1), generator=g).float())).to(torch.bfloat16)
        self.slots = torch.randperm(self.blocks * block_size, generator=g)[: tokens if inserted is None else inserted]
        self.slots[torch.rand(len(self.slots), generator=g) < skip] = -1
        self.positions = torch.randint(0, 4096, (tokens,), generator=g)
        self.table = cos_sin_table(4096)
        self.storage = torch.randint(0, 256, (base + self.blocks * pitch,), generator=g, dtype=torch.uint8)
        self.base, self.pitch = base, pitch

    def cache_of(self, storage, token_bytes):
        return storage[self.base :].as_strided((self.blocks, self.bs * token_bytes), (self.pitch, 1), self.base)

    def run(self, op=insert, token_bytes=368, odd=0):
        """q and the storage after a call; q and kv begin `odd` elements into theirs."""

        def moved(t):
            room = torch.zeros(t.numel() + odd, dtype=t.dtype, device=DEV)
            room[odd:] = t.flatten().to(DEV)
            return room[odd:].view(t.shape)

        q, storage = moved(self.q), self.storage.to(DEV)
        op(q, moved(self.kv), self.cache_of(storage, token_bytes), self.slots.to(DEV), self.positions.to(DEV), self.table.to(DEV), 1e-6, self.bs)
        torch.cuda.synchronize()
        return q.cpu(), storage.cpu()

    def check(self, odd=0):
        q, storage = self.run(odd=odd)
        fp8 = Insertion.__new__(Insertion)
        fp8.__dict__.update(self.__dict__, pitch=self.bs * 584, base=0, storage=torch.zeros(self.blocks * self.bs * 584, dtype=torch.uint8))
        want_q, other = fp8.run(fg.fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert, 584, odd)
        assert torch.equal(q.view(torch.int16), want_q.view(torch.int16))
        want = self.storage.clone()
        cache, of_fp8 = self.cache_of(want, 368), fp8.cache_of(other, 584)
        data, codes = quantised(self.kv[:, :448])
        for t, slot in enumerate(self.slots.tolist()):
            if slot >= 0:
                block, at = cache[slot // self.bs], slot % self.bs
                block[at * 352 : at * 352 + 224] = data[t]
                block[at * 352 + 224 : at * 352 + 352] = of_fp8[slot // self.bs, at * 576 + 448 : at * 576 + 576]
                block[self.bs * 352 + at * 16 :][:14] = codes[t]
                block[self.bs * 352 + at * 16 + 14 :][:2] = 0
        assert torch.equal(storage, want)


@gpu
@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 128), (3, 64), (61, 128), (257, 16), (1000, 3), (33, 0)])
def test_writer(tokens, heads):
    Insertion(tokens, heads, seed=tokens).check()


@gpu
@pytest.mark.parametrize("block_size,extra,base", [(1, 0, 0), (7, 0, 0), (64, 16, 0), (64, 5, 0), (16, 0, 3), (256, 1000, 16), (3, 8, 8)])
def test_writer_block_sizes_pitches_and_bases(block_size, extra, base):
    Insertion(70, 2, block_size, pitch=block_size * 368 + extra, base=base, seed=block_size).check()


@gpu
@pytest.mark.parametrize("odd", [1, 4, 7])
def test_writer_q_and_kv_off_16_bytes(odd):
    Insertion(50, 3, seed=odd).check(odd)


@gpu
@pytest.mark.parametrize("inserted", [0, 1, 30, 64])
def test_writer_with_fewer_slots_than_tokens(inserted):
    Insertion(64, 2, inserted=inserted).check()


@gpu
@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("staging", [0, 1])
def test_writer_launch_modes(mode, staging):
    before = _native.set_pdl(mode), _native.set_table_staging(staging)
    try:
        Insertion(100, 9, seed=4).check()
    finally:
        _native.set_pdl(before[0]), _native.set_table_staging(before[1])


@gpu
@pytest.mark.parametrize("odd", [0, 1])
def test_writer_of_every_magnitude(odd):
    """Every finite bf16 as the largest value of a group, with fractions of it that lie on and beside the borders between e2m1 values."""
    every = torch.arange(0, 0x7F80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).float()
    fractions = torch.tensor([1, -1, 0, -0.0, 5 / 6, 0.5, 7 / 12, 3.5 / 8, 2.5 / 6, 1.75 / 6, 1.25 / 6, 0.75 / 6, 0.25 / 6, 1 / 6, -0.2 / 6, 0.26 / 6, 5 / 8, 5.1 / 8, 2.5 / 8, 1.75 / 8, 1.25 / 8, 0.75 / 8,
                              0.25 / 8, 0.125 / 8, -5 / 8, -3.5 / 8, -0.75 / 8, -0.25 / 8, 3 / 4, 1 / 3, -2 / 3, 1 / 64])
    groups = (every[:, None] * fractions).to(torch.bfloat16)
    tokens = -(-len(groups) // 14)
    groups = torch.cat([groups, groups[: tokens * 14 - len(groups)]])
    i = Insertion(tokens, 0, skip=0.0)
    i.kv = torch.cat([groups.view(tokens, 448), i.kv[:, 448:]], 1)
    i.check(odd)


@gpu
@pytest.mark.parametrize("odd", [0, 1])
def test_writer_of_values_that_are_no_numbers(odd):
    i = Insertion(40, 1, skip=0.0)
    for t, value in enumerate([math.inf, -math.inf, math.nan, -math.nan] * 10):
        i.kv[t, (t * 37) % 448] = value
    i.check(odd)
    data, codes = quantised(i.kv[:, :448])
    assert (codes == 255).sum() == 40 and (data.view(40, 14, 16)[codes == 255] == 0).all()


@gpu
def test_writer_error_is_below_a_fifth_of_the_largest_value():
    """With a = amax, 3 scale < a <= 6 scale.  Above 4, where e2m1 values are 2 apart, an error of the whole scale happens beside 5 only, so where a >= 5
    scale: a / 5; elsewhere half a scale at most, below a / 6."""
    i = Insertion(200, 0, skip=0.0)
    _, storage = i.run()
    rows = mx_rows(i.cache_of(storage, 368), i.bs, i.slots.tolist())[:, :448]
    x = i.kv[:, :448].double()
    top = x.view(-1, 14, 32).abs().amax(-1).repeat_interleave(32, -1)
    assert ((rows - x).abs() <= top / 5).all()


# ---- the attention ----------------------------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("heads", [1, 8, 24, 64, 65, 128, 200])
@pytest.mark.parametrize("lengths,new", [([1], [1]), ([63, 64, 65], [1, 1, 1]), ([300, 5, 129], [1, 1, 1]), ([130, 70, 9], [70, 3, 9])])
def test_causal(heads, lengths, new):
    b = MxBatch(lengths, new, heads, 64, seed=heads)
    check(*b.run(), b.want())


@gpu
@pytest.mark.parametrize("window,first", [(1, 0), (7, 0), (64, 4), (100, 70), (1000, 3), (1 << 40, 1 << 40)])
@pytest.mark.parametrize("heads", [16, 128])
def test_window_and_first_tokens(window, first, heads):
    b = MxBatch([330, 3, 130, 200], [40, 3, 1, 9], heads, 64, seed=1)
    check(*b.run(window, first), b.want(window, first))


@gpu
@pytest.mark.parametrize("block_size,pitch", [(1, None), (7, 7 * 368 + 16), (16, None), (48, None), (256, 256 * 368 + 4096)])
def test_block_sizes_and_pitches(block_size, pitch):
    b = MxBatch([200, 97], [3, 50], 16, block_size, seed=2, pitch=None if pitch is None else -(-pitch // 16) * 16)
    check(*b.run(), b.want())


@gpu
def test_scales_over_the_whole_range():
    b = MxBatch([150, 40], [20, 1], 16, 64, seed=3, extremes=True)
    check(*b.run(), b.want())


@gpu
@pytest.mark.parametrize("code", [0, 1, 2, 125, 126, 127, 128, 250, 252])
def test_every_value_with_a_scale(code):
    """One key, seen alone, with the weight 1: the output is the key itself, so every nibble in every place of a byte comes back exactly (at most 6 * 2^125)."""
    b = MxBatch([16], [16], 1, 16, seed=5)
    b.q.zero_()
    raw = b.cache[b.slot(0, 0) // 16]
    raw[: 16 * 352].view(16, 352)[:, :224] = torch.arange(256, dtype=torch.uint8).roll(code).repeat(14).view(16, 224)
    raw[16 * 352 : 16 * 368].view(16, 16)[:, :14] = code
    out, _ = b.run(window=1, sink=False)
    rows = mx_rows(b.cache, 16, [b.slot(0, j) for j in range(16)])
    assert torch.equal(out[:, 0].double(), rows.to(torch.bfloat16).double())


@gpu
@pytest.mark.parametrize("heads", [8, 64])
def test_groups_that_are_nan(heads):
    """A scale code of 255: rows that see the key are NaN, the others are as if it were not there."""
    b = MxBatch([100, 90], [60, 1], heads, 64, seed=6)
    slot = b.slot(0, 70)
    b.cache[slot // 64, 64 * 352 + (slot % 64) * 16 + 9] = 255
    out, lse = b.run()
    want = b.want()
    assert out[70 - 40 : 60].isnan().all() and lse[70 - 40 : 60].isnan().all()
    keep = [i for i in range(61) if not 30 <= i < 60]
    check(out[keep], lse[keep], [want[i] for i in keep])


@gpu
@pytest.mark.parametrize("code", [253, 254])
def test_values_that_bfloat16_cannot_hold(code):
    """6 * 2^126 and 6 * 2^127: infinite.  Rows that see the key are NaN, all of them or in that dimension; the others are as if it were not there."""
    b = MxBatch([100], [60], 8, 64, seed=6)
    slot = b.slot(0, 70)
    raw, at = b.cache[slot // 64], slot % 64
    raw[at * 352 : at * 352 + 16] = 0
    raw[at * 352 + 5] = 0x07
    raw[64 * 352 + at * 16] = code
    out, lse = b.run()
    assert out[30:, :, 10].isnan().all()
    check(out[:30], lse[:30], b.want()[:30])


@gpu
def test_bytes_that_nobody_sees_do_not_matter():
    """Pages behind the end, later tokens and free slots full of NaN codes and values."""
    b = MxBatch([75, 20], [5, 20], 16, 64, seed=7)
    want = b.want()
    seen = {b.slot(r, j) for r, n in enumerate(b.seq_lens) for j in range(n)}
    for slot in range(b.cache.shape[0] * 64):
        if slot not in seen:
            raw, at = b.cache[slot // 64], slot % 64
            raw[at * 352 : at * 352 + 352] = 0xFF
            raw[64 * 352 + at * 16 :][:16] = 0xFF
    check(*b.run(), want)


@gpu
def test_rows_without_keys_and_pages_outside_the_cache():
    b = MxBatch([0, 5, 64], [2, 1, 1], 8, 64, seed=8, extra_rows=2)
    b.table[2] = -1
    out, lse = b.run()
    assert (out[[0, 1, 3]] == 0).all() and (lse[[0, 1, 3]] == -math.inf).all()
    assert (out[4:] == 7).all() and (lse[4:] == 7).all()
    check(out[2:3], lse[2:3], b.want()[2:3])


@gpu
@pytest.mark.parametrize("tokens,heads,topk", [(1, 128, 512), (5, 16, 200), (3, 64, 1), (7, 130, 1025), (2, 8, 0), (300, 1, 40)])
def test_sparse(tokens, heads, topk):
    g = torch.Generator().manual_seed(tokens)
    cache = make_mx_cache(20, 64, g)
    indices = torch.randint(0, 20 * 64, (tokens, topk), generator=g, dtype=torch.int32)
    indices[torch.rand(tokens, topk, generator=g) < 0.1] = -1
    lens = torch.randint(0, topk + 1, (tokens,), generator=g, dtype=torch.int32)
    lens[0] = topk
    q, sink = torch.randn(tokens, heads, 512, generator=g).to(torch.bfloat16), torch.randn(heads, generator=g)
    lse = torch.empty(tokens, heads, device=DEV)
    out = fg.sparse_latent_attention_mxfp4(q.to(DEV), cache.to(DEV), indices.to(DEV), lens.to(DEV), 64, SCALE, sink.to(DEV), None, lse)
    want = []
    for t in range(tokens):
        slots = [s for s in indices[t, : lens[t]].tolist() if s >= 0]
        want.append(definition(q[t], mx_rows(cache, 64, slots), SCALE, sink))
    check(out.cpu(), lse.cpu(), want)


@gpu
def test_long_context_split_over_the_gpu():
    b = MxBatch([6000, 3000], [1, 1], 8, 64, seed=9)
    check(*b.run(), b.want())


@gpu
def test_strided_queries_and_outputs():
    b = MxBatch([90, 40], [3, 1], 5, 64, seed=10)
    q = torch.zeros(4, 9, 640, dtype=torch.bfloat16, device=DEV)[:, 1:6, 64:576]
    q.copy_(b.q)
    out = torch.full((4, 5, 1024), 3.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.zeros(5, 4, device=DEV).t()
    got, got_lse = b.run(out=out[..., :512], lse=lse, q=q)
    check(got, got_lse, b.want())
    assert (out[..., 512:] == 3).all()


@gpu
def test_cache_beyond_32_bits():
    """A slot whose bytes lie past 2^32."""
    blocks = (1 << 32) // (64 * 368) + 40
    cache = torch.zeros(blocks, 64 * 368, dtype=torch.uint8, device=DEV)
    i = Insertion(3, 4, skip=0.0)
    slots = torch.tensor([blocks * 64 - 1, (blocks - 1) * 64, 5])
    insert(i.q.to(DEV), i.kv.to(DEV), cache, slots.to(DEV), i.positions.to(DEV), i.table.to(DEV), 1e-6, 64)
    far = cache[[0, blocks - 1]].cpu()
    keys = mx_rows(far, 64, [127, 64, 5])
    data, codes = quantised(i.kv[:, :448])
    stored = torch.stack([far[1, 64 * 352 + 63 * 16 :][:14], far[1, 64 * 352 :][:14], far[0, 64 * 352 + 5 * 16 :][:14]])
    assert torch.equal(stored, codes) and torch.equal(far[1, 63 * 352 :][:224], data[0])
    scale = 1e-3 * 2.0 ** -20
    out = fg.sparse_latent_attention_mxfp4(i.q.to(DEV), cache, slots.to(torch.int32).repeat(3, 1).to(DEV), torch.tensor([3, 2, 1], dtype=torch.int32, device=DEV), 64, scale)
    want = [definition(i.q[t], keys[: 3 - t], scale, None) for t in range(3)]
    check(out.cpu(), torch.stack([w[1] for w in want]).float(), want)


# ---- what is refused ----------------------------------------------------------------------------------------------------------------


@gpu
def test_refusals():
    b = MxBatch([90], [2], 4, 64)
    q, cache, table = b.q.to(DEV), b.cache.to(DEV), b.table.to(DEV)
    lens, starts = torch.tensor([90], dtype=torch.int32, device=DEV), b.starts.to(DEV)
    with pytest.raises(AssertionError, match="368"):
        fg.paged_latent_attention_mxfp4(q, cache, table, lens, starts, 65, SCALE)
    with pytest.raises(AssertionError, match="584"):
        fg.paged_latent_attention(q, cache, table, lens, starts, 64, SCALE)
    with pytest.raises(AssertionError):
        fg.sparse_latent_attention_mxfp4(q, cache, table.repeat(2, 1), lens, 64, SCALE)
    with pytest.raises(_native.Dsv4Error):
        fg.paged_latent_attention_mxfp4(q, cache[:, 8:], table, lens, starts, 63, SCALE)
    i = Insertion(4, 2)
    with pytest.raises(AssertionError):
        insert(i.q.to(DEV), i.kv.to(DEV), cache[:, : 64 * 352], i.slots.to(DEV), i.positions.to(DEV), i.table.to(DEV), 1e-6, 64)
