"""Serving steps over a cache in 4 bits, from the lengths of the requests to the attention's output: block tables and slots -> prologue, which writes the
new keys -> attention over the block table -> index bookkeeping -> attention over selected slots -> the blocks of a finished request go back.  Each
stage is checked against its definition fed with the stage before's device result; a decode loop whose state lives on the GPU is captured and replayed."""
from __future__ import annotations

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native
from flaggems_vllm.testing import workloads
from test_latent_attention import check, definition
from test_mxfp4_cache import mx_rows, quantised
from test_paged_batch import extended, released

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BS, BLOCKS, WIDTH, EPS = 16, 60, 12, 1e-6
SCALE = 512 ** -0.5


class Server:
    """The state that a serving loop keeps on the GPU, and its host copy by the definitions."""

    def __init__(self, requests, heads, seed):
        self.g, self.heads, self.n = torch.Generator().manual_seed(seed), heads, requests
        self.context, self.table = [0] * requests, [[-1] * WIDTH for _ in range(requests)]
        self.free, self.num_free = torch.randperm(BLOCKS, generator=self.g).tolist(), BLOCKS
        self.cs, self.sink = workloads.cos_sin_table(1024), torch.randn(heads, generator=self.g)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        self.d_context, self.d_table, self.d_free, self.d_num_free = i32(self.context), i32(self.table), i32(self.free), i32([BLOCKS])
        self.d_cs, self.d_sink = self.cs.to(DEV), self.sink.to(DEV)
        self.cache = torch.zeros(BLOCKS, BS * 368, dtype=torch.uint8, device=DEV)

    def step(self, new, pad=0, topk=20):
        tokens = sum(new) + pad
        q = torch.randn(tokens, self.heads, 512, generator=self.g).to(torch.bfloat16)
        kv = torch.randn(tokens, 512, generator=self.g).to(torch.bfloat16)
        before = self.cache.cpu()
        batch = fg.extend_block_tables(self.d_context, torch.tensor(new, dtype=torch.int32, device=DEV), self.d_table, self.d_free, self.d_num_free, BS, tokens)
        want, self.table = extended(self.context, new, self.table, self.free, self.num_free, BS, tokens)
        for name, t, w in zip(batch._fields, batch, want):
            assert t.tolist() == w, name
        starts, lens, positions, slots, requests, (self.num_free,), _ = want
        # the prologue; q's rows are those of the e4m3 form, the cache's bytes the definition's
        d_q, d_kv = q.to(DEV), kv.to(DEV)
        fg.fused_deepseek_v4_qnorm_rope_kv_rope_mxfp4_insert(d_q, d_kv, self.cache, batch.slot_mapping, batch.position_ids, self.d_cs, EPS, BS)
        other_q, other = q.to(DEV), torch.zeros(BLOCKS, BS * 584, dtype=torch.uint8, device=DEV)
        fg.fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert(other_q, d_kv, other, batch.slot_mapping, batch.position_ids, self.d_cs, EPS, BS)
        assert torch.equal(d_q.view(torch.int16), other_q.view(torch.int16))
        data, codes = quantised(kv[:, :448])
        for t, slot in enumerate(slots):
            if slot >= 0:
                raw, at = before[slot // BS], slot % BS
                raw[at * 352 : at * 352 + 224], raw[at * 352 + 224 : at * 352 + 352] = data[t], other[slot // BS, at * 576 + 448 : at * 576 + 576].cpu()
                raw[BS * 352 + at * 16 :][:14] = codes[t]
        cache = self.cache.cpu()
        assert torch.equal(cache, before)
        # both attentions
        lse, lse_sparse = torch.zeros(tokens, self.heads, device=DEV), torch.zeros(tokens, self.heads, device=DEV)
        out = fg.paged_latent_attention_mxfp4(d_q, self.cache, self.d_table, batch.seq_lens, batch.query_start_loc, BS, SCALE, None, 0, self.d_sink, None, lse)
        picked = torch.full((tokens, topk), -1, dtype=torch.int32)
        for t in range(sum(new)):
            some = torch.randperm(positions[t] + 1, generator=self.g)[:topk].to(torch.int32)
            picked[t, : len(some)] = some
        chosen, counts = fg.compute_global_topk_indices_and_lens(picked.to(DEV), batch.token_to_req_indices, self.d_table, BS)
        out_sparse = fg.sparse_latent_attention_mxfp4(d_q, self.cache, chosen, counts, BS, SCALE, self.d_sink, None, lse_sparse)
        h_q, real = d_q.cpu(), sum(new)
        slot_of = lambda r, p: self.table[r][p // BS] * BS + p % BS  # noqa: E731
        want_paged, want_sparse = [], []
        for t in range(real):
            r = requests[t]
            want_paged.append(definition(h_q[t], mx_rows(cache, BS, [slot_of(r, p) for p in range(positions[t] + 1) if self.table[r][p // BS] >= 0]), SCALE, self.sink))
            want_sparse.append(definition(h_q[t], mx_rows(cache, BS, [slot_of(r, p) for p in picked[t][picked[t] >= 0].tolist()]), SCALE, self.sink))
        if real:
            check(out[:real].cpu(), lse[:real].cpu(), want_paged)
            check(out_sparse[:real].cpu(), lse_sparse[:real].cpu(), want_sparse)
        assert (out_sparse[real:] == 0).all() and _native.device_error() == 0
        self.context, self.d_context, self.d_num_free = lens, batch.seq_lens, batch.num_free

    def finish(self, done):
        finished = [r in done for r in range(self.n)]
        left = fg.release_block_tables(self.d_context, torch.tensor(finished, device=DEV), self.d_table, self.d_free, self.d_num_free, BS)
        self.free, self.num_free = released(self.context, finished, self.table, self.free, self.num_free, BS)
        assert self.d_free.tolist() == self.free and left.tolist() == [self.num_free]
        self.context = [0 if f else c for f, c in zip(finished, self.context)]
        self.d_num_free, self.d_context = left, torch.tensor(self.context, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("heads", [8, 64])
def test_every_stage_matches_its_definition(heads):
    s = Server(4, heads, heads)
    s.step([37, 5, 0, 61])
    s.step([1, 1, 0, 1], pad=2)
    s.step([1, 1, 20, 1])
    s.finish({0, 3})
    s.step([80, 1, 1, 33], pad=1)  # new requests in the rows, and the blocks, of those that ended
    s.finish({1})
    s.step([1, 4, 1, 1])
    used = [e for c, row in zip(s.context, s.table) for e in row[: -(-c // BS)]]
    assert sorted(used + s.free[: s.num_free]) == list(range(BLOCKS))  # no block is lost, none is held twice


def decode(d, out, buffers):
    """A decode step whose lengths, table and stack go on by themselves."""
    batch = fg.extend_block_tables(d["lens"], d["ones"], d["table"], d["free"], d["num_free"], BS, d["ones"].shape[0], out)
    buffers["q"].copy_(d["q"])
    fg.fused_deepseek_v4_qnorm_rope_kv_rope_mxfp4_insert(buffers["q"], d["kv"], d["cache"], batch.slot_mapping, batch.position_ids, d["cs"], EPS, BS)
    fg.paged_latent_attention_mxfp4(buffers["q"], d["cache"], d["table"], batch.seq_lens, batch.query_start_loc, BS, SCALE, None, 0, d["sink"], buffers["out"], buffers["lse"])


@pytest.mark.parametrize("mode", [0, 2])
def test_captured_decode_loop(mode):
    """40 steps replayed from a graph give what the same calls give with a synchronisation behind each, bit for bit; the graph's memory is shared by nobody, and its
    workspace is the call's own."""
    requests, heads, steps = 9, 16, 40
    g = torch.Generator().manual_seed(3)
    previous = _native.set_pdl(mode)
    try:
        results = []
        for captured in (False, True):
            g.manual_seed(3)
            i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
            d = {"lens": i32([0] * requests), "ones": i32([1] * requests), "table": torch.full((requests, 4), -1, dtype=torch.int32, device=DEV), "free": torch.randperm(40, generator=g).to(torch.int32).to(DEV),
                 "num_free": i32([40]), "q": torch.randn(requests, heads, 512, generator=g).to(torch.bfloat16).to(DEV), "kv": torch.randn(requests, 512, generator=g).to(torch.bfloat16).to(DEV),
                 "cache": torch.zeros(40, BS * 368, dtype=torch.uint8, device=DEV), "cs": workloads.cos_sin_table(256).to(DEV), "sink": torch.randn(heads, generator=g).to(DEV)}
            buffers = {"q": torch.empty_like(d["q"]), "out": torch.zeros(requests, heads, 512, dtype=torch.bfloat16, device=DEV), "lse": torch.zeros(requests, heads, device=DEV)}
            out = [torch.zeros(requests + 1, dtype=torch.int32, device=DEV), d["lens"], *(torch.zeros(requests, dtype=torch.int64, device=DEV) for _ in range(2)),
                   torch.zeros(requests, dtype=torch.int32, device=DEV), d["num_free"], torch.zeros(1, dtype=torch.int32, device=DEV)]
            keep = {k: d[k].clone() for k in ("lens", "table", "num_free", "cache")}
            seen = []
            if captured:
                s = torch.cuda.Stream()
                s.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(s):
                    decode(d, out, buffers)
                    for k, t in keep.items():
                        d[k].copy_(t)
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=s):
                        decode(d, out, buffers)
                s.synchronize()
            for _ in range(steps):
                if captured:
                    graph.replay()
                else:
                    decode(d, out, buffers)
                    torch.cuda.synchronize()
                seen.append([buffers["out"].clone(), buffers["lse"].clone(), out[3].clone()])
            torch.cuda.synchronize()
            results.append((seen, {k: d[k].clone() for k in keep}))
        assert _native.device_error() == 0
        for a, b in zip(*(r[0] for r in results)):
            for x, y in zip(a, b):
                assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        for k in results[0][1]:
            assert torch.equal(results[0][1][k], results[1][1][k]), k
        assert results[0][1]["lens"].tolist() == [steps] * requests and results[0][1]["num_free"].item() == 40 - requests * -(-steps // BS)
    finally:
        _native.set_pdl(previous)


@pytest.mark.parametrize("n,requests", [(1, 1), (61, 61), (700, 9), (3000, 3)])
def test_chain_equals_the_synchronised_chain(n, requests):
    """Every call's inputs come from the launch directly in front of it, over buffers that held other values a moment before."""
    g = torch.Generator(device=DEV).manual_seed(n)
    heads, blocks = 8, 2 * (n // BS + requests + 4)
    new = torch.full((requests,), n // requests, dtype=torch.int32, device=DEV)
    new[0] += n - int(new.sum())
    width = int(new.max()) // BS + 6
    sets = []
    for seed in range(2):
        context = torch.randint(0, 40, (requests,), generator=g, device=DEV).to(torch.int32)
        order = torch.randperm(4 * blocks + 3 * requests, generator=g, device=DEV).to(torch.int32)
        table = torch.full((requests, width), -1, dtype=torch.int32, device=DEV)
        table[:, :3] = order[: 3 * requests].view(requests, 3)
        sets.append({"context": context, "table": table, "free": order[3 * requests :].contiguous(), "q": torch.randn(n, heads, 512, generator=g, device=DEV).to(torch.bfloat16),
                     "kv": torch.randn(n, 512, generator=g, device=DEV).to(torch.bfloat16)})
    buffers = {k: torch.zeros_like(t) for k, t in sets[0].items()}
    cache = torch.zeros(4 * blocks + 3 * requests, BS * 368, dtype=torch.uint8, device=DEV)
    num_free = torch.tensor([4 * blocks - 5], dtype=torch.int32, device=DEV)
    cs, done = workloads.cos_sin_table(4096).to(DEV), torch.ones(requests, dtype=torch.bool, device=DEV)

    def chain(s, between):
        for k, t in s.items():
            buffers[k].copy_(t)
        cache.zero_()
        between()
        b = buffers
        batch = fg.extend_block_tables(b["context"], new, b["table"], b["free"], num_free, BS, n)
        between()
        fg.fused_deepseek_v4_qnorm_rope_kv_rope_mxfp4_insert(b["q"], b["kv"], cache, batch.slot_mapping, batch.position_ids, cs, EPS, BS)
        between()
        out = fg.paged_latent_attention_mxfp4(b["q"], cache, b["table"], batch.seq_lens, batch.query_start_loc, BS, SCALE)
        between()
        left = fg.release_block_tables(batch.seq_lens, done, b["table"], b["free"], batch.num_free, BS)
        between()
        again = fg.extend_block_tables(batch.query_start_loc[1:].clone(), new, b["table"], b["free"], left, BS, n)
        return [t.clone() for t in (*batch, b["table"], b["free"], b["q"], cache, out, left, *again)]

    for s in sets + sets:
        fast = chain(s, lambda: None)
        slow = chain(s, torch.cuda.synchronize)
        torch.cuda.synchronize()
        for i, (x, y) in enumerate(zip(fast, slow)):
            assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)), i
    assert _native.device_error() == 0


def test_two_graphs_and_an_eager_call_at_once():
    """Attention calls of two graphs and an eager one on three streams: each has a workspace of its own."""
    from test_mxfp4_cache import MxBatch

    batches = [MxBatch([3000, 900 + 500 * i, 40], [1, 1, 1], 16, 64, seed=20 + i) for i in range(3)]
    held, want = [], []
    for b in batches:
        h = [b.q.to(DEV), b.cache.to(DEV), b.table.to(DEV), torch.tensor(b.seq_lens, dtype=torch.int32, device=DEV), b.starts.to(DEV), 64, SCALE]
        held.append(h)
        want.append(fg.paged_latent_attention_mxfp4(*h).clone())
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(3)]
    for h, s in zip(held[:2], streams):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(fg.paged_latent_attention_mxfp4(*h))
        graphs.append(graph)
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = fg.paged_latent_attention_mxfp4(*held[2])
        torch.cuda.synchronize()
        for got, w in zip(outs + [eager], want):
            assert torch.equal(got, w)
    assert _native.device_error() == 0
