"""The residual norm and both attentions in the order a layer calls them, over one paged cache that already holds the requests' prefixes:
residual + norm + quantisation -> (stand-in projections) -> prologue, which writes the new keys -> attention over the block table with a window
-> index bookkeeping -> attention over the selected slots -> the epilogue's quantiser.  Each stage is checked against its definition fed with
the stage before's device result."""
from __future__ import annotations

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native
from flaggems_vllm.testing import compare, workloads
from oracle import c_oracle
from test_fused_add_rmsnorm_quant_fp8 import definition as norm_definition
from test_fused_add_rmsnorm_quant_fp8 import same
from test_latent_attention import Batch, check, definition, key_rows

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
COLS, GROUP, TOPK, WINDOW, FIRST = 512, 128, 48, 70, 3
EPS = torch.tensor(1e-6).item()
SCALE = 512 ** -0.5


def make_inputs(heads, seed):
    b = Batch([333, 90, 64, 1], [2, 90, 1, 1], heads, 64, seed=seed)
    g = torch.Generator().manual_seed(seed + 100)
    n = b.tokens
    req_of = torch.cat([torch.full((m,), r) for r, m in enumerate(b.new)])
    positions = torch.cat([torch.arange(s - m, s) for s, m in zip(b.seq_lens, b.new)])
    topk = torch.full((n, TOPK), -1, dtype=torch.int32)  # positions of each token's request, none behind its own, no order
    for i in range(n):
        picked = torch.randperm(int(positions[i]) + 1, generator=g)[:TOPK].to(torch.int32)
        topk[i, : len(picked)] = picked
    host = {
        "x": torch.randn(n, COLS, generator=g).to(torch.bfloat16), "residual": torch.randn(n, COLS, generator=g).to(torch.bfloat16),
        "weight": (1 + 0.1 * torch.randn(COLS, generator=g)).to(torch.bfloat16),
        "to_q": (torch.randn(COLS, heads * 512, generator=g) / COLS ** 0.5).to(torch.bfloat16),
        "to_kv": (torch.randn(COLS, 512, generator=g) / COLS ** 0.5).to(torch.bfloat16),
        "cache": b.cache, "table": torch.where(b.table == 1 << 30, 0, b.table), "positions": positions.to(torch.int64),
        "slots": torch.tensor([b.slot(int(r), int(p)) for r, p in zip(req_of, positions)], dtype=torch.int64),
        "seq_lens": torch.tensor(b.seq_lens, dtype=torch.int32), "starts": b.starts, "req_of": req_of.to(torch.int32), "topk": topk,
        "cs": workloads.cos_sin_table(1024), "sink": b.sink,
    }
    return b, host


def to_device(host):
    return {k: v.to(DEV) for k, v in host.items()}


def run(d, heads, buffers):
    n = d["x"].shape[0]
    x_q, scales = fg.fused_add_rmsnorm_quant_fp8(d["x"], buffers["residual"], d["weight"], EPS, GROUP)
    hidden = (x_q.float().view(n, -1, GROUP) * scales[..., None]).view(n, COLS).to(torch.bfloat16)  # stand-in for the projections' products
    q, kv = (hidden @ d["to_q"]).view(n, heads, 512), hidden @ d["to_kv"]
    q_in = q.clone()
    fg.fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert(q, kv, buffers["cache"], d["slots"], d["positions"], d["cs"], EPS, 64)
    lse, lse_sparse = torch.empty(n, heads, device=DEV), torch.empty(n, heads, device=DEV)
    o = fg.paged_latent_attention(q, buffers["cache"], d["table"], d["seq_lens"], d["starts"], 64, SCALE, WINDOW, FIRST, d["sink"], None, lse)
    slots, lens = fg.compute_global_topk_indices_and_lens(d["topk"], d["req_of"], d["table"], 64)
    o_sparse = fg.sparse_latent_attention(q, buffers["cache"], slots, lens, 64, SCALE, d["sink"], None, lse_sparse)
    fp8, scale = fg.fused_inv_rope_fp8_quant(o, d["positions"], d["cs"], 4, heads // 4, tma_aligned_scales=True)
    return {"x_q": x_q, "scales": scales, "q_in": q_in, "kv": kv, "q": q, "o": o, "lse": lse, "slots": slots, "lens": lens, "o_sparse": o_sparse,
            "lse_sparse": lse_sparse, "fp8": fp8, "scale": scale}


def fresh(d):
    return {"residual": d["residual"].clone(), "cache": d["cache"].clone()}


@pytest.mark.parametrize("heads", [16, 64])
def test_every_stage_matches_its_definition(heads):
    b, host = make_inputs(heads, 0)
    d = to_device(host)
    buffers = fresh(d)
    out = {k: t.cpu() for k, t in run(d, heads, buffers).items()}
    cache = buffers["cache"].cpu()
    assert _native.device_error() == 0
    sums, x_q, scales = norm_definition(host["x"], host["residual"], host["weight"], GROUP, False)
    assert same(buffers["residual"], sums) and same(out["x_q"], x_q) and same(out["scales"], scales)
    want_cache, want_q = host["cache"].clone(), out["q_in"].clone()
    c_oracle.prologue(want_q, out["kv"], want_cache, host["slots"], host["positions"], host["cs"], EPS, 64)
    assert torch.equal(cache, want_cache)
    compare.assert_q_close(out["q"], want_q)
    b.cache, b.q = cache, out["q"]
    check(out["o"], out["lse"], b.want(WINDOW, FIRST))
    # the slots behind the selected positions, in the order that the bookkeeping gave them
    want = []
    for i in range(b.tokens):
        positions = host["topk"][i][host["topk"][i] >= 0].tolist()
        assert out["slots"][i, : out["lens"][i]].tolist() == [b.slot(int(host["req_of"][i]), p) for p in positions]
        want.append(definition(out["q"][i], key_rows(cache, 64, out["slots"][i, : out["lens"][i]].tolist()), SCALE, b.sink))
    check(out["o_sparse"], out["lse_sparse"], want)
    want_fp8, want_scale = c_oracle.inv_rope_fp8_quant(out["o"], host["positions"], host["cs"], 4, heads // 4, packed=True)
    assert torch.equal(out["fp8"].view(torch.uint8), want_fp8)
    assert torch.equal(out["scale"].contiguous().view(torch.int32), want_scale.view(torch.int32))


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_run_in_every_launch_mode(mode, graph):
    """Every operator reads what the one in front of it wrote, launched dependently or not: two runs with different inputs take turns, so that
    memory of the allocator holds the other one's values and an early read shows.  All results are reproducible bit for bit."""
    heads = 64
    data = [to_device(make_inputs(heads, seed)[1]) for seed in (1, 2)]
    bytes_of = lambda t: t.contiguous().view(torch.uint8)
    previous = _native.set_pdl(0)
    try:
        want = []
        for d in data:
            buffers = fresh(d)
            out = run(d, heads, buffers)
            torch.cuda.synchronize()
            want.append({k: bytes_of(t).clone() for k, t in {**out, **buffers}.items()})
        _native.set_pdl(mode)
        buffers = [fresh(d) for d in data]
        seen = []

        def turns():
            for turn in range(6):
                i = turn % 2
                for k, t in buffers[i].items():
                    t.copy_(data[i][k])
                seen.append((i, {**run(data[i], heads, buffers[i]), **{k: t.clone() for k, t in buffers[i].items()}}))

        if graph:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                run(data[0], heads, buffers[0])
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured, stream=s):
                    turns()
                for _, results in seen:
                    for t in results.values():
                        t.view(torch.uint8).zero_() if t.is_contiguous() else t.zero_()
                captured.replay()
            s.synchronize()
        else:
            turns()
            torch.cuda.synchronize()
        assert _native.device_error() == 0
        for i, results in seen:
            for k, t in results.items():
                assert torch.equal(bytes_of(t), want[i][k]), k
    finally:
        _native.set_pdl(previous)
