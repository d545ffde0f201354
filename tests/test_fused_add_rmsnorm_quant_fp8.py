"""Residual addition, RMS norm and e4m3 output against the definition in plain torch on the CPU, bit for bit: the mean of squares is formed in
64 bits on both sides (relative error below 2^-48 in any order), its reciprocal root is rounded to 32 once, and every later step is one
IEEE operation in a fixed order.  A row differs only where that root lies within 2^-48 of a rounding border of 32 bits, one row in 2^23."""
from __future__ import annotations

import pytest
import torch

import flaggems_vllm as fg
from flaggems_vllm import _native

gpu = pytest.mark.gpu
DEV = "cuda:0"
EPS = torch.tensor(1e-6).item()  # as the kernel gets it: 32 bits


def definition(x, residual, weight, group, pow2):
    z = x.float() if residual is None else x.float() + residual.float()
    r = (1.0 / torch.sqrt(z.double().square().mean(-1, keepdim=True) + EPS)).float()
    y = (z * r * weight.float()).view(z.shape[0], -1, group)
    scale = y.abs().amax(-1)
    scale = torch.where(scale.isnan(), scale, scale.clamp(min=1e-10)) / 448.0
    if pow2:
        bits = (scale.view(torch.int32) + 0x7FFFFF) & 0x7F800000
        scale = torch.where(scale < 2.0 ** 127, bits.view(torch.float32), scale)
    q = (y / scale.unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(z.shape)
    return z.to(x.dtype), q, scale


def rows(t, n, dtype, pitch, generator, scale=1.0):
    """[t, n] in a buffer of the given pitch, on the GPU, and the same on the CPU."""
    buffer = (torch.randn(max(t, 1), pitch, generator=generator) * scale).to(dtype)
    return buffer.to(DEV)[:t, :n], buffer[:t, :n]


def same(got, want):
    got = got.cpu().contiguous()
    if got.dtype == torch.float8_e4m3fn:
        nan = want.float().isnan()
        assert torch.equal(got.float().isnan(), nan)
        return torch.equal(torch.where(nan, 0.0, got.float()), torch.where(nan, 0.0, want.float()))
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


@gpu
@pytest.mark.parametrize("tokens,cols,group", [(1, 7168, 128), (3, 64, 64), (5, 64, 32), (61, 7168, 128), (149, 1536, 256), (200, 4096, 4096), (7, 32768, 128),
                                               (150, 32768, 64), (2, 8, 8), (1, 1544, 1544), (300, 1544, 1544), (33, 512, 512), (9, 16640, 256), (149, 2304, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pow2", [False, True])
def test_matches_the_definition(tokens, cols, group, dtype, pow2):
    g = torch.Generator().manual_seed(tokens * cols + group)
    x, xc = rows(tokens, cols, dtype, cols, g)
    res, resc = rows(tokens, cols, dtype, cols, g, 3.0)
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(dtype)
    want = definition(xc, resc, w, group, pow2)
    x_q, scales = fg.fused_add_rmsnorm_quant_fp8(x, res, w.to(DEV), EPS, group, False, pow2)
    assert x_q.shape == (tokens, cols) and scales.shape == (tokens, cols // group) and scales.is_contiguous()
    assert same(res, want[0]) and same(scales, want[2]) and same(x_q, want[1])
    assert same(x, xc)


@gpu
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("weight_type", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pitches", [(640, 640), (648, 1024), (2048, 656)])
def test_layouts(with_residual, weight_type, pitches):
    """No residual, weights in 32 bits, rows with gaps (whose bytes stay), column-major scales."""
    g = torch.Generator().manual_seed(3)
    x, xc = rows(37, 640, torch.bfloat16, pitches[0], g)
    res, resc = rows(37, 640, torch.bfloat16, pitches[1], g)
    whole, before = res._base, res._base.clone()
    w = (1 + 0.3 * torch.randn(640, generator=g)).to(weight_type)
    want = definition(xc, resc if with_residual else None, w, 64, False)
    x_q, scales = fg.fused_add_rmsnorm_quant_fp8(x, res if with_residual else None, w.to(DEV), EPS, 64, column_major_scales=True)
    assert scales.shape == (37, 10) and scales.stride() == (1, 37)
    assert same(scales, want[2]) and same(x_q, want[1]) and same(res, want[0] if with_residual else resc)
    assert torch.equal(whole[:, 640:], before[:, 640:])


@gpu
@pytest.mark.parametrize("pow2", [False, True])
def test_special_rows(pow2):
    """Zero rows, huge rows (the sum overflows the tensors' type, not the norm), infinities and NaN: only their row, and of its groups only
    theirs, is affected."""
    g = torch.Generator().manual_seed(4)
    x, r = torch.randn(8, 256, generator=g).to(torch.float16), torch.randn(8, 256, generator=g).to(torch.float16)
    x[1], r[1] = 0.0, 0.0
    x[2], r[2] = 65504.0, 65504.0
    x[3, 70] = float("inf")
    x[4, 200] = float("nan")
    x[5], r[5] = 6e-8, 0.0
    r[6, 0] = float("-inf")
    w = torch.ones(256, dtype=torch.float16)
    w[64:128] = 0.0
    want = definition(x, r, w, 64, pow2)
    res = r.to(DEV)
    x_q, scales = fg.fused_add_rmsnorm_quant_fp8(x.to(DEV), res, w.to(DEV), EPS, 64, False, pow2)
    assert same(res, want[0]) and same(scales, want[2]) and same(x_q, want[1])
    assert torch.isfinite(scales[[0, 1, 2, 5, 7]]).all()


@gpu
def test_empty_other_stream_and_graph():
    g = torch.Generator().manual_seed(5)
    w = torch.ones(512, dtype=torch.bfloat16, device=DEV)
    x_q, scales = fg.fused_add_rmsnorm_quant_fp8(torch.empty(0, 512, dtype=torch.bfloat16, device=DEV), None, w, EPS)
    assert x_q.shape == (0, 512) and scales.shape == (0, 4)
    x, xc = rows(300, 512, torch.bfloat16, 512, g)
    res, resc = rows(300, 512, torch.bfloat16, 512, g)
    kept = res.clone()
    want = definition(xc, resc, w.cpu(), 128, True)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        fg.fused_add_rmsnorm_quant_fp8(x, res.clone(), w, EPS, scale_ue8m0=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            x_q, scales = fg.fused_add_rmsnorm_quant_fp8(x, res, w, EPS, scale_ue8m0=True)
        for _ in range(2):
            res.copy_(kept)
            graph.replay()
    stream.synchronize()
    assert same(res, want[0]) and same(scales, want[2]) and same(x_q, want[1])


@gpu
@pytest.mark.parametrize("offset,pitch", [(1, 520), (4, 520), (0, 513), (0, 516)])
def test_unaligned_rows_are_refused(offset, pitch):
    buffer = torch.zeros(4 * 520 + 16, dtype=torch.bfloat16, device=DEV)
    x = buffer[offset:].as_strided((3, 512), (pitch, 1), offset)
    w = torch.ones(512, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(_native.Dsv4Error):
        fg.fused_add_rmsnorm_quant_fp8(x, None, w, EPS)
    with pytest.raises(_native.Dsv4Error):
        fg.fused_add_rmsnorm_quant_fp8(torch.zeros(3, 512, dtype=torch.bfloat16, device=DEV), x, w, EPS)


@gpu
def test_overlapping_residual_is_refused():
    buffer = torch.zeros(8, 512, dtype=torch.bfloat16, device=DEV)
    w = torch.ones(512, dtype=torch.bfloat16, device=DEV)
    for residual in (buffer[:4], buffer[3:7]):
        with pytest.raises(AssertionError, match="overlap"):
            fg.fused_add_rmsnorm_quant_fp8(buffer[:4], residual, w, EPS)
