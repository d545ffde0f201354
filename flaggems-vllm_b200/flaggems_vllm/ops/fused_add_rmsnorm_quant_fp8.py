"""Residual addition, weighted RMS norm and FP8 e4m3 quantisation of hidden states in one pass: the way into the FP8 projections.

For `x` and `residual` [T, K] in bfloat16 or float16, per row:

    z = x + residual                      (fp32; z = x where residual is None)
    residual <- z                         (in place, rounded to its type)
    y = z / sqrt(mean(z^2) + eps) * weight
    scale = max(max |y|, 1e-10) / 448     per group of `group_size` values, or the power of two at or above it (`scale_ue8m0`)
    x_q = e4m3(y / scale)

Nothing between z and x_q is rounded to 16 bits, and the mean is formed in 64, so scales and bytes do not depend on an order of summation.
Returns (x_q [T, K] float8_e4m3fn, scales [T, K / group_size] float32, transposed storage when `column_major_scales`), as
`per_token_group_quant_fp8` does (src/flaggems_vllm/ops/per_token_group_quant_fp8.py:226-330), whose input this norm would otherwise write.
`group_size`: 32, 64, 128, 256, or K for one scale per token.  A group with a NaN has a NaN scale.  `residual` must not overlap `x` or `weight`.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native
from ..utils.memory import apart

_call = None  # the native front end, looked up once


def _bind():
    global _call
    _call = _native.host_calls().add_rmsnorm_quant
    return _call


def fused_add_rmsnorm_quant_fp8(
    x: torch.Tensor,
    residual: Optional[torch.Tensor],
    weight: torch.Tensor,
    eps: float,
    group_size: int = 128,
    column_major_scales: bool = False,
    scale_ue8m0: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    result = (_call or _bind())(x, residual, weight, eps, group_size, column_major_scales, scale_ue8m0)
    if result is not None:
        return result
    assert x.device.type == "cuda", "this operator has no CPU path"
    assert x.dim() == 2 and x.stride(1) == 1, "x: [tokens, hidden] with unit inner stride"
    assert x.dtype in (torch.bfloat16, torch.float16), "bfloat16 or float16 activations"
    rows, cols = x.shape
    assert group_size in (32, 64, 128, 256) or group_size == cols, "groups of 32, 64, 128 or 256 values, or the whole row"
    assert group_size > 0 and cols % group_size == 0 and cols % 8 == 0, f"the last dimension of `x` {cols} must be divisible by `group_size` {group_size} and by 8"
    assert cols <= 32768, "rows of at most 32768 values"
    if residual is not None:
        assert residual.dim() == 2 and residual.shape == x.shape and residual.dtype == x.dtype and residual.stride(1) == 1, "residual: like x"
        assert residual.device == x.device, "all tensors must be on the same device"
    assert weight.dim() == 1 and weight.shape[0] == cols and weight.is_contiguous(), "weight: [hidden]"
    assert weight.dtype in (x.dtype, torch.float32), "weight: float32 or the type of x"
    assert weight.device == x.device, "all tensors must be on the same device"
    assert rows <= 1 or (x.stride(0) >= cols and (residual is None or residual.stride(0) >= cols)), "rows must not overlap"
    assert residual is None or rows == 0 or apart(x, residual), "residual must not overlap x"
    _native.refuse()


__all__ = ["fused_add_rmsnorm_quant_fp8"]
