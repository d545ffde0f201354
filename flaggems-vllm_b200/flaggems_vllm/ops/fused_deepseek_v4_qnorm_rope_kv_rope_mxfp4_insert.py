"""The attention prologue for a latent cache that is held in 4 bits: q RMSNorm + RoPE, KV RoPE + MXFP4 quantisation + paged insert.

The sibling of `fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert` with the same arguments and effects on q; a cached token takes 368 bytes
instead of 584.  `paged_latent_attention_mxfp4` and `sparse_latent_attention_mxfp4` read the cache.
"""
from __future__ import annotations

import torch

from .. import _native

HEAD_DIM = 512
ROPE_DIM = 64
TOKEN_BYTES = 368  # 448 e2m1 in 224 bytes + 64 bf16 + 16 scale bytes per cached token


def _check_arguments(q, kv, k_cache, slot_mapping, position_ids, cos_sin_cache, cache_block_size):
    assert q.is_contiguous() and kv.is_contiguous()
    num_tokens, _, head_dims = q.shape
    assert head_dims == HEAD_DIM
    assert kv.shape == (num_tokens, HEAD_DIM)
    assert q.dtype == torch.bfloat16 and kv.dtype == torch.bfloat16
    assert k_cache.dtype == torch.uint8
    assert slot_mapping.dim() == 1
    assert slot_mapping.shape[0] <= num_tokens
    assert slot_mapping.dtype == torch.int64
    assert position_ids.shape == (num_tokens,)
    assert position_ids.dtype == torch.int64
    assert cos_sin_cache.dim() == 2 and cos_sin_cache.shape[1] == ROPE_DIM
    assert cos_sin_cache.dtype == torch.float32
    assert k_cache.dim() == 2 and k_cache.stride(1) == 1, "k_cache must be [num_blocks, block_bytes] with unit byte stride"
    assert cache_block_size > 0 and k_cache.shape[1] >= cache_block_size * TOKEN_BYTES, "cache block too small"
    assert slot_mapping.is_contiguous() and position_ids.is_contiguous() and cos_sin_cache.is_contiguous()
    assert q.is_cuda, "this operator has no CPU path: tensors must live on a CUDA device"
    for t in (kv, k_cache, slot_mapping, position_ids, cos_sin_cache):
        assert t.device == q.device, "all tensors must be on the same device"


_call = None  # the native front end, looked up once


def _bind():
    global _call
    _call = _native.host_calls().prologue_mxfp4
    return _call


def fused_deepseek_v4_qnorm_rope_kv_rope_mxfp4_insert(
    q: torch.Tensor,
    kv: torch.Tensor,
    k_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    position_ids: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    eps: float,
    cache_block_size: int,
) -> None:
    """Per-head weight-less RMSNorm + GPT-J RoPE for q (in place), and GPT-J RoPE + MXFP4 quantisation + paged-cache insertion for the latent
    KV, in one kernel launch on the current stream of q's device.

    K-cache block layout: `cache_block_size` token records of 352 bytes (448 e2m1 values, value 2i in the low and 2i + 1 in the high four
    bits of byte i, then 64 bf16), then `cache_block_size` groups of 16 scale bytes (14 UE8M0 codes, one for 32 values each, and two zeros);
    `k_cache.stride(0)` is the block pitch.  Per group of 32 values

        code = ceil(log2(max(amax, 6 * 2^-126) / 6)) + 127,   value = e2m1(x / 2^(code - 127)), to nearest, ties to even

    so a value is off by at most a fifth of its group's maximum, and by at most 2^-128 in a group whose maximum is below 1.25 * 2^-126, for which the
    scale has no smaller step.  Values from 3.5 * 2^126 on, finite ones, are stored as 2^128, which the readers, whose keys are bfloat16, take for infinite.
    e2m1 has neither infinities nor NaN: a group with one gets the code 255, which stands for NaN, and the readers make all 32 values NaN.

    Args:
        q: [num_tokens, num_heads, 512] bfloat16, contiguous, modified in place
        kv: [num_tokens, 512] bfloat16, contiguous, read only
        k_cache: [num_blocks, block_bytes] uint8, modified in place at the mapped slots
        slot_mapping: [num_tokens_insert <= num_tokens] int64; negative entries are skipped
        position_ids: [num_tokens] int64
        cos_sin_cache: [max_pos, 64] float32 (32 cos | 32 sin)
        eps: RMSNorm epsilon
        cache_block_size: tokens per cache block

    Slots and positions are not range-checked on the device.
    """
    if (_call or _bind())(q, kv, k_cache, slot_mapping, position_ids, cos_sin_cache, eps, cache_block_size) is None:
        _check_arguments(q, kv, k_cache, slot_mapping, position_ids, cos_sin_cache, cache_block_size)
        _native.refuse()


__all__ = ["fused_deepseek_v4_qnorm_rope_kv_rope_mxfp4_insert"]
