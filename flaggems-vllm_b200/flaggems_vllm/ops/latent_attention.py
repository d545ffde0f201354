"""Attention over the paged latent cache: what a DeepSeek-V4 layer runs between the prologue, which writes the cache
(`fused_deepseek_v4_qnorm_rope_kv_rope_quant_insert`), and the epilogue (`fused_inv_rope_fp8_quant`).

A cached row of 512 values, shared by all heads, is key and value at once.  Per token and head, over the keys j that the token sees:

    s_j = softmax_scale * q . k_j
    out = sum_j exp(s_j) k_j / (sum_j exp(s_j) + exp(attn_sink[head]))       (the last term where attn_sink is given)
    lse = log sum_j exp(s_j)                                                 (without the sink)

* `paged_latent_attention`: requests with a row of `block_table` each.  Request r has the tokens query_start_loc[r] ..
  query_start_loc[r + 1] - 1 of q, the last of them at position seq_lens[r] - 1 of its sequence, whose keys are in the cache already: a
  chunk of a prompt, or one token per request.  Of these tokens those are computed that q has rows for.  Position p sees j <= p and, with a
  window, of those j > p - window_size or j < num_first_tokens.
* `sparse_latent_attention`: token t sees the cache slots indices[t, : lens[t]], as `compute_global_topk_indices_and_lens` makes them; negative
  entries are skipped.

Scores, sums and both products' accumulators are of 32 bits, cached keys exactly what the cache holds.  The weights exp(s_j) are rounded to bfloat16, in which the
second product takes them (2^-8 of each; their sum is that of the unrounded ones), the exponentials are the hardware's (2^-21), and `out` is rounded once.

`paged_latent_attention_mxfp4` and `sparse_latent_attention_mxfp4` are the same over the cache in 4 bits that
`fused_deepseek_v4_qnorm_rope_kv_rope_mxfp4_insert` writes (368 bytes a token instead of 584).  A scale code of 255 makes its 32 values NaN; values of 2^128 and
more, which bfloat16 cannot hold (scale codes of 253 and 254; written only for magnitudes from 3.5 * 2^126 on), are infinite.

q is bfloat16 [tokens, heads, 512] with unit inner stride, any number of heads; rows, cache and cache blocks on 16-byte boundaries.  `out`
(like q) and `lse` (float32 [tokens, heads]) are written where given; `out` is allocated otherwise, and returned.  Neither may share memory with the
other or with an argument that is read.

A row that sees no key is zero, with an lse of -inf.  Keys that a row does not see do not influence it, whatever their bytes: pages behind a
sequence's end, later tokens of a chunk, entries behind `lens`.  A page or slot outside the cache, and a position behind the block table, is
seen by nobody.  A key with a value that is not finite makes the rows that see it NaN, all of them or, where the score is -inf, at least the
dimensions that are not finite (a row all of whose scores are -inf counts as one that sees no key).  Rows of q behind the last request stay as
they are in `out` and `lse` (in an `out` that was allocated here they are not defined).
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _native
from ..utils.memory import apart, rows_apart

HEAD_DIM, TOKEN_BYTES, TOKEN_BYTES_MXFP4 = 512, 584, 368

_paged = _sparse = _paged_mxfp4 = _sparse_mxfp4 = None  # the native front ends, looked up once


def _bind():
    global _paged, _sparse, _paged_mxfp4, _sparse_mxfp4
    calls = _native.host_calls()
    _paged, _sparse = calls.paged_latent_attention, calls.sparse_latent_attention
    _paged_mxfp4, _sparse_mxfp4 = calls.paged_latent_attention_mxfp4, calls.sparse_latent_attention_mxfp4


def paged_latent_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    cache_block_size: int,
    softmax_scale: float,
    window_size: Optional[int] = None,
    num_first_tokens: int = 0,
    attn_sink: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    if _paged is None:
        _bind()
    result = _paged(q, k_cache, block_table, seq_lens, query_start_loc, cache_block_size, softmax_scale, window_size, num_first_tokens,
                    attn_sink, out, lse)
    if result is not None:
        return result
    _check_paged(q, k_cache, block_table, seq_lens, query_start_loc, cache_block_size, softmax_scale, window_size, num_first_tokens, attn_sink,
                 out, lse, TOKEN_BYTES)
    _native.refuse()


def sparse_latent_attention(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    indices: torch.Tensor,
    lens: torch.Tensor,
    cache_block_size: int,
    softmax_scale: float,
    attn_sink: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    if _sparse is None:
        _bind()
    result = _sparse(q, k_cache, indices, lens, cache_block_size, softmax_scale, attn_sink, out, lse)
    if result is not None:
        return result
    _check_sparse(q, k_cache, indices, lens, cache_block_size, softmax_scale, attn_sink, out, lse, TOKEN_BYTES)
    _native.refuse()


def paged_latent_attention_mxfp4(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    query_start_loc: torch.Tensor,
    cache_block_size: int,
    softmax_scale: float,
    window_size: Optional[int] = None,
    num_first_tokens: int = 0,
    attn_sink: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    if _paged_mxfp4 is None:
        _bind()
    result = _paged_mxfp4(q, k_cache, block_table, seq_lens, query_start_loc, cache_block_size, softmax_scale, window_size,
                          num_first_tokens, attn_sink, out, lse)
    if result is not None:
        return result
    _check_paged(q, k_cache, block_table, seq_lens, query_start_loc, cache_block_size, softmax_scale, window_size, num_first_tokens, attn_sink,
                 out, lse, TOKEN_BYTES_MXFP4)
    _native.refuse()


def sparse_latent_attention_mxfp4(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    indices: torch.Tensor,
    lens: torch.Tensor,
    cache_block_size: int,
    softmax_scale: float,
    attn_sink: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    if _sparse_mxfp4 is None:
        _bind()
    result = _sparse_mxfp4(q, k_cache, indices, lens, cache_block_size, softmax_scale, attn_sink, out, lse)
    if result is not None:
        return result
    _check_sparse(q, k_cache, indices, lens, cache_block_size, softmax_scale, attn_sink, out, lse, TOKEN_BYTES_MXFP4)
    _native.refuse()


def _check_paged(q, k_cache, block_table, seq_lens, query_start_loc, cache_block_size, softmax_scale, window_size, num_first_tokens, attn_sink,
                 out, lse, token_bytes):
    _check(q, k_cache, cache_block_size, softmax_scale, attn_sink, out, lse, token_bytes)
    requests = seq_lens.shape[0]
    for name, t, dims in (("block_table", block_table, 2), ("seq_lens", seq_lens, 1), ("query_start_loc", query_start_loc, 1)):
        assert t.dtype == torch.int32 and t.dim() == dims, f"{name}: int32 of {dims} dimensions"
        assert t.device == q.device, "all tensors must be on the same device"
    assert block_table.stride(1) == 1 and seq_lens.is_contiguous() and query_start_loc.is_contiguous(), "indices with unit stride"
    assert block_table.shape[0] == requests and query_start_loc.shape[0] == requests + 1, "a row of block_table and a start per request, and the end"
    assert window_size is None or int(window_size) >= 1, "a window of at least one token, or None"
    assert int(num_first_tokens) >= 0


def _check_sparse(q, k_cache, indices, lens, cache_block_size, softmax_scale, attn_sink, out, lse, token_bytes):
    _check(q, k_cache, cache_block_size, softmax_scale, attn_sink, out, lse, token_bytes)
    assert indices.dtype == torch.int32 and indices.dim() == 2 and indices.stride(1) == 1, "indices: int32 [tokens, k] with unit inner stride"
    assert lens.dtype == torch.int32 and lens.dim() == 1 and lens.is_contiguous(), "lens: int32 [tokens]"
    assert indices.shape[0] == q.shape[0] and lens.shape[0] == q.shape[0], "a row of indices and a length per token"
    assert indices.device == q.device and lens.device == q.device, "all tensors must be on the same device"


def _check(q, k_cache, cache_block_size, softmax_scale, attn_sink, out, lse, token_bytes):
    assert q.device.type == "cuda", "this operator has no CPU path"
    assert q.dim() == 3 and q.shape[2] == HEAD_DIM and q.dtype == torch.bfloat16 and q.stride(2) == 1, "q: bfloat16 [tokens, heads, 512]"
    assert k_cache.dtype == torch.uint8 and k_cache.dim() == 2 and k_cache.stride(1) == 1, "k_cache: uint8 [blocks, bytes]"
    assert int(cache_block_size) > 0 and k_cache.shape[1] // token_bytes >= int(cache_block_size), f"a cache block holds cache_block_size tokens of {token_bytes} bytes"
    assert k_cache.shape[0] <= 1 or k_cache.stride(0) >= k_cache.shape[1], "cache blocks must not overlap"
    scale = torch.tensor(float(softmax_scale), dtype=torch.float32)
    assert scale > 0 and torch.isfinite(scale * 1.4426950408889634), "a positive softmax_scale, and in 32 bits a number also when it is divided by ln 2"
    tokens, heads = q.shape[:2]
    for t in (k_cache, attn_sink, out, lse):
        assert t is None or t.device == q.device, "all tensors must be on the same device"
    if attn_sink is not None:
        assert attn_sink.dtype == torch.float32 and attn_sink.shape == (heads,) and attn_sink.is_contiguous(), "attn_sink: float32 [heads]"
    if out is not None:
        assert out.dtype == torch.bfloat16 and out.shape == q.shape and out.stride(2) == 1, "out: bfloat16 like q"
    if lse is not None:
        assert lse.dtype == torch.float32 and lse.shape == (tokens, heads), "lse: float32 [tokens, heads]"
    if tokens and heads:
        assert out is None or (apart(out, q) and rows_apart(out)), "out must not overlap q or itself"
        assert lse is None or rows_apart(lse), "lse must not overlap itself"


__all__ = ["paged_latent_attention", "paged_latent_attention_mxfp4", "sparse_latent_attention", "sparse_latent_attention_mxfp4"]
