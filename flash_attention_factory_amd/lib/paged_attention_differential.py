"""``paged_attention_differential.run``: differential attention of a ragged batch over the paged pools.

With q1, q2 the halves of a query row, k1, k2 those of a key row and V's rows whole, a head's result is

    o   = softmax(scale q1 k1^T) V - lambdas[head] softmax(scale q2 k2^T) V
    out = out_scale * norm_weight * o / sqrt(mean(o^2) + norm_eps)

(without ``norm_weight``: ``out_scale * o``), in 32 bits, rounded once.  ``lambdas`` is fp32 ``[heads]``: what a layer has learned,
``exp(lq1 . lk1) - exp(lq2 . lk2) + lambda_init``, one number per head; ``learned_lambda`` computes it.  ``scale`` is that of the
halves, usually ``(head_size / 2) ** -0.5``, ``out_scale`` usually ``1 - lambda_init``.  The batch, the pools and the other
arguments are those of ``paged_attention_ragged``; pools hold 16-bit values or int8 with scales.

Returns the kernel time in microseconds as a one-element list, or ``[]`` with ``timed=False`` (asynchronous on the current stream).
"""
from __future__ import annotations

from typing import List, Optional

import torch

from .. import _cabi
from . import _ragged
from .paged_attention_ragged import call


def learned_lambda(lq1: torch.Tensor, lk1: torch.Tensor, lq2: torch.Tensor, lk2: torch.Tensor, lambda_init: float,
                   num_heads: int) -> torch.Tensor:
    """fp32 ``[heads]`` from a layer's four vectors ``[head_size / 2]`` (or ``[heads, head_size / 2]``), once after loading."""
    lam = torch.exp((lq1.float() * lk1.float()).sum(-1)) - torch.exp((lq2.float() * lk2.float()).sum(-1)) + lambda_init
    return lam.expand(num_heads).contiguous()


def run(out: torch.Tensor, query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
        block_tables: torch.Tensor, query_start: torch.Tensor, context_lens: torch.Tensor, scale: float,
        lambdas: torch.Tensor, norm_weight: Optional[torch.Tensor], max_query_len: int, max_context_len: int = 0,
        norm_eps: float = 1e-5, out_scale: float = 1.0, k_scales: Optional[torch.Tensor] = None,
        v_scales: Optional[torch.Tensor] = None, window_left: int = -1, *, timed: bool = True) -> List[float]:
    L = _cabi.load()
    sh = _ragged.attention_shape(out, query, key_cache, value_cache, block_tables, query_start, context_lens, max_query_len,
                                 max_context_len)
    _cabi.require_same_device("query", query, (("lambdas", lambdas), ("norm_weight", norm_weight), ("k_scales", k_scales),
                                               ("v_scales", v_scales)))
    if lambdas.dtype != torch.float32 or lambdas.numel() != sh.num_heads or not lambdas.is_contiguous():
        raise _ragged.bad(f"lambdas must be contiguous fp32 [{sh.num_heads}]")
    if norm_weight is not None and (norm_weight.dtype != torch.float32 or norm_weight.numel() != sh.head_size
                                    or not norm_weight.is_contiguous()):
        raise _ragged.bad(f"norm_weight must be contiguous fp32 [{sh.head_size}]")
    op = _cabi.Options()
    if window_left >= 0:
        op.mask_flags |= _cabi.FA_MASK_WINDOW
        op.window_left = _ragged.bound(window_left)
    if sh.cache_dtype == _cabi.FA_KV_CACHE_16BIT and k_scales is not None:
        raise _ragged.bad("k_scales / v_scales belong to byte pools", _cabi.FA_ERR_UNSUPPORTED_DTYPE)
    op.kv_scale_mode = _ragged.check_scales(k_scales, v_scales, sh.num_kv_heads, sh.num_pool_blocks)
    op.k_scales, op.v_scales = _ragged.pointer(k_scales), _ragged.pointer(v_scales)
    extra = (lambdas.data_ptr(), _ragged.pointer(norm_weight), float(norm_eps), float(out_scale))
    return call(L.fa_paged_attention_differential, 2, extra, out, query, key_cache, value_cache, block_tables, query_start,
                context_lens, scale, sh, op, timed)
