"""``paged_attention_ragged.run``: causal attention of a ragged batch of new tokens over the paged pools.

``query`` / ``out`` are ``[tokens, heads, head_size]`` (fp16 or bf16; ``query`` may have token and head strides), the new tokens of
all sequences one behind the other: whole prompts, pieces of prompts and single tokens of running sequences in one call.  Token j of
a sequence's n new ones sits at position ``context_lens[s] - n + j`` and sees the keys up to there, which must be in the pools
already (``kv_cache_append`` puts them there).  ``max_query_len`` bounds the new tokens of a sequence, ``max_context_len`` its keys (0:
what the block table holds).

Pools: 16-bit of the queries' type; FP8 with ``fp8_scale``; or bytes (FP8 or int8) with ``k_scales`` / ``v_scales``, not negative, of
``[kv_heads]`` or ``[blocks, kv_heads]``.  ``sinks``, ``alibi_slopes``, ``softcap`` (> 0) and ``window_left`` (>= 0) act when they are
passed.  The reference has the single-token case only (paged_attention_loop.cpp:21-84); its ``attention_ref`` (test_paged.py:40-168)
says what the modifiers mean.

Returns the kernel time in microseconds as a one-element list, or ``[]`` with ``timed=False`` (asynchronous on the current stream).
"""
from __future__ import annotations

import ctypes
from typing import List, Optional

import torch

from .. import _cabi
from . import _ragged
from ._run import current_stream


def run(out: torch.Tensor, query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
        block_tables: torch.Tensor, query_start: torch.Tensor, context_lens: torch.Tensor, scale: float,
        max_query_len: int, max_context_len: int = 0, fp8_scale: float = 1.0, k_scales: Optional[torch.Tensor] = None,
        v_scales: Optional[torch.Tensor] = None, sinks: Optional[torch.Tensor] = None,
        alibi_slopes: Optional[torch.Tensor] = None, softcap: float = 0.0, window_left: int = -1, *,
        timed: bool = True) -> List[float]:
    L = _cabi.load()
    sh = _ragged.attention_shape(out, query, key_cache, value_cache, block_tables, query_start, context_lens, max_query_len,
                                 max_context_len)
    _cabi.require_same_device("query", query, (("sinks", sinks), ("alibi_slopes", alibi_slopes), ("k_scales", k_scales),
                                               ("v_scales", v_scales)))
    op = _cabi.Options()
    if sinks is not None:
        if sinks.dtype != query.dtype or sinks.numel() != sh.num_heads or not sinks.is_contiguous():
            raise _ragged.bad(f"sinks must be a contiguous [{sh.num_heads}] tensor of the query dtype")
        op.sinks = sinks.data_ptr()
    if alibi_slopes is not None:
        if alibi_slopes.dtype != torch.float32 or alibi_slopes.numel() != sh.num_heads or not alibi_slopes.is_contiguous():
            raise _ragged.bad(f"alibi_slopes must be contiguous fp32 [{sh.num_heads}]")
        op.alibi_slopes = alibi_slopes.data_ptr()
        op.mask_flags |= _cabi.FA_MASK_ALIBI
    if softcap > 0.0:
        op.mask_flags |= _cabi.FA_MASK_SOFTCAP
        op.softcap = softcap
    if window_left >= 0:
        op.mask_flags |= _cabi.FA_MASK_WINDOW
        op.window_left = _ragged.bound(window_left)
    if sh.cache_dtype == _cabi.FA_KV_CACHE_16BIT and k_scales is not None:
        raise _ragged.bad("k_scales / v_scales belong to byte pools", _cabi.FA_ERR_UNSUPPORTED_DTYPE)
    op.fp8_scale = fp8_scale
    op.kv_scale_mode = _ragged.check_scales(k_scales, v_scales, sh.num_kv_heads, sh.num_pool_blocks)
    op.k_scales, op.v_scales = _ragged.pointer(k_scales), _ragged.pointer(v_scales)
    return call(L.fa_paged_attention_ragged, 1, (), out, query, key_cache, value_cache, block_tables, query_start, context_lens, scale,
                sh, op, timed)


def call(entry, maps: int, extra: tuple, out, query, key_cache, value_cache, block_tables, query_start, context_lens, scale: float,
         sh: _cabi.RaggedShape, op: _cabi.Options, timed: bool) -> List[float]:
    """The C call, with its workspace from PyTorch's stream-ordered allocator."""
    op.stream = current_stream(query.device)
    elapsed = ctypes.c_float(0.0)
    op.elapsed_us = ctypes.pointer(elapsed) if timed else None
    with torch.cuda.device(query.device):
        need = _cabi.load().fa_paged_attention_ragged_workspace_bytes(ctypes.byref(sh), maps)
        space = torch.empty(need, dtype=torch.uint8, device=query.device) if need > 0 else None
        _cabi.check(entry(out.data_ptr(), query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), block_tables.data_ptr(),
                          query_start.data_ptr(), context_lens.data_ptr(), float(scale), *extra, _ragged.pointer(space), need,
                          ctypes.byref(sh), ctypes.byref(op)))
    return [elapsed.value] if timed else []
