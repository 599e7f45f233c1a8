"""``kv_cache_append.run``: the new tokens of a ragged batch into the paged pools, queries and keys rotated on the way.

``key`` / ``value`` are ``[tokens, kv_heads, head_size]``, ``query`` ``[tokens, heads, head_size]`` (optional; rotated into
``query_out``, which may be ``query`` itself), all fp16 or all bf16, with any token and head strides (parts of one fused
projection, say).  ``cos_sin`` is fp32 ``[positions, rotary_dim]``: the cosines of a position's angles, then their sines; the first
``rotary_dim`` elements of a row are rotated, pairs being ``rotary_dim / 2`` apart, or neighbours with ``interleaved=True``; None
rotates nothing.  Token j of a sequence's n new ones is stored at position ``context_lens[s] - n + j``.

Pools are ``[blocks, block_size, kv_heads, head_size]`` views: 16-bit of the rows' type; FP8 with a scalar ``fp8_scale`` or
``k_scales`` / ``v_scales`` of ``[kv_heads]``; or int8 with ``k_scales`` / ``v_scales`` of ``[blocks, kv_heads]``, which are kept up
to date: a block's scale grows to what its new rows ask for, and the rows that it held are rounded again.  A block whose first
row is new starts afresh.  Upstream has no such step (its tests fill pools with tensor casts, test_paged_fp8cache.py:171-203).

Returns the kernel time in microseconds as a one-element list, or ``[]`` with ``timed=False`` (asynchronous on the current stream).
"""
from __future__ import annotations

import ctypes
from typing import List, Optional

import torch

from .. import _cabi
from . import _ragged
from ._run import current_stream


def run(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
        block_tables: torch.Tensor, query_start: torch.Tensor, context_lens: torch.Tensor,
        cos_sin: Optional[torch.Tensor] = None, query: Optional[torch.Tensor] = None,
        query_out: Optional[torch.Tensor] = None, k_scales: Optional[torch.Tensor] = None,
        v_scales: Optional[torch.Tensor] = None, fp8_scale: float = 1.0, interleaved: bool = False, *,
        timed: bool = True) -> List[float]:
    L = _cabi.load()
    if not key.is_cuda:
        raise RuntimeError("the append runs on the GPU only: `key` is not a device tensor")
    _cabi.require_same_device("key", key, (("value", value), ("key_cache", key_cache), ("value_cache", value_cache),
                                           ("block_tables", block_tables), ("query_start", query_start),
                                           ("context_lens", context_lens), ("cos_sin", cos_sin), ("query", query),
                                           ("query_out", query_out), ("k_scales", k_scales), ("v_scales", v_scales)))
    sh = _cabi.KvAppendShape()
    sh.src_dtype = _ragged.dtype_of("key", key)
    for name, t in (("value", value), ("query", query), ("query_out", query_out)):
        if t is not None and t.dtype != key.dtype:
            raise _ragged.bad(f"{name} must be of key's type, {key.dtype}", _cabi.FA_ERR_UNSUPPORTED_DTYPE)
    for name, t in (("key", key), ("value", value), ("query", query), ("query_out", query_out)):
        if t is not None and (t.dim() != 3 or t.stride(2) != 1 or t.size(0) != key.size(0) or t.size(2) != key.size(2)):
            raise _ragged.bad(f"{name} must be [tokens, heads, head_size] as key is, with a contiguous last dimension")
    if value.shape != key.shape:
        raise _ragged.bad("value must have the shape of key")
    if (query is None) != (query_out is None) or (query is not None and query.shape != query_out.shape):
        raise _ragged.bad("query and query_out come together, in one shape")
    _ragged.check_pools(key_cache, value_cache, key.size(1), key.size(2))
    sh.cache_dtype = _ragged.cache_dtype_of(key_cache, value_cache, key.dtype)
    sh.num_seqs = _ragged.check_batch(block_tables, query_start, context_lens)
    sh.num_tokens, sh.num_kv_heads, sh.head_size = key.shape
    sh.num_pool_blocks, sh.block_size = key_cache.shape[:2]
    sh.max_blocks_per_seq = block_tables.size(1)
    sh.kv_block_stride, sh.kv_token_stride, sh.kv_head_stride = key_cache.stride()[:3]
    sh.key_token_stride, sh.key_head_stride = key.stride()[:2]
    sh.value_token_stride, sh.value_head_stride = value.stride()[:2]
    if query is not None:
        sh.num_heads = query.size(1)
        sh.query_token_stride, sh.query_head_stride = query.stride()[:2]
        sh.query_out_token_stride, sh.query_out_head_stride = query_out.stride()[:2]
    if cos_sin is not None:
        if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous():
            raise _ragged.bad("cos_sin must be contiguous fp32 [positions, rotary_dim]")
        sh.max_positions, sh.rotary_dim = cos_sin.shape
        if sh.rotary_dim == 0 or sh.max_positions == 0:
            raise _ragged.bad("cos_sin must hold at least one position and one pair")
    sh.interleaved = int(interleaved)
    sh.fp8_scale = fp8_scale
    if sh.cache_dtype == _cabi.FA_KV_CACHE_16BIT and k_scales is not None:
        raise _ragged.bad("k_scales / v_scales belong to byte pools", _cabi.FA_ERR_UNSUPPORTED_DTYPE)
    sh.kv_scale_mode = _ragged.check_scales(k_scales, v_scales, sh.num_kv_heads, sh.num_pool_blocks)
    elapsed = ctypes.c_float(0.0)
    op = _cabi.Options()
    op.stream = current_stream(key.device)
    op.elapsed_us = ctypes.pointer(elapsed) if timed else None
    with torch.cuda.device(key.device):
        _cabi.check(L.fa_kv_cache_append(_ragged.pointer(query), _ragged.pointer(query_out), key.data_ptr(), value.data_ptr(),
                                         key_cache.data_ptr(), value_cache.data_ptr(), _ragged.pointer(cos_sin),
                                         block_tables.data_ptr(), query_start.data_ptr(), context_lens.data_ptr(),
                                         _ragged.pointer(k_scales), _ragged.pointer(v_scales), ctypes.byref(sh), ctypes.byref(op)))
    return [elapsed.value] if timed else []
