"""What the modules for ragged batches share: checks of the tensors that describe a batch and its pools, and the shape struct.

A ragged batch brings the new tokens of all its sequences one behind the other: ``query_start`` (int32 ``[seqs + 1]``) says which
are whose, ``context_lens`` (int32 ``[seqs]``) counts each sequence's keys with its new tokens.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _cabi

_BYTE_CACHES = {torch.float8_e5m2: _cabi.FA_KV_CACHE_E5M2, torch.float8_e4m3fn: _cabi.FA_KV_CACHE_E4M3,
                torch.uint8: _cabi.FA_KV_CACHE_E5M2, torch.int8: _cabi.FA_KV_CACHE_I8}


def bad(message: str, code: int = _cabi.FA_ERR_BAD_SHAPE) -> _cabi.PagedAttentionError:
    return _cabi.PagedAttentionError(code, message)


def dtype_of(name: str, t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return _cabi.FA_DTYPE_BF16
    if t.dtype == torch.float16:
        return _cabi.FA_DTYPE_F16
    raise bad(f"{name} must be fp16 or bf16, not {t.dtype}", _cabi.FA_ERR_UNSUPPORTED_DTYPE)


def cache_dtype_of(key_cache: torch.Tensor, value_cache: torch.Tensor, row_type: torch.dtype) -> int:
    """fa_kv_cache_dtype of a pair of pools: 16-bit pools hold the rows' own type."""
    if value_cache.dtype != key_cache.dtype or (key_cache.dtype != row_type and key_cache.dtype not in _BYTE_CACHES):
        raise bad(f"cache dtypes {key_cache.dtype}, {value_cache.dtype} are neither both {row_type} nor one byte format",
                  _cabi.FA_ERR_UNSUPPORTED_DTYPE)
    return _BYTE_CACHES.get(key_cache.dtype, _cabi.FA_KV_CACHE_16BIT)


def check_pools(key_cache: torch.Tensor, value_cache: torch.Tensor, kv_heads: Optional[int], head_size: int) -> None:
    if key_cache.dim() != 4 or key_cache.stride(3) != 1 or value_cache.stride() != key_cache.stride() \
            or key_cache.size(3) != head_size or kv_heads not in (None, key_cache.size(2)):
        raise bad("caches must be 4-D [blocks, block_size, kv_heads, head_size] views that match the rows, with a contiguous last "
                  "dimension and equal strides")
    _cabi.require_value_pool(key_cache, value_cache)


def check_batch(block_tables: torch.Tensor, query_start: torch.Tensor, context_lens: torch.Tensor) -> int:
    """Number of sequences."""
    for name, t in (("block_tables", block_tables), ("query_start", query_start), ("context_lens", context_lens)):
        if t.dtype != torch.int32:
            raise bad(f"{name} must be int32", _cabi.FA_ERR_UNSUPPORTED_DTYPE)
        if not t.is_contiguous():
            raise bad(f"{name} must be contiguous")
    S = context_lens.numel()
    if context_lens.dim() != 1 or block_tables.dim() != 2 or block_tables.size(0) != S or query_start.dim() != 1 \
            or query_start.numel() != S + 1:
        raise bad(f"block_tables must be [{S}, max_blocks_per_seq], query_start [{S + 1}] and context_lens [{S}]")
    return S


def check_scales(k_scales: Optional[torch.Tensor], v_scales: Optional[torch.Tensor], kv_heads: int, blocks: int) -> int:
    """fa_kv_scale of a pair of scale tensors (None: one scalar)."""
    if (k_scales is None) != (v_scales is None):
        raise bad("k_scales and v_scales come together", _cabi.FA_ERR_NULL_POINTER)
    if k_scales is None:
        return _cabi.FA_KV_SCALE_TENSOR
    for t in (k_scales, v_scales):
        if t.dtype != torch.float32 or not t.is_contiguous() or t.shape != k_scales.shape:
            raise bad("k_scales / v_scales must be contiguous fp32 device tensors of one shape")
    if tuple(k_scales.shape) == (kv_heads,):
        return _cabi.FA_KV_SCALE_HEAD
    if tuple(k_scales.shape) == (blocks, kv_heads):
        return _cabi.FA_KV_SCALE_BLOCK
    raise bad(f"scales of shape {tuple(k_scales.shape)} are neither [{kv_heads}] (per kv head) nor [{blocks}, {kv_heads}] "
              "(per block and kv head)")


def bound(v: int) -> int:
    """A bound of the caller's (a window, a number of keys) for a 32-bit field: beyond 2^31 - 1 it bounds nothing more."""
    return max(-1, min(int(v), 0x7fffffff))


def pointer(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def attention_shape(out: torch.Tensor, query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                    block_tables: torch.Tensor, query_start: torch.Tensor, context_lens: torch.Tensor, max_query_len: int,
                    max_context_len: int) -> _cabi.RaggedShape:
    """The shape struct of an attention over a ragged batch, every tensor checked."""
    if not query.is_cuda:
        raise RuntimeError("paged attention runs on the GPU only: `query` is not a device tensor")
    _cabi.require_same_device("query", query, (("out", out), ("key_cache", key_cache), ("value_cache", value_cache),
                                               ("block_tables", block_tables), ("query_start", query_start),
                                               ("context_lens", context_lens)))
    sh = _cabi.RaggedShape()
    sh.q_dtype = dtype_of("query", query)
    if query.dim() != 3 or (query.size(2) > 1 and query.stride(2) != 1):
        raise bad("query must be [tokens, heads, head_size] with a contiguous last dimension")
    if out.dtype != query.dtype or out.shape != query.shape or not out.is_contiguous():
        raise bad("out must be contiguous, of the shape and type of query")
    check_pools(key_cache, value_cache, None, query.size(2))
    sh.cache_dtype = cache_dtype_of(key_cache, value_cache, query.dtype)
    sh.num_seqs = check_batch(block_tables, query_start, context_lens)
    sh.num_tokens, sh.num_heads, sh.head_size = query.shape
    sh.num_pool_blocks, sh.block_size, sh.num_kv_heads = key_cache.shape[:3]
    sh.max_blocks_per_seq = block_tables.size(1)
    sh.kv_block_stride, sh.kv_token_stride, sh.kv_head_stride = key_cache.stride()[:3]
    sh.query_token_stride, sh.query_head_stride = query.stride()[:2]
    sh.max_query_len, sh.max_context_len = bound(max_query_len), bound(max_context_len)
    return sh
