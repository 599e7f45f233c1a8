"""What the modules for latent attention share: checks of a latent pool and its scales.

A latent pool is ``[blocks, block_size, latent + rope]``: each token's latent (256 or 512 elements) and its rotated key part (64), once for
all heads; 16-bit of the queries' type, or ``float8_e4m3fn`` with fp32 ``scales`` ``[blocks, block_size]``, one for each row.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _cabi
from ._ragged import bad

ROPE = 64


def check_pool(cache: torch.Tensor, scales: Optional[torch.Tensor], row_type: torch.dtype) -> int:
    """fa_kv_cache_dtype of a latent pool that serves rows of ``row_type``, its scales checked."""
    if cache.dim() != 3 or cache.stride(2) != 1 or cache.size(2) <= ROPE:
        raise bad(f"cache must be [blocks, block_size, latent + {ROPE}] with a contiguous last dimension")
    if cache.dtype == row_type:
        if scales is not None:
            raise bad("scales belong to FP8 pools", _cabi.FA_ERR_UNSUPPORTED_DTYPE)
        return _cabi.FA_KV_CACHE_16BIT
    if cache.dtype != torch.float8_e4m3fn:
        raise bad(f"cache must be {row_type} or float8_e4m3fn, not {cache.dtype}", _cabi.FA_ERR_UNSUPPORTED_DTYPE)
    if scales is None:
        raise bad("FP8 pools need scales", _cabi.FA_ERR_NULL_POINTER)
    if scales.dtype != torch.float32 or not scales.is_contiguous() or scales.shape != cache.shape[:2]:
        raise bad(f"scales must be contiguous fp32 {list(cache.shape[:2])}, one for each row of the pool")
    return _cabi.FA_KV_CACHE_E4M3


def check_rows(name: str, t: torch.Tensor, shape, dtype: torch.dtype) -> None:
    if t.dtype != dtype:
        raise bad(f"{name} must be {dtype}, not {t.dtype}", _cabi.FA_ERR_UNSUPPORTED_DTYPE)
    if tuple(t.shape) != tuple(shape) or (t.size(-1) > 1 and t.stride(-1) != 1):
        raise bad(f"{name} must be {list(shape)} with a contiguous last dimension")
