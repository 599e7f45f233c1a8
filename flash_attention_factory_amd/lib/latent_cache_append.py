"""``latent_cache_append.run``: the new tokens of a ragged batch into a latent pool, normalised and rotated on the way.

``latent`` is ``[tokens, latent]``, ``rope_key`` ``[tokens, 64]`` (parts of one projection, say), ``query_rope`` ``[tokens, heads, 64]``
(optional: the rotated parts of the queries, rotated into ``query_rope_out``, which may be ``query_rope`` itself), all fp16 or all bf16.
With ``norm_weight`` (fp32 ``[latent]``) a latent c is stored as ``c / sqrt(mean(c^2) + norm_eps) * norm_weight``; without, as it is.
``cos_sin`` is fp32 ``[positions, 64]``: the cosines of a position's angles, then their sines; pairs are 32 apart, or neighbours
with ``interleaved=True``; None rotates nothing.  Token j of a sequence's n new ones is stored at position ``context_lens[s] - n + j``.

``cache`` is ``[blocks, block_size, latent + 64]``, 16-bit of the rows' type, or ``float8_e4m3fn`` with ``scales`` (fp32 ``[blocks,
block_size]``), which are written with the rows: the least power of two that brings a row's largest magnitude to 448 or less.  Upstream has
no such step.

Returns the kernel time in microseconds as a one-element list, or ``[]`` with ``timed=False`` (asynchronous on the current stream).
"""
from __future__ import annotations

import ctypes
from typing import List, Optional

import torch

from .. import _cabi
from . import _latent, _ragged
from ._run import current_stream


def run(latent: torch.Tensor, rope_key: torch.Tensor, cache: torch.Tensor, block_tables: torch.Tensor, query_start: torch.Tensor,
        context_lens: torch.Tensor, norm_weight: Optional[torch.Tensor] = None, cos_sin: Optional[torch.Tensor] = None,
        query_rope: Optional[torch.Tensor] = None, query_rope_out: Optional[torch.Tensor] = None,
        scales: Optional[torch.Tensor] = None, norm_eps: float = 1e-6, interleaved: bool = False, *, timed: bool = True) -> List[float]:
    L = _cabi.load()
    if not latent.is_cuda:
        raise RuntimeError("the append runs on the GPU only: `latent` is not a device tensor")
    _cabi.require_same_device("latent", latent, (("rope_key", rope_key), ("cache", cache), ("block_tables", block_tables),
                                                 ("query_start", query_start), ("context_lens", context_lens),
                                                 ("norm_weight", norm_weight), ("cos_sin", cos_sin), ("query_rope", query_rope),
                                                 ("query_rope_out", query_rope_out), ("scales", scales)))
    sh = _cabi.LatentAppendShape()
    sh.src_dtype = _ragged.dtype_of("latent", latent)
    sh.cache_dtype = _latent.check_pool(cache, scales, latent.dtype)
    tokens, width = latent.size(0), cache.size(2) - _latent.ROPE
    _latent.check_rows("latent", latent, (tokens, width), latent.dtype)
    _latent.check_rows("rope_key", rope_key, (tokens, _latent.ROPE), latent.dtype)
    if (query_rope is None) != (query_rope_out is None):
        raise _ragged.bad("query_rope and query_rope_out come together")
    if query_rope is not None:
        for name, t in (("query_rope", query_rope), ("query_rope_out", query_rope_out)):
            _latent.check_rows(name, t, (tokens, query_rope.size(1) if query_rope.dim() == 3 else -1, _latent.ROPE), latent.dtype)
        sh.num_heads = query_rope.size(1)
        sh.query_token_stride, sh.query_head_stride = query_rope.stride()[:2]
        sh.query_out_token_stride, sh.query_out_head_stride = query_rope_out.stride()[:2]
    if norm_weight is not None and (norm_weight.dtype != torch.float32 or not norm_weight.is_contiguous() or tuple(norm_weight.shape) != (width,)):
        raise _ragged.bad(f"norm_weight must be contiguous fp32 [{width}]")
    if cos_sin is not None:
        if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.size(1) != _latent.ROPE \
                or cos_sin.size(0) == 0:
            raise _ragged.bad(f"cos_sin must be contiguous fp32 [positions, {_latent.ROPE}] with at least one position")
        sh.max_positions = cos_sin.size(0)
    sh.num_seqs = _ragged.check_batch(block_tables, query_start, context_lens)
    sh.num_tokens, sh.latent_dim, sh.rope_dim = tokens, width, _latent.ROPE
    sh.num_pool_blocks, sh.block_size = cache.shape[:2]
    sh.max_blocks_per_seq = block_tables.size(1)
    sh.block_stride, sh.token_stride = cache.stride()[:2]
    sh.latent_token_stride, sh.rope_key_token_stride = latent.stride(0), rope_key.stride(0)
    sh.interleaved, sh.norm_eps = int(interleaved), norm_eps
    elapsed = ctypes.c_float(0.0)
    op = _cabi.Options()
    op.stream = current_stream(latent.device)
    op.elapsed_us = ctypes.pointer(elapsed) if timed else None
    with torch.cuda.device(latent.device):
        _cabi.check(L.fa_latent_cache_append(latent.data_ptr(), rope_key.data_ptr(), cache.data_ptr(), _ragged.pointer(norm_weight),
                                             _ragged.pointer(cos_sin), _ragged.pointer(query_rope), _ragged.pointer(query_rope_out),
                                             _ragged.pointer(scales), block_tables.data_ptr(), query_start.data_ptr(),
                                             context_lens.data_ptr(), ctypes.byref(sh), ctypes.byref(op)))
    return [elapsed.value] if timed else []
