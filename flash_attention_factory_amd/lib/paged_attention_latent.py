"""``paged_attention_latent.run``: attention of a ragged batch over a latent pool itself, all heads over the same rows.

The products that expand a cached latent c into a head's keys and values are absorbed: ``query_latent`` (``[tokens, heads, latent]``) is
the head's query times the key part of that product, and what comes out (``out``, of the same shape) goes through the value
part afterwards.  With r the cached rotated part:

    s = scale (query_latent . c + query_rope . r),   out = sum of softmax(s) c

``query_rope`` is ``[tokens, heads, 64]``.  All three may have any token and head strides (heads outermost, as batched products leave
them; parts of a projection's rows).  ``cache`` is ``[blocks, block_size, latent + 64]``, 16-bit of the queries' type, or
``float8_e4m3fn`` with ``scales`` (fp32 ``[blocks, block_size]``).  Causal: token j of a sequence's n sees the keys up to position
``context_lens[s] - n + j``.  ``max_query_len`` and ``max_context_len`` (0: what the table holds) are bounds the host knows.  Upstream
has no such kernel.

Returns the kernel time in microseconds as a one-element list, or ``[]`` with ``timed=False`` (asynchronous on the current stream).
"""
from __future__ import annotations

import ctypes
from typing import List, Optional

import torch

from .. import _cabi
from . import _latent, _ragged
from ._run import current_stream


def run(out: torch.Tensor, query_latent: torch.Tensor, query_rope: torch.Tensor, cache: torch.Tensor, block_tables: torch.Tensor,
        query_start: torch.Tensor, context_lens: torch.Tensor, scale: float, max_query_len: int, max_context_len: int = 0,
        scales: Optional[torch.Tensor] = None, *, timed: bool = True) -> List[float]:
    L = _cabi.load()
    if not query_latent.is_cuda:
        raise RuntimeError("latent attention runs on the GPU only: `query_latent` is not a device tensor")
    _cabi.require_same_device("query_latent", query_latent, (("out", out), ("query_rope", query_rope), ("cache", cache),
                                                             ("block_tables", block_tables), ("query_start", query_start),
                                                             ("context_lens", context_lens), ("scales", scales)))
    sh = _cabi.LatentAttentionShape()
    sh.q_dtype = _ragged.dtype_of("query_latent", query_latent)
    sh.cache_dtype = _latent.check_pool(cache, scales, query_latent.dtype)
    if query_latent.dim() != 3:
        raise _ragged.bad("query_latent must be [tokens, heads, latent]")
    tokens, heads, width = query_latent.size(0), query_latent.size(1), cache.size(2) - _latent.ROPE
    for name, t, last in (("query_latent", query_latent, width), ("out", out, width), ("query_rope", query_rope, _latent.ROPE)):
        _latent.check_rows(name, t, (tokens, heads, last), query_latent.dtype)
    sh.num_seqs = _ragged.check_batch(block_tables, query_start, context_lens)
    sh.num_tokens, sh.num_heads, sh.latent_dim, sh.rope_dim = tokens, heads, width, _latent.ROPE
    sh.num_pool_blocks, sh.block_size = cache.shape[:2]
    sh.max_blocks_per_seq = block_tables.size(1)
    sh.block_stride, sh.token_stride = cache.stride()[:2]
    sh.query_latent_token_stride, sh.query_latent_head_stride = query_latent.stride()[:2]
    sh.query_rope_token_stride, sh.query_rope_head_stride = query_rope.stride()[:2]
    sh.out_token_stride, sh.out_head_stride = out.stride()[:2]
    sh.max_query_len, sh.max_context_len = _ragged.bound(max_query_len), _ragged.bound(max_context_len)
    elapsed = ctypes.c_float(0.0)
    op = _cabi.Options()
    op.stream = current_stream(query_latent.device)
    op.elapsed_us = ctypes.pointer(elapsed) if timed else None
    with torch.cuda.device(query_latent.device):
        need = L.fa_paged_attention_latent_workspace_bytes(ctypes.byref(sh))
        space = torch.empty(need, dtype=torch.uint8, device=query_latent.device) if need > 0 else None
        _cabi.check(L.fa_paged_attention_latent(out.data_ptr(), query_latent.data_ptr(), query_rope.data_ptr(), cache.data_ptr(),
                                                _ragged.pointer(scales), block_tables.data_ptr(), query_start.data_ptr(),
                                                context_lens.data_ptr(), scale, _ragged.pointer(space), need, ctypes.byref(sh),
                                                ctypes.byref(op)))
    return [elapsed.value] if timed else []
