"""``attention_latent_expanded.run``: causal attention of a ragged batch over keys and values that a product has expanded from latents.

``query`` is ``[tokens, heads, D + 64]``, ``key`` and ``value`` ``[keys, heads, D]`` (parts of one product's rows, say; D is 64 or 128),
``rope_key`` ``[keys, 64]``, shared by the heads; all fp16 or all bf16, any token and head strides.  Sequence s has the tokens
``query_start[s] ..`` and the keys ``key_start[s] ..`` (int32 ``[seqs + 1]``); its last token is at its last key, and a token sees the keys
up to its own:

    s = scale (query[:D] . key + query[D:] . rope_key),   out = sum of softmax(s) value

Values of a new token that are infinite or NaN can reach earlier new tokens of its sequence, nothing reaches another sequence.
``max_query_len`` and ``max_key_len`` (0: all keys) are bounds the host knows.  The form for prompts, where expanding every key once costs less
than attending latents that are four times as wide.  Upstream has no such kernel.

Returns the kernel time in microseconds as a one-element list, or ``[]`` with ``timed=False`` (asynchronous on the current stream).
"""
from __future__ import annotations

import ctypes
from typing import List

import torch

from .. import _cabi
from . import _latent, _ragged
from ._run import current_stream


def run(out: torch.Tensor, query: torch.Tensor, key: torch.Tensor, rope_key: torch.Tensor, value: torch.Tensor, query_start: torch.Tensor,
        key_start: torch.Tensor, scale: float, max_query_len: int, max_key_len: int = 0, *, timed: bool = True) -> List[float]:
    L = _cabi.load()
    if not query.is_cuda:
        raise RuntimeError("latent attention runs on the GPU only: `query` is not a device tensor")
    _cabi.require_same_device("query", query, (("out", out), ("key", key), ("rope_key", rope_key), ("value", value),
                                               ("query_start", query_start), ("key_start", key_start)))
    sh = _cabi.LatentExpandedShape()
    sh.dtype = _ragged.dtype_of("query", query)
    if query.dim() != 3 or key.dim() != 3:
        raise _ragged.bad("query must be [tokens, heads, D + 64] and key [keys, heads, D]")
    (tokens, heads, _), (keys, _, D) = query.shape, key.shape
    for name, t, shape in (("query", query, (tokens, heads, D + _latent.ROPE)), ("out", out, (tokens, heads, D)), ("key", key, (keys, heads, D)),
                           ("value", value, (keys, heads, D)), ("rope_key", rope_key, (keys, _latent.ROPE))):
        _latent.check_rows(name, t, shape, query.dtype)
    for name, t in (("query_start", query_start), ("key_start", key_start)):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.dim() != 1 or t.numel() < 1:
            raise _ragged.bad(f"{name} must be contiguous int32 [seqs + 1]", _cabi.FA_ERR_UNSUPPORTED_DTYPE)
    if key_start.numel() != query_start.numel():
        raise _ragged.bad("query_start and key_start must have one length")
    sh.num_seqs = query_start.numel() - 1
    sh.num_tokens, sh.num_keys, sh.num_heads, sh.head_size, sh.rope_dim = tokens, keys, heads, D, _latent.ROPE
    sh.query_token_stride, sh.query_head_stride = query.stride()[:2]
    sh.key_token_stride, sh.key_head_stride = key.stride()[:2]
    sh.rope_key_token_stride = rope_key.stride(0)
    sh.value_token_stride, sh.value_head_stride = value.stride()[:2]
    sh.out_token_stride, sh.out_head_stride = out.stride()[:2]
    sh.max_query_len, sh.max_key_len = _ragged.bound(max_query_len), _ragged.bound(max_key_len)
    elapsed = ctypes.c_float(0.0)
    op = _cabi.Options()
    op.stream = current_stream(query.device)
    op.elapsed_us = ctypes.pointer(elapsed) if timed else None
    with torch.cuda.device(query.device):
        need = L.fa_attention_latent_expanded_workspace_bytes(ctypes.byref(sh))
        space = torch.empty(need, dtype=torch.uint8, device=query.device) if need > 0 else None
        _cabi.check(L.fa_attention_latent_expanded(out.data_ptr(), query.data_ptr(), key.data_ptr(), rope_key.data_ptr(), value.data_ptr(),
                                                   query_start.data_ptr(), key_start.data_ptr(), scale, _ragged.pointer(space), need,
                                                   ctypes.byref(sh), ctypes.byref(op)))
    return [elapsed.value] if timed else []
