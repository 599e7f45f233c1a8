"""``latent_cache_gather.run``: rows of a latent pool, read back as dense 16-bit rows: what the product that expands them into keys and
values takes.

Row ``row_start[s] + i`` of ``out`` (``[rows, latent + 64]``, fp16 or bf16, any row stride) becomes key ``first_keys[s] + i`` of sequence s
(``row_start`` int32 ``[seqs + 1]``, ``first_keys`` int32 ``[seqs]``, None: 0), times its scale where ``cache`` is ``float8_e4m3fn``.  A
16-bit pool is of ``out``'s type.  A key that the block table or the pool does not have gives zeros; rows behind the last
sequence's stay as they are.  Upstream has no such step.

Returns the kernel time in microseconds as a one-element list, or ``[]`` with ``timed=False`` (asynchronous on the current stream).
"""
from __future__ import annotations

import ctypes
from typing import List, Optional

import torch

from .. import _cabi
from . import _latent, _ragged
from ._run import current_stream


def run(out: torch.Tensor, cache: torch.Tensor, block_tables: torch.Tensor, row_start: torch.Tensor,
        first_keys: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None, *, timed: bool = True) -> List[float]:
    L = _cabi.load()
    if not out.is_cuda:
        raise RuntimeError("the read-back runs on the GPU only: `out` is not a device tensor")
    _cabi.require_same_device("out", out, (("cache", cache), ("block_tables", block_tables), ("row_start", row_start),
                                           ("first_keys", first_keys), ("scales", scales)))
    sh = _cabi.LatentGatherShape()
    sh.out_dtype = _ragged.dtype_of("out", out)
    sh.cache_dtype = _latent.check_pool(cache, scales, out.dtype)
    _latent.check_rows("out", out, (out.size(0), cache.size(2)), out.dtype)
    for name, t, dims in (("block_tables", block_tables, 2), ("row_start", row_start, 1), ("first_keys", first_keys, 1)):
        if t is not None and (t.dtype != torch.int32 or not t.is_contiguous() or t.dim() != dims):
            raise _ragged.bad(f"{name} must be contiguous int32 of {dims} dimension(s)", _cabi.FA_ERR_UNSUPPORTED_DTYPE)
    S = block_tables.size(0)
    if row_start.numel() != S + 1 or (first_keys is not None and first_keys.numel() != S):
        raise _ragged.bad(f"row_start must be [{S + 1}] and first_keys [{S}] for block_tables of {S} sequences")
    sh.num_seqs, sh.num_rows = S, out.size(0)
    sh.latent_dim, sh.rope_dim = cache.size(2) - _latent.ROPE, _latent.ROPE
    sh.num_pool_blocks, sh.block_size = cache.shape[:2]
    sh.max_blocks_per_seq = block_tables.size(1)
    sh.block_stride, sh.token_stride = cache.stride()[:2]
    sh.out_stride = out.stride(0)
    elapsed = ctypes.c_float(0.0)
    op = _cabi.Options()
    op.stream = current_stream(out.device)
    op.elapsed_us = ctypes.pointer(elapsed) if timed else None
    with torch.cuda.device(out.device):
        _cabi.check(L.fa_latent_cache_gather(out.data_ptr(), cache.data_ptr(), _ragged.pointer(scales), block_tables.data_ptr(),
                                             row_start.data_ptr(), _ragged.pointer(first_keys), ctypes.byref(sh), ctypes.byref(op)))
    return [elapsed.value] if timed else []
