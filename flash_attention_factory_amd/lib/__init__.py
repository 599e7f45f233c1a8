"""The four modules the upstream tests import (``from lib import paged_attention_loop``,
test_paged.py:2-3, test_paged_fp8cache.py:2-3), each exposing ``run(...)``, and
``kv_cache_write`` -- the step upstream has only as test code
(test_paged_fp8cache.py:171-203) that fills the pools those four read.  ``kv_cache_append``,
``paged_attention_ragged`` and ``paged_attention_differential`` serve ragged batches: any number of new tokens per sequence.
``latent_cache_append``, ``latent_cache_gather``, ``paged_attention_latent`` and ``attention_latent_expanded`` do so for models
whose keys and values come from one latent vector per token."""
from . import (attention_latent_expanded, kv_cache_append, kv_cache_write, latent_cache_append, latent_cache_gather,
               paged_attention_differential, paged_attention_fp8_loop, paged_attention_fp8_reduce, paged_attention_latent,
               paged_attention_loop, paged_attention_ragged, paged_attention_reduce)

__all__ = ["paged_attention_loop", "paged_attention_reduce", "paged_attention_fp8_loop",
           "paged_attention_fp8_reduce", "kv_cache_write", "kv_cache_append", "paged_attention_ragged",
           "paged_attention_differential", "latent_cache_append", "latent_cache_gather", "paged_attention_latent",
           "attention_latent_expanded"]
