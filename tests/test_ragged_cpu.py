"""CPU-only checks of the entries for ragged batches: symbols, struct layouts, refusals (validate_only launches nothing)."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from flash_attention_factory_amd import _cabi, torch_ops
from flash_attention_factory_amd.lib import kv_cache_append, paged_attention_differential, paged_attention_ragged

import _ragged as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P16 = 1 << 20  # an aligned address that nothing follows


def test_header_symbols_are_exported():
    header = open(os.path.join(ROOT, "include", "fa_ragged.h")).read()
    declared = set(re.findall(r"\b(fa_[a-z0-9_]+)\s*\(", header[header.index('extern "C"'):]))
    assert declared == set(_cabi.RAGGED_EXPORTS)
    L = _cabi.load()
    assert all(hasattr(L, name) for name in declared)


def test_structs_agree_with_the_compiler(tmp_path):
    fields = [("fa_kv_cache_append_shape", _cabi.KvAppendShape), ("fa_ragged_shape", _cabi.RaggedShape)]
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "fa_ragged.h"', "int main(void) {"]
    for name, cls in fields:
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    lines += [f'printf("i8 %d\\n", FA_KV_CACHE_I8);', "fa_ragged_shape a = FA_RAGGED_SHAPE_INIT;",
              "fa_kv_cache_append_shape b = FA_KV_CACHE_APPEND_SHAPE_INIT;", 'printf("init %u %u\\n", a.struct_size, b.struct_size);',
              "return 0; }"]
    source = tmp_path / "sizes.c"
    source.write_text("\n".join(lines))
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    said = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split("\n")
    want = []
    for name, cls in fields:
        want.append(f"{name} {ctypes.sizeof(cls)}")
        want += [f"{name}.{f[0]} {getattr(cls, f[0]).offset}" for f in cls._fields_]
    want += [f"i8 {_cabi.FA_KV_CACHE_I8}", f"init {ctypes.sizeof(_cabi.RaggedShape)} {ctypes.sizeof(_cabi.KvAppendShape)}"]
    assert said[:-1] == want


def _options(**fields):
    op = _cabi.Options()
    op.validate_only = 1
    for name, value in fields.items():
        setattr(op, name, value)
    return op


def _ragged_shape(**fields):
    sh = _cabi.RaggedShape()
    for name, value in dict(num_seqs=2, num_tokens=5, num_heads=8, num_kv_heads=2, head_size=128, block_size=16, max_blocks_per_seq=4,
                            kv_block_stride=16 * 2 * 128, kv_token_stride=256, kv_head_stride=128, query_token_stride=1024,
                            query_head_stride=128, q_dtype=0, cache_dtype=0, num_pool_blocks=9, max_query_len=4,
                            max_context_len=60).items():
        setattr(sh, name, value)
    for name, value in fields.items():
        setattr(sh, name, value)
    return sh


def _attend(sh, op, differential=False, **args):
    L = _cabi.load()
    a = dict(out=P16, query=P16, keys=P16, values=P16, tables=P16, start=P16, lens=P16, scale=0.1, lambdas=P16, weight=P16, eps=1e-5,
             space=P16)
    a.update(args)
    first = (a["out"], a["query"], a["keys"], a["values"], a["tables"], a["start"], a["lens"], a["scale"])
    if differential:
        return L.fa_paged_attention_differential(*first, a["lambdas"], a["weight"], a["eps"], 1.0, a["space"], 1 << 40, ctypes.byref(sh),
                                                 ctypes.byref(op))
    return L.fa_paged_attention_ragged(*first, a["space"], 1 << 40, ctypes.byref(sh), ctypes.byref(op))


def test_attention_accepts_what_it_says():
    assert _attend(_ragged_shape(), _options()) == _cabi.FA_OK
    assert _attend(_ragged_shape(cache_dtype=3), _options(kv_scale_mode=2, k_scales=P16, v_scales=P16)) == _cabi.FA_OK
    assert _attend(_ragged_shape(cache_dtype=2, head_size=64), _options(fp8_scale=0.5, mask_flags=7, softcap=1.0, alibi_slopes=P16)) == _cabi.FA_OK
    assert _attend(_ragged_shape(num_tokens=0), _options(), out=None, query=None) == _cabi.FA_OK
    assert _attend(_ragged_shape(), _options(mask_flags=4, window_left=3), differential=True) == _cabi.FA_OK
    assert _attend(_ragged_shape(), _options(), differential=True, weight=None) == _cabi.FA_OK


@pytest.mark.parametrize("shape,options,args,code,text", [
    (dict(head_size=96), {}, {}, _cabi.FA_ERR_UNSUPPORTED_HEAD_OR_BLOCK_SIZE, "head size"),
    (dict(block_size=24), {}, {}, _cabi.FA_ERR_UNSUPPORTED_HEAD_OR_BLOCK_SIZE, "block size"),
    (dict(num_heads=7), {}, {}, _cabi.FA_ERR_UNSUPPORTED_GROUP, "queries per token"),
    (dict(num_heads=64), {}, {}, _cabi.FA_ERR_UNSUPPORTED_GROUP, "queries per token"),
    (dict(q_dtype=2), {}, {}, _cabi.FA_ERR_UNSUPPORTED_DTYPE, "q_dtype"),
    (dict(cache_dtype=4), {}, {}, _cabi.FA_ERR_UNSUPPORTED_DTYPE, "cache_dtype"),
    (dict(cache_dtype=3), {}, {}, _cabi.FA_ERR_BAD_SHAPE, "integers need"),
    (dict(cache_dtype=3), dict(kv_scale_mode=2, k_scales=P16), {}, _cabi.FA_ERR_NULL_POINTER, "v_scales"),
    (dict(cache_dtype=1), dict(kv_scale_mode=5), {}, _cabi.FA_ERR_BAD_SHAPE, "kv_scale_mode"),
    (dict(max_query_len=0), {}, {}, _cabi.FA_ERR_BAD_SHAPE, "max_query_len"),
    (dict(num_pool_blocks=0), {}, {}, _cabi.FA_ERR_BAD_SHAPE, "num_pool_blocks"),
    (dict(kv_token_stride=100), {}, {}, _cabi.FA_ERR_BAD_SHAPE, "kv strides"),
    (dict(kv_token_stride=260), {}, {}, _cabi.FA_ERR_BAD_SHAPE, "16 bytes"),
    (dict(query_token_stride=1020), {}, {}, _cabi.FA_ERR_BAD_SHAPE, "query strides"),
    (dict(max_blocks_per_seq=1 << 27), {}, {}, _cabi.FA_ERR_BAD_SHAPE, "2^30"),
    (dict(num_seqs=1 << 20, max_blocks_per_seq=1 << 20), {}, {}, _cabi.FA_ERR_BAD_SHAPE, "too large"),
    (dict(struct_size=40), {}, {}, _cabi.FA_ERR_BAD_SHAPE, "struct_size"),
    ({}, dict(mask_flags=8), {}, _cabi.FA_ERR_BAD_SHAPE, "mask_flags"),
    ({}, dict(mask_flags=1), {}, _cabi.FA_ERR_NULL_POINTER, "alibi_slopes"),
    ({}, dict(mask_flags=2), {}, _cabi.FA_ERR_BAD_SHAPE, "softcap"),
    ({}, dict(mask_flags=4, window_left=-1), {}, _cabi.FA_ERR_BAD_SHAPE, "window_left"),
    ({}, dict(query_len=2), {}, _cabi.FA_ERR_BAD_SHAPE, "query_start"),
    ({}, {}, dict(keys=None), _cabi.FA_ERR_NULL_POINTER, "non-NULL"),
    ({}, {}, dict(query=P16 + 2), _cabi.FA_ERR_BAD_SHAPE, "aligned"),
    ({}, {}, dict(lens=P16 + 2), _cabi.FA_ERR_BAD_SHAPE, "aligned"),
    ({}, {}, dict(scale=float("nan")), _cabi.FA_ERR_BAD_SHAPE, "scale"),
    ({}, {}, dict(scale=float("inf")), _cabi.FA_ERR_BAD_SHAPE, "scale"),
])
def test_attention_refuses(shape, options, args, code, text):
    for differential in (False, True):
        assert _attend(_ragged_shape(**shape), _options(**options), differential, **args) == code or (
            differential and (shape.get("cache_dtype") == 1 or options.get("mask_flags") in (1, 2)))
        assert text in _cabi.load().fa_last_error().decode() or differential


@pytest.mark.parametrize("shape,options,args,code", [
    (dict(cache_dtype=1), {}, {}, _cabi.FA_ERR_UNSUPPORTED_DTYPE), ({}, dict(sinks=P16), {}, _cabi.FA_ERR_BAD_SHAPE),
    ({}, dict(mask_flags=2, softcap=1.0), {}, _cabi.FA_ERR_BAD_SHAPE), ({}, {}, dict(lambdas=None), _cabi.FA_ERR_NULL_POINTER),
    ({}, {}, dict(weight=P16 + 4), _cabi.FA_ERR_BAD_SHAPE), ({}, {}, dict(eps=-1.0), _cabi.FA_ERR_BAD_SHAPE),
    ({}, {}, dict(eps=float("nan")), _cabi.FA_ERR_BAD_SHAPE)])
def test_differential_refuses(shape, options, args, code):
    assert _attend(_ragged_shape(**shape), _options(**options), True, **args) == code


def _append(shape=None, options=None, **args):
    sh = _cabi.KvAppendShape()
    for name, value in {**dict(num_seqs=2, num_tokens=5, num_heads=8, num_kv_heads=2, head_size=128, block_size=16, max_blocks_per_seq=4,
                               kv_block_stride=16 * 2 * 128, kv_token_stride=256, kv_head_stride=128, query_token_stride=1536,
                               query_head_stride=128, query_out_token_stride=1024, query_out_head_stride=128, key_token_stride=1536,
                               key_head_stride=128, value_token_stride=1536, value_head_stride=128, num_pool_blocks=9, max_positions=64,
                               rotary_dim=128), **(shape or {})}.items():
        setattr(sh, name, value)
    a = {**dict.fromkeys(("query", "query_out", "key", "value", "keys", "values", "table", "tables", "start", "lens", "ks", "vs"), P16), **args}
    return _cabi.load().fa_kv_cache_append(*a.values(), ctypes.byref(sh), ctypes.byref(_options(**(options or {}))))


def test_append_accepts_what_it_says():
    assert _append() == _cabi.FA_OK
    assert _append(query=None, query_out=None, table=None, shape=dict(rotary_dim=0, num_heads=0)) == _cabi.FA_OK
    assert _append(shape=dict(cache_dtype=3, kv_scale_mode=2)) == _cabi.FA_OK
    assert _append(shape=dict(cache_dtype=1, kv_scale_mode=1)) == _cabi.FA_OK
    assert _append(shape=dict(num_tokens=0), key=None, value=None) == _cabi.FA_OK


@pytest.mark.parametrize("shape,args,code", [
    (dict(head_size=72, rotary_dim=0), {}, _cabi.FA_ERR_UNSUPPORTED_HEAD_OR_BLOCK_SIZE),
    (dict(block_size=8), {}, _cabi.FA_ERR_UNSUPPORTED_HEAD_OR_BLOCK_SIZE),
    (dict(rotary_dim=24), {}, _cabi.FA_ERR_BAD_SHAPE),
    (dict(rotary_dim=144), {}, _cabi.FA_ERR_BAD_SHAPE),
    (dict(max_positions=0), {}, _cabi.FA_ERR_NULL_POINTER),
    ({}, dict(table=None), _cabi.FA_ERR_NULL_POINTER),
    ({}, dict(query_out=None), _cabi.FA_ERR_NULL_POINTER),
    ({}, dict(value=None), _cabi.FA_ERR_NULL_POINTER),
    (dict(cache_dtype=3), {}, _cabi.FA_ERR_BAD_SHAPE),
    (dict(cache_dtype=1, kv_scale_mode=2), {}, _cabi.FA_ERR_BAD_SHAPE),
    (dict(kv_scale_mode=1), {}, _cabi.FA_ERR_BAD_SHAPE),
    (dict(cache_dtype=3, kv_scale_mode=2), dict(ks=None), _cabi.FA_ERR_NULL_POINTER),
    (dict(cache_dtype=9), {}, _cabi.FA_ERR_UNSUPPORTED_DTYPE),
    (dict(src_dtype=3), {}, _cabi.FA_ERR_UNSUPPORTED_DTYPE),
    (dict(key_head_stride=60), {}, _cabi.FA_ERR_BAD_SHAPE),
    (dict(kv_block_stride=0), {}, _cabi.FA_ERR_BAD_SHAPE),
    (dict(num_pool_blocks=0), {}, _cabi.FA_ERR_BAD_SHAPE),
    ({}, dict(key=P16 + 8), _cabi.FA_ERR_BAD_SHAPE),
])
def test_append_refuses(shape, args, code):
    assert _append(shape, **args) == code


def test_host_tensors_are_refused():
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    pool = torch.zeros(3, 16, 2, 64, dtype=torch.float16)
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU only"):
        paged_attention_ragged.run(q, q, pool, pool, ints[None], ints, ints[:1], 0.1, 2)
    with pytest.raises(RuntimeError, match="on the GPU only"):
        paged_attention_differential.run(q, q, pool, pool, ints[None], ints, ints[:1], 0.1, torch.ones(4), None, 2)
    with pytest.raises(RuntimeError, match="on the GPU only"):
        kv_cache_append.run(q[:, :2], q[:, :2], pool, pool, ints[None], ints, ints[:1])
    for name in ("kv_cache_append", "paged_attention_ragged", "paged_attention_differential"):
        assert hasattr(torch.ops.fa_amd, name) and name in torch_ops._NAMES


def test_fakes_trace():
    q = torch.zeros(2, 4, 64, dtype=torch.float16, device="meta")
    pool = torch.zeros(3, 16, 2, 64, dtype=torch.float16, device="meta")
    ints = torch.zeros(2, dtype=torch.int32, device="meta")
    assert torch.ops.fa_amd.paged_attention_ragged(q, q, pool, pool, ints[None], ints, ints[:1], 0.1, 2) is None
    assert torch.ops.fa_amd.kv_cache_append(q[:, :2], q[:, :2], pool, pool, ints[None], ints, ints[:1]) is None


def test_the_plain_forms_agree_with_a_softmax_over_one_sequence():
    """The 64-bit forms that the kernels are tested against, against torch's own on a dense sequence."""
    batch = R.Batch([7], [5], B=16)
    g = torch.Generator().manual_seed(0)
    q, k, v = torch.randn(7, 4, 64, generator=g), torch.randn(12, 2, 64, generator=g), torch.randn(12, 2, 64, generator=g)
    pools = [torch.zeros(batch.blocks, 16, 2, 64, dtype=torch.float64) for _ in range(2)]
    for pool, x in zip(pools, (k, v)):
        pool[batch.tables[0, 0].long(), :12] = x.double()
    want = torch.nn.functional.scaled_dot_product_attention(
        q.double().transpose(0, 1), k.double().repeat_interleave(2, 1).transpose(0, 1), v.double().repeat_interleave(2, 1).transpose(0, 1),
        attn_mask=torch.arange(12)[None] <= torch.arange(5, 12)[:, None]).transpose(0, 1)
    (got, bound), = R.attention(batch, q, *pools, 0.125)
    assert torch.allclose(got, want, atol=1e-12) and bool((bound >= got.abs() - 1e-12).all())
    one, two = R.attention(batch, q, *pools, 0.2, maps=2)
    o = R.differential([one, two], torch.full((4,), 0.5), None, 0.0, 2.0)
    assert torch.allclose(o, 2.0 * (one[0] - 0.5 * two[0]))
