"""CPU-only checks of the entries for latent attention: symbols, struct layouts, refusals (validate_only launches nothing), plain forms."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from flash_attention_factory_amd import _cabi, torch_ops
from flash_attention_factory_amd.lib import (_latent, attention_latent_expanded, latent_cache_append, latent_cache_gather,
                                             paged_attention_latent)

import _latent as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P16 = 1 << 20  # an aligned address that nothing follows
BAD, NULL, TYPE, SIZE = (_cabi.FA_ERR_BAD_SHAPE, _cabi.FA_ERR_NULL_POINTER, _cabi.FA_ERR_UNSUPPORTED_DTYPE,
                         _cabi.FA_ERR_UNSUPPORTED_HEAD_OR_BLOCK_SIZE)


def test_header_symbols_are_exported():
    header = open(os.path.join(ROOT, "include", "fa_latent.h")).read()
    declared = set(re.findall(r"\b(fa_[a-z0-9_]+)\s*\(", header[header.index('extern "C"'):]))
    assert declared == set(_cabi.LATENT_EXPORTS)
    L = _cabi.load()
    assert all(hasattr(L, name) for name in declared)


def test_structs_agree_with_the_compiler(tmp_path):
    structs = [("append", _cabi.LatentAppendShape), ("gather", _cabi.LatentGatherShape), ("attention", _cabi.LatentAttentionShape),
               ("expanded", _cabi.LatentExpandedShape)]
    lines, want = ["#include <stddef.h>", "#include <stdio.h>", '#include "fa_latent.h"', "int main(void) {"], []
    for name, cls in structs:
        c = f"fa_latent_{name}_shape"
        lines.append(f'{c} {name} = FA_LATENT_{name.upper()}_SHAPE_INIT; printf("{c} %zu %u\\n", sizeof({c}), {name}.struct_size);')
        lines += [f'printf("{c}.{f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in cls._fields_]
        want.append(f"{c} {ctypes.sizeof(cls)} {cls().struct_size}")
        want += [f"{c}.{f[0]} {getattr(cls, f[0]).offset}" for f in cls._fields_]
    source = tmp_path / "sizes.c"
    source.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    said = subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split("\n")
    assert said[:-1] == want


def _filled(struct, fields, changes):
    for name, value in {**fields, **changes}.items():
        setattr(struct, name, value)
    return struct


def _validate():
    op = _cabi.Options()
    op.validate_only = 1
    return ctypes.byref(op)


POOL = dict(latent_dim=512, rope_dim=64, block_size=16, max_blocks_per_seq=4, block_stride=16 * 576, token_stride=576, num_pool_blocks=9, cache_dtype=0)


def _append(shape=None, **args):
    sh = _filled(_cabi.LatentAppendShape(), dict(POOL, num_seqs=2, num_tokens=5, num_heads=8, latent_token_stride=576, rope_key_token_stride=576,
                                                 query_token_stride=1536, query_head_stride=192, query_out_token_stride=512,
                                                 query_out_head_stride=64, max_positions=64, norm_eps=1e-6), shape or {})
    a = {**dict.fromkeys(("latent", "rope", "cache", "weight", "cos_sin", "query", "query_out", "scales", "tables", "start", "lens"), P16), **args}
    return _cabi.load().fa_latent_cache_append(*a.values(), ctypes.byref(sh), _validate())


def _gather(shape=None, **args):
    sh = _filled(_cabi.LatentGatherShape(), dict(POOL, num_seqs=2, num_rows=5, out_stride=576), shape or {})
    a = {**dict.fromkeys(("out", "cache", "scales", "tables", "start", "first"), P16), **args}
    return _cabi.load().fa_latent_cache_gather(*a.values(), ctypes.byref(sh), _validate())


def _attend(shape=None, **args):
    sh = _filled(_cabi.LatentAttentionShape(), dict(POOL, num_seqs=2, num_tokens=5, num_heads=8, query_latent_token_stride=4096,
                                                    query_latent_head_stride=512, query_rope_token_stride=1536, query_rope_head_stride=192,
                                                    out_token_stride=4096, out_head_stride=512, max_query_len=4, max_context_len=60), shape or {})
    a = {**dict.fromkeys(("out", "ql", "qr", "cache", "scales", "tables", "start", "lens"), P16), "scale": 0.1, "space": P16, **args}
    return _cabi.load().fa_paged_attention_latent(*a.values(), 1 << 40, ctypes.byref(sh), _validate())


def _expand(shape=None, **args):
    sh = _filled(_cabi.LatentExpandedShape(), dict(num_seqs=2, num_tokens=5, num_keys=50, num_heads=8, head_size=128, rope_dim=64, query_token_stride=1536,
                                                   query_head_stride=192, key_token_stride=2048, key_head_stride=256, rope_key_token_stride=576,
                                                   value_token_stride=2048, value_head_stride=256, out_token_stride=1024, out_head_stride=128,
                                                   max_query_len=4, max_key_len=30), shape or {})
    a = {**dict.fromkeys(("out", "query", "key", "rope", "value", "start", "key_start"), P16), "scale": 0.1, "space": P16, **args}
    return _cabi.load().fa_attention_latent_expanded(*a.values(), 1 << 40, ctypes.byref(sh), _validate())


def test_entries_accept_what_they_say():
    for entry in (_append, _gather, _attend, _expand):
        assert entry() == _cabi.FA_OK
    for entry in (_append, _gather, _attend):
        assert entry(dict(cache_dtype=2)) == _cabi.FA_OK
        assert entry(dict(latent_dim=256, block_size=64)) == _cabi.FA_OK
        assert entry(scales=None) == _cabi.FA_OK  # a 16-bit pool needs none
    assert _append(query=None, query_out=None, cos_sin=None, weight=None, shape=dict(max_positions=0, num_heads=0)) == _cabi.FA_OK
    assert _append(dict(num_tokens=0), latent=None, rope=None) == _cabi.FA_OK
    assert _gather(first=None) == _cabi.FA_OK
    assert _attend(dict(num_tokens=0), out=None, ql=None) == _cabi.FA_OK
    assert _attend(dict(num_heads=128, max_context_len=0), scale=-0.5) == _cabi.FA_OK
    assert _expand(dict(num_keys=0), key=None, rope=None, value=None) == _cabi.FA_OK
    assert _expand(dict(head_size=64)) == _cabi.FA_OK


@pytest.mark.parametrize("shape,code,text", [
    (dict(latent_dim=384), SIZE, "latent_dim"), (dict(rope_dim=32), SIZE, "rope_dim"), (dict(block_size=24), SIZE, "block_size"),
    (dict(block_size=8), SIZE, "block_size"), (dict(cache_dtype=1), TYPE, "cache_dtype"), (dict(cache_dtype=3), TYPE, "cache_dtype"),
    (dict(max_blocks_per_seq=0), BAD, "positive"), (dict(num_pool_blocks=0), BAD, "positive"), (dict(max_blocks_per_seq=1 << 27), BAD, "2^30"),
    (dict(block_stride=0), BAD, "pool strides"), (dict(token_stride=512), BAD, "pool strides"), (dict(token_stride=580), BAD, "16 bytes"),
    (dict(cache_dtype=2, token_stride=584), BAD, "16 bytes"), (dict(block_stride=1 << 40), BAD, "too large"), (dict(num_seqs=-1), BAD, "num_seqs"),
    (dict(struct_size=40), BAD, "struct_size"), (dict(struct_size=4096), BAD, "struct_size"),
])
def test_pools_that_are_refused(shape, code, text):
    for entry in (_append, _gather, _attend):
        assert entry(shape) == code, entry
        assert text in _cabi.load().fa_last_error().decode()


@pytest.mark.parametrize("entry,shape,args,code,text", [
    (_append, {}, dict(latent=None), NULL, "latent"), (_append, {}, dict(query_out=None), NULL, "come together"),
    (_append, dict(cache_dtype=2), dict(scales=None), NULL, "scales"), (_append, {}, dict(cos_sin=None), NULL, "cos_sin"),
    (_append, dict(src_dtype=2), {}, TYPE, "src_dtype"), (_append, dict(latent_token_stride=504), {}, BAD, "latent strides"),
    (_append, dict(rope_key_token_stride=60), {}, BAD, "rope_key strides"), (_append, dict(query_head_stride=68), {}, BAD, "query strides"),
    (_append, dict(num_heads=0), {}, BAD, "num_heads"), (_append, {}, dict(weight=P16 + 4), BAD, "aligned"), (_append, {}, dict(lens=P16 + 2), BAD, "aligned"),
    (_append, dict(norm_eps=-1.0), {}, BAD, "norm_eps"), (_append, dict(norm_eps=float("nan")), {}, BAD, "norm_eps"),
    (_append, dict(max_positions=-1), {}, BAD, "max_positions"),
    (_gather, {}, dict(start=None), NULL, "row_start"), (_gather, dict(cache_dtype=2), dict(scales=None), NULL, "scales"),
    (_gather, dict(out_dtype=5), {}, TYPE, "out_dtype"), (_gather, dict(out_stride=568), {}, BAD, "out strides"), (_gather, {}, dict(out=P16 + 8), BAD, "aligned"),
    (_gather, {}, dict(first=P16 + 2), BAD, "aligned"), (_gather, dict(num_rows=-1), {}, BAD, "num_rows"),
    (_attend, {}, dict(qr=None), NULL, "query_rope"), (_attend, dict(cache_dtype=2), dict(scales=None), NULL, "scales"),
    (_attend, dict(q_dtype=3), {}, TYPE, "q_dtype"), (_attend, dict(num_heads=0), {}, BAD, "num_heads"), (_attend, dict(max_query_len=0), {}, BAD, "max_query_len"),
    (_attend, dict(max_context_len=-1), {}, BAD, "max_context_len"), (_attend, dict(query_latent_head_stride=256), {}, BAD, "query_latent"),
    (_attend, dict(out_token_stride=4100), {}, BAD, "out"), (_attend, dict(query_rope_head_stride=32), {}, BAD, "query_rope strides"),
    (_attend, {}, dict(scale=float("inf")), BAD, "scale"), (_attend, {}, dict(scale=float("nan")), BAD, "scale"),
    (_attend, {}, dict(ql=P16 + 8), BAD, "aligned"), (_attend, dict(num_tokens=1 << 30), {}, BAD, "too large"),
    (_attend, dict(num_seqs=1 << 20, num_tokens=1 << 20, num_heads=128, max_blocks_per_seq=1 << 25), {}, BAD, "too large"),
    (_expand, dict(head_size=96), {}, SIZE, "head_size"), (_expand, dict(rope_dim=128), {}, SIZE, "rope_dim"), (_expand, dict(dtype=2), {}, TYPE, "dtype"),
    (_expand, {}, dict(value=None), NULL, "value"), (_expand, {}, dict(key_start=None), NULL, "key_start"),
    (_expand, dict(query_head_stride=128), {}, BAD, "query strides"), (_expand, dict(key_token_stride=2044), {}, BAD, "key, value and out"),
    (_expand, dict(rope_key_token_stride=8), {}, BAD, "rope_key strides"), (_expand, dict(value_token_stride=1 << 27), {}, BAD, "2^26"),
    (_expand, dict(max_key_len=-1), {}, BAD, "max_key_len"), (_expand, dict(num_keys=1 << 30), {}, BAD, "too large"),
    (_expand, {}, dict(rope=P16 + 2), BAD, "aligned"), (_expand, {}, dict(scale=float("nan")), BAD, "scale"), (_expand, dict(struct_size=8), {}, BAD, "struct_size"),
])
def test_calls_that_are_refused(entry, shape, args, code, text):
    assert entry(shape, **args) == code
    assert text in _cabi.load().fa_last_error().decode()


def test_host_tensors_are_refused():
    x, pool, ints = torch.zeros(2, 4, 512, dtype=torch.float16), torch.zeros(3, 16, 576, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    calls = ((latent_cache_append.run, (x[:, 0], x[:, 0, :64], pool, ints[None], ints, ints[:1])), (latent_cache_gather.run, (pool[0], pool, ints[None], ints)),
             (paged_attention_latent.run, (x, x, x[..., :64], pool, ints[None], ints, ints[:1], 0.1, 2)),
             (attention_latent_expanded.run, (x[..., :128], x[..., :192], x[..., :128], x[:, 0, :64], x[..., :128], ints, ints, 0.1, 2)))
    for run, arguments in calls:
        with pytest.raises(RuntimeError, match="on the GPU only"):
            run(*arguments)


@pytest.mark.parametrize("cache,scales,text", [
    (torch.zeros(3, 16, 64, dtype=torch.float16), None, "latent"), (torch.zeros(3, 16, 4, 576, dtype=torch.float16), None, "latent"),
    (torch.zeros(3, 16, 576, dtype=torch.bfloat16), None, "not torch.bfloat16"), (torch.zeros(3, 16, 576).to(torch.float8_e5m2), None, "float8"),
    (torch.zeros(3, 16, 576).to(torch.float8_e4m3fn), None, "need scales"), (torch.zeros(3, 16, 576, dtype=torch.float16), torch.ones(3, 16), "belong"),
    (torch.zeros(3, 16, 576).to(torch.float8_e4m3fn), torch.ones(3), "one for each row"),
    (torch.zeros(3, 16, 576).to(torch.float8_e4m3fn), torch.ones(3, 16, dtype=torch.float16), "one for each row"),
    (torch.zeros(3, 576, 16, dtype=torch.float16).transpose(1, 2), None, "contiguous last"),
])
def test_pool_tensors_that_are_refused(cache, scales, text):
    with pytest.raises(_cabi.PagedAttentionError, match=text):
        _latent.check_pool(cache, scales, torch.float16)


def test_operators_are_registered_and_trace():
    for name in ("latent_cache_append", "latent_cache_gather", "paged_attention_latent", "attention_latent_expanded"):
        assert hasattr(torch.ops.fa_amd, name) and name in torch_ops._NAMES
    x, pool, ints = (torch.zeros(s, dtype=t, device="meta") for s, t in (((2, 4, 512), torch.float16), ((3, 16, 576), torch.float16), ((2,), torch.int32)))
    assert torch.ops.fa_amd.paged_attention_latent(x, x, x[..., :64], pool, ints[None], ints, ints[:1], 0.1, 2) is None
    assert torch.ops.fa_amd.latent_cache_append(x[:, 0], x[:, 0, :64], pool, ints[None], ints, ints[:1]) is None
    assert torch.ops.fa_amd.latent_cache_gather(x[:, 0], pool, ints[None], ints) is None
    assert torch.ops.fa_amd.attention_latent_expanded(x[..., :128], x[..., :192], x[..., :128], x[:, 0, :64], x[..., :128], ints, ints, 0.1, 2) is None


def test_the_absorbed_form_is_the_expanded_one():
    """The identity that the two forms rest on, in the plain forms that the kernels are tested against: (q W_k) . c = q . (W_k c)."""
    g = torch.Generator().manual_seed(0)
    n, old, H, D, L = 5, 9, 3, 64, 256
    batch = R.Batch([n], [old], 16)
    _, _, values = R.pool(batch, L, "16", torch.float16)
    values = values[..., :L + R.ROPE]
    wk, wv = (torch.randn(H, D, L, generator=g).double() for _ in range(2))
    q, qr = torch.randn(n, H, D, generator=g).double(), torch.randn(n, H, R.ROPE, generator=g).double()
    t = torch.arange(n + old)
    rows = values[batch.tables[0, t // 16].long(), t % 16]
    ql = torch.matmul(q.transpose(0, 1), wk).transpose(0, 1)
    o, _ = R.absorbed(batch, ql, qr, values, 0.01)
    got = torch.matmul(o.transpose(0, 1), wv.transpose(1, 2)).transpose(0, 1)
    key, value = (torch.matmul(rows[:, :L], w.transpose(1, 2)).transpose(0, 1) for w in (wk, wv))
    want, _ = R.expanded(torch.cat([q, qr], -1), key, rows[:, L:], value, [0, n], [0, n + old], 0.01)
    assert torch.allclose(got, want, rtol=1e-9, atol=1e-9)
    # ... and the expanded one is torch's own attention
    full = torch.cat([key, rows[:, None, L:].expand(-1, H, -1)], -1)
    sdpa = torch.nn.functional.scaled_dot_product_attention(
        torch.cat([q, qr], -1).transpose(0, 1), full.transpose(0, 1), value.transpose(0, 1), scale=0.01,
        attn_mask=torch.arange(n + old)[None] <= torch.arange(old, old + n)[:, None]).transpose(0, 1)
    assert torch.allclose(want, sdpa, rtol=1e-9, atol=1e-9)
