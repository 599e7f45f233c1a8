"""Ragged attention and differential attention against their 64-bit forms; unused rows of the pools, unused blocks' scales and
unused table entries hold what must never matter (NaN, ids of no block)."""
import math

import pytest
import torch

from flash_attention_factory_amd import torch_ops  # noqa: F401
from flash_attention_factory_amd.lib import paged_attention_differential, paged_attention_ragged

import _ragged as R

pytestmark = pytest.mark.gpu

F8 = {"e5m2": torch.float8_e5m2, "e4m3": torch.float8_e4m3fn}
BATCHES = {
    "one_token": ([1], [0]),
    "decode": ([1] * 6, [0, 1, 62, 127, 128, 515]),
    "edges": ([63, 64, 65, 1, 2, 128], [1, 64, 0, 63, 126, 63]),
    "mixed": ([1, 70, 0, 3, 1, 150], [300, 10, 20, 129, 0, 77]),
    "long": ([40, 1], [1500, 2100]),
}


def _pools(batch, Hk, D, kv, dtype, layout, seed, scales="block", spread=0.3):
    """(device pool, its values in 64 bits with zeros where nothing may be read, scales) for K and V."""
    g = torch.Generator().manual_seed(seed)
    NB, B = batch.blocks, batch.B
    got = []
    for _ in range(2):
        x = torch.randn(NB, B, Hk, D, generator=g)
        unused = ~batch.used[:, :, None, None].expand_as(x)
        s = None
        if kv == "16":
            pool = x.to(dtype)
            value = pool.double()
            pool = pool.masked_fill(unused, float("nan"))
        else:
            raw = (x * 40).round().clamp(-127, 127).to(torch.int8) if kv == "i8" else x.to(F8[kv])
            value = raw.double()
            if scales == "block":
                s = (0.025 if kv == "i8" else 1.0) * torch.exp(spread * torch.randn(NB, Hk, generator=g))
                value = value * s.double()[:, None, :, None]
                s = s.masked_fill(~batch.used.any(1)[:, None], float("nan"))
            elif scales == "head":
                s = (0.025 if kv == "i8" else 1.0) * (0.5 + torch.rand(Hk, generator=g))
                value = value * s.double()[None, None, :, None]
            junk = torch.full_like(raw, 100) if kv == "i8" else torch.full(raw.shape, 0x7f, dtype=torch.uint8).view(raw.dtype)
            pool = torch.where(unused, junk.view(torch.uint8), raw.view(torch.uint8)).view(raw.dtype)
        if layout == "head":
            pool = pool.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        got.append((pool.cuda(), value.masked_fill(unused, 0.0), None if s is None else s.cuda()))
    return got


def _query(batch, H, D, dtype, seed, size=1.0):
    """Queries as part of a wider row: token and head strides of their own."""
    g = torch.Generator().manual_seed(seed + 77)
    return (size * torch.randn(batch.T, H + 3, D + 8, generator=g)).to(dtype)[:, 1:H + 1, :D]


def _strided(q):
    """The same view on the device (copying it alone would make it contiguous)."""
    whole = torch.zeros(q.size(0), q.size(1) + 2, q.size(2) + 8, dtype=q.dtype, device="cuda")
    part = whole[:, 1:-1, :q.size(2)]
    part.copy_(q)
    return part


def _close(got, want, bound):
    off = (got.double().cpu() - want).abs() - bound
    assert not torch.isnan(got).any()
    assert bool((off <= 0.0).all()), f"off by {float((got.double().cpu() - want).abs().max())}, {float(off.max())} beyond the bound"


def _ragged(batch, H, Hk, D, kv, dtype, *, layout="head", seed=3, scales="block", scale=None, most=None, longest=0, q_size=1.0,
            window=-1, softcap=0.0, alibi=False, sinks=False, fp8_scale=1.0, spread=0.3, call="op"):
    query = _query(batch, H, D, dtype, seed, q_size)
    (kp, k, ks), (vp, v, vs) = _pools(batch, Hk, D, kv, dtype, layout, seed, scales, spread)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    slopes = torch.exp2(-8.0 * torch.arange(1, H + 1) / H) if alibi else None
    sink = torch.linspace(-1.0, 2.0, H).to(dtype) if sinks else None
    tables, start, lens = batch.on("cuda")
    out = torch.full((batch.T, H, D), float("nan"), dtype=dtype, device="cuda")
    args = (out, _strided(query), kp, vp, tables, start, lens, scale, most or max(1, max(batch.new)), longest)
    more = dict(fp8_scale=fp8_scale, k_scales=ks, v_scales=vs, sinks=None if sink is None else sink.cuda(),
                alibi_slopes=None if slopes is None else slopes.cuda(), softcap=softcap, window_left=window)
    if call == "op":
        torch.ops.fa_amd.paged_attention_ragged(*args, **more)
    else:
        us = paged_attention_ragged.run(*args, **more)
        assert len(us) == 1 and (us[0] > 0 or batch.T == 0)
    torch.cuda.synchronize()
    maps = R.attention(batch, query, k * fp8_scale, v * fp8_scale, scale, window=window, softcap=softcap, slopes=slopes, sinks=sink)
    operand = dtype if kv == "16" else torch.float16
    _close(out, maps[0][0], R.attention_bound(maps, dtype, operand))
    return out


@pytest.mark.parametrize("name", sorted(BATCHES))
@pytest.mark.parametrize("kv", ["16", "i8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_formats(name, kv, dtype, D):
    _ragged(R.Batch(*BATCHES[name], B=16), 8, 2, D, kv, dtype)


@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 1), (16, 1), (7, 7), (10, 2), (32, 2)])
@pytest.mark.parametrize("kv", ["16", "i8"])
def test_head_counts(H, Hk, kv):
    _ragged(R.Batch(*BATCHES["mixed"], B=16), H, Hk, 128, kv, torch.bfloat16)


@pytest.mark.parametrize("B", [32, 64, 256])
@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("kv", ["16", "i8"])
def test_blocks_and_layouts(B, layout, kv):
    _ragged(R.Batch(*BATCHES["mixed"], B=B), 4, 2, 128, kv, torch.float16, layout=layout)


@pytest.mark.parametrize("name", ["decode", "mixed"])
@pytest.mark.parametrize("kv", ["16", "i8"])
@pytest.mark.parametrize("mods", [dict(sinks=True), dict(window=0), dict(window=63), dict(window=100, sinks=True), dict(softcap=2.5),
                                  dict(alibi=True), dict(softcap=5.0, alibi=True, window=70, sinks=True)])
def test_modifiers(name, kv, mods):
    _ragged(R.Batch(*BATCHES[name], B=16), 8, 2, 64, kv, torch.float16, **mods)


@pytest.mark.parametrize("kv,scales,fp8_scale", [("e5m2", None, 1.0), ("e5m2", None, 0.5), ("e4m3", None, 2.0), ("e5m2", "head", 1.0),
                                                 ("i8", "head", 1.0), ("e5m2", "block", 1.0)])
@pytest.mark.parametrize("name", ["decode", "mixed"])
def test_scales(kv, scales, fp8_scale, name):
    _ragged(R.Batch(*BATCHES[name], B=16), 4, 2, 128, kv, torch.bfloat16, scales=scales, fp8_scale=fp8_scale, call="run")


@pytest.mark.parametrize("name", ["decode", "mixed", "long"])
def test_block_scales_of_very_different_size(name):
    """V scales that differ by orders of magnitude from block to block, in both directions."""
    _ragged(R.Batch(*BATCHES[name], B=16), 4, 2, 128, "i8", torch.bfloat16, spread=3.0, q_size=0.2)


@pytest.mark.parametrize("size", [1e-20, 1e20])
@pytest.mark.parametrize("name", ["decode", "mixed"])
def test_bf16_queries_beyond_fp16(size, name):
    """bf16 queries that fp16 could not hold, over integers, with the scale that brings the scores back."""
    _ragged(R.Batch(*BATCHES[name], B=16), 4, 2, 64, "i8", torch.bfloat16, q_size=size, scale=0.125 / size)


@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("name", ["decode", "mixed"])
@pytest.mark.parametrize("kv", ["16", "i8"])
def test_scales_of_the_scores(scale, name, kv):
    _ragged(R.Batch(*BATCHES[name], B=16), 4, 2, 64, kv, torch.bfloat16, scale=scale)


@pytest.mark.parametrize("kv", ["16", "i8"])
@pytest.mark.parametrize("new,old,lens", [([5, 40, 3], [0, 0, 0], [2, 25, 0]), ([1, 1], [0, 0], [0, 1])])
def test_tokens_that_see_nothing(kv, new, old, lens):
    """Contexts shorter than the new tokens, and none at all: zeros."""
    batch = R.Batch(new, old, B=16, lens=lens)
    out = _ragged(batch, 4, 2, 64, kv, torch.float16)
    assert bool((out[0] == 0).all())
    _ragged(batch, 4, 2, 64, kv, torch.float16, sinks=True)


@pytest.mark.parametrize("kv", ["16", "i8"])
def test_many_sequences(kv):
    n = 150
    new = [0 if k % 11 == 0 else 1 + (k * 5) % 3 if k % 7 else 40 for k in range(n)]
    _ragged(R.Batch(new, [(k * 37) % 200 for k in range(n)], B=16), 4, 2, 64, kv, torch.float16)


def test_one_long_sequence_is_cut():
    _ragged(R.Batch([1], [9001], B=16), 8, 1, 128, "i8", torch.bfloat16)
    _ragged(R.Batch([33], [6007], B=16), 8, 1, 128, "16", torch.bfloat16)
    _ragged(R.Batch([33], [6007], B=16), 8, 1, 128, "i8", torch.float16, sinks=True, longest=6040)


def test_bounds_that_are_wider_than_the_batch():
    batch = R.Batch(*BATCHES["mixed"], B=16)
    _ragged(batch, 4, 2, 128, "16", torch.float16, most=1000, longest=100000)
    _ragged(R.Batch(*BATCHES["decode"], B=16), 4, 2, 128, "i8", torch.float16, most=7, longest=100000)


def test_same_bits_every_time():
    a = _ragged(R.Batch(*BATCHES["long"], B=16), 8, 2, 128, "i8", torch.float16)
    for _ in range(3):
        assert torch.equal(a, _ragged(R.Batch(*BATCHES["long"], B=16), 8, 2, 128, "i8", torch.float16))


def test_nothing_asked():
    _ragged(R.Batch([0, 0], [3, 0], B=16), 4, 2, 64, "16", torch.float16, call="run")


def _differential(batch, H, Hk, D, kv, dtype, *, layout="head", seed=5, window=-1, norm=True, eps=1e-5, out_scale=0.8, longest=0, call="op"):
    query = _query(batch, H, D, dtype, seed)
    (kp, k, ks), (vp, v, vs) = _pools(batch, Hk, D, kv, dtype, layout, seed)
    scale = (D // 2) ** -0.5
    g = torch.Generator().manual_seed(seed)
    lambdas = 0.2 + 0.6 * torch.rand(H, generator=g)
    weight = 1.0 + 0.2 * torch.randn(D, generator=g) if norm else None
    tables, start, lens = batch.on("cuda")
    out = torch.full((batch.T, H, D), float("nan"), dtype=dtype, device="cuda")
    args = (out, _strided(query), kp, vp, tables, start, lens, scale, lambdas.cuda(), None if weight is None else weight.cuda(),
            max(1, max(batch.new)), longest)
    more = dict(norm_eps=eps, out_scale=out_scale, k_scales=ks, v_scales=vs, window_left=window)
    if call == "op":
        torch.ops.fa_amd.paged_attention_differential(*args, **more)
    else:
        assert paged_attention_differential.run(*args, **more)[0] > 0
    torch.cuda.synchronize()
    maps = R.attention(batch, query, k, v, scale, maps=2, window=window)
    want = R.differential(maps, lambdas, weight, eps, out_scale)
    operand = dtype if kv == "16" else torch.float16
    _close(out, want, R.attention_bound(maps, dtype, operand, lambdas, weight, eps, out_scale))
    return out


@pytest.mark.parametrize("name", sorted(BATCHES))
@pytest.mark.parametrize("kv", ["16", "i8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_differential_formats(name, kv, dtype, D):
    _differential(R.Batch(*BATCHES[name], B=16), 4, 2, D, kv, dtype)


@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 1), (8, 1), (16, 1), (6, 3)])
@pytest.mark.parametrize("window", [-1, 40])
def test_differential_head_counts(H, Hk, window):
    _differential(R.Batch(*BATCHES["mixed"], B=32), H, Hk, 128, "16", torch.float16, layout="token", window=window)


@pytest.mark.parametrize("name", ["decode", "mixed"])
@pytest.mark.parametrize("eps,out_scale", [(0.0, 1.0), (1e-2, -0.5)])
def test_differential_without_norm_and_with_other_constants(name, eps, out_scale):
    batch = R.Batch(*BATCHES[name], B=16)
    _differential(batch, 4, 2, 64, "16", torch.bfloat16, norm=False, out_scale=out_scale)
    if eps > 0:
        _differential(batch, 4, 2, 64, "16", torch.bfloat16, eps=eps, out_scale=out_scale, call="run")


def test_differential_one_long_sequence_is_cut():
    _differential(R.Batch([1], [9001], B=16), 4, 1, 128, "16", torch.bfloat16)
    _differential(R.Batch([33], [6007], B=16), 4, 1, 128, "i8", torch.float16, longest=6040)


def test_differential_rows_that_see_nothing():
    out = _differential(R.Batch([5, 40, 1], [0, 0, 0], B=16, lens=[2, 25, 0]), 4, 2, 64, "16", torch.float16)
    assert bool((out[:3] == 0).all()) and bool((out[-1] == 0).all())


def test_learned_lambda():
    g = torch.Generator().manual_seed(1)
    v = [0.1 * torch.randn(32, generator=g) for _ in range(4)]
    got = paged_attention_differential.learned_lambda(*v, 0.3, 5)
    want = math.exp(float(v[0].double() @ v[1].double())) - math.exp(float(v[2].double() @ v[3].double())) + 0.3
    assert got.shape == (5,) and got.dtype == torch.float32 and float((got.double() - want).abs().max()) < 1e-6


@pytest.mark.parametrize("which", ["ragged", "differential"])
def test_another_stream_and_graphs(which):
    """Captured once and replayed between eager work: every replay gives the eager result for the inputs of its time."""
    batch = R.Batch(*BATCHES["mixed"], B=16)
    H, Hk, D, dtype = 4, 2, 128, torch.float16
    query = _query(batch, H, D, dtype, 9).cuda()
    (kp, _, _), (vp, _, _) = _pools(batch, Hk, D, "16", dtype, "head", 9)
    tables, start, lens = batch.on("cuda")
    out = torch.zeros(batch.T, H, D, dtype=dtype, device="cuda")
    lambdas, weight = torch.full((H,), 0.4, device="cuda"), torch.ones(D, device="cuda")

    def call():
        if which == "ragged":
            torch.ops.fa_amd.paged_attention_ragged(out, query, kp, vp, tables, start, lens, 0.09, max(batch.new))
        else:
            torch.ops.fa_amd.paged_attention_differential(out, query, kp, vp, tables, start, lens, 0.125, lambdas, weight, max(batch.new))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for k in range(4):
        query.copy_(_query(batch, H, D, dtype, 20 + k))
        call()
        torch.cuda.synchronize()
        want = out.clone()
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
