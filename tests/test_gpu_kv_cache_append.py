"""The ragged append against its formula, bit for bit: 32-bit operations that are rounded one by one have one result."""
import pytest
import torch

from flash_attention_factory_amd import torch_ops  # noqa: F401
from flash_attention_factory_amd.lib import kv_cache_append

import _ragged as R

pytestmark = pytest.mark.gpu

BATCHES = {
    "one_token": ([1], [0]),
    "decode": ([1] * 7, [0, 1, 14, 15, 16, 100, 333]),
    "ragged": ([5, 0, 1, 40, 16, 0, 33], [0, 9, 31, 7, 48, 16, 3]),
    "prompts": ([130, 257], [0, 45]),
}


def _inputs(batch, H, Hk, D, dtype, seed, spread=0.0):
    """Rows of one fused projection, as a model has them; ``spread``: tokens of different magnitudes."""
    g = torch.Generator().manual_seed(seed)
    fused = torch.randn(batch.T, H + 2 * Hk, D, generator=g) * torch.exp(spread * torch.randn(batch.T, 1, 1, generator=g))
    return fused.to(dtype)


def _pools(kv, batch, Hk, D, dtype, layout, seed):
    g = torch.Generator().manual_seed(seed)
    NB, B = batch.blocks, batch.B
    shape = (NB, Hk, B, D) if layout == "head" else (NB, B, Hk, D)
    pools, scales = [], []
    for _ in range(2):
        if kv == "i8":
            pools.append(torch.randint(-127, 128, shape, generator=g, dtype=torch.int8))
            scales.append(0.002 + 0.03 * torch.rand(NB, Hk, generator=g))
        elif kv == "16":
            pools.append(torch.randn(shape, generator=g).to(dtype))
        else:
            pools.append(torch.randn(shape, generator=g).to({"e5m2": torch.float8_e5m2, "e4m3": torch.float8_e4m3fn}[kv]))
    return pools, scales


def _view(pool, layout):
    return pool.permute(0, 2, 1, 3) if layout == "head" else pool


def _bits(t):
    return t.view(torch.int16) if t.dtype in (torch.float16, torch.bfloat16) else t.view(torch.uint8)


def _check(batch, H, Hk, D, dtype, kv, layout, rot, interleaved, *, seed=1, spread=0.5, head_scales=False, queries=True, call="op"):
    dev = torch.device("cuda")
    fused = _inputs(batch, H, Hk, D, dtype, seed, spread)
    pools, scales = _pools(kv, batch, Hk, D, dtype, layout, seed + 1)
    table = R.angle_table(max(max(batch.lens), 1), rot) if rot else None
    fp8_scale = 1.0
    if kv in ("e5m2", "e4m3"):
        if head_scales:
            g = torch.Generator().manual_seed(seed)
            scales = [0.5 + torch.rand(Hk, generator=g) for _ in range(2)]
        else:
            fp8_scale = 0.75
    d_fused = fused.to(dev)
    d_pools, d_scales = [p.to(dev) for p in pools], [s.to(dev) for s in scales]
    d_out = torch.full((batch.T, H, D), 7.0, dtype=dtype, device=dev)
    tables, start, lens = batch.on(dev)
    args = (d_fused[:, H:H + Hk], d_fused[:, H + Hk:], *(_view(p, layout) for p in d_pools), tables, start, lens,
            None if table is None else table.to(dev), d_fused[:, :H] if queries else None, d_out if queries else None,
            *(d_scales or (None, None)), fp8_scale, interleaved)
    if call == "op":
        torch.ops.fa_amd.kv_cache_append(*args)
    else:
        us = kv_cache_append.run(*args)
        assert len(us) == 1 and us[0] > 0
    torch.cuda.synchronize()
    want = R.append(batch, fused[:, H:H + Hk], fused[:, H + Hk:], *(_view(p, layout) for p in pools), table, interleaved,
                    *(scales or (None, None)), fp8_scale, fused[:, :H] if queries else None)
    for got, ref in zip(d_pools, pools):
        assert torch.equal(_bits(got.cpu()), _bits(ref))
    for got, ref in zip(d_scales, scales):
        assert torch.equal(got.cpu(), ref)
    if queries:
        assert torch.equal(_bits(d_out.cpu()), _bits(want))
    else:
        assert bool((d_out == 7.0).all())
    return d_pools, d_scales


@pytest.mark.parametrize("name", sorted(BATCHES))
@pytest.mark.parametrize("kv", ["16", "i8", "e5m2", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_formats(name, kv, dtype):
    _check(R.Batch(*BATCHES[name], B=16), 8, 2, 128, dtype, kv, "head", 128, False)


@pytest.mark.parametrize("D,rot,interleaved", [(64, 64, False), (64, 32, True), (128, 16, False), (128, 128, True), (96, 48, False),
                                               (256, 64, True), (16, 16, False), (80, 0, False)])
@pytest.mark.parametrize("kv", ["16", "i8"])
def test_head_sizes_and_rotations(D, rot, interleaved, kv):
    _check(R.Batch(*BATCHES["ragged"], B=32), 6, 3, D, torch.float16, kv, "token", rot, interleaved)


@pytest.mark.parametrize("B", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("layout", ["head", "token"])
def test_integer_blocks_of_every_size(B, D, layout):
    """Blocks that one wavefront, two or four hold in registers, and larger ones that are read twice."""
    _check(R.Batch([300, 1, 17, 64], [77, 5, 130, 0], B=B), 4, 2, D, torch.bfloat16, "i8", layout, D // 2, False)


def test_many_tokens_of_integers():
    """Over 1024 tokens a work-group looks for block owners among a block's worth of tokens."""
    _check(R.Batch([1, 700, 0, 1, 513, 15], [16, 3, 9, 15, 16, 1], B=16), 4, 2, 64, torch.float16, "i8", "head", 64, False)


def test_many_sequences():
    n = 300
    new = [(k * 7) % 3 for k in range(n)]
    _check(R.Batch(new, [(k * 11) % 50 for k in range(n)], B=16), 2, 1, 64, torch.bfloat16, "i8", "head", 64, False)
    _check(R.Batch(new, [(k * 11) % 50 for k in range(n)], B=16), 2, 1, 64, torch.bfloat16, "16", "head", 64, False)


@pytest.mark.parametrize("growth", [0.25, 4.0])
def test_scales_grow_and_stay(growth):
    """Token by token into the same blocks, each of `growth` times the magnitude: scales that grow every time, or never."""
    dev = torch.device("cuda")
    Hk, D, B, steps = 3, 64, 16, 20
    g = torch.Generator().manual_seed(5)
    pools = [torch.zeros(4, B, Hk, D, dtype=torch.int8) for _ in range(2)]
    scales = [torch.full((4, Hk), float("nan")) for _ in range(2)]  # a fresh block's old scale counts for nothing
    d_pools, d_scales = [p.to(dev) for p in pools], [s.to(dev) for s in scales]
    for step in range(steps):
        batch = R.Batch([1, 1], [step, step], B=B, lens=[step + 1, step + 1], spare=4)
        batch.tables = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32)
        rows = (torch.randn(2, 2 * Hk, D, generator=g) * growth ** (step % 5)).to(torch.bfloat16)
        tables, start, lens = batch.on(dev)
        torch.ops.fa_amd.kv_cache_append(rows[:, :Hk].to(dev), rows[:, Hk:].to(dev), *d_pools, tables, start, lens, None, None, None, *d_scales)
        R.append(batch, rows[:, :Hk], rows[:, Hk:], *pools, None, False, *scales)
        for got, ref in zip(d_pools + d_scales, pools + scales):
            assert torch.equal(torch.nan_to_num(got.cpu(), nan=-1.0) if got.is_floating_point() else got.cpu(),
                               torch.nan_to_num(ref, nan=-1.0) if ref.is_floating_point() else ref)


def test_zeros_and_what_is_not_a_number():
    """A block of zeros gets the least scale; NaN becomes 0 and does not count for the scale."""
    dev = torch.device("cuda")
    rows = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    rows[1, 0, 3], rows[1, 0, 5] = float("nan"), 2.0
    pools = [torch.full((2, 16, 1, 64), 9, dtype=torch.int8, device=dev) for _ in range(2)]
    scales = [torch.ones(2, 1, device=dev) for _ in range(2)]
    tables = torch.tensor([[0], [1]], dtype=torch.int32, device=dev)
    start, lens = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev), torch.tensor([1, 1], dtype=torch.int32, device=dev)
    torch.ops.fa_amd.kv_cache_append(rows[:, :1].to(dev), rows[:, 1:].to(dev), *pools, tables, start, lens, None, None, None, *scales)
    assert scales[0].flatten().tolist() == [2.0 ** -126, float(torch.tensor(2.0) * torch.tensor(1.0 / 127.0))]
    assert scales[1].flatten().tolist() == [2.0 ** -126] * 2
    assert bool((pools[0][0, 0] == 0).all()) and pools[0][1, 0, 0, 3] == 0 and pools[0][1, 0, 0, 5] == 127
    assert bool((pools[0][:, 1:] == 9).all())


@pytest.mark.parametrize("kv", ["16", "i8"])
def test_tokens_without_a_place(kv):
    """Negative positions, contexts beyond the table and block ids outside the pool: nothing is stored, the rest is."""
    batch = R.Batch([6, 20, 4], [0, 0, 12], B=16, lens=[4, 20, 16])
    batch.tables[1, 0] = batch.blocks + 5
    batch.tables[2, 0] = -1
    _check(batch, 2, 2, 64, torch.float16, kv, "head", 64, False)


def test_queries_in_place_and_left_out():
    dev = torch.device("cuda")
    batch = R.Batch([3, 9], [4, 0], B=16)
    q = torch.randn(batch.T, 4, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    kv = torch.randn(batch.T, 2, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    table = R.angle_table(16, 128)
    pools = [torch.zeros(batch.blocks, 16, 1, 128, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    d_q, (tables, start, lens) = q.to(dev), batch.on(dev)
    torch.ops.fa_amd.kv_cache_append(kv[:, :1].to(dev), kv[:, 1:].to(dev), *pools, tables, start, lens, table.to(dev), d_q, d_q)
    ref = [torch.zeros(batch.blocks, 16, 1, 128, dtype=torch.bfloat16) for _ in range(2)]
    want = R.append(batch, kv[:, :1], kv[:, 1:], *ref, table, False, query=q)
    assert torch.equal(d_q.cpu().view(torch.int16), want.view(torch.int16))
    _check(batch, 4, 2, 128, torch.float16, "i8", "head", 64, False, queries=False)
    _check(batch, 4, 2, 128, torch.float16, "16", "token", 64, True, queries=False, call="run")


@pytest.mark.parametrize("kv", ["e5m2", "e4m3"])
def test_fp8_scales_of_heads(kv):
    _check(R.Batch(*BATCHES["ragged"], B=16), 4, 2, 128, torch.bfloat16, kv, "head", 128, False, head_scales=True, call="run")


def test_nothing_to_append():
    batch = R.Batch([0, 0], [5, 0], B=16)
    _check(batch, 4, 2, 64, torch.float16, "i8", "head", 64, False, call="op")


def test_another_stream():
    side = torch.cuda.Stream()
    batch = R.Batch(*BATCHES["ragged"], B=16)
    with torch.cuda.stream(side):
        _check(batch, 4, 2, 128, torch.float16, "i8", "head", 128, False)
