"""Ragged append and attention at the edges of what a call may hold: rows and scales of zeros, lengths that the table or the caller's
bounds do not cover, sinks far above the scores, blocks longer than a step."""
import math

import pytest
import torch

from flash_attention_factory_amd import torch_ops  # noqa: F401

import _ragged as R
from test_gpu_ragged_attention import _close, _pools, _query, _strided

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -126  # the scale that the append gives to a block of zeros


def _attend(batch, query, pools, scale, *, maps=1, most=None, longest=0, window=-1, sinks=None, slopes=None, lambdas=None, weight=None,
            eps=1e-5, out_scale=1.0, fp8_scale=1.0, softcap=0.0):
    """The operator's result; rows that it leaves alone are NaN."""
    (kp, _, ks), (vp, _, vs) = pools
    dev = "cuda"
    tables, start, lens = batch.on(dev)
    out = torch.full(query.shape, float("nan"), dtype=query.dtype, device=dev)
    args = (out, _strided(query), kp, vp, tables.contiguous(), start, lens, scale)
    most = most or max(1, max(batch.new))
    if maps == 1:
        torch.ops.fa_amd.paged_attention_ragged(*args, most, longest, fp8_scale=fp8_scale, k_scales=ks, v_scales=vs,
                                                sinks=None if sinks is None else sinks.to(dev),
                                                alibi_slopes=None if slopes is None else slopes.to(dev), softcap=softcap,
                                                window_left=window)
    else:
        torch.ops.fa_amd.paged_attention_differential(*args, lambdas.to(dev), None if weight is None else weight.to(dev), most, longest,
                                                      norm_eps=eps, out_scale=out_scale, k_scales=ks, v_scales=vs, window_left=window)
    torch.cuda.synchronize()
    return out


# ---- factors of zero ----

@pytest.mark.parametrize("new,old", [([40, 1], [0, 30]), ([40], [100]), ([1, 3], [20, 47])])
@pytest.mark.parametrize("maps", [1, 2])
def test_rows_of_zeros_from_the_append(new, old, maps):
    """Padding: keys, values and queries of zeros, put into integer pools by the append itself."""
    batch = R.Batch(new, [0] * len(old), B=16, lens=[n + o for n, o in zip(new, old)])
    fill = R.Batch([n + o for n, o in zip(new, old)], [0] * len(old), B=16)
    fill.tables = batch.tables
    H, Hk, D, dtype, dev = 4, 2, 64, torch.bfloat16, "cuda"
    pools = [torch.full((batch.blocks, 16, Hk, D), 55, dtype=torch.int8, device=dev) for _ in range(2)]
    scales = [torch.full((batch.blocks, Hk), float("nan"), device=dev) for _ in range(2)]
    tables, start, lens = fill.on(dev)
    rows = torch.zeros(fill.T, Hk, D, dtype=dtype, device=dev)
    values = torch.ones(fill.T, Hk, D, dtype=dtype, device=dev)
    torch.ops.fa_amd.kv_cache_append(rows, values, *pools, tables, start, lens, None, None, None, *scales)
    for size in (0.0, 1e-6, 1.0):
        query = torch.full((batch.T, H, D), size, dtype=dtype)
        out = _attend(batch, query, [(pools[0], None, scales[0]), (pools[1], None, scales[1])], 0.125, maps=maps,
                      lambdas=torch.full((H,), 0.25))
        # every key counts the same, and every value is 1: 127 steps of 1 / 127 in 32 bits
        want = 1.0 if maps == 1 else 0.75
        assert bool(((out.float() - want).abs() < 2.0 ** -8).all())


@pytest.mark.parametrize("name", ["mixed", "decode"])
@pytest.mark.parametrize("k_scale", [LEAST, 0.0])
@pytest.mark.parametrize("scale", [0.0, 1e-33, 0.125, -0.125])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_key_scales_down_to_zero(name, k_scale, scale, dtype):
    """Some blocks' keys count for nothing (scores of 0 with them), whatever the scale of the scores and the queries' size."""
    batch = R.Batch(*{"mixed": ([1, 70, 0, 3, 1, 150], [300, 10, 20, 129, 0, 77]), "decode": ([1] * 6, [0, 1, 62, 127, 128, 515])}[name], B=16)
    H, Hk, D = 4, 2, 64
    (kp, k, ks), (vp, v, vs) = _pools(batch, Hk, D, "i8", dtype, "head", 3)
    some = torch.arange(batch.blocks) % 3 == 0
    there = some & batch.used.any(1)
    ks[there.cuda()] = k_scale
    k = k.masked_fill(some[:, None, None, None], 0.0)
    query = _query(batch, H, D, dtype, 3)
    query[::5] = 0
    out = _attend(batch, query, [(kp, k, ks), (vp, v, vs)], scale)
    maps = R.attention(batch, query, k, v, scale)
    _close(out, maps[0][0], R.attention_bound(maps, dtype, torch.float16))
    lambdas = torch.full((H,), 0.3)
    out = _attend(batch, query, [(kp, k, ks), (vp, v, vs)], scale, maps=2, lambdas=lambdas)
    maps = R.attention(batch, query, k, v, scale, maps=2)
    _close(out, R.differential(maps, lambdas, None, 0.0, 1.0), R.attention_bound(maps, dtype, torch.float16, lambdas))


# ---- blocks longer than a step of 64 keys, with a pool that ends with them ----

@pytest.mark.parametrize("B", [128, 256])
@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("kv", ["i8", "e4m3"])
def test_long_blocks_with_more_loading_threads_than_keys(B, layout, kv):
    """Rows of 64 bytes and eight wavefronts: twice as many threads as a step has keys to load."""
    batch = R.Batch([70, 1, 45], [1700, 300, 3], B=B, spare=0)
    H, Hk, D, dtype = 16, 2, 64, torch.float16
    query = _query(batch, H, D, dtype, 4)
    pools = _pools(batch, Hk, D, kv, dtype, layout, 4)
    (_, k, _), (_, v, _) = pools
    out = _attend(batch, query, pools, 0.125)
    maps = R.attention(batch, query, k, v, 0.125)
    _close(out, maps[0][0], R.attention_bound(maps, dtype, torch.float16))
    if kv == "i8":
        lambdas = torch.full((H,), 0.4)
        out = _attend(batch, query, pools, 0.125, maps=2, lambdas=lambdas)
        maps = R.attention(batch, query, k, v, 0.125, maps=2)
        _close(out, R.differential(maps, lambdas, None, 0.0, 1.0), R.attention_bound(maps, dtype, torch.float16, lambdas))


# ---- tokens beyond the block table ----

def _narrow(batch, columns):
    batch.tables = batch.tables[:, :columns].contiguous()
    return batch


@pytest.mark.parametrize("kv", ["16", "i8"])
@pytest.mark.parametrize("new,lens,columns", [([1], [33], 2), ([1, 40, 5], [40, 45, 31], 2), ([70, 2], [100, 65], 4), ([3], [80], 2)])
def test_append_beyond_the_table_is_left_out(kv, new, lens, columns):
    """Tokens at positions past the table's columns are not stored; those before are, at their own positions."""
    H, Hk, D, dtype, dev = 2, 2, 64, torch.float16, "cuda"
    batch = R.Batch(new, [0] * len(new), B=16, lens=lens)
    whole = batch.tables.clone()
    _narrow(batch, columns)
    g = torch.Generator().manual_seed(6)
    fused = torch.randn(batch.T, H + 2 * Hk, D, generator=g).to(dtype)
    shape = (batch.blocks, 16, Hk, D)
    if kv == "i8":
        pools = [torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2)]
        scales = [0.002 + 0.03 * torch.rand(batch.blocks, Hk, generator=g) for _ in range(2)]
    else:
        pools, scales = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)], []
    table = R.angle_table(max(lens), D)
    d_fused, d_pools, d_scales = fused.to(dev), [p.to(dev) for p in pools], [s.to(dev) for s in scales]
    d_out = torch.zeros(batch.T, H, D, dtype=dtype, device=dev)
    torch.ops.fa_amd.kv_cache_append(d_fused[:, H:H + Hk], d_fused[:, H + Hk:], *d_pools, *batch.on(dev), table.to(dev), d_fused[:, :H],
                                     d_out, *(d_scales or (None, None)))
    # the plain form on the wide table, with ids of no block beyond the narrow one
    batch.tables = torch.where(torch.arange(whole.size(1))[None] < columns, whole, torch.full_like(whole, 1 << 30))
    want = R.append(batch, fused[:, H:H + Hk], fused[:, H + Hk:], *pools, table, False, *(scales or (None, None)), query=fused[:, :H])
    for got, ref in zip(d_pools + d_scales, pools + scales):
        assert torch.equal(got.cpu(), ref)
    assert torch.equal(d_out.cpu(), want)


@pytest.mark.parametrize("new,old", [([3, 50], [20, 40]), ([1, 4], [0, 300])])
@pytest.mark.parametrize("kv", ["16", "i8"])
def test_append_of_more_tokens_in_query_start_than_rows(new, old, kv):
    """Arrays with fewer rows than query_start counts: the rows that are there keep their positions."""
    Hk, D, dtype, dev = 2, 64, torch.float16, "cuda"
    batch = R.Batch(new, old, B=16)
    rows = batch.T - 2
    fewer = R.Batch(new[:-1] + [new[-1] - 2], old, B=16)
    fewer.tables = batch.tables
    g = torch.Generator().manual_seed(11)
    fused = torch.randn(rows, 2 * Hk, D, generator=g).to(dtype)
    shape = (batch.blocks, 16, Hk, D)
    if kv == "i8":
        pools = [torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2)]
        scales = [0.002 + 0.03 * torch.rand(batch.blocks, Hk, generator=g) for _ in range(2)]
    else:
        pools, scales = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)], []
    table = R.angle_table(max(batch.lens), D)
    d_rows, d_pools, d_scales = fused.to(dev), [p.to(dev) for p in pools], [x.to(dev) for x in scales]
    torch.ops.fa_amd.kv_cache_append(d_rows[:, :Hk], d_rows[:, Hk:], *d_pools, *batch.on(dev), table.to(dev), None, None,
                                     *(d_scales or (None, None)))
    R.append(fewer, fused[:, :Hk], fused[:, Hk:], *pools, table, False, *(scales or (None, None)))
    for got, ref in zip(d_pools + d_scales, pools + scales):
        assert torch.equal(got.cpu(), ref)


def _beyond(batch, query, k, v, scale, columns, maps=1, window=-1, slopes=None):
    """64-bit form for tables of `columns` columns: tokens past it attend from its last position."""
    T, H, D = query.shape
    Hk, B, d = k.size(2), batch.B, D // maps
    got = [(torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)) for _ in range(maps)]
    for s, (n, ctx) in enumerate(zip(batch.new, batch.lens)):
        a, keys = int(batch.start[s]), min(ctx, columns * B)
        t, pos = torch.arange(keys), torch.arange(ctx - n, ctx).clamp_max(keys - 1)
        ids = batch.tables[s, t // B].long()
        sees = t[None] <= pos[:, None]
        if window >= 0:
            sees &= t[None] >= pos[:, None] - window
        for h in range(H):
            rows, vals = k[ids, t % B, h // (H // Hk)], v[ids, t % B, h // (H // Hk)]
            for m in range(maps):
                x = query[a:a + n, h, m * d:(m + 1) * d].double() @ rows[:, m * d:(m + 1) * d].T * scale
                if slopes is not None:
                    x = x + float(slopes[h]) * (t[None] - pos[:, None])
                x = x.masked_fill(~sees, -math.inf)
                p = torch.softmax(x, -1).masked_fill(~sees, 0.0)
                got[m][0][a:a + n, h] = p @ vals
                got[m][1][a:a + n, h] = p @ vals.abs()
    return got


@pytest.mark.parametrize("kv", ["16", "i8"])
@pytest.mark.parametrize("new,lens,columns", [([1, 1], [40, 33], 2), ([1, 2], [1300, 1290], 80), ([40, 7], [47, 20], 2),
                                              ([300], [1500], 80), ([90, 30], [100, 60], 2)])
@pytest.mark.parametrize("window", [-1, 12])
def test_attention_beyond_the_table_sees_what_is_there(kv, new, lens, columns, window):
    H, Hk, D, dtype = 4, 2, 64, torch.float16
    batch = R.Batch(new, [0] * len(new), B=16, lens=lens)
    query = _query(batch, H, D, dtype, 8)
    # rows past the narrow table's are not to be read
    wide = batch.tables.clone()
    for s in range(len(new)):
        for block in wide[s, columns:].tolist():
            if 0 <= block < batch.blocks:
                batch.used[block] = False
    pools = _pools(batch, Hk, D, kv, dtype, "head", 8)
    (_, k, _), (_, v, _) = pools
    _narrow(batch, columns)
    slopes = torch.tensor([0.5, 0.1, 0.02, 0.0])
    for more in ({}, {"slopes": slopes}):
        out = _attend(batch, query, pools, 0.125, window=window, **more)
        maps = _beyond(batch, query, k, v, 0.125, columns, window=window, **more)
        _close(out, maps[0][0], R.attention_bound(maps, dtype, dtype))
    lambdas = torch.full((H,), 0.4)
    out = _attend(batch, query, pools, 0.17, maps=2, lambdas=lambdas, window=window)
    maps = _beyond(batch, query, k, v, 0.17, columns, maps=2, window=window)
    _close(out, R.differential(maps, lambdas, None, 0.0, 1.0), R.attention_bound(maps, dtype, dtype, lambdas))


# ---- more new tokens than the call's bounds allow ----

@pytest.mark.parametrize("kv", ["16", "i8"])
@pytest.mark.parametrize("most", [1, 3, 30, 200])
@pytest.mark.parametrize("maps", [1, 2])
def test_tokens_beyond_max_query_len_are_left_out(kv, most, maps):
    """The first `most` tokens of a sequence are right, the rest of `out` stays as it was."""
    H, Hk, D, dtype = 4, 2, 64, torch.float16
    batch = R.Batch([40, 1, 300, 5], [7, 100, 650, 0], B=16)
    query = _query(batch, H, D, dtype, 9)
    pools = _pools(batch, Hk, D, kv, dtype, "head", 9)
    (_, k, _), (_, v, _) = pools
    lambdas = torch.full((H,), 0.4)
    out = _attend(batch, query, pools, 0.125, maps=maps, most=most, lambdas=lambdas, window=70 if most == 30 else -1)
    refs = R.attention(batch, query, k, v, 0.125, maps=maps, window=70 if most == 30 else -1)
    want = refs[0][0] if maps == 1 else R.differential(refs, lambdas, None, 0.0, 1.0)
    bound = R.attention_bound(refs, dtype, dtype, None if maps == 1 else lambdas)
    kept = torch.cat([torch.arange(n) < most for n in batch.new])
    assert bool(torch.isnan(out.cpu()[~kept]).all())
    _close(out.cpu()[kept], want[kept], bound[kept])


@pytest.mark.parametrize("new,old", [([3, 50], [20, 40]), ([1, 4], [0, 300])])
def test_more_tokens_in_query_start_than_rows(new, old):
    """Arrays with fewer rows than query_start counts: the rows that are there keep their positions."""
    H, Hk, D, dtype, dev = 4, 2, 64, torch.float16, "cuda"
    batch = R.Batch(new, old, B=16)
    rows = batch.T - 2
    query = _query(batch, H, D, dtype, 10)
    pools = _pools(batch, Hk, D, "16", dtype, "head", 10)
    (kp, k, _), (vp, v, _) = pools
    out = _attend(batch, query[:rows], pools, 0.125, most=max(new))
    refs = R.attention(batch, query, k, v, 0.125)
    _close(out, refs[0][0][:rows], R.attention_bound(refs, dtype, dtype)[:rows])


# ---- nothing to normalise ----

@pytest.mark.parametrize("new,old,lens", [([5, 3], [0, 0], [2, 0]), ([5, 40, 1], [0, 0, 0], [2, 25, 0]), ([2, 1], [0, 700], [1, 701]),
                                          ([2, 1], [0, 700], [0, 701])])
@pytest.mark.parametrize("longest", [0, 10000])
def test_differential_without_epsilon_and_without_keys(new, old, lens, longest):
    """norm_eps may be 0: tokens that see nothing are zeros, the others are normalised."""
    H, Hk, D, dtype = 4, 2, 64, torch.float16
    batch = R.Batch(new, old, B=16, lens=lens)
    query = _query(batch, H, D, dtype, 12)
    pools = _pools(batch, Hk, D, "16", dtype, "head", 12)
    (_, k, _), (_, v, _) = pools
    lambdas, weight = torch.full((H,), 0.3), 1.0 + 0.1 * torch.randn(D, generator=torch.Generator().manual_seed(1))
    out = _attend(batch, query, pools, 0.17, maps=2, lambdas=lambdas, weight=weight, eps=0.0, out_scale=0.8, longest=longest)
    refs = R.attention(batch, query, k, v, 0.17, maps=2)
    blind = (refs[0][1] == 0).all(-1).all(-1)
    assert bool(blind.any()) and bool((out.cpu()[blind] == 0).all())
    want = R.differential(refs, lambdas, weight, 0.0, 0.8)
    bound = R.attention_bound(refs, dtype, dtype, lambdas, weight, 0.0, 0.8)
    _close(out.cpu()[~blind], want[~blind], bound[~blind])


# ---- sinks far above the scores ----

@pytest.mark.parametrize("kv,dtype", [("16", torch.float16), ("16", torch.bfloat16), ("i8", torch.bfloat16), ("e4m3", torch.bfloat16)])
@pytest.mark.parametrize("new,old", [([1, 2], [400, 450]), ([1, 1], [1500, 900]), ([40, 3], [700, 900]), ([33], [3000])])
def test_sinks_far_above_the_scores(kv, dtype, new, old):
    """A sink takes its share of the sum and leaves the bits of the others' weights alone."""
    H, Hk, D = 8, 2, 64
    batch = R.Batch(new, old, B=16)
    query = _query(batch, H, D, dtype, 13, 0.1)
    pools = _pools(batch, Hk, D, kv, dtype, "head", 13)
    (_, k, _), (_, v, _) = pools
    v = v.abs()  # sums that do not cancel
    if kv == "16":
        pools[1] = (pools[1][0].abs(), None, None)
    elif kv == "i8":
        pools[1] = (pools[1][0].abs(), None, pools[1][2])
    else:
        pools[1] = ((pools[1][0].view(torch.uint8) & 0x7f).view(pools[1][0].dtype), None, pools[1][2])
    sinks = torch.linspace(8.0, 15.0, H).to(dtype)
    out = _attend(batch, query, pools, 0.125, sinks=sinks)
    refs = R.attention(batch, query, k, v, 0.125, sinks=sinks)
    bound = R.attention_bound(refs, dtype, dtype if kv == "16" else torch.float16) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    _close(out, refs[0][0], bound)


# ---- value scales of very different size ----

@pytest.mark.parametrize("new,old", [([1] * 4, [100, 40, 300, 800]), ([40, 1, 70], [100, 200, 20]), ([33], [1500])])
@pytest.mark.parametrize("small,zeros", [(LEAST, True), (2.0 ** -100, False), (0.0, True)])
@pytest.mark.parametrize("every", [2, 5])
def test_value_scales_that_lie_binary_orders_apart(new, old, small, zeros, every):
    """Blocks of zero (or hardly any) values among others: their keys count in the sum like all the others."""
    H, Hk, D, dtype = 8, 2, 64, torch.bfloat16
    batch = R.Batch(new, old, B=16)
    query = _query(batch, H, D, dtype, 14)
    pools = _pools(batch, Hk, D, "i8", dtype, "head", 14)
    (kp, k, ks), (vp, v, vs) = pools
    some = torch.arange(batch.blocks) % every == 0
    there = (some & batch.used.any(1)).cuda()
    vs[there] = small
    if zeros:
        vp[there] = 0
    v = v.masked_fill(some[:, None, None, None], 0.0)
    for maps in (1, 2):
        lambdas = torch.full((H,), 0.4)
        out = _attend(batch, query, [(kp, k, ks), (vp, v, vs)], 0.125, maps=maps, lambdas=lambdas)
        refs = R.attention(batch, query, k, v, 0.125, maps=maps)
        if maps == 1:
            _close(out, refs[0][0], R.attention_bound(refs, dtype, torch.float16))
        else:
            _close(out, R.differential(refs, lambdas, None, 0.0, 1.0), R.attention_bound(refs, dtype, torch.float16, lambdas))


# ---- the difference of two maps that are nearly alike ----

def _alike(batch, H, Hk, D, dtype, seed):
    """Queries whose halves differ by some hundredths, keys whose halves are the same: the maps differ little, and the rounding of
    their weights has nothing in common."""
    g = torch.Generator().manual_seed(seed)
    half = 0.3 * torch.randn(batch.T, H, D // 2, generator=g)
    query = torch.cat([half, half + 0.03 * torch.randn(batch.T, H, D // 2, generator=g)], -1).to(dtype)
    k = torch.randn(batch.blocks, batch.B, Hk, D // 2, generator=g)
    k = torch.cat([k, k], -1).to(dtype)
    v = torch.randn(batch.blocks, batch.B, Hk, D, generator=g).to(dtype)
    return query, k, v


def _alike_bound(refs, lambdas, dtype, weights):
    """Normalised difference (no epsilon, no weights of the norm): weights in two parts carry the square of one rounding, sums
    of 32 products of about 1 in 32 bits and their exponentials 2e-5; the result is rounded to its type once."""
    (o1, a1), (o2, a2) = refs
    o = o1 - lambdas.double()[:, None] * o2
    e = (weights + 2e-5) * (a1 + lambdas.double()[:, None] * a2)
    rms = torch.sqrt((o * o).mean(-1, keepdim=True) + 1e-5)
    off = e.square().mean(-1, keepdim=True).sqrt() / rms
    return (e + o.abs() * off * 1.1 + R.UNIT[dtype] * o.abs()) / rms + 1e-6


@pytest.mark.parametrize("dtype,new,old", [(torch.bfloat16, [1, 2, 1], [5, 9, 30]), (torch.float16, [1, 2, 1], [5, 9, 30]),
                                           (torch.bfloat16, [20, 33], [0, 0]), (torch.bfloat16, [1], [700])])
def test_weights_in_two_parts(dtype, new, old):
    """Over 16-bit pools the weights of two maps go to the matrix cores in two parts (prompts of fp16: in one)."""
    H, Hk, D = 4, 2, 64
    batch = R.Batch(new, old, B=16)
    query, k, v = _alike(batch, H, Hk, D, dtype, 15)
    lambdas = torch.full((H,), 0.95)
    refs = R.attention(batch, query, k.double(), v.double(), 0.17, maps=2)
    out = _attend(batch, query, [(k.cuda(), None, None), (v.cuda(), None, None)], 0.17, maps=2, lambdas=lambdas, weight=torch.ones(D))
    want = R.differential(refs, lambdas, torch.ones(D), 1e-5, 1.0)
    _close(out, want, _alike_bound(refs, lambdas, dtype, R.UNIT[dtype] ** 2))



# ---- many sequences ----

@pytest.mark.parametrize("B", [16, 64])
@pytest.mark.parametrize("n", [1100, 1700])
def test_append_of_many_single_tokens(B, n):
    """Sequences of one token each, or hardly more, every one of which owns its block: a work-group each, and several to one."""
    Hk, D, dtype, dev = 1, 64, torch.bfloat16, "cuda"
    batch = R.Batch([1 if k % 9 else 2 for k in range(n)], [(k * 13) % 40 for k in range(n)], B=B)
    g = torch.Generator().manual_seed(16)
    fused = torch.randn(batch.T, 2 * Hk, D, generator=g).to(dtype)
    pools = [torch.randint(-127, 128, (batch.blocks, B, Hk, D), generator=g, dtype=torch.int8) for _ in range(2)]
    scales = [0.002 + 0.03 * torch.rand(batch.blocks, Hk, generator=g) for _ in range(2)]
    d_rows, d_pools, d_scales = fused.to(dev), [p.to(dev) for p in pools], [s.to(dev) for s in scales]
    torch.ops.fa_amd.kv_cache_append(d_rows[:, :Hk], d_rows[:, Hk:], *d_pools, *batch.on(dev), None, None, None, *d_scales)
    R.append(batch, fused[:, :Hk], fused[:, Hk:], *pools, None, False, *scales)
    for got, ref in zip(d_pools + d_scales, pools + scales):
        assert torch.equal(got.cpu(), ref)


# ---- bounds beyond 32 bits ----

@pytest.mark.parametrize("new,old", [([1, 2], [40, 30]), ([40, 1], [50, 7])])
@pytest.mark.parametrize("maps", [1, 2])
def test_bounds_beyond_32_bits_bound_nothing(new, old, maps):
    """A window, a number of tokens or keys of 2^32 and a few is not one of those few."""
    H, Hk, D, dtype = 4, 2, 64, torch.float16
    batch = R.Batch(new, old, B=16)
    query = _query(batch, H, D, dtype, 17)
    pools = _pools(batch, Hk, D, "16", dtype, "head", 17)
    (_, k, _), (_, v, _) = pools
    lambdas = torch.full((H,), 0.4)
    out = _attend(batch, query, pools, 0.125, maps=maps, lambdas=lambdas, most=(1 << 32) + 1, longest=(1 << 32) + 3, window=(1 << 32) + 5)
    refs = R.attention(batch, query, k, v, 0.125, maps=maps)
    want = refs[0][0] if maps == 1 else R.differential(refs, lambdas, None, 0.0, 1.0)
    _close(out, want, R.attention_bound(refs, dtype, dtype, None if maps == 1 else lambdas))


# ---- a scalar scale below zero ----

@pytest.mark.parametrize("kv", ["e5m2", "e4m3"])
@pytest.mark.parametrize("new,old", [([1, 2], [40, 300]), ([40, 1], [50, 7]), ([33], [1500])])
@pytest.mark.parametrize("scale", [0.125, -0.125])
@pytest.mark.parametrize("softcap", [0.0, 3.0])
def test_scalar_scale_below_zero(kv, new, old, scale, softcap):
    """fp8_scale multiplies keys and values, whatever its sign, as in the other operators over FP8 pools."""
    H, Hk, D, dtype = 4, 2, 64, torch.bfloat16
    batch = R.Batch(new, old, B=16)
    query = _query(batch, H, D, dtype, 18, 8.0)  # scores that spread over tens of binary orders
    pools = _pools(batch, Hk, D, kv, dtype, "head", 18, None)
    (_, k, _), (_, v, _) = pools
    out = _attend(batch, query, pools, scale, fp8_scale=-0.5, softcap=softcap)
    refs = R.attention(batch, query, k * -0.5, v * -0.5, scale, softcap=softcap)
    _close(out, refs[0][0], R.attention_bound(refs, dtype, torch.float16))


# ---- halves of rows ----

@pytest.mark.parametrize("layout", ["head", "token"])
def test_append_of_halves_that_are_rotated_for_themselves(layout):
    """Two calls over the halves of rows and 16-bit pools: pairs a quarter of a row apart."""
    H, Hk, D, dtype, dev = 4, 2, 128, torch.bfloat16, "cuda"
    batch = R.Batch([3, 40, 1], [14, 0, 77], B=16)
    g = torch.Generator().manual_seed(19)
    fused = torch.randn(batch.T, H + 2 * Hk, D, generator=g).to(dtype)
    table = R.angle_table(max(batch.lens), D // 2)
    shape = (batch.blocks, Hk, 16, D) if layout == "head" else (batch.blocks, 16, Hk, D)
    pools = [torch.randn(shape, generator=g).to(dtype) for _ in range(2)]
    views = [p.permute(0, 2, 1, 3) if layout == "head" else p for p in pools]
    d_fused, d_pools, d_table = fused.to(dev), [p.to(dev) for p in pools], table.to(dev)
    d_views = [p.permute(0, 2, 1, 3) if layout == "head" else p for p in d_pools]
    q, k, v = d_fused.split([H, Hk, Hk], 1)
    want = []
    for half in (slice(0, D // 2), slice(D // 2, D)):
        torch.ops.fa_amd.kv_cache_append(k[..., half], v[..., half], *(p[..., half] for p in d_views), *batch.on(dev), d_table,
                                         q[..., half], q[..., half])
        want.append(R.append(batch, fused[:, H:H + Hk, half], fused[:, H + Hk:, half], *(p[..., half] for p in views), table, False,
                             query=fused[:, :H, half]))
    for got, ref in zip(d_pools, pools):
        assert torch.equal(got.cpu(), ref)
    assert torch.equal(d_fused[:, :H].cpu(), torch.cat(want, -1))
