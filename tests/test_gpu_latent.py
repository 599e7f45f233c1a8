"""Latent attention on the GPU against the plain 64-bit forms: append, read-back, absorbed and expanded attention, types, sizes, masks."""
import math

import pytest
import torch

from flash_attention_factory_amd import torch_ops  # noqa: F401
from flash_attention_factory_amd.lib import attention_latent_expanded, paged_attention_latent

import _latent as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.fa_amd
F16, BF16 = torch.float16, torch.bfloat16


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


# ---- append ----

def _append(dtype, kind, L, B, H, new, old, interleaved, norm=True, rotate=True, in_place=False, lens=None):
    batch = R.Batch(new, old, B, seed=3, lens=lens)
    T = batch.T
    down = randn(T, L + R.ROPE + 8, seed=1, dtype=dtype)  # latent and key part in one row, which is wider than both
    down[:, L:] *= 3.0
    q = randn(T, H, 128 + R.ROPE, seed=2, dtype=dtype)
    weight = 1.0 + 0.2 * randn(L, seed=4) if norm else None
    table = R.angle_table(max(8, max(batch.lens)), R.ROPE) if rotate else None
    cache = randn(batch.blocks, B, L + R.ROPE, seed=5).to(dtype if kind == "16" else torch.float8_e4m3fn)
    scales = None if kind == "16" else torch.rand(batch.blocks, B, generator=torch.Generator().manual_seed(6)) + 0.5
    d = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    dd, dq, dc, ds = d(down), d(q), d(cache), d(scales)
    out = dq[..., 128:] if in_place else torch.full((T, H, R.ROPE), 7.0, dtype=dtype, device=DEV)
    ops.latent_cache_append(dd[:, :L], dd[:, L:L + R.ROPE], dc, *batch.on(DEV), d(weight), d(table), dq[..., 128:], out, ds, norm_eps=1e-5,
                            interleaved=interleaved)
    u = R.UNIT[dtype]
    written = torch.zeros(batch.blocks, B, dtype=torch.bool)
    got, got_scales, got_q = dc.cpu(), d(ds).cpu() if ds is not None else None, out.cpu()
    for s, (n, ctx) in enumerate(zip(batch.new, batch.lens)):
        if n == 0:
            continue
        a = int(batch.start[s])
        pos = torch.arange(ctx - n, ctx)
        angles = None if table is None else table[pos.clamp(0, table.size(0) - 1)]
        want_q = R.rotated(q[a:a + n, :, 128:], angles, interleaved)
        assert bool(((got_q[a:a + n].double() - want_q).abs() <= u * want_q.abs() + 4 * 2.0 ** -24 * 8).all())
        x = down[a:a + n, :L].double()
        if norm:
            x = x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-5) * weight.double()
        rope = R.rotated(down[a:a + n, None, L:L + R.ROPE], angles, interleaved)[:, 0]
        row = torch.cat([x, rope], 1)
        kept = pos >= 0
        kept &= pos // B < batch.tables.size(1)
        ids, at = batch.tables[s, (pos.clamp_min(0) // B).clamp_max(batch.tables.size(1) - 1)].long(), pos % B
        kept &= (ids >= 0) & (ids < batch.blocks)
        ids, at, row = ids[kept], at[kept], row[kept]
        written[ids, at] = True
        if kind == "16":
            # one rounding, after some 32-bit operations (the mean of squares, a root, two products: 8 roundings of 2^-24)
            assert bool(((got[ids, at].double() - row).abs() <= (u + 8 * 2.0 ** -24) * row.abs() + 4 * 2.0 ** -24 * 20).all())
        else:
            scale = R.row_scale(row.abs().amax(1))
            assert torch.equal(got_scales[ids, at], scale)
            value = got[ids, at].double() * scale.double()[:, None]
            # half a step of 2^-3 relative, or of the subnormal numbers' 2^-9
            assert bool(((value - row).abs() <= (2.0 ** -4 + 1e-5) * row.abs() + 2.0 ** -10 * scale.double()[:, None] * 1.001).all())
    same = got.view(torch.uint8 if kind != "16" else torch.int16) == cache.view(torch.uint8 if kind != "16" else torch.int16)
    assert bool(same[~written].all()), "rows without a new token have changed"
    if scales is not None:
        assert torch.equal(got_scales[~written], scales[~written])


@pytest.mark.parametrize("dtype,kind,L,B,H,new,old,interleaved", [
    (F16, "16", 512, 16, 16, [1, 1, 1], [0, 15, 200], False),
    (BF16, "16", 256, 32, 3, [5, 0, 33, 1], [3, 9, 0, 64], True),
    (BF16, "e4m3", 512, 64, 128, [1] * 9, list(range(0, 900, 100)), True),
    (F16, "e4m3", 256, 16, 1, [70, 2, 1], [7, 0, 31], False),
    (F16, "e4m3", 512, 16, 5, [1] * 300, [3] * 300, False),
])
def test_append(dtype, kind, L, B, H, new, old, interleaved):
    _append(dtype, kind, L, B, H, new, old, interleaved)


@pytest.mark.parametrize("kind", ["16", "e4m3"])
def test_append_without_norm_or_rotation_and_in_place(kind):
    _append(BF16, kind, 512, 16, 4, [3, 2], [1, 40], False, norm=False)
    _append(F16, kind, 256, 16, 4, [3, 2], [1, 40], True, rotate=False)
    _append(F16, kind, 512, 16, 4, [30, 2], [1, 40], True, in_place=True)


@pytest.mark.parametrize("kind", ["16", "e4m3"])
def test_append_leaves_out_tokens_without_a_place(kind):
    # three tokens at negative positions
    _append(BF16, kind, 512, 16, 2, [5, 2], [0, 4], False, lens=[2, 6])


def test_append_of_zeros_and_small_rows():
    batch = R.Batch([3], [0], 16, seed=0)
    x = torch.zeros(3, 576, dtype=BF16)
    x[1] = 2.0 ** -120
    x[2, 0] = 448.0 * 2 ** 10
    cache, scales = torch.zeros(batch.blocks, 16, 576, device=DEV).to(torch.float8_e4m3fn), torch.zeros(batch.blocks, 16, device=DEV)
    dx = x.to(DEV)
    ops.latent_cache_append(dx[:, :512], dx[:, 512:], cache, *batch.on(DEV), scales=scales)
    block = int(batch.tables[0, 0])
    assert scales[block, :3].tolist() == [2.0 ** -100, 2.0 ** -100, 2.0 ** 10]
    assert float(cache[block, 2, 0].float()) == 448.0 and float(cache[block, :2].float().abs().max()) == 0.0


# ---- read-back ----

@pytest.mark.parametrize("dtype,kind,L,B,lens,first", [
    (F16, "16", 512, 16, [1, 0, 37, 200], None), (BF16, "16", 256, 64, [65, 3], [4, 60]), (BF16, "e4m3", 512, 32, [100, 1, 0, 33], [0, 31, 5, 1]),
    (F16, "e4m3", 256, 16, [17000], None), (BF16, "e4m3", 512, 16, [9] * 300, [1] * 300),
])
def test_gather(dtype, kind, L, B, lens, first):
    batch = R.Batch([n + (first[s] if first else 0) for s, n in enumerate(lens)], [0] * len(lens), B, seed=1)
    cache, scales, _ = R.pool(batch, L, kind, dtype)
    N = sum(lens)
    out = torch.full((N + 3, L + R.ROPE + 8), 5.0, dtype=dtype, device=DEV)  # rows wider than asked for, and three behind the last sequence
    start = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)
    ops.latent_cache_gather(out[:, :L + R.ROPE], cache.to(DEV), batch.tables.to(DEV), start,
                            None if first is None else torch.tensor(first, dtype=torch.int32, device=DEV), None if scales is None else scales.to(DEV))
    want = torch.full((N + 3, L + R.ROPE + 8), 5.0, dtype=dtype)
    at = 0
    for s, n in enumerate(lens):
        t = torch.arange(n) + (first[s] if first else 0)
        ids = batch.tables[s, t // B].long()
        rows = cache[ids, t % B]
        want[at:at + n, :L + R.ROPE] = rows if scales is None else (rows.float() * scales[ids, t % B][:, None]).to(dtype)
        at += n
    assert torch.equal(out.cpu(), want)


def test_gather_of_keys_that_are_not_there():
    batch = R.Batch([20, 20], [0, 0], 16, seed=1)
    cache, _, _ = R.pool(batch, 256, "16", F16)
    batch.tables[1, 0] = batch.blocks  # outside the pool
    out = torch.full((90, 320), 5.0, dtype=F16, device=DEV)
    ops.latent_cache_gather(out, cache.to(DEV), batch.tables.to(DEV), torch.tensor([0, 50, 90], dtype=torch.int32, device=DEV),
                            torch.tensor([-5, 0], dtype=torch.int32, device=DEV))
    got = out.cpu()
    real = cache[batch.tables[0, torch.arange(20) // 16].long(), torch.arange(20) % 16]
    assert torch.equal(got[5:25], real) and float(got[:5].abs().max()) == 0.0
    assert float(got[37:50].abs().max()) == 0.0  # past the table's columns (2 blocks of 16)
    assert float(got[50:66].abs().max()) == 0.0
    assert torch.equal(got[66:70], cache[int(batch.tables[1, 1]), :4])


# ---- absorbed attention ----

def _absorbed(dtype, kind, L, H, B, new, old, *, scale=None, lens=None, size=1.0, layout="heads", most=None, longest=None, seed=0, call=None, table=None):
    batch = R.Batch(new, old, B, seed=seed, lens=lens)
    if table is not None:
        batch.tables = batch.tables[:, :table].contiguous()
    cache, scales, values = R.pool(batch, L, kind, dtype, seed=seed + 1)
    T, spare = batch.T, 2
    scale = (L + R.ROPE) ** -0.5 if scale is None else scale
    shape = (H, T + spare, L) if layout == "heads" else (T + spare, H, L)
    ql = (size * randn(*shape, seed=seed + 2)).to(dtype).to(DEV)
    out = torch.full(shape, 9.0, dtype=dtype, device=DEV)
    if layout == "heads":
        ql, out = ql.transpose(0, 1), out.transpose(0, 1)
    qr = (size * randn(T + spare, H, 128 + R.ROPE, seed=seed + 3)).to(dtype).to(DEV)[..., 128:]
    arguments = (out, ql, qr, cache.to(DEV), *batch.on(DEV), scale, most or max(1, max(new)), max(batch.lens) if longest is None else longest)
    (call or ops.paged_attention_latent)(*arguments, scales=None if scales is None else scales.to(DEV))
    got = out.cpu().double()
    want, sizes = R.absorbed(batch, ql[:T].cpu(), qr[:T].cpu(), values, scale, most)
    untouched = torch.isnan(want)
    assert bool((got[:T][untouched] == 9.0).all()) and bool((got[T:] == 9.0).all()), "rows that belong to no token have changed"
    want = torch.where(untouched, got[:T], want)
    bound = R.bound(want, sizes, dtype, scores=4.0 * max(1.0, size))
    off = (got[:T] - want).abs()
    assert not torch.isnan(got).any()
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.2f} of the bound"


ABSORBED = [
    (F16, "16", 512, 16, 16, [1, 1, 1], [0, 7, 300]),
    (BF16, "16", 512, 128, 64, [1] * 6, [0, 30, 31, 32, 33, 1000]),
    (F16, "16", 256, 20, 16, [1, 1], [100, 517]),
    (BF16, "16", 256, 8, 32, [3, 0, 1, 17], [250, 3, 700, 0]),
    (F16, "e4m3", 512, 16, 16, [1, 1, 1], [0, 40, 2000]),
    (BF16, "e4m3", 512, 64, 64, [1] * 5, [5, 64, 128, 129, 900]),
    (F16, "e4m3", 256, 5, 16, [4, 1, 9], [31, 0, 600]),
    (BF16, "e4m3", 256, 40, 32, [1, 1], [333, 12]),
    (F16, "16", 512, 128, 16, [2, 1, 9], [600, 1, 77]),       # several tiles of 128 rows
    (BF16, "e4m3", 512, 128, 16, [5, 1], [900, 20]),
    (F16, "e4m3", 512, 128, 64, [1, 3], [3000, 10]),
    (F16, "16", 512, 1, 16, [1], [0]),                        # one row, one key
]


@pytest.mark.parametrize("dtype,kind,L,H,B,new,old", ABSORBED)
def test_absorbed(dtype, kind, L, H, B, new, old):
    _absorbed(dtype, kind, L, H, B, new, old)


@pytest.mark.parametrize("dtype,kind,H", [(BF16, "16", 16), (F16, "e4m3", 16), (BF16, "e4m3", 48), (F16, "16", 128)])
def test_absorbed_one_long_context_over_many_work_groups(dtype, kind, H):
    _absorbed(dtype, kind, 512, H, 64, [1], [20011])


@pytest.mark.parametrize("kind", ["16", "e4m3"])
def test_absorbed_more_sequences_than_lanes(kind):
    _absorbed(BF16, kind, 256, 4, 16, [1, 2, 0, 1, 3] * 30, [5, 300, 9, 0, 41] * 30)


@pytest.mark.parametrize("kind", ["16", "e4m3"])
def test_absorbed_short_calls(kind):
    _absorbed(F16, kind, 512, 16, 16, [1, 1, 4, 0], [0, 16, 31, 0], longest=64)
    _absorbed(BF16, kind, 512, 128, 16, [1, 1, 4, 0], [0, 200, 31, 0], longest=256)


@pytest.mark.parametrize("kind", ["16", "e4m3"])
def test_absorbed_tokens_that_see_nothing(kind):
    _absorbed(F16, kind, 512, 16, 16, [5, 2], [0, 100], lens=[2, 102])  # three tokens before key 0
    _absorbed(BF16, kind, 256, 64, 16, [3], [0], lens=[0])


@pytest.mark.parametrize("kind", ["16", "e4m3"])
def test_absorbed_bounds(kind):
    _absorbed(F16, kind, 256, 16, 16, [7, 1, 4], [300, 2, 90], most=3)                  # tokens beyond max_query_len are left out
    _absorbed(F16, kind, 256, 16, 16, [2, 1], [300, 2], longest=0)                      # as far as the table goes
    _absorbed(F16, kind, 256, 16, 16, [2, 1], [90, 2], table=3)                         # ... where the lengths go further


@pytest.mark.parametrize("dtype,kind", [(F16, "16"), (BF16, "16"), (F16, "e4m3"), (BF16, "e4m3")])
def test_absorbed_scores_of_any_size(dtype, kind):
    _absorbed(dtype, kind, 512, 16, 16, [1, 2], [900, 333], size=4.0, layout="tokens")  # references move
    _absorbed(dtype, kind, 256, 16, 16, [1], [500], scale=-0.06)
    _absorbed(dtype, kind, 256, 70, 16, [1], [500], scale=0.0)


def test_absorbed_references_move_at_any_key():
    """A key that outweighs all others, at each place within a step and at the ends of steps and shares."""
    L, H, n = 512, 128, 700
    for at in (0, 1, 15, 16, 31, 32, 63, 255, 256, 511, 698, 699):
        for dtype in (F16, BF16):
            batch = R.Batch([1], [n - 1], 16, seed=at)
            rows = 0.05 * randn(batch.blocks, 16, L + R.ROPE, seed=at)
            rows[int(batch.tables[0, at // 16]), at % 16] = 1.0
            q = torch.full((1, H, L + R.ROPE), 1.0)
            rows, q = rows.to(dtype), q.to(dtype)
            out = torch.empty(1, H, L, dtype=dtype, device=DEV)
            dq = q.to(DEV)
            ops.paged_attention_latent(out, dq[..., :L], dq[..., L:], rows.to(DEV), *batch.on(DEV), 0.1, 1, n)
            assert float((out.double() - 1.0).abs().max()) < 1e-2, (at, dtype)  # exp(-50) of the others


def test_absorbed_rows_of_zeros_and_small_scales():
    """Scales binary orders apart: rows of zeros have the least scale, and weigh as much as others."""
    L, H = 256, 16
    batch = R.Batch([1], [199], 16, seed=0)
    for dtype in (F16, BF16):
        cache, scales, values = R.pool(batch, L, "e4m3", dtype)
        for t in range(0, 200, 3):
            block, at = int(batch.tables[0, t // 16]), t % 16
            cache.view(torch.uint8)[block, at] = 0
            scales[block, at] = 2.0 ** -100
            values[block, at] = 0.0
        ql, qr = randn(1, H, L, seed=1, dtype=dtype), randn(1, H, R.ROPE, seed=2, dtype=dtype)
        want, sizes = R.absorbed(batch, ql, qr, values, 0.06)
        out = torch.empty(1, H, L, dtype=dtype, device=DEV)
        ops.paged_attention_latent(out, ql.to(DEV), qr.to(DEV), cache.to(DEV), *batch.on(DEV), 0.06, 1, 200, scales.to(DEV))
        assert bool(((out.cpu().double() - want).abs() <= R.bound(want, sizes, dtype)).all())


def test_absorbed_infinite_and_nan_rows():
    """Rows that a token sees spread; rows that it does not see do not."""
    L, H = 512, 16
    batch = R.Batch([2], [70], 16, seed=0)
    cache, _, _ = R.pool(batch, L, "16", BF16)
    cache[int(batch.tables[0, 71 // 16]), 71 % 16] = math.nan  # the last token's own
    ql, qr = randn(2, H, L, seed=1, dtype=BF16).to(DEV), randn(2, H, R.ROPE, seed=2, dtype=BF16).to(DEV)
    out = torch.empty(2, H, L, dtype=BF16, device=DEV)
    ops.paged_attention_latent(out, ql, qr, cache.to(DEV), *batch.on(DEV), 0.04, 2, 72)
    assert bool(torch.isnan(out[1]).all())


def test_absorbed_through_lib():
    def call(*arguments, scales):
        us = paged_attention_latent.run(*arguments, scales)
        assert len(us) == 1 and us[0] > 0.0
    _absorbed(BF16, "e4m3", 512, 16, 16, [1, 3], [900, 10], call=call)


# ---- expanded attention ----

def _expanded(dtype, D, H, new, keys, *, scale=None, size=1.0, most=None, longest=None, heads_first=False, seed=0):
    T, N, spare = sum(new), sum(keys), 2
    start, key_start = ([0] + torch.tensor(x).cumsum(0).tolist() for x in (new, keys))
    scale = (D + R.ROPE) ** -0.5 if scale is None else scale
    q = (size * randn(T + spare, H, D + R.ROPE, seed=seed)).to(dtype).to(DEV)
    both = randn(N + 1, H, 2 * D, seed=seed + 1, dtype=dtype)
    both[N:] = math.nan
    rope = randn(N + 1, 96, seed=seed + 2, dtype=dtype)
    rope[N:] = math.nan
    out = torch.full((H, T + spare, D) if heads_first else (T + spare, H, D), 9.0, dtype=dtype, device=DEV)
    out = out.transpose(0, 1) if heads_first else out
    d_both, d_rope = both.to(DEV), rope.to(DEV)
    ops.attention_latent_expanded(out, q, d_both[:N, :, :D], d_rope[:N, 32:], d_both[:N, :, D:], torch.tensor(start, dtype=torch.int32, device=DEV),
                                  torch.tensor(key_start, dtype=torch.int32, device=DEV), scale, most or max(1, max(new)),
                                  max(keys) if longest is None else longest)
    got = out.cpu().double()
    want, sizes = R.expanded(q[:T].cpu(), both[:N, :, :D], rope[:N, 32:], both[:N, :, D:], start, key_start, scale, most)
    untouched = torch.isnan(want)
    assert bool((got[:T][untouched] == 9.0).all()) and bool((got[T:] == 9.0).all()), "rows that belong to no token have changed"
    want = torch.where(untouched, got[:T], want)
    bound = R.bound(want, sizes, dtype, scores=4.0 * max(1.0, size))
    off = (got[:T] - want).abs()
    assert not torch.isnan(got).any()
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.2f} of the bound"


@pytest.mark.parametrize("dtype,D,H,new,keys", [
    (F16, 128, 4, [1], [1]), (BF16, 128, 3, [5, 64, 1], [5, 64, 1]), (F16, 64, 5, [33, 0, 127], [33, 0, 127]),
    (BF16, 64, 2, [300], [300]), (F16, 128, 2, [129, 65], [1000, 65]), (BF16, 128, 16, [1, 1, 40], [700, 63, 64]),
    (F16, 128, 2, [513], [1700]), (BF16, 64, 3, [200, 256, 257], [1800, 256, 2000]),
])
def test_expanded(dtype, D, H, new, keys):
    _expanded(dtype, D, H, new, keys)


@pytest.mark.parametrize("dtype,D,new,keys", [(F16, 128, [3], [9000]), (BF16, 64, [70, 1], [6000, 5000]), (BF16, 128, [300], [12001])])
def test_expanded_few_tokens_after_many_keys(dtype, D, new, keys):
    _expanded(dtype, D, 2, new, keys)


def test_expanded_many_tiles():
    _expanded(BF16, 128, 8, [700, 1100, 3, 900], [700, 1900, 3, 1600])  # a work-group for each tile, eight wavefronts
    _expanded(F16, 64, 24, [100] * 30, [100] * 30)


def test_expanded_more_sequences_than_lanes():
    _expanded(F16, 64, 2, [1, 0, 9, 130] * 20, [17, 3, 9, 200] * 20)


def test_expanded_tokens_that_see_nothing():
    _expanded(F16, 128, 2, [7, 5], [3, 0])
    _expanded(BF16, 64, 2, [300], [20])


def test_expanded_bounds():
    _expanded(F16, 64, 2, [40, 3, 200], [60, 3, 300], most=33)
    _expanded(F16, 64, 2, [40, 3], [60, 3], longest=0)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_expanded_scores_of_any_size(dtype):
    _expanded(dtype, 128, 2, [150], [400], size=4.0, heads_first=True)
    _expanded(dtype, 64, 2, [20], [100], scale=-0.1)
    _expanded(dtype, 64, 2, [20], [100], scale=0.0)


def test_expanded_later_keys_may_be_anything():
    """Keys and values behind a sequence's own are another's: nothing of them reaches it."""
    q = randn(6, 2, 128, seed=0, dtype=F16).to(DEV)
    both, rope = randn(200, 2, 128, seed=1, dtype=F16), randn(200, 64, seed=2, dtype=F16)
    both[70:], rope[70:] = math.nan, math.nan
    starts = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 5, 6], [0, 70, 200])]
    out = torch.empty(6, 2, 64, dtype=F16, device=DEV)
    d, r = both.to(DEV), rope.to(DEV)
    ops.attention_latent_expanded(out, q, d[..., :64], r, d[..., 64:], *starts, 0.1, 5, 130)
    want, sizes = R.expanded(q[:5].cpu(), both[:70, :, :64], rope[:70], both[:70, :, 64:], [0, 5], [0, 70], 0.1)
    assert bool(((out[:5].cpu().double() - want).abs() <= R.bound(want, sizes, F16)).all())
    assert bool(torch.isnan(out[5]).all())


def test_expanded_through_lib():
    x = randn(9, 2, 192, seed=0, dtype=BF16).to(DEV)
    k, r = randn(9, 2, 256, seed=1, dtype=BF16).to(DEV), randn(9, 64, seed=2, dtype=BF16).to(DEV)
    start = torch.tensor([0, 9], dtype=torch.int32, device=DEV)
    a, b = torch.empty(9, 2, 128, dtype=BF16, device=DEV), torch.empty(9, 2, 128, dtype=BF16, device=DEV)
    us = attention_latent_expanded.run(a, x, k[..., :128], r, k[..., 128:], start, start, 0.07, 9)
    ops.attention_latent_expanded(b, x, k[..., :128], r, k[..., 128:], start, start, 0.07, 9)
    assert len(us) == 1 and us[0] > 0.0 and torch.equal(a, b)
