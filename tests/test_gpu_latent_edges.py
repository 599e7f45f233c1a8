"""Latent pools at the ends of what they hold: rows of very large numbers, infinities and NaN beside a sequence's own rows."""
import pytest
import torch

from flash_attention_factory_amd import torch_ops  # noqa: F401

import _latent as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.fa_amd
F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def randn(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("L", [256, 512])
def test_rows_of_large_numbers_in_fp8_pools(L):
    """Rows up to the largest of bf16 are stored, read back and attended like others: their scales go up to 2^120."""
    n, H = 90, 16
    batch = R.Batch([n], [0], 16)
    x = randn(n, L + R.ROPE, seed=1).clamp(-3.9, 3.9)
    exponents = 96 + torch.arange(n) % 31  # up to 3.9 * 2^126
    x = (x * 2.0 ** exponents[:, None].double()).to(BF16)
    cache = torch.zeros(batch.blocks, 16, L + R.ROPE, device=DEV).to(E4M3)
    scales = torch.zeros(batch.blocks, 16, device=DEV)
    d = x.to(DEV)
    ops.latent_cache_append(d[:, :L], d[:, L:], cache, *batch.on(DEV), scales=scales)
    t = torch.arange(n)
    ids = batch.tables[0, t // 16].long()
    scale = R.row_scale(x.double().abs().amax(1))
    assert torch.equal(scales.cpu()[ids, t % 16], scale) and float(scale.max()) > 2.0 ** 110
    rows = cache.cpu()[ids, t % 16].double() * scale.double()[:, None]
    # half a step: 2^-4 relative, or of the subnormal numbers' 2^-9
    assert bool(((rows - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * scale.double()[:, None]).all())
    back = torch.empty(n, L + R.ROPE, dtype=BF16, device=DEV)
    ops.latent_cache_gather(back, cache, batch.tables.to(DEV), torch.tensor([0, n], dtype=torch.int32, device=DEV), scales=scales)
    assert torch.equal(back.cpu().double(), rows.to(BF16).double())
    # with weights from a normalised latent: the factors are what is large
    weight = 2.0 ** 112 * (1.0 + 0.1 * randn(L, seed=2))
    y = randn(n, L + R.ROPE, seed=3).to(F16)
    d = y.to(DEV)
    ops.latent_cache_append(d[:, :L], d[:, L:], cache, *batch.on(DEV), weight.to(DEV), None, None, None, scales, norm_eps=1e-6)
    c = y[:, :L].double()
    c = c / torch.sqrt(c.square().mean(1, keepdim=True) + 1e-6) * weight.double()
    scale = scales.cpu()[ids, t % 16].double()
    assert torch.equal(scale, R.row_scale(c.abs().amax(1)).double())
    assert bool(((cache.cpu()[ids, t % 16, :L].double() * scale[:, None] - c).abs() <= (2.0 ** -4 + 1e-5) * c.abs() + 2.0 ** -10 * 1.001 * scale[:, None]).all())


def test_attention_over_rows_of_large_numbers():
    n, H, L = 90, 16, 512
    batch = R.Batch([1], [n - 1], 16)
    x = (randn(batch.blocks, 16, L + R.ROPE, seed=1) * 2.0 ** 110).to(BF16)
    scales = R.row_scale(x.double().abs().amax(-1))
    cache = (x.double() / scales.double()[..., None]).float().to(E4M3)
    assert float(scales.max()) > 2.0 ** 100
    ql, qr = ((randn(1, H, m, seed=2 + m) * 2.0 ** -110).to(BF16) for m in (L, R.ROPE))
    want, sizes = R.absorbed(batch, ql, qr, cache.double() * scales.double()[..., None], 0.04)
    out = torch.empty(1, H, L, dtype=BF16, device=DEV)
    ops.paged_attention_latent(out, ql.to(DEV), qr.to(DEV), cache.to(DEV), *batch.on(DEV), 0.04, 1, n, scales.to(DEV))
    assert bool(((out.cpu().double() - want).abs() <= R.bound(want, sizes, BF16)).all())


@pytest.mark.parametrize("kind", ["16", "e4m3"])
@pytest.mark.parametrize("H,new,old", [(16, [1, 1], [70, 300]), (32, [1, 2], [63, 40]), (64, [3, 1], [0, 257]), (128, [1, 5], [300, 31])])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_of_others_and_behind_the_last_key_do_not_reach_a_sequence(kind, H, new, old, bad):
    """Whatever lies in the pool behind a sequence's last key or in another sequence's blocks, its results are the same bit for bit."""
    L, B = 512, 16
    batch = R.Batch(new, old, B)
    cache, scales, _ = R.pool(batch, L, kind, BF16, junk=False)
    ql, qr = randn(batch.T, H, L, seed=1).to(BF16).to(DEV), randn(batch.T, H, R.ROPE, seed=2).to(BF16).to(DEV)

    def run(rows, its_scales):
        out = torch.empty(batch.T, H, L, dtype=BF16, device=DEV)
        ops.paged_attention_latent(out, ql, qr, rows.to(DEV), *batch.on(DEV), 0.04, max(new), max(batch.lens),
                                   None if its_scales is None else its_scales.to(DEV))
        return out
    want = run(cache, scales)
    assert not torch.isnan(want).any()
    for s in range(2):
        mine = torch.zeros(batch.blocks, B, dtype=torch.bool)
        for t in range(batch.lens[s]):
            mine[int(batch.tables[s, t // B]), t % B] = True
        spoilt = cache.clone()
        spoilt_scales = None if scales is None else scales.clone()
        if kind == "16":
            spoilt[~mine] = bad
        else:  # E4M3 has no infinities: bytes of NaN, and scales that are not finite
            spoilt.view(torch.uint8)[~mine] = 0x7f
            spoilt_scales[~mine] = bad
        a, b = int(batch.start[s]), int(batch.start[s + 1])
        assert torch.equal(run(spoilt, spoilt_scales)[a:b], want[a:b])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new,keys", [([3, 5], [70, 64]), ([200, 40], [700, 41])])
def test_expanded_rows_of_others_do_not_reach_a_sequence(D, new, keys):
    H, N = 3, sum(keys)
    starts = [torch.tensor([0, x[0], sum(x)], dtype=torch.int32, device=DEV) for x in (new, keys)]
    q = randn(sum(new), H, D + R.ROPE, seed=1).to(BF16).to(DEV)
    both, rope = randn(N, H, 2 * D, seed=2).to(BF16).to(DEV), randn(N, R.ROPE, seed=3).to(BF16).to(DEV)

    def run(x, r):
        out = torch.empty(sum(new), H, D, dtype=BF16, device=DEV)
        ops.attention_latent_expanded(out, q, x[..., :D], r, x[..., D:], *starts, 0.07, max(new), max(keys))
        return out
    want = run(both, rope)
    assert not torch.isnan(want).any()
    for s, others in ((0, slice(keys[0], N)), (1, slice(0, keys[0]))):
        x, r = both.clone(), rope.clone()
        x[others], r[others] = float("nan"), float("inf")
        mine = slice(0, new[0]) if s == 0 else slice(new[0], sum(new))
        assert torch.equal(run(x, r)[mine], want[mine])


@pytest.mark.parametrize("kind", ["16", "e4m3"])
@pytest.mark.parametrize("H,new,most", [(128, [1, 3, 2, 0, 4], 2), (64, [9, 1, 2], 4), (128, [2, 6, 4, 4], 4)])
def test_unequal_sequences_whose_total_is_that_of_equal_ones(kind, H, new, most):
    """num_tokens = sequences x max_query_len, but some bring less and the longer ones are cut: tiles side by side that some do not have."""
    L, old = 512, [300 + 77 * k for k in range(len(new))]
    assert sum(new) == most * len(new)
    batch = R.Batch(new, old, 16)
    cache, scales, values = R.pool(batch, L, kind, F16)
    ql, qr = randn(batch.T, H, L, seed=1).to(F16), randn(batch.T, H, R.ROPE, seed=2).to(F16)
    want, sizes = R.absorbed(batch, ql, qr, values, 0.04, most)
    out = torch.full((batch.T, H, L), 9.0, dtype=F16, device=DEV)
    ops.paged_attention_latent(out, ql.to(DEV), qr.to(DEV), cache.to(DEV), *batch.on(DEV), 0.04, most, max(batch.lens),
                               None if scales is None else scales.to(DEV))
    got, left_out = out.cpu().double(), torch.isnan(want)
    assert bool((got[left_out] == 9.0).all())
    assert bool(((got - want).abs() <= R.bound(want, sizes, F16))[~left_out].all())
