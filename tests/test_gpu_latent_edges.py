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
