"""Plain 64-bit forms of latent attention, sequence by sequence on the CPU, and inputs to try it on."""
import math

import torch

from _ragged import UNIT, Batch, angle_table  # noqa: F401

ROPE = 64


def pool(batch, L, kind, dtype, seed=0, junk=True):
    """A latent pool [blocks, B, L + 64], its scales (FP8: rows of different sizes) and its values in 64 bits.  Rows that hold no key, and their
    scales, are NaN."""
    g = torch.Generator().manual_seed(seed)
    rows = torch.randn(batch.blocks, batch.B, L + ROPE, generator=g)
    if kind == "16":
        cache, scales = rows.to(dtype), None
        values = cache.double()
    else:
        rows = rows * torch.exp(torch.randn(batch.blocks, batch.B, 1, generator=g))
        scales = row_scale(rows.abs().amax(-1))
        cache = (rows / scales[..., None]).to(torch.float8_e4m3fn)
        # back to a size that keeps scores of the order of 1, and no powers of two
        scales = scales * 1.1 / rows.square().mean(-1).sqrt()
        values = cache.double() * scales.double()[..., None]
    if junk:
        empty = ~batch.used
        if kind == "16":
            cache[empty] = math.nan
        else:
            cache.view(torch.uint8)[empty] = 0x7f
            scales[empty] = math.nan
        values[empty] = 0.0
    return cache, scales, values


def row_scale(most):
    """The least power of two, 2^-100 or more, that brings a row's largest magnitude to 448 or less."""
    return torch.tensor([2.0 ** max(-100, math.ceil(math.log2(m / 448.0))) if m > 0 else 2.0 ** -100 for m in most.double().flatten().tolist()],
                        dtype=torch.float32).view(most.shape)


def weights(x, pos):
    """Softmax weights of scores x [heads, n, keys] of tokens at the positions pos: those that see nothing get zeros."""
    key = torch.arange(x.size(-1))
    x = x.masked_fill(key[None, None] > pos[None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    return p / total.masked_fill(total == 0, 1.0)


def absorbed(batch, ql, qr, values, scale, most=None):
    """[T, H, L] in 64 bits, and the same with |c| (what rounding errors are proportional to); rows of no token are NaN."""
    T, H, L = ql.shape
    out, size = torch.full((T, H, L), math.nan, dtype=torch.float64), torch.zeros((T, H, L), dtype=torch.float64)
    columns = batch.tables.size(1) * batch.B
    for s, (n, ctx) in enumerate(zip(batch.new, batch.lens)):
        a, first = int(batch.start[s]), ctx - n
        n = n if most is None else min(n, most)
        if n == 0:
            continue
        keys = max(0, min(first + n, columns))
        pos = torch.arange(first, first + n).clamp_max(keys - 1)
        t = torch.arange(keys)
        rows = values[batch.tables[s, t // batch.B].long(), t % batch.B]
        q = torch.cat([ql[a:a + n], qr[a:a + n]], -1).double().transpose(0, 1)
        p = weights(q @ rows.T * scale, pos) if keys else torch.zeros(H, n, 0, dtype=torch.float64)
        out[a:a + n], size[a:a + n] = (p @ rows[:, :L]).transpose(0, 1), (p @ rows[:, :L].abs()).transpose(0, 1)
    return out, size


def expanded(query, key, rope, value, start, key_start, scale, most=None):
    T, H, _ = query.shape
    D = key.size(2)
    out, size = torch.full((T, H, D), math.nan, dtype=torch.float64), torch.zeros((T, H, D), dtype=torch.float64)
    for s in range(len(start) - 1):
        a, n, k0, m = start[s], start[s + 1] - start[s], key_start[s], key_start[s + 1] - key_start[s]
        first = m - n
        n = n if most is None else min(n, most)
        if n == 0:
            continue
        k = torch.cat([key[k0:k0 + m], rope[k0:k0 + m, None].expand(m, H, ROPE)], -1).double().permute(1, 2, 0)
        p = weights(query[a:a + n].double().transpose(0, 1) @ k * scale, torch.arange(first, first + n)) if m else torch.zeros(H, n, 0, dtype=torch.float64)
        v = value[k0:k0 + m].double().transpose(0, 1)
        out[a:a + n], size[a:a + n] = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
    return out, size


def bound(want, size, dtype, scores=4.0):
    """Largest error of a result.  Weights are rounded once (relative error UNIT each, so UNIT * sum p|v| in a result); a score is a sum of up
    to 576 products in 32 bits, off by up to 576 * 2^-24 of the sum of their magnitudes, which is some ten times the scores (`scores`:
    the largest that weigh), and that is the weight's relative error, as is the 32-bit exponential's; the result is rounded once."""
    u = UNIT[dtype]
    return (u + 576 * 2.0 ** -24 * 10 * scores / 10 + 5e-5) * size + u * want.abs() + 1e-6


def rotated(x, angles, interleaved):
    """Rows [n, heads, 64] in 64 bits, as complex numbers times exp(i angle)."""
    x = x.double()
    if angles is None:
        return x
    half = x.size(-1) // 2
    phase = torch.complex(angles[:, :half].double(), angles[:, half:].double())[:, None]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    z = torch.complex(a.contiguous(), b.contiguous()) * phase
    return torch.view_as_real(z).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)
