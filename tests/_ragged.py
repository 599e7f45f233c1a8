"""Plain 64-bit forms of the operators for ragged batches, sequence by sequence on the CPU, and batches to try them on."""
import math

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # relative error of one rounding: 11 and 8 significant bits


class Batch:
    """Sequences of ``new[s]`` tokens after ``old[s]`` ones: tables of random blocks; unused entries name no block of the pool."""

    def __init__(self, new, old, B, seed=0, spare=3, lens=None):
        g = torch.Generator().manual_seed(seed)
        self.new, self.B = list(new), B
        self.lens = [n + o for n, o in zip(new, old)] if lens is None else list(lens)
        per = [max(0, -(-n // B)) for n in self.lens]
        self.blocks = sum(per) + spare
        order = torch.randperm(self.blocks, generator=g)
        self.tables = torch.full((len(new), max(1, max(per))), 1 << 30, dtype=torch.int32)
        self.tables[:, 1::2] = -7
        at = 0
        for s, n in enumerate(per):
            self.tables[s, :n] = order[at:at + n].to(torch.int32)
            at += n
        self.start = torch.tensor([0] + list(torch.tensor(self.new).cumsum(0)), dtype=torch.int32)
        self.T = sum(self.new)
        self.used = torch.zeros((self.blocks, B), dtype=torch.bool)  # rows that hold a key
        for s, n in enumerate(self.lens):
            for t in range(n):
                self.used[int(self.tables[s, t // B]), t % B] = True

    def on(self, dev):
        return self.tables.to(dev), self.start.to(dev), torch.tensor(self.lens, dtype=torch.int32, device=dev)


def attention(batch, query, keys, values, scale, *, maps=1, window=-1, softcap=0.0, slopes=None, sinks=None):
    """[T, H, D] in 64 bits from pools of values [blocks, B, Hk, D] in 64 bits: one result per map, and the same with |V|
    (what the result's rounding errors are proportional to)."""
    T, H, D = query.shape
    Hk, B, d = keys.size(2), batch.B, D // maps
    got = [(torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, D, dtype=torch.float64)) for _ in range(maps)]
    for s, (n, ctx) in enumerate(zip(batch.new, batch.lens)):
        a = int(batch.start[s])
        if n == 0 or ctx <= 0:
            continue
        t = torch.arange(ctx)
        ids = batch.tables[s, t // B].long()
        pos = torch.arange(ctx - n, ctx)
        sees = t[None, :] <= pos[:, None]
        if window >= 0:
            sees &= t[None, :] >= pos[:, None] - window
        for h in range(H):
            kvh = h // (H // Hk)
            k, v = keys[ids, t % B, kvh], values[ids, t % B, kvh]
            for m in range(maps):
                x = query[a:a + n, h, m * d:(m + 1) * d].double() @ k[:, m * d:(m + 1) * d].T * scale
                if softcap > 0:
                    x = softcap * torch.tanh(x / softcap)
                if slopes is not None:
                    x = x + float(slopes[h]) * (t[None, :] - pos[:, None])
                x = x.masked_fill(~sees, -math.inf)
                top = x.amax(1, keepdim=True)
                if sinks is not None:
                    top = top.clamp_min(float(sinks[h]))
                top = top.masked_fill(top == -math.inf, 0.0)
                p = torch.exp(x - top)
                total = p.sum(1, keepdim=True)
                if sinks is not None:
                    total = total + torch.exp(float(sinks[h]) - top)
                p = p / total.masked_fill(total == 0, 1.0)
                p = p.masked_fill(~sees, 0.0)
                got[m][0][a:a + n, h] = p @ v
                got[m][1][a:a + n, h] = p @ v.abs()
    return got


def differential(maps, lambdas, weight, eps, out_scale):
    (o1, _), (o2, _) = maps
    o = o1 - lambdas.double()[:, None] * o2
    if weight is None:
        return o * out_scale
    return o / torch.sqrt((o * o).mean(-1, keepdim=True) + eps) * weight.double() * out_scale


def attention_bound(maps, out_type, operand_type, lambdas=None, weight=None, eps=0.0, out_scale=1.0):
    """Largest error of a result.  Probabilities are rounded to the operand type (relative error u each, so u * sum p|v| in a
    result), scores and exponentials carry about 1e-4 of relative error at the sizes tried (128 products of about 1 in 32 bits,
    a 32-bit exponential, softcap's reciprocal), the result is rounded to its type once."""
    u, v = UNIT[operand_type] + 2e-4, UNIT[out_type]
    if lambdas is None:
        (o, a), = maps
        return u * a + v * o.abs() + 1e-6
    e = u * (maps[0][1] + lambdas.double().abs()[:, None] * maps[1][1])
    o = maps[0][0] - lambdas.double()[:, None] * maps[1][0]
    if weight is None:
        return abs(out_scale) * (e + v * o.abs()) + 1e-6
    # the norm's own relative error is at most |e| / |o| over the row, and it multiplies every element
    rms = torch.sqrt((o * o).mean(-1, keepdim=True) + eps)
    off = e.square().mean(-1, keepdim=True).sqrt() / rms
    mul = weight.double().abs() * abs(out_scale) / rms
    return mul * (e + o.abs() * off * 1.1 + v * o.abs()) + 1e-6


def rotated(x, angles, interleaved):
    """In 32 bits, each operation rounded by itself: x [n, heads, D], angles [n, R] (cosines, then sines)."""
    if angles is None:
        return x.float()
    half = angles.size(1) // 2
    cos, sin = angles[:, None, :half], angles[:, None, half:]
    x = x.float().clone()
    a, b = (x[..., 0:2 * half:2].clone(), x[..., 1:2 * half:2].clone()) if interleaved else (x[..., :half].clone(), x[..., half:2 * half].clone())
    p, q = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        x[..., 0:2 * half:2], x[..., 1:2 * half:2] = p, q
    else:
        x[..., :half], x[..., half:2 * half] = p, q
    return x


def append(batch, key, value, keys, values, table, interleaved, k_scales=None, v_scales=None, fp8_scale=1.0, query=None):
    """What the append leaves in the pools (and scales), written in place; returns the rotated queries."""
    out = None if query is None else torch.zeros_like(query)
    B = batch.B
    for s, (n, ctx) in enumerate(zip(batch.new, batch.lens)):
        if n == 0:
            continue
        a = int(batch.start[s])
        pos = torch.arange(ctx - n, ctx)
        angles = None if table is None else table[pos.clamp(0, table.size(0) - 1)]
        if query is not None:
            out[a:a + n] = rotated(query[a:a + n], angles, interleaved).to(query.dtype)
        for rows, pool, scales in ((rotated(key[a:a + n], angles, interleaved), keys, k_scales), (value[a:a + n].float(), values, v_scales)):
            for col in range(max(0, ctx - n) // B, -(-ctx // B)):
                block = int(batch.tables[s, col])
                if not 0 <= block < pool.size(0):
                    continue
                here = (pos >= col * B) & (pos < (col + 1) * B) & (pos >= 0)
                if not bool(here.any()):
                    continue
                at, x = pos[here] - col * B, rows[here]
                if pool.dtype != torch.int8:
                    if pool.dtype in (torch.float16, torch.bfloat16):
                        pool[block, at] = x.to(pool.dtype)
                    else:
                        mul = torch.tensor(1.0) / (torch.tensor(fp8_scale, dtype=torch.float32) if scales is None else scales[:, None])
                        pool.view(torch.uint8)[block, at] = (x * mul).to(pool.dtype).view(torch.uint8)
                    continue
                first = int(at[0])
                had = torch.zeros_like(scales[block]) if first == 0 else scales[block].clone()
                most = x.abs().amax((0, 2))
                new = torch.maximum(torch.maximum(had, most * torch.tensor(1.0 / 127.0, dtype=torch.float32)), torch.tensor(2.0 ** -126))
                ratio = (had / new)[:, None]
                if first > 0:
                    pool[block, :first] = (pool[block, :first].float() * ratio).round().clamp(-127, 127).to(torch.int8)
                pool[block, at] = (x * (1.0 / new)[:, None]).round().clamp(-127, 127).to(torch.int8)
                scales[block] = new
    return out


def angle_table(positions, rotary):
    a = torch.arange(positions).double()[:, None] * 10000.0 ** (-torch.arange(0, rotary, 2).double() / rotary)[None, :]
    return torch.cat([a.cos(), a.sin()], 1).float()
