"""The operators around a paged cache that is filled and read in ragged batches, as cases that can be timed and compared.

  kind "append"        new tokens of every sequence: queries and keys are rotated by their positions, keys and values go to
                       their places in the paged pools; pools of 8-bit integers keep a scale for each block and kv head, which
                       grows (and what the block holds is rounded again) when a new token asks for it
  kind "scaled"        attention of the new tokens over such 8-bit pools, causal, any number of new tokens per sequence
  kind "differential"  the difference of two softmax maps over one paged cache, each head's result normalised

The fields of a case:

  q            type of queries, keys, values and outputs: "fp16" or "bf16"
  kv           the pools: "16" (the same type), "i8" (integers, a scale for each block and kv head) or "e4m3"
  S, H, Hk, D, B   sequences, query heads, kv heads, elements of a cache row, tokens per block
  rows         pool layout: "head" [blocks, kv_heads, block, D] or "token" [blocks, block, kv_heads, D]
  new_lo .. new_hi   new tokens of a sequence (spread over the logarithm);  singles: how many sequences bring one token instead
  old_lo .. old_hi   tokens that are in the cache already
  rot, interleaved   rotated dims of a row, and whether a pair is two neighbours or lies half the rotated dims apart
  window, sinks      how many earlier keys a token sees (-1: all), and one more logit per head without a value

Lengths are functions of the case alone, so that every seed deals the same work to other blocks.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_DEFAULTS = dict(kind="append", q="bf16", kv="16", S=1, H=8, Hk=8, D=128, B=16, rows="head", new_lo=1, new_hi=1, singles=0,
                 old_lo=0, old_hi=0, rot=128, interleaved=False, window=-1, sinks=False)
_LEAST_SCALE = 2.0 ** -126
_NORM_EPS = 1e-5
_LAMBDA_INIT = 0.2


def _case(**fields):
    return {**_DEFAULTS, **fields}


def listed():
    return [
        # the smallest decode step: a few short sequences of a small model put one token each into 16-bit pools
        _case(name="append_few_short", kind="append", q="fp16", S=4, H=8, Hk=8, D=64, rot=64, old_lo=1, old_hi=255),
        # a decode batch of grouped-query heads over 8-bit pools
        _case(name="append_i8_batch", kind="append", kv="i8", S=128, H=64, Hk=8, old_lo=64, old_hi=4096),
        # prompts of several users, 16-bit pools, half of each row rotated, pairs of neighbours
        _case(name="append_prompts", kind="append", S=9, H=32, Hk=8, rot=64, interleaved=True, new_lo=301, new_hi=5003),
        # pieces of long prompts into 8-bit pools, token-major, blocks of 64
        _case(name="append_i8_pieces", kind="append", q="fp16", kv="i8", S=7, H=32, Hk=8, B=64, rows="token", new_lo=2048,
              new_hi=4096, old_lo=1001, old_hi=8192),
        # a handful of users with a few thousand tokens each: latency of one token
        _case(name="scaled_few_users", kind="scaled", kv="i8", S=3, H=32, Hk=8, old_lo=900, old_hi=4096),
        # a large serving mix: one token each over long 8-bit caches
        _case(name="scaled_i8_mix", kind="scaled", kv="i8", S=128, H=64, Hk=8, old_lo=512, old_hi=32768),
        # prompts next to running sequences, in one batch
        _case(name="scaled_mixed_batch", kind="scaled", q="fp16", kv="i8", S=19, H=32, Hk=8, singles=13, new_lo=127, new_hi=700,
              old_lo=33, old_hi=4096, sinks=True),
        # a piece of a long document: the largest product
        _case(name="scaled_e4m3_document", kind="scaled", kv="e4m3", S=1, H=32, Hk=8, new_lo=4096, new_hi=4096, old_lo=12288,
              old_hi=12288),
        # one user, small heads: the smallest differential step
        _case(name="differential_short", kind="differential", q="fp16", S=2, H=8, Hk=8, D=64, old_lo=31, old_hi=256),
        # a decode batch over 16-bit caches
        _case(name="differential_batch", kind="differential", S=32, H=16, Hk=8, old_lo=512, old_hi=8192),
        # one user with a long document
        _case(name="differential_one_long", kind="differential", S=1, H=16, Hk=4, old_lo=30010, old_hi=30010),
        # prompts of several users
        _case(name="differential_prompts", kind="differential", q="fp16", S=5, H=16, Hk=4, new_lo=513, new_hi=2003),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(["append", "scaled", "differential"])
        D = rng.choice([128, 128, 64])
        heads = rng.choice([1, 2, 4, 5, 8, 8, 16])
        group = rng.choice([1, 2, 3, 4, 4, 7, 8] if kind != "differential" else [1, 2, 2, 3, 4])
        c = _case(kind=kind, q=rng.choice(["fp16", "bf16"]), S=_log_int(rng, 1, 160), H=group * heads, Hk=heads, D=D,
                  B=rng.choice([16, 16, 32, 64]), rows=rng.choice(["head", "head", "token"]), old_hi=_log_int(rng, 1, 32768))
        c["kv"] = {"append": rng.choice(["16", "i8", "i8"]), "scaled": rng.choice(["i8", "i8", "e4m3"]),
                   "differential": rng.choice(["16", "16", "i8"])}[kind]
        c["old_lo"] = int(c["old_hi"] * rng.uniform(0.0, 0.9))
        if rng.random() < 0.5:  # prompts, some of them with single tokens beside them
            c["new_hi"] = _log_int(rng, 2, 5000)
            c["new_lo"] = max(1, int(c["new_hi"] * rng.uniform(0.1, 1.0)))
            c["singles"] = rng.choice([0, 0, c["S"] // 2])
        if kind == "append":
            c["rot"] = rng.choice([D, D, D // 2, D // 4])
            c["interleaved"] = rng.random() < 0.3
        else:
            c["window"] = rng.choice([-1, -1, -1, 511, 1023])
            c["sinks"] = kind == "scaled" and rng.random() < 0.25
        w = work(c)
        new, old = _lengths(c)
        padded = c["S"] * max(new) * c["H"] * (max(old) + max(new)) * (2 if kind == "differential" else 1)
        if w["bytes"] <= 0.8e9 and w["flops"] <= 0.9e12 and padded <= 1.5e9 and sum(old) + sum(new) <= 1 << 20:
            return c


def _lengths(case):
    """New tokens and tokens before them, of every sequence: quantiles of log-uniform spreads, in orders that do not go together."""
    n = case["S"]
    at = [(k + 0.5) / n for k in range(n)]

    def spread(lo, hi, u):
        return min(hi, int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** u)) - 1)

    new = [max(1, spread(case["new_lo"], case["new_hi"], (u * 7.0 + 0.31) % 1.0)) for u in at]
    old = [max(0, spread(case["old_lo"], case["old_hi"], (u * 5.0 + 0.17) % 1.0)) for u in at]
    for k in range(case["singles"]):  # they lie between the others
        new[(k * 3 + 1) % n if n % 3 else k] = 1
    return new, old


def work(case):
    c = case
    new, old = _lengths(c)
    T, kv_bytes = sum(new), 2 if c["kv"] == "16" else 1
    row = 2 * c["Hk"] * c["D"]  # elements of one token's K and V rows
    queries = 2 * T * c["H"] * c["D"] * 2
    if c["kind"] == "append":
        table = max(n + o for n, o in zip(new, old)) if max(new) > 1 else T  # rows of the table of angles
        touched = sum((o + n - 1) // c["B"] - o // c["B"] + 1 for n, o in zip(new, old))
        scales = 2 * touched * c["Hk"] * 4 * 2 if c["kv"] == "i8" else 0
        return {"bytes": queries + T * row * (2 + kv_bytes) + min(table, T) * c["rot"] * 4 + touched * 4 + c["S"] * 8 + scales,
                "flops": 3 * T * (c["H"] + c["Hk"]) * c["rot"]}
    seen = pairs = entries = 0
    for n, o in zip(new, old):
        first = 0 if c["window"] < 0 else max(0, o - c["window"])  # the first key that some token sees
        seen += o + n - first
        entries += (o + n - 1) // c["B"] - first // c["B"] + 1
        if c["window"] < 0:
            pairs += n * o + n * (n + 1) // 2
        else:
            full = min(n, max(0, c["window"] + 1 - o))  # tokens that see everything before them
            pairs += full * o + full * (full + 1) // 2 + (n - full) * (c["window"] + 1)
    total = queries + seen * row * kv_bytes + entries * 4 + c["S"] * 8
    if c["kv"] != "16":
        total += entries * c["Hk"] * 8
    return {"bytes": total, "flops": pairs * c["H"] * c["D"] * (6 if c["kind"] == "differential" else 4)}


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    S, H, Hk, D, B = c["S"], c["H"], c["Hk"], c["D"], c["B"]
    dtype = _TYPES[c["q"]]
    new, old = (torch.tensor(x, dtype=torch.int64) for x in _lengths(c))
    lens = new + old
    T = int(new.sum())
    start = torch.zeros(S + 1, dtype=torch.int32)
    start[1:] = torch.cumsum(new, 0)
    per_seq = (lens + B - 1) // B
    need = int(per_seq.sum())
    blocks = need + need // 16 + 1
    tables = torch.zeros((S, int(per_seq.max())), dtype=torch.int32)
    tables[torch.arange(tables.size(1))[None, :] < per_seq[:, None]] = torch.randperm(blocks, generator=host)[:need].to(torch.int32)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float16)

    s = dict(case=c, tables=tables.to(dev), start=start.to(dev), lens=lens.to(torch.int32).to(dev), most_new=int(new.max()),
             longest=int(lens.max()), k_scales=None, v_scales=None)
    shape = (blocks, Hk, B, D) if c["rows"] == "head" else (blocks, B, Hk, D)
    pools = []
    for which in ("k_scales", "v_scales"):
        values = normal(*shape)
        if c["kv"] == "16":
            pools.append(values.to(dtype))
            continue
        # 8 bits: a block's largest value sits at the end of the range, the blocks' scales differ
        most = values.abs().amax((2, 3) if c["rows"] == "head" else (1, 3)).float().clamp_min(1e-3)
        unit = (most / (127.0 if c["kv"] == "i8" else 448.0)).contiguous()
        per = unit[:, :, None, None] if c["rows"] == "head" else unit[:, None, :, None]
        values = values / per.half()
        pools.append(values.clamp_(-127, 127).round_().to(torch.int8) if c["kv"] == "i8" else
                     values.clamp_(-448, 448).to(torch.float8_e4m3fn))
        s[which] = unit * torch.exp(0.3 * normal(blocks, Hk).float())
    s["pools"] = pools
    # the views that the entry points take: [blocks, block_size, kv_heads, D]
    s["keys"], s["values"] = (p.permute(0, 2, 1, 3) if c["rows"] == "head" else p for p in pools)
    if c["kind"] == "append":
        # queries, keys and values as a projection leaves them: side by side in one row per token
        fused = normal(T, H + 2 * Hk, D).to(dtype)
        s["query"], s["new_keys"], s["new_values"] = fused[:, :H], fused[:, H:H + Hk], fused[:, H + Hk:]
        s["query_out"] = torch.zeros((T, H, D), dtype=dtype, device=dev)
        angles = torch.arange(s["longest"], device=dev).double()[:, None] * \
            10000.0 ** (-torch.arange(0, c["rot"], 2, device=dev).double() / c["rot"])[None, :]
        s["cos_sin"] = torch.cat([angles.cos(), angles.sin()], 1).float()
        return s
    s["query"] = normal(T, H, D).to(dtype)
    s["out"] = torch.zeros((T, H, D), dtype=dtype, device=dev)
    s["scale"] = 1.0 / math.sqrt(D if c["kind"] == "scaled" else D // 2)
    s["sinks"] = normal(H).to(dtype) if c["sinks"] else None
    if c["kind"] == "differential":
        s["lambdas"] = _LAMBDA_INIT + 0.3 * torch.rand(H, generator=g, device=dev)
        s["norm_weight"] = 1.0 + 0.1 * normal(D).float()
    return s


# ---- the operators in their plain form: elementary operations in 32 bits, rounded once at the end ----

def _tokens(s):
    """Sequence, place among the sequence's new tokens, and position of every new token."""
    t = torch.arange(s["query"].size(0), device=s["start"].device)
    seq = torch.searchsorted(s["start"][1:].contiguous(), t.to(torch.int32), right=True)
    start = s["start"].long()
    j = t - start[seq]
    return seq, j, s["lens"].long()[seq] - (start[seq + 1] - start[seq]) + j


def _rotated(x, angles, rot, interleaved):
    x = x.float()
    cos, sin = angles[:, None, :rot // 2], angles[:, None, rot // 2:]
    pairs, rest = x[..., :rot], x[..., rot:]
    a, b = (pairs[..., 0::2], pairs[..., 1::2]) if interleaved else (pairs[..., :rot // 2], pairs[..., rot // 2:])
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([turned, rest], -1)


def _place(rows, cache, scales, block, row):
    """The rows at their places of the pool; with a scale for each block and head, what was there is rounded again where it grew."""
    if scales is None:
        cache[block, row] = rows.to(cache.dtype)
        return
    NB, B, Hk, _ = cache.shape
    most = torch.zeros((NB, Hk), device=rows.device)
    most.scatter_reduce_(0, block[:, None].expand(-1, Hk), rows.abs().amax(-1), "amax")
    first = torch.full((NB,), B, device=rows.device)  # the first row of a block that is new
    first.scatter_reduce_(0, block, row, "amin")
    touched = (first < B)[:, None]
    before = torch.where((first == 0)[:, None], torch.zeros_like(scales), scales)  # what a block held for others counts no more
    after = torch.maximum(torch.maximum(before, most / 127.0), torch.full_like(before, _LEAST_SCALE))
    ratio = torch.where(touched, before / after, torch.ones_like(scales))
    again = (cache.float() * ratio[:, None, :, None]).round_().clamp_(-127, 127).to(torch.int8)
    kept = torch.arange(B, device=rows.device)[None, :] < torch.where(first < B, first, torch.zeros_like(first))[:, None]
    cache.copy_(torch.where(kept[:, :, None, None], again, cache))
    scales.copy_(torch.where(touched, after, scales))
    cache[block, row] = (rows * (1.0 / scales)[block][..., None]).round_().clamp_(-127, 127).to(torch.int8)


def _append_plain(s):
    c = s["case"]
    seq, _, at = _tokens(s)
    angles = s["cos_sin"][at]
    s["query_out"].copy_(_rotated(s["query"], angles, c["rot"], c["interleaved"]))
    block, row = s["tables"][seq, at // c["B"]].long(), at % c["B"]
    _place(_rotated(s["new_keys"], angles, c["rot"], c["interleaved"]), s["keys"], s["k_scales"], block, row)
    _place(s["new_values"].float(), s["values"], s["v_scales"], block, row)


def _gathered(s):
    """Queries [S, new, H, D] and the rows of K and V [S, Hk, keys, D] of every sequence, and which keys a query sees."""
    c = s["case"]
    n, long = s["most_new"], s["longest"]
    key = torch.arange(long, device=s["tables"].device)
    block = s["tables"][:, key // c["B"]].long()  # [S, keys]
    got = []
    for pool, scales in ((s["keys"], s["k_scales"]), (s["values"], s["v_scales"])):
        rows = pool[block, key % c["B"]].float()
        if scales is not None:
            rows *= scales[block][..., None]
        got.append(rows.transpose(1, 2).contiguous())
    start, lens = s["start"].long(), s["lens"].long()
    j = torch.arange(n, device=key.device)
    token = (start[:-1, None] + j).clamp_max(s["query"].size(0) - 1)
    at = (lens - (start[1:] - start[:-1]))[:, None] + j  # [S, new]
    sees = (key <= at[..., None]) & (key < lens[:, None, None])
    if c["window"] >= 0:
        sees &= key >= at[..., None] - c["window"]
    return s["query"].float()[token], *got, sees


def _softmax_rows(q, k, v, sees, scale, sinks):
    """One softmax map applied to V: q [S, new, H, d], k [S, Hk, keys, d], v [S, Hk, keys, D] -> [S, new, H, D]."""
    S, n, H, d = q.shape
    Hk = k.size(1)
    x = torch.matmul(q.view(S, n, Hk, H // Hk, d).transpose(1, 2).reshape(S, Hk, -1, d), k.transpose(2, 3))
    x = x.view(S, Hk, n, H // Hk, -1).mul_(scale).masked_fill_(~sees[:, None, :, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    if sinks is not None:
        sinks = sinks.float().view(1, Hk, 1, -1, 1)
        top = torch.maximum(top, sinks)
    top = top.masked_fill(top == -math.inf, 0.0)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks - top)
    o = torch.matmul(x.view(S, Hk, n * (H // Hk), -1), v).view(S, Hk, n, H // Hk, -1)
    return (o / total.masked_fill(total == 0.0, 1.0)).transpose(1, 2).reshape(S, n, H, -1)


def _attend_plain(s):
    q, k, v, sees = _gathered(s)
    if s["case"]["kind"] == "scaled":
        o = _softmax_rows(q, k, v, sees, s["scale"], s["sinks"])
    else:
        d = q.size(-1) // 2
        o = _softmax_rows(q[..., :d], k[..., :d], v, sees, s["scale"], None)
        o = o - s["lambdas"][:, None] * _softmax_rows(q[..., d:], k[..., d:], v, sees, s["scale"], None)
        o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + _NORM_EPS) * s["norm_weight"] * (1.0 - _LAMBDA_INIT)
    seq, j, _ = _tokens(s)
    s["out"].copy_(o[seq, j])


# ---- the calls that a user makes of the framework ----

def _append_own(s):
    torch.ops.fa_amd.kv_cache_append(
        s["new_keys"], s["new_values"], s["keys"], s["values"], s["tables"], s["start"], s["lens"], s["cos_sin"], s["query"],
        s["query_out"], s["k_scales"], s["v_scales"], interleaved=s["case"]["interleaved"])


def _scaled_own(s):
    torch.ops.fa_amd.paged_attention_ragged(
        s["out"], s["query"], s["keys"], s["values"], s["tables"], s["start"], s["lens"], s["scale"], s["most_new"], s["longest"],
        k_scales=s["k_scales"], v_scales=s["v_scales"], sinks=s["sinks"], window_left=s["case"]["window"])


def _differential_own(s):
    torch.ops.fa_amd.paged_attention_differential(
        s["out"], s["query"], s["keys"], s["values"], s["tables"], s["start"], s["lens"], s["scale"], s["lambdas"],
        s["norm_weight"], s["most_new"], s["longest"], norm_eps=_NORM_EPS, out_scale=1.0 - _LAMBDA_INIT, k_scales=s["k_scales"],
        v_scales=s["v_scales"], window_left=s["case"]["window"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        from flash_attention_factory_amd import torch_ops  # noqa: F401  (registers torch.ops.fa_amd)
        {"append": _append_own, "scaled": _scaled_own, "differential": _differential_own}[kind](state)
    else:
        (_append_plain if kind == "append" else _attend_plain)(state)
    if kind != "append":
        return state["out"]
    # integers are compared as what they are, number for number, beside the scales that they are multiples of: their products
    # would cost a pass over the pools that no program makes
    got = {"query": state["query_out"], "keys": state["pools"][0], "values": state["pools"][1]}
    if state["k_scales"] is not None:
        got.update(k_scales=state["k_scales"], v_scales=state["v_scales"])
    return got


# ---- the same in 64 bits, sequence by sequence ----

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(case, s) if case["kind"] == "append" else _exact_attend(case, s)


def _turn(x, angles, interleaved):
    """Rows [tokens, heads, D] in 64 bits, as complex numbers times exp(i angle)."""
    half = angles.size(1) // 2
    phase = torch.complex(angles[:, :half].double(), angles[:, half:].double())[:, None, :]
    x = x.double().clone()
    if interleaved:
        z = torch.complex(x[..., 0:2 * half:2].clone(), x[..., 1:2 * half:2].clone()) * phase
        x[..., 0:2 * half:2], x[..., 1:2 * half:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half].clone(), x[..., half:2 * half].clone()) * phase
        x[..., :half], x[..., half:2 * half] = z.real, z.imag
    return x


def _exact_append(c, s):
    start, lens, tables = s["start"].tolist(), s["lens"].tolist(), s["tables"].long()
    B = c["B"]
    query, pools = [], [p.double() if c["kv"] == "16" else None for p in s["pools"]]
    scales = [None if x is None else x.double().clone() for x in (s["k_scales"], s["v_scales"])]
    for q in range(c["S"]):
        a, b = start[q], start[q + 1]
        at = torch.arange(lens[q] - (b - a), lens[q], device=tables.device)
        angles = s["cos_sin"][at]
        query.append(_turn(s["query"][a:b], angles, c["interleaved"]))
        block = tables[q, at // B]
        for which, rows in enumerate((_turn(s["new_keys"][a:b], angles, c["interleaved"]), s["new_values"][a:b].double())):
            if c["kv"] == "16":
                (pools[which].transpose(1, 2) if c["rows"] == "head" else pools[which])[block, at % B] = rows
                continue
            first, last = int(at[0]) // B, int(at[-1]) // B
            most = torch.zeros((last - first + 1, c["Hk"]), dtype=torch.float64, device=rows.device)
            most.scatter_reduce_(0, (at // B - first)[:, None].expand(-1, c["Hk"]), rows.abs().amax(-1), "amax")
            ids = tables[q, first:last + 1]
            had = scales[which][ids]
            if int(at[0]) % B == 0:
                had[0] = 0.0
            had[1:] = 0.0
            scales[which][ids] = torch.maximum(had, most / 127.0).clamp_min(_LEAST_SCALE)
    got = {"query": torch.cat(query), "keys": pools[0], "values": pools[1]}
    if scales[0] is not None:
        got.update(k_scales=scales[0], v_scales=scales[1])
    return got


def _exact_attend(c, s):
    start, lens, tables = s["start"].tolist(), s["lens"].tolist(), s["tables"].long()
    H, Hk, D = c["H"], c["Hk"], c["D"]
    maps = 1 if c["kind"] == "scaled" else 2
    d = D // maps
    out = torch.zeros((start[-1], H, D), dtype=torch.float64, device=tables.device)
    for q in range(c["S"]):
        n, a = lens[q], start[q]
        key = torch.arange(n, device=tables.device)
        ids = tables[q, key // c["B"]]
        at = torch.arange(n - (start[q + 1] - a), n, device=tables.device)
        sees = key[None, :] <= at[:, None]
        if c["window"] >= 0:
            sees &= key[None, :] + c["window"] >= at[:, None]
        for h in range(Hk):
            k, v = (p[ids, key % c["B"], h].double() * (1.0 if x is None else x[ids, h, None].double())
                    for p, x in ((s["keys"], s["k_scales"]), (s["values"], s["v_scales"])))
            for head in range(h * (H // Hk), (h + 1) * (H // Hk)):
                o = 0.0
                for m in range(maps):
                    x = s["query"][a:start[q + 1], head, m * d:(m + 1) * d].double() @ k[:, m * d:(m + 1) * d].T * s["scale"]
                    x = x.masked_fill(~sees, -math.inf)
                    if s["sinks"] is not None:
                        x = torch.cat([x, s["sinks"][head].double().expand(x.size(0), 1)], 1)
                    p = torch.softmax(x, -1)[:, :n]
                    o = o + (p @ v) * (1.0 if m == 0 else -s["lambdas"][head].double())
                if maps == 2:
                    o = o / torch.sqrt((o * o).mean(-1, keepdim=True) + _NORM_EPS) * s["norm_weight"].double() * (1.0 - _LAMBDA_INIT)
                out[a:start[q + 1], head] = o
    return out
