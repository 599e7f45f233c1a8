"""Latent attention -- one shared latent vector and one rotated key part a token -- as cases that can be timed and compared.

  kind "append"    new tokens of every sequence: the latent is normalised, its key part and the queries' are rotated by their
                   positions, latent and key part go side by side to the token's row of the paged pool; an FP8 pool keeps a scale for each row
  kind "gather"    the cached rows of every sequence, read back as dense 16-bit rows (what the expanding product takes)
  kind "absorbed"  attention of the new tokens over the pool itself, the up-projections absorbed into the queries: the row is the
                   key of all heads, and its latent part the value
  kind "expanded"  attention over keys and values that have been expanded for each head, the rotated key part shared by the heads

The fields of a case:

  q            type of queries, latents and outputs: "fp16" or "bf16"
  kv           the pool: "16" (the same type) or "e4m3" (bytes, a scale for each row)
  S, H         sequences, query heads
  L, R         elements of the latent and of the rotated part
  D            elements of an expanded key (without its rotated part) and value
  B            tokens per block
  new_lo .. new_hi   new tokens of a sequence (spread over the logarithm);  singles: how many sequences bring one token instead
  old_lo .. old_hi   tokens before them
  interleaved  whether a rotated pair is two neighbours, or lies R / 2 apart

Lengths are functions of the case alone, so that every seed deals the same work to other blocks.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_DEFAULTS = dict(kind="absorbed", q="bf16", kv="16", S=1, H=16, L=512, R=64, D=128, B=16, new_lo=1, new_hi=1, singles=0, old_lo=0,
                 old_hi=0, interleaved=False)
_EPS = 1e-6


def _case(**fields):
    return {**_DEFAULTS, **fields}


def listed():
    return [
        # the smallest decode step: a few short sequences put one token each into a 16-bit pool
        _case(name="append_few_short", kind="append", q="fp16", S=4, H=16, old_lo=1, old_hi=255),
        # a decode batch with many heads over an FP8 pool
        _case(name="append_e4m3_batch", kind="append", kv="e4m3", S=128, H=128, old_lo=64, old_hi=4096, interleaved=True),
        # prompts of several users
        _case(name="append_e4m3_prompts", kind="append", kv="e4m3", S=9, H=32, B=64, new_lo=301, new_hi=5003, interleaved=True),
        # the context of a few short conversations
        _case(name="gather_few_short", kind="gather", q="fp16", S=3, old_lo=100, old_hi=900),
        # long contexts before their next pieces are attended
        _case(name="gather_e4m3_contexts", kind="gather", kv="e4m3", S=21, B=64, old_lo=1001, old_hi=24000),
        # a handful of users, a share of the heads: latency of one token
        _case(name="absorbed_few_users", kind="absorbed", S=3, H=16, old_lo=900, old_hi=4096),
        # a decode batch with all of many heads
        _case(name="absorbed_many_heads", kind="absorbed", S=64, H=128, old_lo=512, old_hi=16384),
        # a large serving mix with a share of the heads over a long FP8 cache
        _case(name="absorbed_e4m3_mix", kind="absorbed", kv="e4m3", S=128, H=16, B=64, old_lo=512, old_hi=32768),
        # drafted tokens verified, a few for each sequence
        _case(name="absorbed_drafts", kind="absorbed", q="fp16", kv="e4m3", S=13, H=64, new_lo=2, new_hi=6, old_lo=301, old_hi=9000),
        # short prompts of a small model
        _case(name="expanded_short", kind="expanded", q="fp16", S=5, H=16, D=64, new_lo=17, new_hi=257),
        # prompts of several users
        _case(name="expanded_prompts", kind="expanded", S=6, H=32, new_lo=513, new_hi=4003),
        # a piece of a long document: the largest product
        _case(name="expanded_document", kind="expanded", S=1, H=32, new_lo=4096, new_hi=4096, old_lo=12288, old_hi=12288),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        kind = rng.choice(["append", "gather", "absorbed", "absorbed", "absorbed", "expanded", "expanded"])
        c = _case(kind=kind, q=rng.choice(["fp16", "bf16"]), kv=rng.choice(["16", "e4m3"]), S=_log_int(rng, 1, 160),
                  H=rng.choice([5, 8, 16, 16, 20, 32, 40, 64, 128]), L=rng.choice([512, 512, 256]), D=rng.choice([128, 128, 64]),
                  B=rng.choice([16, 32, 64]), old_hi=_log_int(rng, 1, 32768), interleaved=rng.random() < 0.5)
        c["old_lo"] = int(c["old_hi"] * rng.uniform(0.0, 0.9))
        if kind == "expanded" or (kind == "append" and rng.random() < 0.5):  # prompts and pieces of them
            c["new_hi"] = _log_int(rng, 2, 5000)
            c["new_lo"] = max(1, int(c["new_hi"] * rng.uniform(0.1, 1.0)))
            c["singles"] = rng.choice([0, 0, c["S"] // 2])
            if rng.random() < 0.5:
                c["old_lo"] = c["old_hi"] = 0
        elif kind == "absorbed" and rng.random() < 0.4:  # drafted tokens, short pieces
            c["new_hi"] = _log_int(rng, 2, 64)
            c["new_lo"] = max(1, int(c["new_hi"] * rng.uniform(0.1, 1.0)))
            c["singles"] = rng.choice([0, 0, c["S"] // 2])
        w = work(c)
        new, old = _lengths(c)
        scores = c["S"] * c["H"] * max(new) * (max(new) + max(old))
        rows = c["S"] * (max(new) + max(old)) * (c["L"] + c["R"] if kind != "expanded" else c["H"] * (2 * c["D"] + c["R"]))
        if w["bytes"] <= 1.2e9 and w["flops"] <= 1.1e12 and scores <= 2.1e9 and rows <= 2.5e9:
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
    T, width = sum(new), c["L"] + c["R"]
    row = width * 2 if c["kv"] == "16" else width + 4
    if c["kind"] == "append":
        table = max(n + o for n, o in zip(new, old)) if max(new) > 1 else T  # rows of the table of angles
        touched = sum((o + n - 1) // c["B"] - o // c["B"] + 1 for n, o in zip(new, old))
        return {"bytes": T * (width * 2 + row) + 2 * T * c["H"] * c["R"] * 2 + min(table, T) * c["R"] * 4 + c["L"] * 4 + touched * 4 + c["S"] * 8,
                "flops": T * (4 * c["L"] + 3 * (c["H"] + 1) * c["R"])}
    if c["kind"] == "gather":
        rows = sum(old)
        entries = sum(-(-o // c["B"]) for o in old)
        return {"bytes": rows * (row + width * 2) + entries * 4 + c["S"] * 4, "flops": rows * width if c["kv"] != "16" else 0}
    keys = sum(n + o for n, o in zip(new, old))
    pairs = sum(n * o + n * (n + 1) // 2 for n, o in zip(new, old))
    if c["kind"] == "absorbed":
        entries = sum(-(-(n + o) // c["B"]) for n, o in zip(new, old))
        return {"bytes": T * c["H"] * (width + c["L"]) * 2 + keys * row + entries * 4 + c["S"] * 8,
                "flops": pairs * c["H"] * 2 * (width + c["L"])}
    return {"bytes": T * c["H"] * (2 * c["D"] + c["R"]) * 2 + keys * (c["H"] * 2 * c["D"] + c["R"]) * 2 + c["S"] * 8,
            "flops": pairs * c["H"] * 2 * (2 * c["D"] + c["R"])}


def prepare(case, seed):
    c = case
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    host = torch.Generator()
    host.manual_seed(seed)
    S, H, L, R, D, B = c["S"], c["H"], c["L"], c["R"], c["D"], c["B"]
    dtype = _TYPES[c["q"]]
    new, old = (torch.tensor(x, dtype=torch.int64) for x in _lengths(c))
    lens = old if c["kind"] == "gather" else new + old
    T, N = int(new.sum()), int(lens.sum())

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float16)

    def upto(counts):
        at = torch.zeros(S + 1, dtype=torch.int32)
        at[1:] = torch.cumsum(counts, 0)
        return at.to(dev)

    s = dict(case=c, start=upto(new), keys_at=upto(lens), lens=lens.to(torch.int32).to(dev), most_new=int(new.max()), longest=int(lens.max()),
             scale=1.0 / math.sqrt(D + R), scales=None)
    if c["kind"] == "expanded":
        s["query"] = normal(T, H, D + R).to(dtype)
        # keys and values as the expanding product leaves them: side by side for each head
        s["expanded"] = normal(N, H, 2 * D).to(dtype)
        s["rope_key"] = normal(N, L + R).to(dtype)[:, L:]
        s["out"] = torch.zeros((T, H, D), dtype=dtype, device=dev)
        return s
    per_seq = (lens + B - 1) // B
    need = int(per_seq.sum())
    blocks = need + need // 16 + 1
    tables = torch.zeros((S, max(1, int(per_seq.max()))), dtype=torch.int32)
    tables[torch.arange(tables.size(1))[None, :] < per_seq[:, None]] = torch.randperm(blocks, generator=host)[:need].to(torch.int32)
    s["tables"] = tables.to(dev)
    rows = normal(blocks, B, L + R)
    if c["kv"] == "16":
        s["cache"] = rows.to(dtype)
    else:  # rows of different sizes, each with the power of two that brings its largest value to the end of the range
        rows = rows.float() * torch.exp(normal(blocks, B, 1).float())
        s["scales"] = _row_scale(rows.abs().amax(-1))
        s["cache"] = (rows / s["scales"][..., None]).to(torch.float8_e4m3fn)
        # the size that a normalised latent has
        s["scales"] = s["scales"] * torch.exp2(torch.round(-torch.log2(rows.square().mean(-1).sqrt())))
    if c["kind"] == "append":
        # latent and key part as the compressing product leaves them, side by side; the rotated parts of the queries' heads
        down = normal(T, L + R).to(dtype)
        s["latent"], s["rope_key"] = down[:, :L], down[:, L:]
        s["norm_weight"] = 1.0 + 0.1 * normal(L).float()
        s["query_rope"] = normal(T, H, D + R).to(dtype)[..., D:]
        s["query_out"] = torch.zeros((T, H, R), dtype=dtype, device=dev)
        angles = torch.arange(s["longest"], device=dev).double()[:, None] * \
            10000.0 ** (-torch.arange(0, R, 2, device=dev).double() / R)[None, :]
        s["cos_sin"] = torch.cat([angles.cos(), angles.sin()], 1).float()
    elif c["kind"] == "gather":
        s["out"] = torch.zeros((N, L + R), dtype=dtype, device=dev)
    else:
        # queries as the absorbing products leave them: heads outermost; the rotated parts within the rows of the projection.  A latent
        # query is a sum over D elements with weights that keep the scores of the order of 1
        s["query_latent"] = (normal(H, T, L) * math.sqrt(D / L)).to(dtype).transpose(0, 1)
        s["query_rope"] = normal(T, H, D + R).to(dtype)[..., D:]
        s["out"] = torch.zeros((H, T, L), dtype=dtype, device=dev).transpose(0, 1)
    return s


# ---- the operators in their plain form: elementary operations in 32 bits, rounded once at the end ----

def _row_scale(most):
    """The least power of two, 2^-100 or more, that brings a row's largest value to 448 or less."""
    part, power = torch.frexp(most / 448.0)
    return torch.exp2(torch.where(most > 0, power - (part == 0.5).to(power.dtype), torch.full_like(power, -100)).clamp(-100, 100).float())


def _tokens(start, n):
    """Which sequence a row belongs to, and its place among the sequence's rows."""
    t = torch.arange(n, device=start.device)
    seq = torch.searchsorted(start[1:].contiguous(), t.to(torch.int32), right=True)
    return seq, t - start.long()[seq]


def _rotated(x, angles, interleaved):
    x = x.float()
    half = x.size(-1) // 2
    cos, sin = angles[..., :half], angles[..., half:]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    p, q = a * cos - b * sin, b * cos + a * sin
    return torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)


def _append_plain(s):
    c = s["case"]
    seq, j = _tokens(s["start"], s["latent"].size(0))
    start = s["start"].long()
    at = s["lens"].long()[seq] - (start[seq + 1] - start[seq]) + j
    angles = s["cos_sin"][at]
    x = s["latent"].float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * s["norm_weight"]
    row = torch.cat([x, _rotated(s["rope_key"], angles, c["interleaved"])], -1)
    s["query_out"].copy_(_rotated(s["query_rope"], angles[:, None], c["interleaved"]))
    block, place = s["tables"][seq, at // c["B"]].long(), at % c["B"]
    if s["scales"] is not None:
        scale = _row_scale(row.abs().amax(-1))
        s["scales"][block, place] = scale
        row = row / scale[:, None]
    s["cache"][block, place] = row.to(s["cache"].dtype)


def _cached(s, seq, key):
    """Rows of the pool in 32 bits."""
    block, place = s["tables"][seq, key // s["case"]["B"]].long(), key % s["case"]["B"]
    rows = s["cache"][block, place].float()
    return rows if s["scales"] is None else rows * s["scales"][block, place][..., None]


def _gather_plain(s):
    s["out"].copy_(_cached(s, *_tokens(s["keys_at"], s["out"].size(0))))


def _padded(s):
    """[S, new] rows of the token arrays and [S, new, keys] which keys a token sees."""
    n, long = s["most_new"], s["longest"]
    start, lens = s["start"].long(), s["lens"].long()
    j, key = torch.arange(n, device=start.device), torch.arange(long, device=start.device)
    token = (start[:-1, None] + j).clamp_max(int(s["out"].size(0)) - 1)
    at = (lens - (start[1:] - start[:-1]))[:, None] + j
    return token, (key <= at[..., None]) & (key < lens[:, None, None])


def _weights(x, scale, sees):
    """Softmax over the last dimension of scores x [S, H, new, keys], those that are not seen left out: weights and their sums."""
    x = x.mul_(scale).masked_fill_(~sees[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = x.sum(-1, keepdim=True)
    return x, total.masked_fill_(total == 0.0, 1.0)


def _absorbed_plain(s):
    c = s["case"]
    S, H, L = c["S"], c["H"], c["L"]
    token, sees = _padded(s)
    n, long = token.size(1), s["longest"]
    key = torch.arange(long, device=token.device)
    k = _cached(s, torch.arange(S, device=key.device)[:, None], key[None])  # [S, keys, L + R]
    q = torch.cat([s["query_latent"].float(), s["query_rope"].float()], -1)[token]  # [S, new, H, L + R]
    x = torch.matmul(q.transpose(1, 2).reshape(S, H * n, -1), k.transpose(1, 2).contiguous())
    x, total = _weights(x.view(S, H, n, long), s["scale"], sees)
    o = torch.matmul(x.view(S, H * n, long), k[..., :L].contiguous()).view(S, H, n, L) / total
    seq, j = _tokens(s["start"], s["out"].size(0))
    s["out"].copy_(o[seq, :, j])


def _expanded_plain(s):
    c = s["case"]
    H, D = c["H"], c["D"]
    token, sees = _padded(s)
    S, n, long = sees.shape
    key = (s["keys_at"].long()[:-1, None] + torch.arange(long, device=token.device)).clamp_max(s["expanded"].size(0) - 1)
    expanded = s["expanded"].float()[key].transpose(1, 2)  # [S, H, keys, 2 D]
    shared = s["rope_key"].float()[key][:, None].expand(S, H, long, -1)
    k = torch.cat([expanded[..., :D], shared], -1).transpose(2, 3).contiguous()
    x, total = _weights(torch.matmul(s["query"].float()[token].transpose(1, 2).contiguous(), k), s["scale"], sees)
    o = torch.matmul(x, expanded[..., D:].contiguous()) / total
    seq, j = _tokens(s["start"], s["out"].size(0))
    s["out"].copy_(o[seq, :, j])


# ---- the calls that a user makes of the framework ----

def _append_own(s):
    torch.ops.fa_amd.latent_cache_append(
        s["latent"], s["rope_key"], s["cache"], s["tables"], s["start"], s["lens"], s["norm_weight"], s["cos_sin"], s["query_rope"],
        s["query_out"], s["scales"], norm_eps=_EPS, interleaved=s["case"]["interleaved"])


def _gather_own(s):
    torch.ops.fa_amd.latent_cache_gather(s["out"], s["cache"], s["tables"], s["keys_at"], scales=s["scales"])


def _absorbed_own(s):
    torch.ops.fa_amd.paged_attention_latent(
        s["out"], s["query_latent"], s["query_rope"], s["cache"], s["tables"], s["start"], s["lens"], s["scale"], s["most_new"],
        s["longest"], scales=s["scales"])


def _expanded_own(s):
    D = s["case"]["D"]
    torch.ops.fa_amd.attention_latent_expanded(
        s["out"], s["query"], s["expanded"][..., :D], s["rope_key"], s["expanded"][..., D:], s["start"], s["keys_at"], s["scale"],
        s["most_new"], s["longest"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        from flash_attention_factory_amd import torch_ops  # noqa: F401  (registers torch.ops.fa_amd)
        {"append": _append_own, "gather": _gather_own, "absorbed": _absorbed_own, "expanded": _expanded_own}[kind](state)
    else:
        {"append": _append_plain, "gather": _gather_plain, "absorbed": _absorbed_plain, "expanded": _expanded_plain}[kind](state)
    if kind != "append":
        return state["out"]
    # an FP8 pool is returned as it is, beside the scales that its rows are multiples of: their products would cost a pass over the
    # pool that no program makes
    got = {"query": state["query_out"], "cache": state["cache"]}
    if state["scales"] is not None:
        got["scales"] = state["scales"]
    return got


# ---- the same in 64 bits, sequence by sequence ----

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "gather": _exact_gather, "absorbed": _exact_absorbed, "expanded": _exact_expanded}[case["kind"]](case, s)


def _turn(x, angles, interleaved):
    """Rows [tokens, heads, R] in 64 bits, as complex numbers times exp(i angle)."""
    x = x.double()
    half = x.size(-1) // 2
    phase = torch.complex(angles[:, :half].double(), angles[:, half:].double())[:, None, :]
    z = (torch.complex(x[..., 0::2].contiguous(), x[..., 1::2].contiguous()) if interleaved else
         torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous())) * phase
    return torch.view_as_real(z).flatten(-2) if interleaved else torch.cat([z.real, z.imag], -1)


def _exact_append(c, s):
    start, lens, tables = s["start"].tolist(), s["lens"].tolist(), s["tables"].long()
    B = c["B"]
    cache, query = s["cache"].double(), []
    scales = None if s["scales"] is None else s["scales"].double()
    for q in range(c["S"]):
        a, b = start[q], start[q + 1]
        at = torch.arange(lens[q] - (b - a), lens[q], device=tables.device)
        angles = s["cos_sin"][at]
        query.append(_turn(s["query_rope"][a:b], angles, c["interleaved"]))
        x = s["latent"][a:b].double()
        x = x / torch.sqrt(x.pow(2).sum(1, keepdim=True) / c["L"] + _EPS) * s["norm_weight"].double()
        row = torch.cat([x, _turn(s["rope_key"][a:b, None], angles, c["interleaved"])[:, 0]], 1)
        ids = tables[q, at // B]
        if scales is not None:  # a pool of bytes holds multiples of the row's scale
            unit = 2.0 ** torch.ceil(torch.log2(row.abs().amax(1) / 448.0))
            scales[ids, at % B] = unit
            row = row / unit[:, None]
        cache[ids, at % B] = row
    got = {"query": torch.cat(query), "cache": cache}
    if scales is not None:
        got["scales"] = scales
    return got


def _exact_rows(c, s, q, n):
    at = torch.arange(n, device=s["tables"].device)
    ids = s["tables"][q, at // c["B"]].long()
    rows = s["cache"][ids, at % c["B"]].double()
    return rows if s["scales"] is None else rows * s["scales"][ids, at % c["B"]].double()[:, None]


def _exact_gather(c, s):
    return torch.cat([_exact_rows(c, s, q, n) for q, n in enumerate(s["lens"].tolist())])


def _exact_softmax(x, n, ctx):
    """Causal weights of scores x [n, ctx]: the last token sees every key."""
    at = torch.arange(ctx - n, ctx, device=x.device)
    return torch.softmax(x.masked_fill(torch.arange(ctx, device=x.device)[None] > at[:, None], -math.inf), -1)


def _exact_absorbed(c, s):
    start = s["start"].tolist()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=s["out"].device)
    for q, ctx in enumerate(s["lens"].tolist()):
        a, b = start[q], start[q + 1]
        rows = _exact_rows(c, s, q, ctx)
        for h in range(c["H"]):
            x = s["query_latent"][a:b, h].double() @ rows[:, :c["L"]].T + s["query_rope"][a:b, h].double() @ rows[:, c["L"]:].T
            out[a:b, h] = _exact_softmax(x * s["scale"], b - a, ctx) @ rows[:, :c["L"]]
    return out


def _exact_expanded(c, s):
    start, keys_at = s["start"].tolist(), s["keys_at"].tolist()
    D = c["D"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=s["out"].device)
    for q in range(c["S"]):
        a, b, k0, k1 = start[q], start[q + 1], keys_at[q], keys_at[q + 1]
        shared = s["rope_key"][k0:k1].double()
        for h in range(c["H"]):
            x = s["query"][a:b, h, :D].double() @ s["expanded"][k0:k1, h, :D].double().T + s["query"][a:b, h, D:].double() @ shared.T
            out[a:b, h] = _exact_softmax(x * s["scale"], b - a, k1 - k0) @ s["expanded"][k0:k1, h, D:].double()
    return out
