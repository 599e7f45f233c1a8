"""Latent attention as a server uses it: its operators together, tall and cut tiles, captured graphs, other streams, large and strided pools."""
import math

import pytest
import torch

from flash_attention_factory_amd import torch_ops  # noqa: F401

import _latent as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.fa_amd
F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


class Case:
    """A batch, its pool and queries on the GPU, and what attention of them is in 64 bits."""

    def __init__(self, dtype, kind, L, H, B, new, old, columns=0, seed=0, size=1.0):
        self.batch = batch = R.Batch(new, old, B, seed=seed)
        self.H, self.L, self.dtype = H, L, dtype
        cache, scales, values = R.pool(batch, L, kind, dtype, seed=seed + 1)
        if columns > batch.tables.size(1):  # a table with room for longer contexts: its other entries name no block
            more = torch.full((len(new), columns - batch.tables.size(1)), 1 << 30, dtype=torch.int32)
            batch.tables = torch.cat([batch.tables, more], 1)
        self.cache, self.scales = cache.to(DEV), None if scales is None else scales.to(DEV)
        self.ql = (size * randn(H, batch.T, L, seed=seed + 2)).to(dtype).to(DEV).transpose(0, 1)
        self.qr = (size * randn(batch.T, H, 192, seed=seed + 3)).to(dtype).to(DEV)[..., 128:]
        self.scale = (L + R.ROPE) ** -0.5
        self.on = batch.on(DEV)
        self.values, self.size = values, size

    def run(self, out=None, longest=None, scales=None):
        out = torch.full((self.batch.T, self.H, self.L), 9.0, dtype=self.dtype, device=DEV) if out is None else out
        ops.paged_attention_latent(out, self.ql, self.qr, self.cache, *self.on, self.scale, max(1, max(self.batch.new)),
                                   max(self.batch.lens) if longest is None else longest, self.scales)
        return out

    def check(self, out):
        want, sizes = R.absorbed(self.batch, self.ql.cpu(), self.qr.cpu(), self.values, self.scale)
        got = out.cpu().double()
        off = (got - want).abs() / R.bound(want, sizes, self.dtype, scores=4.0 * max(1.0, self.size))
        assert not torch.isnan(got).any() and float(off.max()) <= 1.0, f"off by {float(off.max()):.2f} of the bound"


# The table, and so the longest context that the call has to reckon with, decides with the rows how tall tiles are: 16 sequences of 128 rows
# and 32768 keys are work for tiles of 128 rows.
TALL = [(BF16, "16", 512, 128, [1] * 16, [0, 1, 30, 31, 32, 33, 63, 64, 95, 400, 7, 511, 640, 1000, 250, 3]),
        (F16, "16", 256, 70, [2, 1] * 20, [5, 300, 64, 31] * 10),
        (F16, "e4m3", 512, 128, [1] * 16, [0, 1, 30, 31, 32, 33, 63, 64, 95, 400, 7, 511, 640, 1000, 250, 3]),
        (BF16, "e4m3", 256, 128, [3, 1, 2, 4] * 4, [97, 0, 700, 31] * 4),
        (BF16, "e4m3", 512, 64, [4] * 10, [60, 0, 129, 31, 900] * 2),      # equal, two tiles each: side by side
        (F16, "16", 512, 128, [4] * 4, [200, 3, 1100, 64])]                # four


@pytest.mark.parametrize("dtype,kind,L,H,new,old", TALL)
def test_tall_tiles(dtype, kind, L, H, new, old):
    c = Case(dtype, kind, L, H, 64, new, old, columns=1024)
    c.check(c.run(longest=65536))


@pytest.mark.parametrize("kind", ["16", "e4m3"])
def test_tall_tiles_with_moving_references(kind):
    c = Case(BF16, kind, 512, 128, 64, [1] * 16, [900, 41] * 8, columns=1024, size=4.0)
    c.check(c.run(longest=65536))


@pytest.mark.parametrize("kind", ["16", "e4m3"])
@pytest.mark.parametrize("H,new,old", [(128, [3, 7, 1, 16] * 5, [0, 9, 90, 16] * 5), (40, [30, 64, 1], [4, 100, 255]), (64, [64] * 6, [0] * 6)])
def test_whole_tiles_of_short_contexts(kind, H, new, old):
    new, old = list(new), [min(o, 256 - n) for n, o in zip(new, old)]
    c = Case(F16, kind, 512, H, 32, new, old)
    c.check(c.run())


@pytest.mark.parametrize("kind", ["16", "e4m3"])
@pytest.mark.parametrize("H,keys", [(16, 257), (16, 320), (5, 4100), (64, 700), (128, 290), (128, 5000)])
def test_one_sequence_cut_into_pieces(kind, H, keys):
    c = Case(BF16, kind, 512, H, 16, [1], [keys - 1])
    c.check(c.run())


@pytest.mark.parametrize("kind,H", [("16", 16), ("e4m3", 16), ("16", 64), ("e4m3", 64), ("e4m3", 128)])
def test_results_are_the_same_every_time(kind, H):
    c = Case(F16, kind, 512, H, 16, [1, 3, 1, 2, 1], [700, 90, 1500, 31, 400])
    first = c.run()
    for _ in range(5):
        assert torch.equal(c.run(), first)


def test_blocks_that_several_sequences_share():
    """A common beginning: the same blocks in several rows of the table, and twice in one."""
    c = Case(BF16, "16", 512, 16, 16, [1] * 4, [199] * 4)
    tables = c.batch.tables.clone()
    tables[1:, :6] = tables[0, :6]
    tables[2, 6] = tables[2, 0]
    c.batch.tables, c.on = tables, (tables.to(DEV), *c.on[1:])
    c.check(c.run())


@pytest.mark.parametrize("kind", ["16", "e4m3"])
def test_rows_and_blocks_farther_apart_than_they_need(kind):
    for L, H in ((512, 16), (256, 128)):
        c = Case(F16, kind, L, H, 16, [1, 2], [300, 40])
        dense = c.run()
        n, B, W = c.cache.shape
        wide = torch.full((n, B + 1, W + 48), 3.0, dtype=F16 if kind == "16" else torch.float32, device=DEV).to(c.cache.dtype)[:, :B, :W]
        wide.copy_(c.cache)
        c.cache = wide
        assert torch.equal(c.run(), dense)


def test_queries_and_results_in_any_layout():
    c = Case(F16, "16", 512, 20, 16, [1, 5], [300, 40])
    want = c.run()
    T, H, L = want.shape
    both = torch.zeros(T, H, L + R.ROPE, dtype=F16, device=DEV)  # latent and rotated part of a query side by side
    both[..., :L], both[..., L:] = c.ql, c.qr
    c.ql, c.qr = both[..., :L], both[..., L:]
    for shape, turn in (((T, H, L + 8), False), ((H, T, L), True), ((H, T, L + 64), True)):
        out = torch.zeros(shape, dtype=F16, device=DEV)
        out = (out.transpose(0, 1) if turn else out)[..., :L]
        assert torch.equal(c.run(out), want)


@pytest.mark.parametrize("kind", ["16", "e4m3"])
def test_a_pool_of_more_than_four_gib(kind):
    """Offsets past 32 bits: the last blocks of a large pool."""
    L, B, H = 512, 64, 16
    itemsize = 2 if kind == "16" else 1
    blocks = (1 << 32) // (B * (L + R.ROPE) * itemsize) + 40
    cache = torch.empty((blocks, B, L + R.ROPE), dtype=BF16 if kind == "16" else E4M3, device=DEV)
    scales = None if kind == "16" else torch.empty((blocks, B), device=DEV)
    new, old = [2, 1], [150, 700]
    small = Case(BF16, kind, L, H, B, new, old)
    far = small.batch.tables.clone()
    for s, n in enumerate(small.batch.lens):
        for k in range(-(-n // B)):
            block = int(small.batch.tables[s, k])
            far[s, k] = blocks - 1 - block
            cache[blocks - 1 - block] = small.cache[block]
            if scales is not None:
                scales[blocks - 1 - block] = small.scales[block]
    want = small.run()
    d_far = far.to(DEV)
    out = torch.zeros_like(want)
    ops.paged_attention_latent(out, small.ql, small.qr, cache, d_far, *small.on[1:], small.scale, 2, 701, scales)
    assert torch.equal(out, want)
    # new rows there, and read back
    T = sum(new)
    down = randn(T, L + R.ROPE, seed=9, dtype=BF16).to(DEV)
    ops.latent_cache_append(down[:, :L], down[:, L:], cache, d_far, *small.on[1:], scales=scales)
    ops.latent_cache_append(down[:, :L], down[:, L:], small.cache, *small.on, scales=small.scales)
    start = torch.tensor([0, 152, 853], dtype=torch.int32, device=DEV)
    rows = [torch.zeros(853, L + R.ROPE, dtype=BF16, device=DEV) for _ in range(2)]
    ops.latent_cache_gather(rows[0], cache, d_far, start, scales=scales)
    ops.latent_cache_gather(rows[1], small.cache, small.on[0], start, scales=small.scales)
    assert torch.equal(rows[0], rows[1]) and bool((rows[0][151] != 0).any())


# ---- the operators together ----

class Layer:
    """One layer of latent attention: the products around the operators are plain matrix products."""

    def __init__(self, dtype, kind, H, D, L, B, S, columns, interleaved):
        self.H, self.D, self.L, self.B, self.interleaved, self.dtype = H, D, L, B, interleaved, dtype
        self.up_k = (randn(H, D, L, seed=1) / math.sqrt(L)).to(dtype).to(DEV)  # k = up_k c, v = up_v c
        self.up_v = (randn(H, D, L, seed=2) / math.sqrt(L)).to(dtype).to(DEV)
        self.weight = (1.0 + 0.1 * randn(L, seed=3)).to(DEV)
        self.table = R.angle_table(columns * B, R.ROPE).to(DEV)
        blocks = S * columns
        self.cache = torch.zeros(blocks, B, L + R.ROPE, dtype=dtype if kind == "16" else torch.float32, device=DEV)
        self.cache = self.cache if kind == "16" else self.cache.to(E4M3)
        self.scales = None if kind == "16" else torch.ones(blocks, B, device=DEV)
        order = torch.randperm(blocks, generator=torch.Generator().manual_seed(4)).to(torch.int32)
        self.tables = order.view(S, columns).to(DEV)
        self.scale = (D + R.ROPE) ** -0.5

    def append(self, down, query, start, lens):
        ops.latent_cache_append(down[:, :self.L], down[:, self.L:], self.cache, self.tables, start, lens, self.weight, self.table,
                                query[..., self.D:], query[..., self.D:], self.scales, interleaved=self.interleaved)

    def absorbed(self, query, start, lens, most, longest):
        ql = torch.bmm(query[..., :self.D].transpose(0, 1).contiguous(), self.up_k).transpose(0, 1)
        out = torch.empty(self.H, query.size(0), self.L, dtype=self.dtype, device=DEV).transpose(0, 1)
        ops.paged_attention_latent(out, ql, query[..., self.D:], self.cache, self.tables, start, lens, self.scale, most, longest, self.scales)
        return torch.bmm(out.transpose(0, 1), self.up_v.transpose(1, 2).contiguous()).transpose(0, 1)

    def expanded(self, query, start, keys_at, most, longest, N):
        rows = torch.empty(N, self.L + R.ROPE, dtype=self.dtype, device=DEV)
        ops.latent_cache_gather(rows, self.cache, self.tables, keys_at, scales=self.scales)
        up = torch.cat([self.up_k, self.up_v], 1).view(self.H * 2 * self.D, self.L)
        both = (rows[:, :self.L] @ up.t()).view(N, self.H, 2 * self.D)
        out = torch.empty(query.size(0), self.H, self.D, dtype=self.dtype, device=DEV)
        ops.attention_latent_expanded(out, query, both[..., :self.D], rows[:, self.L:], both[..., self.D:], start, keys_at, self.scale, most, longest)
        return out

    def exact(self, down, query, interleaved):
        """One whole sequence in 64 bits: down [n, L + 64], query [n, H, D + 64], before the append."""
        n = down.size(0)
        x = down[:, :self.L].double()
        c = x / torch.sqrt(x.square().mean(1, keepdim=True) + 1e-6) * self.weight.double().cpu()
        angles = self.table[:n].cpu()
        r = R.rotated(down[:, None, self.L:], angles, interleaved)[:, 0]
        qr = R.rotated(query[..., self.D:], angles, interleaved)
        k = torch.einsum("hdl,nl->hnd", self.up_k.double().cpu(), c)
        v = torch.einsum("hdl,nl->hnd", self.up_v.double().cpu(), c)
        s = torch.einsum("nhd,hmd->hnm", query[..., :self.D].double(), k) + torch.einsum("nhr,mr->hnm", qr, r)
        p = R.weights(s * self.scale, torch.arange(n))
        return torch.einsum("hnm,hmd->nhd", p, v), torch.einsum("hnm,hmd->nhd", p, v.abs())


def _starts(counts):
    return torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype,kind,H,D,L,interleaved", [(BF16, "16", 16, 128, 512, False), (F16, "e4m3", 8, 64, 256, True), (BF16, "e4m3", 40, 128, 512, True)])
def test_prompts_pieces_and_single_tokens_of_a_layer(dtype, kind, H, D, L, interleaved):
    """Prompts through the expanded form, further pieces and single tokens through the absorbed form, against each request alone in 64 bits."""
    whole = [90, 33, 200, 1]
    S, columns, B = len(whole), 16, 16
    layer = Layer(dtype, kind, H, D, L, B, S, columns, interleaved)
    downs = [randn(n, L + R.ROPE, seed=10 + s, dtype=dtype) for s, n in enumerate(whole)]
    queries = [randn(n, H, D + R.ROPE, seed=20 + s, dtype=dtype) for s, n in enumerate(whole)]
    got = [[] for _ in whole]
    done = [0] * S
    for step, size in enumerate((30, 1, 1, 40, 1, 200)):  # the first and the fourth as prompts are: expanded
        new = [min(size, n - d) for n, d in zip(whole, done)]
        if not any(new):
            continue
        down = torch.cat([x[d:d + n] for x, d, n in zip(downs, done, new)]).to(DEV)
        query = torch.cat([x[d:d + n] for x, d, n in zip(queries, done, new)]).to(DEV)
        done = [d + n for d, n in zip(done, new)]
        lens, start = torch.tensor(done, dtype=torch.int32, device=DEV), _starts(new)
        layer.append(down, query, start, lens)
        if step in (0, 3):
            out = layer.expanded(query, start, _starts(done), max(new), max(done), sum(done))
        else:
            out = layer.absorbed(query, start, lens, max(new), max(done))
        for s, part in enumerate(out.cpu().split(new)):
            got[s].append(part)
    # Roundings on the way, relative to the rows' size (u: of the type, k: of the cached bytes): latents, queries, their products, weights and
    # results some eight u, cached rows k, which move scores by k / sqrt(dim) times their size of about sqrt(2) and add k to values.
    u, k = R.UNIT[dtype], 2.0 ** -4 if kind == "e4m3" else 0.0
    for s in range(S):
        want, _ = layer.exact(downs[s], queries[s], interleaved)
        off = (torch.cat(got[s]).double() - want).norm(dim=-1) / want.norm(dim=-1)
        assert float(off.max()) <= 8 * u + 2 * k, (s, float(off.max()))


def _replays(make, n=4):
    """make(step) fills the inputs in place and gives the call; the call is captured once and replayed with every step's inputs."""
    call, fill, result = make()
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph, call, fill, result


def test_captured_steps():
    """A decode step (append, then attention) and a prompt step in two graphs, replayed in turns with eager work between them."""
    H, D, L, B, S, columns = 16, 128, 512, 16, 5, 40

    def decode():
        layer = Layer(BF16, "e4m3", H, D, L, B, S, columns, True)
        layer.cache.copy_(randn(S * columns, B, L + R.ROPE, seed=7).to(DEV).to(E4M3))
        down, query = torch.empty(S, L + R.ROPE, dtype=BF16, device=DEV), torch.empty(S, H, D + R.ROPE, dtype=BF16, device=DEV)
        lens, start = torch.empty(S, dtype=torch.int32, device=DEV), _starts([1] * S)
        out = torch.empty(S, H, D, dtype=BF16, device=DEV)

        def call():
            q = query.clone()
            layer.append(down, q, start, lens)
            out.copy_(layer.absorbed(q, start, lens, 1, columns * B))

        def fill(step):
            down.copy_(randn(*down.shape, seed=100 + step, dtype=BF16))
            query.copy_(randn(*query.shape, seed=200 + step, dtype=BF16))
            lens.copy_(torch.tensor([1 + step, 300 + step, 17, 600 + step, 64 + step], dtype=torch.int32))
        return call, fill, out

    def prompt():
        n, N = 70, 5 * 70
        query, both = torch.empty(N, H, D + R.ROPE, dtype=F16, device=DEV), torch.empty(N, H, 2 * D, dtype=F16, device=DEV)
        rope, out, start = torch.empty(N, R.ROPE, dtype=F16, device=DEV), torch.empty(N, H, D, dtype=F16, device=DEV), _starts([n] * 5)

        def call():
            ops.attention_latent_expanded(out, query, both[..., :D], rope, both[..., D:], start, start, 0.07, n, n)

        def fill(step):
            for k, x in enumerate((query, both, rope)):
                x.copy_(randn(*x.shape, seed=300 + 10 * step + k, dtype=F16))
        return call, fill, out

    graphs = [_replays(decode), _replays(prompt)]
    for step in range(5):
        for graph, _, fill, out in graphs:
            fill(step)
            graph.replay()
        got = [out.clone() for *_, out in graphs]
        torch.cuda.synchronize()
        for k, (_, call, fill, out) in enumerate(graphs):
            out.fill_(7.0)
            call()
            assert torch.equal(out, got[k]), (step, k)


def test_calls_on_two_streams():
    """Two calls at once, each with its own workspace."""
    cases = [Case(F16, "e4m3", 512, 16, 16, [1] * 8, [900 + 31 * k for k in range(8)], seed=5), Case(BF16, "16", 512, 64, 16, [1] * 8, [700 + 29 * k for k in range(8)], seed=9)]
    want = [c.run() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[] for _ in cases]
    for _ in range(10):
        for k, c in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                outs[k].append(c.run())
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o, want[k]) for o in outs[k])
