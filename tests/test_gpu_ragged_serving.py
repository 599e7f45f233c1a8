"""The operators together, as the serving example runs them: a batch of requests in pieces gives what each request gives alone."""
import pytest
import torch

from flash_attention_factory_amd import serving_example as E

pytestmark = pytest.mark.gpu


def _tables(lens):
    at, tables = 0, []
    for n in lens:
        blocks = -(-n // E.BLOCK)
        tables.append(list(range(at, at + blocks)))
        at += blocks
    return tables


# Rounding: bf16 rows carry up to 2^-8 of their size in each of some ten roundings a layer, int8 caches a step of 1/127 of a block's
# largest value (three to four standard deviations), 0.9 % of the rows' size as noise, again for each time that a block's scale
# grew.  Four layers of it stay under a tenth of the rows' norm; a key in the wrong place or a wrong mask changes rows by about their norm.
BOUND = 0.1


def test_pieces_give_what_whole_prompts_give():
    lens = [1, 37, 300, 64, 513]
    generator = torch.Generator().manual_seed(2)
    prompts = [torch.randint(E.VOCABULARY, (n,), generator=generator).tolist() for n in lens]
    tables = _tables(lens)
    whole = E.Server(len(lens), 640).step(prompts, tables, lens)
    server = E.Server(len(lens), 640)
    rows, done = [[] for _ in lens], [0] * len(lens)
    size = 1
    while any(d < n for d, n in zip(done, lens)):  # pieces of 1, 3, 9, .. tokens, requests that are through drop out
        batch = [s for s in range(len(lens)) if done[s] < lens[s]]
        tokens = [prompts[s][done[s]:done[s] + size] for s in batch]
        for s, t in zip(batch, tokens):
            done[s] += len(t)
        x = server.step(tokens, [tables[s] for s in batch], [done[s] for s in batch])
        for s, part in zip(batch, x.split([len(t) for t in tokens])):
            rows[s].append(part)
        size *= 3
    got = torch.cat([torch.cat(r) for r in rows]).double()
    want = whole.double()
    assert not torch.isnan(got).any()
    off = (got - want).norm(dim=-1) / want.norm(dim=-1)
    assert float(off.max()) < BOUND, float(off.max())


def test_a_request_alone_and_among_others():
    generator = torch.Generator().manual_seed(3)
    prompts = [torch.randint(E.VOCABULARY, (n,), generator=generator).tolist() for n in (3, 90, 200)]
    server = E.Server(4, 256)
    blocks = len(server.free)
    answers = server.serve(prompts, 5, piece=64)
    assert [len(a) for a in answers] == [5, 5, 5] and len(server.free) == blocks
    x = server.step([prompts[1]], [list(range(6))], [90])
    first = int((x[-1] @ server.embedding.t()).argmax())
    assert answers[1][0] == first
