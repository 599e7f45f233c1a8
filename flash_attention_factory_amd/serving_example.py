"""The ragged operators as a server uses them: ``python -m flash_attention_factory_amd.serving_example``.

A small decoder of random weights answers requests of different lengths.  Every step is one ragged batch: running requests bring
the token they have just made, new ones a piece of their prompt.  Each layer makes two calls of the library beside the
plain products -- ``kv_cache_append`` (rotation of queries and keys, keys and values into the pools) and the attention over
the pools (one kernel, or two) -- and the layers differ on purpose: even ones keep int8 pools with a scale per block and attend with
``paged_attention_ragged``, odd ones keep 16-bit pools and attend with ``paged_attention_differential``.
"""
from __future__ import annotations

import time
from typing import List, Sequence

import torch

from . import torch_ops  # noqa: F401  (registers torch.ops.fa_amd)
from .lib.paged_attention_differential import learned_lambda

HIDDEN, HEADS, KV_HEADS, HEAD_SIZE, BLOCK, VOCABULARY = 512, 8, 2, 64, 16, 1000


def angle_table(positions: int, rotary_dim: int, device) -> torch.Tensor:
    """fp32 [positions, rotary_dim]: cosines of a position's angles, then their sines."""
    rate = 10000.0 ** (-torch.arange(0, rotary_dim, 2, device=device) / rotary_dim)
    angles = torch.arange(positions, device=device)[:, None] * rate[None]
    return torch.cat([angles.cos(), angles.sin()], 1).float().contiguous()


class Layer:
    def __init__(self, differential: bool, blocks: int, generator: torch.Generator, dtype: torch.dtype, device):
        def weight(rows, columns):
            return (torch.randn(rows, columns, generator=generator) / rows ** 0.5).to(dtype).to(device)

        self.differential = differential
        self.qkv = weight(HIDDEN, (HEADS + 2 * KV_HEADS) * HEAD_SIZE)
        self.out = weight(HEADS * HEAD_SIZE, HIDDEN)
        pool = (blocks, KV_HEADS, BLOCK, HEAD_SIZE)
        kind = dtype if differential else torch.int8
        self.keys, self.values = (torch.zeros(pool, dtype=kind, device=device).permute(0, 2, 1, 3) for _ in range(2))
        self.k_scales = self.v_scales = None
        if differential:
            vectors = [0.1 * torch.randn(HEAD_SIZE // 2, generator=generator) for _ in range(4)]
            self.lambdas = learned_lambda(*vectors, 0.35, HEADS).to(device)
            self.norm = torch.ones(HEAD_SIZE, device=device)
        else:
            self.k_scales, self.v_scales = (torch.zeros(blocks, KV_HEADS, device=device) for _ in range(2))

    def __call__(self, x, tables, start, lens, table, max_new, max_len):
        rows = torch.nn.functional.rms_norm(x, (HIDDEN,)) @ self.qkv
        heads = rows.view(-1, HEADS + 2 * KV_HEADS, HEAD_SIZE)
        q, k, v = heads.split([HEADS, KV_HEADS, KV_HEADS], 1)
        # halves of a differential row are queries of their own: positions turn neighbouring pairs, which stay within a half
        torch.ops.fa_amd.kv_cache_append(k, v, self.keys, self.values, tables, start, lens, table, q, q, self.k_scales,
                                         self.v_scales, interleaved=self.differential)
        y = torch.empty(x.size(0), HEADS, HEAD_SIZE, dtype=x.dtype, device=x.device)
        if self.differential:
            torch.ops.fa_amd.paged_attention_differential(y, q, self.keys, self.values, tables, start, lens, (HEAD_SIZE // 2) ** -0.5,
                                                          self.lambdas, self.norm, max_new, max_len, out_scale=0.65)
        else:
            torch.ops.fa_amd.paged_attention_ragged(y, q, self.keys, self.values, tables, start, lens, HEAD_SIZE ** -0.5, max_new,
                                                    max_len, k_scales=self.k_scales, v_scales=self.v_scales)
        return x + y.view(-1, HEADS * HEAD_SIZE) @ self.out


class Server:
    def __init__(self, max_requests: int, max_length: int, layers: int = 4, dtype: torch.dtype = torch.bfloat16, seed: int = 0,
                 device: str = "cuda"):
        generator = torch.Generator().manual_seed(seed)
        self.columns = -(-max_length // BLOCK)
        blocks = max_requests * self.columns
        self.device, self.max_length = device, max_length
        self.free = torch.randperm(blocks, generator=generator).tolist()
        self.layers = [Layer(k % 2 == 1, blocks, generator, dtype, device) for k in range(layers)]
        self.embedding = torch.randn(VOCABULARY, HIDDEN, generator=generator).to(dtype).to(device)
        self.angles = angle_table(max_length, HEAD_SIZE, device)

    def step(self, tokens: Sequence[Sequence[int]], tables: Sequence[Sequence[int]], lens: Sequence[int]) -> torch.Tensor:
        """New tokens, block tables and lengths (with the new tokens) of a batch -> hidden rows of all new tokens."""
        counts = [len(t) for t in tokens]
        table = torch.zeros(len(tables), self.columns, dtype=torch.int32)
        for s, blocks in enumerate(tables):
            table[s, :len(blocks)] = torch.tensor(blocks, dtype=torch.int32)
        start = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
        ids = torch.tensor([i for t in tokens for i in t])
        x = self.embedding[ids.to(self.device)]
        batch = (table.to(self.device), start.to(self.device), torch.tensor(lens, dtype=torch.int32).to(self.device))
        for layer in self.layers:
            x = layer(x, *batch, self.angles, max(counts), max(lens))
        return x

    def serve(self, prompts: Sequence[Sequence[int]], answer: int, piece: int = 256) -> List[List[int]]:
        """Greedy answers of ``answer`` tokens; a step takes at most ``piece`` tokens of each prompt."""
        lengths = [len(prompt) + max(answer, 1) - 1 for prompt in prompts]  # tokens in the pools at the end
        if piece < 1 or not all(prompts) or max(lengths, default=0) > self.max_length:
            raise ValueError(f"prompts hold at least one token, with their answers at most {self.max_length}, and a piece one")
        if sum(-(-n // BLOCK) for n in lengths) > len(self.free):
            raise ValueError(f"the requests need more blocks than the {len(self.free)} that are free")
        answers: List[List[int]] = [[] for _ in prompts]
        tables: List[List[int]] = [[] for _ in prompts]
        done = [0] * len(prompts)  # tokens in the pools
        while True:
            batch, tokens = [], []
            for s, prompt in enumerate(prompts):
                if len(answers[s]) < answer:
                    batch.append(s)
                    tokens.append(list(prompt[done[s]:done[s] + piece]) if done[s] < len(prompt) else answers[s][-1:])
            if not batch:
                return answers
            for s, new in zip(batch, tokens):
                done[s] += len(new)
                while len(tables[s]) * BLOCK < done[s]:
                    tables[s].append(self.free.pop())
            x = self.step(tokens, [tables[s] for s in batch], [done[s] for s in batch])
            last = torch.tensor([len(t) for t in tokens]).cumsum(0) - 1
            best = (x[last.to(self.device)] @ self.embedding.t()).argmax(-1).tolist()
            for s, token in zip(batch, best):
                if done[s] >= len(prompts[s]):
                    answers[s].append(token)
                    if len(answers[s]) == answer:
                        self.free.extend(tables[s])
                        tables[s] = []


def main() -> None:
    generator = torch.Generator().manual_seed(1)
    prompts = [torch.randint(VOCABULARY, (n,), generator=generator).tolist() for n in (5, 130, 700, 41, 1500, 16)]
    server = Server(len(prompts), 2048)
    server.serve(prompts, 2)
    torch.cuda.synchronize()
    begin = time.perf_counter()
    answers = server.serve(prompts, 32)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - begin
    tokens = sum(len(p) for p in prompts) + sum(len(a) for a in answers)
    print(f"{len(prompts)} requests, {tokens} tokens in {seconds * 1e3:.1f} ms")
    for prompt, answer in zip(prompts, answers):
        print(f"  {len(prompt):5d} tokens -> {answer[:8]} ...")


if __name__ == "__main__":
    main()
