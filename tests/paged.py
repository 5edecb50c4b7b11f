"""A paged cache filled at random, for tests of what reads and writes it."""
import math

import numpy as np
import torch

from attention_plain import to64
from diskmule_b200 import _native as N
from diskmule_b200.attention import KvCache

KIND = {torch.bfloat16: N.BF16, torch.float16: N.F16}


def ints(values):
    return torch.tensor(np.asarray(values, np.int64), dtype=torch.int32, device="cuda")


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


class Paged:
    """Sequences of the lengths `lens` in shuffled pages; whatever no sequence holds is NaN."""

    def __init__(self, ctx, dtype, kv, dim, page, lens, layers=2, seed=0, spare=3, rows=0, max_pages=0):
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        order = np.random.RandomState(seed).permutation(pages)
        rows = rows or len(lens)
        table = np.full((rows, max_pages or max(need + [1]) + 1), -1)
        references = np.zeros(pages)
        shape = (pages, layers, 2, kv, page, dim)
        self.memory = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        gen, at = generator(seed + 1), 0
        for i, n in enumerate(need):
            ids = order[at:at + n]
            table[i, :n] = ids
            references[ids] = 1
            at += n
            for j, p in enumerate(ids):
                used = min(page, lens[i] - j * page)
                self.memory[p, :, :, :, :used] = normal(gen, (layers, 2, kv, used, dim), dtype)
        self.table, self.references = ints(table), ints(references)
        self.lengths = ints(list(lens) + [0] * (rows - len(lens)))
        self.lens, self.page, self.kv, self.dim, self.layers = list(lens), page, kv, dim, layers
        self.cache = KvCache(ctx, type=KIND[dtype], layers=layers, kv_heads=kv, head_dim=dim,
                             page_tokens=page, pages=pages, max_sequences=rows, max_pages=table.shape[1],
                             memory=self.memory.data_ptr(), page_table=self.table.data_ptr(),
                             lengths=self.lengths.data_ptr(), references=self.references.data_ptr())

    def tokens(self, s, layer):
        """Keys and values of a sequence in 64 bits: [2][kv][tokens][dim]."""
        ids = self.table[s, :-(-self.lens[s] // self.page)].long()
        x = to64(self.memory[ids, layer]).transpose(1, 2, 0, 3, 4)
        return x.reshape(2, self.kv, -1, self.dim)[:, :, :self.lens[s]]

    def at(self, s, j):
        """Page and row of token j."""
        return int(self.table[s, j // self.page]), j % self.page


def seen(p, n, window, sinks):
    """The keys that position p of n tokens sees, as an index array."""
    j = np.arange(max(0, min(n, p + 1)))
    return j[(j > p - window) | (j < sinks)] if window else j
