"""Attention and the paged cache written out in 64 bits and plain loops, with the error
bounds that follow from the kernels' roundings."""
import math

import numpy as np
import torch

# half a unit in the last place, relative: 2^-8 and 2^-11
EPS = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}


def row(q, k, v, scale, eps):
    """One query row: q [d], k and v [n, d] (64 bits) -> out, lse, bounds of both.

    The bound on out: the result is rounded once (eps |out|), each weight is rounded once
    to 16 bits before the product (eps sum p|v| / l; weights below the f16 normal range
    round by at most 2^-25 of the largest), and weights carry the f32 error of their score:
    (d + 4) 2^-24 sum|q k| scale, twice (numerator and denominator), plus a few units of
    2^-22 from exp2 and the sums' n 2^-24. The bound on lse is the score's and the sum's."""
    n, d = k.shape
    if n == 0:
        return np.zeros(v.shape[1]), -math.inf, np.zeros(v.shape[1]), 0.0
    s = k @ q * scale
    m = s.max()
    p = np.exp(s - m)
    l = p.sum()
    out = p @ v / l
    spread = p @ np.abs(v) / l
    ds = (d + 4) * 2.0 ** -24 * (np.abs(k) @ np.abs(q)).max() * scale + np.abs(s).max() * 2.0 ** -22
    rel = ds + 2.0 ** -21 + n * 2.0 ** -24
    bound = 1.02 * eps * (np.abs(out) + spread) + 2 * rel * spread + 2.0 ** -24
    bound += n * 2.0 ** -25 * np.abs(v).max() / l
    return out, m + math.log(l), bound, rel + 2.0 ** -20 * (1 + abs(m))


def to64(t):
    return t.detach().to(torch.float64).cpu().numpy()


def check_rows(got, lse, rows, where):
    """got [.., d] (16-bit tensor) and lse against a list of (index, row(...))."""
    g = to64(got)
    e = None if lse is None else to64(lse)
    for index, (out, ref_lse, bound, lse_bound) in rows:
        err = np.abs(g[index] - out)
        assert np.all(err <= bound), (
            f"{where} row {index}: off by {np.nanmax(err)} at {int(np.nanargmax(err - bound))}, "
            f"allowed {bound[int(np.nanargmax(err - bound))]}")
        if e is not None:
            if math.isinf(ref_lse):
                assert e[index] == ref_lse, f"{where} lse {index}: {e[index]}, not {ref_lse}"
            else:
                assert abs(e[index] - ref_lse) <= lse_bound, (
                    f"{where} lse {index}: {e[index]} and {ref_lse}, allowed {lse_bound}")


class PlainCache:
    """The cache's bookkeeping as the header words it, one sequence and page at a time."""

    def __init__(self, pool, page_tokens, max_sequences, max_pages):
        self.pool, self.P = pool, page_tokens          # numpy [pages][layers][2][heads][P][d]
        self.table = np.full((max_sequences, max_pages), -1, np.int32)
        self.lengths = np.zeros(max_sequences, np.int32)
        self.refs = np.zeros(pool.shape[0], np.int32)

    def pages(self, s):
        return -(-int(self.lengths[s]) // self.P)

    def take(self, count):
        free = np.nonzero(self.refs == 0)[0]
        return None if len(free) < count else list(free[:count])

    def extend(self, seqs, counts):
        need = [-(-int(self.lengths[s] + c) // self.P) - self.pages(s) for s, c in zip(seqs, counts)]
        fresh = self.take(sum(need))
        if fresh is None:
            return False
        for s, c, n in zip(seqs, counts, need):
            for j in range(n):
                page = fresh.pop(0)
                self.table[s, self.pages(s) + j] = page
                self.refs[page] = 1
            self.lengths[s] += c
        return True

    def token(self, s, j):
        return int(self.table[s, j // self.P]), j % self.P

    def write(self, layer, k, v, seqs, offsets):
        for i, s in enumerate(seqs):
            for t in range(offsets[i], offsets[i + 1]):
                page, r = self.token(s, int(self.lengths[s]) - (offsets[i + 1] - t))
                self.pool[page, layer, 0, :, r] = k[t]
                self.pool[page, layer, 1, :, r] = v[t]

    def fork(self, parents, children):
        need = [int(self.lengths[p]) % self.P != 0 for p in parents]
        fresh = self.take(sum(need))
        if fresh is None:
            return False
        for p, c, n in zip(parents, children, need):
            full = int(self.lengths[p]) // self.P
            self.table[c, :full] = self.table[p, :full]
            for page in self.table[p, :full]:
                self.refs[page] += 1
            if n:
                page, used = fresh.pop(0), int(self.lengths[p]) % self.P
                self.pool[page, :, :, :, :used] = self.pool[self.table[p, full], :, :, :, :used]
                self.table[c, full] = page
                self.refs[page] = 1
            self.lengths[c] = self.lengths[p]
        return True

    def compact(self, seqs, keeps):
        stay = []
        for s, keep in zip(seqs, keeps):
            same = 0
            while same < len(keep) and keep[same] == same:
                same += 1
            n = same // self.P
            if same == len(keep):
                n = -(-same // self.P)
                if same % self.P and self.refs[self.table[s, n - 1]] > 1:
                    n -= 1
            stay.append(n)
        need = [-(-len(keep) // self.P) - n for keep, n in zip(keeps, stay)]
        fresh = self.take(sum(need))
        if fresh is None:
            return False
        gone = []
        for s, keep, n, f in zip(seqs, keeps, stay, need):
            new = list(self.table[s, :n])
            for j in range(n * self.P, len(keep)):
                if j % self.P == 0:
                    new.append(fresh.pop(0))
                page, r = self.token(s, keep[j])
                self.pool[new[-1], :, :, :, j % self.P] = self.pool[page, :, :, :, r]
            gone += list(self.table[s, n:self.pages(s)])
            for page in new[n:]:
                self.refs[page] = 1
            self.table[s] = -1
            self.table[s, :len(new)] = new
            self.lengths[s] = len(keep)
        for page in gone:
            self.refs[page] -= 1
        return True

    def free(self, seqs):
        for s in seqs:
            for page in self.table[s, :self.pages(s)]:
                self.refs[page] -= 1
            self.table[s] = -1
            self.lengths[s] = 0
