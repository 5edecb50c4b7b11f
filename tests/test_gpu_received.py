"""Received weight where a row or an entry gives nothing, and how near its sums come."""
import math

import numpy as np
import pytest
import torch

from attention_plain import to64
from diskmule_b200 import CudaContext, DmError, _native as N
from diskmule_b200.attention import attention_status
from paged import Paged, generator, ints, normal
from test_gpu_chunk import run_chunk
from test_gpu_evict import received, run_weights, statistics

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = CudaContext(0)
    yield c
    c.close()


def sums(pool, q, lse, new, rows=None, layer=1, **more):
    w = torch.zeros(pool.table.shape[0], max(pool.lens), device="cuda")
    run_weights(pool, q, lse, new, w, layer=layer, rows=rows, **more)
    attention_status(pool.cache._ctx)
    return w


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new,lens,heads,dim,window,sinks", [
    ([6], [400], 4, 64, 0, 0), ([1, 2], [300, 900], 8, 128, 0, 0), ([128, 40], [700, 500], 8, 64, 0, 0),
    ([128], [700], 8, 128, 200, 4), ([70], [900], 4, 256, 0, 0), ([9, 3], [200, 90], 192, 64, 0, 0)])
def test_rows_without_statistics(ctx, new, lens, heads, dim, window, sinks, value, dtype):
    """A row whose lse is -infinity gives nothing whatever its query holds: padding, say. (192
    heads over 2 are a group that tiles do not take.)"""
    pool = Paged(ctx, dtype, 2, dim, 16, lens)
    q = normal(generator(2), (sum(new), heads, dim), dtype)
    lse = torch.full(q.shape[:2], 6.0, device="cuda")
    lse[::3] = -math.inf
    lse[1:, 1] = -math.inf
    want = sums(pool, q, lse, new, window=window, sinks=sinks)
    assert torch.isfinite(want).all() and want.sum() > 0
    q[lse == -math.inf] = value
    assert torch.equal(sums(pool, q, lse, new, window=window, sinks=sinks), want)


def test_broadcast_rows_without_statistics(ctx):
    """The same on the tiles of queries that no tensor map holds."""
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, [400])
    q = torch.full((1, 8, 64), math.nan, dtype=torch.bfloat16, device="cuda")
    q[:, :5] = normal(generator(2), (1, 5, 64), torch.bfloat16)
    q = q.expand(50, 8, 64)
    lse = torch.full((50, 8), 6.0, device="cuda")
    lse[:, 5:] = -math.inf
    got = sums(pool, q, lse, [50])
    want, bound = received(pool, q.nan_to_num(0.0), lse, [50], 1, 0, 0, 0.125, None)
    assert np.all(np.abs(to64(got) - want) <= bound)


@pytest.mark.parametrize("heads", [4, 130])
@pytest.mark.parametrize("new,rows,counted,status", [
    ([0, 5, 0, 3], [0, 0, 0, 1], {0: (0, 5), 1: (5, 3)}, 0),       # idle places that name a busy row
    ([0, 5, 3], [1, 1, 1], {1: (0, 5)}, N.KV_BAD_SEQUENCE),        # the first one with rows counts
    ([4, 0, 2], [7, 0, 0], {0: (4, 2)}, 0)])
def test_entries_without_rows_take_nobodys_place(ctx, new, rows, counted, status, heads):
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, [300, 200])
    q = normal(generator(3), (sum(new), heads, 64), torch.bfloat16, 2.0)
    lse = statistics(pool, q, new, 1, 0, 0, 0.125, rows)
    got = to64(sums(pool, q, lse, new, rows=rows))
    assert pool.cache.status() == status
    for row in range(2):
        if row not in counted:
            assert np.all(got[row] == 0)
            continue
        at, n = counted[row]
        want, bound = received(pool, q[at:at + n], lse[at:at + n], [n], 1, 0, 0, 0.125, [row])
        assert np.all(np.abs(got[row] - want[row]) <= bound[row])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,heads", [(1, 4), (70, 4), (5, 72)])
def test_exact_products(ctx, rows, heads, dim, dtype):
    """Queries and keys of small integers, whose products and partial sums are exact: what is left
    is the exponent's one rounding (2^-24 of it), the exponential's two units of 2^-23 and four of
    2^-24 for the factors, and the sum's. Nothing in it grows with the score alone."""
    n = 200
    pool = Paged(ctx, dtype, 1, dim, 64, [n], layers=1, seed=1)
    g = generator(3)
    shape = tuple(pool.memory[pool.table[0, :4].long(), 0, 0].shape)
    pool.memory[pool.table[0, :4].long(), 0, 0] = torch.randint(-4, 5, shape, generator=g, device="cuda").to(dtype)
    q = torch.randint(-8, 9, (rows, heads, dim), generator=g, device="cuda").to(dtype)
    lse = statistics(pool, q, [rows], 0, 0, 0, dim ** -0.5, None)
    got = to64(sums(pool, q, lse, [rows], layer=0))[0]
    K, Q, E = pool.tokens(0, 0)[0, 0], to64(q), to64(lse)
    want, bound, terms = np.zeros(n), np.zeros(n), np.zeros(n)
    for t in range(rows):
        seen = n - rows + t + 1
        x = K[:seen] @ Q[t].T * dim ** -0.5 - E[t]
        want[:seen] += np.exp(x).sum(1)
        bound[:seen] += (np.exp(x) * (2.0 ** -22 + (np.abs(x) + 4) * 2.0 ** -24)).sum(1)
        terms[:seen] += heads
    # weights below the smallest normal number are gone
    assert np.all(np.abs(got - want) <= bound + want * terms * 2.0 ** -24 + terms * 2.0 ** -126)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_weights_with_the_statistics_of_chunks(ctx, dim, dtype):
    """With the lse that chunks return a row's weights come to one: both have the same scores. What
    is left is lse's three roundings (sum, logarithm, to nats), 2^-24 of it each at most, and a few
    units (2^-21) of exponentials and sums."""
    new, lens = [300, 200], [700, 900]
    pool = Paged(ctx, dtype, 2, dim, 64, lens, layers=1, seed=dim)
    q = normal(generator(5), (sum(new), 8, dim), dtype, 8.0)
    lse = run_chunk(pool, q, new, layer=0)[1]
    total = to64(sums(pool, q, lse, new, layer=0)).sum()
    each = total / (sum(new) * 8)
    assert abs(each - 1) <= 3 * 2.0 ** -24 * float(lse.abs().mean()) + 2.0 ** -21


def test_too_many_rows(ctx):
    """Rows are counted in 32 bits, up to a whole tile of them: refused before anything is read."""
    pool = Paged(ctx, torch.bfloat16, 1, 64, 16, [300])
    q = normal(generator(1), (1, 1, 64), torch.bfloat16)
    lse, o = torch.zeros(1, device="cuda"), ints([0, 1])
    weights = torch.zeros(1, 304, device="cuda")
    for heads, tokens in ((127, 16909320), (126, 17043521), (72, 1 << 25), (2, 1073741823)):
        with pytest.raises(DmError) as e:
            pool.cache.token_weights(layer=0, heads=heads, q=q.data_ptr(), lse=lse.data_ptr(), offsets=o.data_ptr(),
                                     n=1, tokens=tokens, max_length=300, weights=weights.data_ptr(), weights_stride=304)
        assert e.value.status == N.ERR_OVERFLOW
    assert weights.sum() == 0
