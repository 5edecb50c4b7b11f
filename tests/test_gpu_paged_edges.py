"""Chunks, rotation, received weight and eviction at their edges: waits that run out, offsets
beyond 32 bits, bounds of zero, layouts that no tensor map holds, runs of all of them together."""
import math

import numpy as np
import pytest
import torch

from attention_plain import EPS, to64
from diskmule_b200 import CudaContext, DmError, _native as N
from diskmule_b200.attention import KvCache, Rope, attention_status, offsets, rotate
from paged import KIND, Paged, generator, ints, normal
from test_gpu_chunk import check_chunk, run_chunk
from test_gpu_evict import received, run_weights, statistics

pytestmark = pytest.mark.gpu

LIMITS = [1, 500, 2000, 8000, 30000]


@pytest.fixture(scope="module")
def ctx():
    c = CudaContext(0)
    yield c
    c.close()


def out_of_time(ctx, run, want):
    """Calls whose waits may run out: reported, and the next call is right again."""
    late = 0
    try:
        for limit in LIMITS:
            N.check(N.lib().dm_selftest_attention_wait(ctx.handle, limit))
            got = run()
            try:
                attention_status(ctx)
            except DmError as e:
                assert e.status == N.ERR_TIMEOUT
                late += 1
            else:
                assert all(torch.equal(a, b) for a, b in zip(got, want))
            N.check(N.lib().dm_selftest_attention_wait(ctx.handle, 0))
            assert all(torch.equal(a, b) for a, b in zip(run(), want))
            attention_status(ctx)
    finally:
        N.check(N.lib().dm_selftest_attention_wait(ctx.handle, 0))
    return late


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,lens", [([1, 3], [900, 4000]), ([300, 1, 900], [2500, 3000, 900]), ([1] * 40, [1500] * 40)])
def test_chunk_out_of_time(ctx, dim, new, lens):
    pool = Paged(ctx, torch.bfloat16, 2, dim, 16, lens, layers=2)
    q = normal(generator(dim), (sum(new), 8, dim), torch.bfloat16, 2.0)
    run = lambda: run_chunk(pool, q, new)
    want = run()
    out_of_time(ctx, run, want)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,lens", [([1, 1], [900, 4000]), ([100, 7], [2500, 300]), ([12] * 20, [700] * 20)])
@pytest.mark.parametrize("broadcast", [False, True])
def test_weights_out_of_time(ctx, dim, new, lens, broadcast):
    pool = Paged(ctx, torch.float16, 2, dim, 16, lens, layers=2)
    q = normal(generator(dim), (sum(new), 8, dim), torch.float16, 2.0)
    if broadcast:  # blocks without tensor memory
        q = q[:1].expand(sum(new), 8, dim)
    lse = torch.full((sum(new), 8), 9.0, device="cuda")

    def run():
        weights = torch.zeros(len(lens), max(lens), device="cuda")
        run_weights(pool, q, lse, new, weights)
        return (weights,)

    out_of_time(ctx, run, run())


def test_bounds_of_zero(ctx):
    """max_length 0: sequences have no tokens. Rows of zeros and -infinity, nothing received."""
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, [100, 50])
    q = normal(generator(1), (5, 4, 64), torch.bfloat16)
    out, lse = run_chunk(pool, q, [3, 2], max_length=0)
    assert (out == 0).all() and (lse == -math.inf).all()
    weights = torch.zeros(2, 112, device="cuda")
    run_weights(pool, q, lse, [3, 2], weights, max_length=0)
    assert weights.abs().sum() == 0
    empty = Paged(ctx, torch.bfloat16, 2, 64, 16, [0, 0])
    out, lse = run_chunk(empty, q, [3, 2])
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("new,lens,heads,kv,dim", [([30], [700], 4, 2, 64), ([5, 70], [300, 90], 6, 2, 128),
                                                   ([9], [500], 4, 1, 256), ([3], [200], 72, 1, 64)])
def test_weights_of_broadcast_queries_and_wide_groups(ctx, new, lens, heads, kv, dim):
    pool = Paged(ctx, torch.bfloat16, kv, dim, 16, lens)
    q = normal(generator(2), (1 if heads < 70 else sum(new), heads, dim), torch.bfloat16, 2.0).expand(sum(new), heads, dim)
    lse = statistics(pool, q, new, 1, 0, 0, dim ** -0.5, None)
    weights = torch.zeros(len(lens), max(lens), device="cuda")
    run_weights(pool, q, lse, new, weights)
    want, bound = received(pool, q, lse, new, 1, 0, 0, dim ** -0.5, None)
    assert np.all(np.abs(to64(weights) - want) <= bound)


class Far:
    """A pool of more than 2^32 bytes and 2^31 values, used at its far end only."""

    def __init__(self, ctx, lens, kv=2, dim=128, page=64, layers=2):
        page_bytes = layers * 2 * kv * page * dim * 2
        pages = (1 << 32) // page_bytes + 500
        self.memory = torch.empty(pages * page_bytes // 2, dtype=torch.bfloat16, device="cuda").view(pages, layers, 2, kv, page, dim)
        need = [-(-n // page) for n in lens]
        table, at = np.full((len(lens), max(need) + 1), -1), pages
        for i, n in enumerate(need):
            at -= n
            table[i, :n] = np.arange(at, at + n)
        self.memory[at:].normal_(generator=generator(1))
        self.table, self.lengths = ints(table), ints(lens)
        self.references = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.references[:at - 40] = 1
        self.references[at:] = 1
        self.lens, self.page, self.kv, self.dim, self.layers = lens, page, kv, dim, layers
        self.cache = KvCache(ctx, type=N.BF16, layers=layers, kv_heads=kv, head_dim=dim, page_tokens=page, pages=pages,
                             max_sequences=len(lens), max_pages=table.shape[1], memory=self.memory.data_ptr(),
                             page_table=self.table.data_ptr(), lengths=self.lengths.data_ptr(),
                             references=self.references.data_ptr())

    tokens = Paged.tokens
    at = Paged.at


def test_pools_beyond_32_bits(ctx):
    pool = Far(ctx, [500, 1300])
    for new in ([1, 3], [200, 70]):
        q = normal(generator(3), (sum(new), 4, 128), torch.bfloat16, 2.0)
        out, lse = run_chunk(pool, q, new)
        check_chunk(pool, q, new, out, lse, some=4)
        weights = torch.zeros(2, 1344, device="cuda")
        run_weights(pool, q, lse, new, weights)
        want, bound = received(pool, q, lse, new, 1, 0, 0, 128 ** -0.5, None)
        assert np.all(np.abs(to64(weights)[:, :1300] - want) <= bound)
    k = normal(generator(4), (5, 4, 128), torch.bfloat16)
    off = ints([0, 2, 5])
    rotate(ctx, None, type=N.BF16, kv_heads=2, head_dim=128, tokens=5, k=k.data_ptr(), v=k[:, 2:].data_ptr(),
           k_stride=(512, 128), v_stride=(512, 128), cache=pool.cache, layer=1, offsets=off.data_ptr(), n=2)
    for s, t, j in ((0, 0, 498), (0, 1, 499), (1, 2, 1297), (1, 4, 1299)):
        page, r = pool.at(s, j)
        assert torch.equal(pool.memory[page, 1, 0, :, r], k[t, :2]) and torch.equal(pool.memory[page, 1, 1, :, r], k[t, 2:])
    before = pool.tokens(1, 0)
    rows, keep, at = ints([1]), ints([0] * 400), ints([0, 0])
    w = weights[1].cpu().numpy().copy()
    pool.cache.evict(sequences=rows.data_ptr(), n=1, budget=400, sinks=4, recent=50, weights=weights.data_ptr(),
                     weights_stride=1344, keep_offsets=at.data_ptr(), keep=keep.data_ptr())
    assert pool.cache.status() == 0 and int(pool.lengths[1]) == 400
    pool.lens = [500, 400]
    stays = keep.cpu().numpy()
    assert np.array_equal(pool.tokens(1, 0), before[:, :, stays])
    assert np.array_equal(weights[1, :400].cpu().numpy(), w[stays]) and weights[1, 400:1300].abs().sum() == 0


def test_a_long_chat(ctx):
    """All of it as a serving loop runs it: pieces of a prompt are rotated into the cache, attended and
    weighed, the sequence is cut down, and tokens go on at their own positions. Against one pass in
    64 bits over the tokens that are there."""
    heads, kv, dim, total, budget = 8, 2, 64, 900, 300
    g = generator(7)
    qkv = normal(g, (total + 8, heads + 2 * kv, dim), torch.bfloat16, 1.5)
    cache_rows = 3
    pool = Paged(ctx, torch.bfloat16, kv, dim, 16, [0], layers=1, rows=cache_rows, spare=200, max_pages=70)
    rope = Rope(ctx, dim, theta=1e4)
    weights = torch.zeros(cache_rows, 70 * 16, device="cuda")
    row, st = ints([1]), (qkv.stride(0), qkv.stride(1))
    outs, lses, qs = [], [], []

    def feed(a, b, length):
        n = b - a
        x, off, count = qkv[a:b], ints([0, n]), ints([n])
        pool.cache.extend(row.data_ptr(), count.data_ptr(), 1)
        q = torch.empty(n, heads, dim, dtype=torch.bfloat16, device="cuda")
        p = ints([list(range(a, b))])
        rotate(ctx, rope, type=N.BF16, heads=heads, kv_heads=kv, head_dim=dim, tokens=n, q=x.data_ptr(),
               k=x[:, heads:].data_ptr(), v=x[:, heads + kv:].data_ptr(), q_stride=st, k_stride=st, v_stride=st,
               q_out=q.data_ptr(), cache=pool.cache, layer=0, sequences=row.data_ptr(), offsets=off.data_ptr(), n=1,
               positions=p.data_ptr(), norm_q=True, norm_k=True)
        out, lse = torch.empty_like(q), torch.empty(n, heads, device="cuda")
        need = pool.cache.chunk_workspace(heads, 1, n, length + n)
        work = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
        pool.cache.chunk_attention(layer=0, heads=heads, q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
                                   sequences=row.data_ptr(), offsets=off.data_ptr(), n=1, tokens=n, max_length=length + n,
                                   workspace=work.data_ptr(), workspace_bytes=need)
        pool.cache.token_weights(layer=0, heads=heads, q=q.data_ptr(), lse=lse.data_ptr(), sequences=row.data_ptr(),
                                 offsets=off.data_ptr(), n=1, tokens=n, max_length=length + n, weights=weights.data_ptr(),
                                 weights_stride=weights.stride(0))
        return q, out, lse

    at = 0
    for piece in (400, 1, 299, 200):
        q, out, lse = feed(at, at + piece, at)
        at += piece
        qs.append(q), outs.append(out), lses.append(lse)
    torch.cuda.synchronize()
    pool.lens = [0, total, 0]
    q, out, lse = torch.cat(qs), torch.cat(outs), torch.cat(lses)
    check_chunk(pool, q, [total], out, lse, layer=0, rows=[1])
    want, bound = received(pool, q, lse, [total], 0, 0, 0, dim ** -0.5, [1])
    assert np.all(np.abs(to64(weights)[1, :total] - want[1]) <= bound[1] + 2.0 ** -22 * want[1])
    # half of it goes; the rest stays as it was
    before, w = pool.tokens(1, 0), weights[1].cpu().numpy().copy()
    keep, off = ints([0] * budget), ints([0, 0])
    pool.cache.evict(sequences=row.data_ptr(), n=1, budget=budget, sinks=4, recent=64, weights=weights.data_ptr(),
                     weights_stride=weights.stride(0), keep_offsets=off.data_ptr(), keep=keep.data_ptr())
    torch.cuda.synchronize()
    pool.lens = [0, budget, 0]
    stays = keep.cpu().numpy()
    assert np.array_equal(stays[:4], np.arange(4)) and np.array_equal(stays[-64:], np.arange(total - 64, total))
    middle = np.setdiff1d(np.arange(4, total - 64), stays)
    assert w[stays[4:-64]].min() >= w[middle].max()
    assert np.array_equal(pool.tokens(1, 0), before[:, :, stays])
    # and a draft of eight goes on at position `total`
    q, out, lse = feed(total, total + 8, budget)
    torch.cuda.synchronize()
    pool.lens = [0, budget + 8, 0]
    check_chunk(pool, q, [8], out, lse, layer=0, rows=[1])
    assert pool.cache.status() == 0


def test_captured_weights_and_eviction(ctx):
    """Clusters in a graph: replayed after lengths, offsets and sums have changed, as direct calls."""
    lens = [3000, 20000]
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, lens, layers=1, spare=1400, max_pages=1300)
    q = normal(generator(2), (40, 8, 64), torch.bfloat16, 2.0)
    lse = torch.full((40, 8), 12.0, device="cuda")
    weights = torch.zeros(2, 1300 * 16, device="cuda")
    o, rows, side = ints([0, 1, 40]), ints([0, 1]), torch.cuda.Stream()
    keep, off = ints([0] * 2 * 2500), ints([0] * 3)

    def calls(stream):
        pool.cache.token_weights(layer=0, heads=8, q=q.data_ptr(), lse=lse.data_ptr(), offsets=o.data_ptr(), n=2, tokens=40,
                                 max_length=20800, weights=weights.data_ptr(), weights_stride=weights.stride(0), stream=stream)
        pool.cache.evict(sequences=rows.data_ptr(), n=2, budget=2500, sinks=4, recent=64, weights=weights.data_ptr(),
                         weights_stride=weights.stride(0), keep_offsets=off.data_ptr(), keep=keep.data_ptr(), stream=stream)

    start = [t.clone() for t in (pool.memory, pool.table, pool.lengths, pool.references)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        calls(side.cuda_stream)
    for new, shorter in (([1, 39], 0), ([0, 3], 11), ([40, 0], 700)):
        got = []
        for run in (g.replay, lambda: calls(0)):
            for t, s in zip((pool.memory, pool.table, pool.lengths, pool.references), start):
                t.copy_(s)
            pool.lengths.sub_(shorter)
            o.copy_(ints(offsets(new)))
            weights.copy_(torch.rand(weights.shape, generator=generator(5), device="cuda"))
            keep.zero_()
            run()
            torch.cuda.synchronize()
            got.append([t.clone().view(torch.int16) if t.dtype == torch.bfloat16 else t.clone()
                        for t in (pool.memory, pool.table, pool.lengths, pool.references, weights, keep, off)])
        assert pool.cache.status() == 0
        for a, b in zip(*got):
            assert torch.equal(a, b)
        assert got[0][2].tolist() == [min(2500, n - shorter) for n in lens]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [31, 33, 2500])
def test_many_entries(ctx, dim, n):
    """Entries without rows between a few with many: items and tokens are found behind all of them."""
    some = {0: 1, 7: 150, n // 2: 3, n - 2: 70, n - 1: 1}
    new, lens = [some.get(i, 0) for i in range(n)], [some.get(i, 0) + 90 if i in some or i < 20 else 0 for i in range(n)]
    pool = Paged(ctx, torch.bfloat16, 2, dim, 16, lens)
    q = normal(generator(n), (sum(new), 4, dim), torch.bfloat16, 2.0)
    for window, sinks in ((0, 0), (40, 3)):
        out, lse = run_chunk(pool, q, new, window=window, sinks=sinks)
        check_chunk(pool, q, new, out, lse, window=window, sinks=sinks)
    out, lse = run_chunk(pool, q, new)
    weights = torch.zeros(n, max(lens), device="cuda")
    run_weights(pool, q, lse, new, weights)
    want, bound = received(pool, q, lse, new, 1, 0, 0, dim ** -0.5, None)
    assert np.all(np.abs(to64(weights) - want) <= bound)


@pytest.mark.parametrize("dtype,value", [(torch.bfloat16, float("inf")), (torch.float16, float("nan"))])
@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 4)])
def test_hidden_values_of_wide_heads(ctx, dtype, value, dim, window, sinks):
    """Tokens that are not finite, hidden from some rows by the order of tokens or by the window: rows
    that do not see them are what they are without, also where several hundred rows do see them."""
    n, a = 1500, 700
    pool = Paged(ctx, dtype, 1, dim, 64, [n])
    q = normal(generator(2), (a, 4, dim), dtype, 2.0)
    before, lse0 = run_chunk(pool, q, [a], window=window, sinks=sinks)
    check_chunk(pool, q, [a], before, lse0, window=window, sinks=sinks)
    hit = 1150  # of position 350 among the rows
    page, r = pool.at(0, hit)
    pool.memory[page, 1, :, :, r] = value
    out, lse = run_chunk(pool, q, [a], window=window, sinks=sinks)
    sees = np.zeros(a, bool)
    sees[hit - (n - a):(hit - (n - a) + window if window else a)] = True
    free = torch.tensor(~sees, device="cuda")
    assert torch.equal(out[free], before[free]) and torch.equal(lse[free], lse0[free])
    pool.memory[page, 1, 0, :, r] = 0
    pool.memory[page, 1, 1, :, r] = 0
    pool.memory[page, 1, 1, 0, r, dim - 3] = value
    out, _ = run_chunk(pool, q, [a], window=window, sinks=sinks)
    assert not torch.isfinite(out[~free, :, dim - 3]).any()
    out[~free, :, dim - 3] = 0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype,value", [(torch.bfloat16, float("nan")), (torch.float16, float("inf"))])
@pytest.mark.parametrize("dim,kv,heads", [(64, 8, 32), (128, 8, 32), (96, 4, 20)])
@pytest.mark.parametrize("n,window,sinks", [(700, 0, 0), (700, 200, 6), (91, 0, 0), (1501, 1000, 0)])
def test_hidden_values_of_many_short_entries(ctx, dtype, value, dim, kv, heads, n, window, sinks):
    """The same for entries of few rows, in the first and the last tiles that some of them see."""
    a, count, which = 30, 12, 5
    pool = Paged(ctx, dtype, kv, dim, 16, [n] * count)
    q = normal(generator(2), (a * count, heads, dim), dtype, 2.0)
    before, lse0 = run_chunk(pool, q, [a] * count, window=window, sinks=sinks)
    check_chunk(pool, q, [a] * count, before, lse0, window=window, sinks=sinks, some=4)
    first = n - a  # position of the entry's first row
    for hit in (n - 10, first - window + 12 if window else n - 1):
        page, r = pool.at(which, hit)
        kept = pool.memory[page, 1, :, :, r].clone()
        pool.memory[page, 1, :, :, r] = value
        out, lse = run_chunk(pool, q, [a] * count, window=window, sinks=sinks)
        sees = np.zeros((count, a), bool)
        for t in range(a):
            sees[which, t] = hit <= first + t and (not window or hit > first + t - window or hit < sinks)
        assert 0 < sees.sum() < a
        sees = torch.tensor(sees.reshape(-1), device="cuda")
        assert torch.equal(out[~sees], before[~sees]) and torch.equal(lse[~sees], lse0[~sees])
        pool.memory[page, 1, 0, :, r] = 0
        pool.memory[page, 1, 1, :, r] = 0
        pool.memory[page, 1, 1, 0, r, dim - 3] = value
        out, _ = run_chunk(pool, q, [a] * count, window=window, sinks=sinks)
        group = heads // kv
        assert not torch.isfinite(out[sees, :group, dim - 3]).any()
        out[sees, :group, dim - 3] = 0
        assert torch.isfinite(out).all()
        pool.memory[page, 1, :, :, r] = kept


def test_rising_and_falling_scores_of_short_entries(ctx):
    """Scores that rise or fall from key to key, so that halves of a row's tiles differ by powers of two."""
    n, a, count = 1000, 20, 16
    for dim in (64, 128):
        pool = Paged(ctx, torch.bfloat16, 4, dim, 16, [n] * count)
        for s in range(count):
            ids = pool.table[s, :-(-n // 16)].long()
            x = torch.zeros(len(ids) * 16, device="cuda")
            x[:n] = torch.arange(n, device="cuda") / 8
            pool.memory[ids, 1, 0] = 0
            pool.memory[ids, 1, 0, :, :, 0] = x.view(-1, 1, 16).to(torch.bfloat16).expand(-1, 4, 16)
        q = torch.zeros(a * count, 16, dim, dtype=torch.bfloat16, device="cuda")
        q[:, 0::2, 0], q[:, 1::2, 0] = 8.0, -8.0
        out, lse = run_chunk(pool, q, [a] * count)
        check_chunk(pool, q, [a] * count, out, lse, some=3)
