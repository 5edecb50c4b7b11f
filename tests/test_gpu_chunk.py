"""dm_attention_chunk against attention written out in 64 bits."""
import math

import numpy as np
import pytest
import torch

from attention_plain import EPS, check_rows, row, to64
from diskmule_b200 import CudaContext, DmError, _native as N
from diskmule_b200.attention import attention_status, offsets
from paged import KIND, Paged, generator, ints, normal, seen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = CudaContext(0)
    yield c
    c.close()


def run_chunk(pool, q, new, layer=1, window=0, sinks=0, rows=None, scale=0.0, tokens=None, max_length=None,
              out=None, lse=True, offset=None, stream=0):
    """out and lse start as NaN."""
    heads = q.shape[1]
    out = torch.full_like(q, float("nan")) if out is None else out
    e = torch.full(q.shape[:2], float("nan"), device="cuda") if lse else None
    o = ints(offsets(new) if offset is None else offset)
    r = None if rows is None else ints(rows)
    tokens = q.shape[0] if tokens is None else tokens
    max_length = max(pool.lens + [1]) if max_length is None else max_length
    need = pool.cache.chunk_workspace(heads, len(new), tokens, max_length, window=window, sinks=sinks)
    work = torch.full((max(16, need) // 4 + 4,), float("nan"), device="cuda")
    pool.cache.chunk_attention(layer=layer, heads=heads, q=q.data_ptr(), out=out.data_ptr(),
                               lse=e.data_ptr() if lse else 0, sequences=r.data_ptr() if r is not None else 0,
                               offsets=o.data_ptr(), n=len(new), tokens=tokens, max_length=max_length,
                               window=window, sinks=sinks, scale=scale, q_stride=(q.stride(0), q.stride(1)),
                               out_stride=(out.stride(0), out.stride(1)), workspace=work.data_ptr(),
                               workspace_bytes=need, stream=stream)
    torch.cuda.synchronize()
    return out, e


def check_chunk(pool, q, new, out, lse, layer=1, window=0, sinks=0, rows=None, scale=0.0, some=12, bits=0):
    heads = q.shape[1]
    g = heads // pool.kv
    scale = scale or 1.0 / math.sqrt(q.shape[2])
    Q, want, at = to64(q), [], 0
    for i, a in enumerate(new):
        s = i if rows is None else rows[i]
        n = pool.lens[s] if 0 <= s < len(pool.lens) else 0
        kv = pool.tokens(s, layer) if n else np.zeros((2, pool.kv, 0, q.shape[2]))
        tokens = range(a) if a <= some else sorted(
            {0, 1, a - 1, a // 2} | {int(x) for x in np.random.RandomState(a + n).randint(0, a, some)})
        for t in tokens:
            keys = seen(n - a + t, n, window, sinks)
            for h in range(heads):
                want.append(((at + t, h), row(Q[at + t, h], kv[0, h // g, keys], kv[1, h // g, keys], scale,
                                              EPS[q.dtype])))
        at += a
    check_rows(out, lse, want, "chunk")
    assert torch.isnan(out[at:]).all()  # rows behind the last entry
    attention_status(pool.cache._ctx)
    assert pool.cache.status() == bits


CHUNKS = [
    # new tokens, tokens with them, heads, kv heads, dim, page, window, sinks
    ([1], [1], 1, 1, 64, 16, 0, 0),
    ([1, 1, 1], [7, 300, 64], 8, 2, 64, 16, 0, 0),
    ([5, 3, 6, 5], [305, 80, 647, 905], 8, 2, 64, 16, 0, 0),
    ([1], [9000], 32, 8, 128, 64, 0, 0),                     # a long axis cut in parts
    ([2], [3001], 2, 1, 256, 32, 0, 0),
    ([40, 0, 1, 0, 17], [40, 50, 333, 0, 90], 6, 2, 80, 16, 0, 0),  # a prompt; entries without rows
    ([9, 30], [5, 0], 4, 2, 128, 16, 0, 0),                  # more rows than tokens
    ([200], [900], 7, 1, 96, 128, 0, 0),
    ([513], [2000], 4, 4, 128, 64, 0, 0),
    ([300, 1, 129, 1], [4000, 2500, 129, 77], 16, 2, 128, 32, 0, 0),
    ([257], [700], 2, 1, 256, 16, 0, 0),
    ([20], [300], 128, 1, 64, 16, 0, 0),                     # the widest group
    ([1, 33], [700, 60], 2, 2, 8, 16, 0, 0),
    # windows, sinks
    ([1, 1], [4000, 90], 8, 2, 128, 16, 100, 4),
    ([64, 1, 300], [500, 3000, 300], 8, 2, 64, 32, 128, 1),
    ([300], [2500], 4, 1, 256, 16, 200, 0),
    ([300], [2500], 4, 1, 256, 16, 200, 40),
    ([150, 150], [1000, 150], 5, 1, 128, 16, 1, 0),          # a token sees itself
    ([150, 9], [1000, 40], 4, 2, 128, 64, 33, 500),          # more sinks than a sequence has tokens
    ([700], [5000], 2, 2, 128, 16, 1000, 81),                # sinks that end inside a tile
    ([260], [3000], 8, 4, 80, 16, 77, 17),
    ([40], [2000], 4, 2, 64, 16, 1990, 12),                  # the window almost reaches the sinks
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,lens,heads,kv,dim,page,window,sinks", CHUNKS)
def test_chunk(ctx, new, lens, heads, kv, dim, page, window, sinks, dtype):
    pool = Paged(ctx, dtype, kv, dim, page, lens, seed=sum(lens))
    q = normal(generator(3), (sum(new) + 2, heads, dim), dtype, 2.0)
    out, lse = run_chunk(pool, q, new, window=window, sinks=sinks)
    check_chunk(pool, q, new, out, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("new,lens,heads,kv,dim,window,sinks", [
    ([1024], [12000], 16, 2, 128, 0, 0), ([3000, 700], [3000, 9000], 8, 1, 64, 0, 0),
    ([1500], [6000], 4, 1, 256, 700, 9), ([2001] + [1] * 20, [4001] + [100 + 97 * i for i in range(20)], 32, 8, 128, 0, 0),
    ([64] * 40, [64 + 60 * i for i in range(40)], 16, 4, 128, 500, 4)])
def test_chunk_long(ctx, new, lens, heads, kv, dim, window, sinks):
    pool = Paged(ctx, torch.bfloat16, kv, dim, 64, lens, layers=1, seed=5)
    q = normal(generator(4), (sum(new), heads, dim), torch.bfloat16, 2.0)
    out, lse = run_chunk(pool, q, new, layer=0, window=window, sinks=sinks)
    check_chunk(pool, q, new, out, lse, layer=0, window=window, sinks=sinks, some=4)


@pytest.mark.parametrize("new,lens", [([1, 5, 2], [300, 80, 1700]), ([140, 3], [1000, 333])])
def test_strides_rows_scale_and_bounds(ctx, new, lens):
    """Queries out of a fused projection, outputs with gaps, entries in another order and one
    twice, bounds above what there is, no lse."""
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, lens, rows=6, seed=8)
    n = sum(new) + new[0]
    fused = normal(generator(9), (n + 5, 12, 64), torch.bfloat16, 2.0)
    q = fused[:, 2:10]
    out = torch.full((n + 5, 8, 72), float("nan"), dtype=torch.bfloat16, device="cuda")[..., :64]
    order = list(range(len(lens)))[::-1] + [len(lens) - 1]
    chunks = [new[i] for i in order[:-1]] + [new[0]]
    assert sum(chunks) == n
    out, lse = run_chunk(pool, q, chunks, rows=order, scale=0.3, out=out, max_length=10 ** 6)
    check_chunk(pool, q, chunks, out, lse, rows=order, scale=0.3)
    again = torch.full_like(out, float("nan"))
    run_chunk(pool, q, chunks, rows=order, scale=0.3, out=again, lse=False, max_length=10 ** 6)
    assert torch.equal(out.nan_to_num(7.0), again.nan_to_num(7.0))


def test_heads_first_queries(ctx):
    """[heads, tokens, dim] tensors seen as [tokens, heads, dim]."""
    new, lens = [130, 7], [400, 900]
    pool = Paged(ctx, torch.float16, 2, 128, 32, lens)
    q = normal(generator(2), (8, 137, 128), torch.float16, 2.0).transpose(0, 1)
    out = torch.full((8, 137, 128), float("nan"), dtype=torch.float16, device="cuda").transpose(0, 1)
    out, lse = run_chunk(pool, q, new, out=out)
    check_chunk(pool, q, new, out, lse)


def test_broadcast_queries(ctx):
    """One query for all rows and heads: strides of zero."""
    new, lens = [150], [700]
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, lens)
    q = normal(generator(2), (1, 1, 64), torch.bfloat16).expand(150, 4, 64)
    out = torch.full((150, 4, 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    e = torch.empty(150, 4, device="cuda")
    o = ints(offsets(new))
    need = pool.cache.chunk_workspace(4, 1, 150, 700)
    work = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    # a stride of zero along one axis; along both it would mean contiguous
    q2 = normal(generator(2), (1, 4, 64), torch.bfloat16).expand(150, 4, 64)
    pool.cache.chunk_attention(layer=1, heads=4, q=q2.data_ptr(), out=out.data_ptr(), lse=e.data_ptr(),
                               offsets=o.data_ptr(), n=1, tokens=150, max_length=700, q_stride=(0, 64),
                               workspace=work.data_ptr(), workspace_bytes=need)
    torch.cuda.synchronize()
    check_chunk(pool, q2, new, out, e)


@pytest.mark.parametrize("new", [[1, 2], [200, 20]])
def test_entries_outside_the_table_and_bad_pages(ctx, new):
    """They see nothing; a page outside the pool reads as zeros and is reported."""
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, [500, 300])
    q = normal(generator(2), (sum(new) + 1, 4, 64), torch.bfloat16, 2.0)
    out, lse = run_chunk(pool, q, new, rows=[0, 7], max_length=500)
    check_chunk(pool, q, new, out, lse, rows=[0, 7])
    for bad in (pool.memory.shape[0], -1):
        pool.table[0, 3] = bad
        ids = pool.table[0].tolist()
        out, lse = run_chunk(pool, q, new)
        zero = pool.tokens
        def tokens(s, layer):
            kv = zero(s, layer)
            if s == 0:
                kv[:, :, 48:64] = 0
            return kv
        pool.table[0, 3] = 0  # for the oracle's gather; zeroed above
        pool.tokens = tokens
        check_chunk(pool, q, new, out, lse, bits=N.KV_BAD_TOKEN)
        pool.tokens = zero


@pytest.mark.parametrize("dtype,value", [(torch.bfloat16, float("nan")), (torch.float16, float("inf"))])
@pytest.mark.parametrize("new,window,sinks", [([3], 0, 0), ([200], 0, 0), ([2], 60, 4), ([200], 60, 4), ([200], 60, 100)])
def test_hidden_values_have_no_influence(ctx, dtype, value, new, window, sinks):
    """Keys and values that some rows see and others don't, not finite: rows that do not see
    them are what they are without."""
    n, dim = 600, 64
    pool = Paged(ctx, dtype, 2, dim, 16, [n])
    q = normal(generator(2), (new[0], 4, dim), dtype, 2.0)
    before, lse0 = run_chunk(pool, q, new, window=window, sinks=sinks)
    check_chunk(pool, q, new, before, lse0, window=window, sinks=sinks)
    # token n - 2 is hidden from all but the last two; token 30 from all, if there is a window
    # (or seen by all, as a sink)
    hit = {n - 2} | ({30} if window and sinks <= 30 else set())
    for j in hit:
        page, r = pool.at(0, j)
        pool.memory[page, 1, :, :, r] = value
    out, lse = run_chunk(pool, q, new, window=window, sinks=sinks)
    free = new[0] - 2
    assert torch.equal(out[:free], before[:free]) and torch.equal(lse[:free], lse0[:free])
    # the values alone, through the weights of rows that see them
    for j in hit:
        page, r = pool.at(0, j)
        pool.memory[page, 1, 0, :, r] = 0
        pool.memory[page, 1, 1, :, r] = 0
        pool.memory[page, 1, 1, 0, r, 5] = value
    out, _ = run_chunk(pool, q, new, window=window, sinks=sinks)
    assert not torch.isfinite(out[free:, :2, 5]).any()
    out[free:, :2, 5] = 0
    assert torch.isfinite(out).all()


def test_growing_scores(ctx):
    """Scores that rise from key to key, so that the running maximum never settles."""
    n, new = 900, [300]
    for dim in (64, 128, 256):
        pool = Paged(ctx, torch.bfloat16, 1, dim, 32, [n])
        for j in range(n):
            page, r = pool.at(0, j)
            pool.memory[page, 1, 0, 0, r] = 0
            pool.memory[page, 1, 0, 0, r, 0] = j / 8
        q = torch.zeros(300, 2, dim, dtype=torch.bfloat16, device="cuda")
        q[:, 0, 0], q[:, 1, 0] = 8.0, -8.0
        out, lse = run_chunk(pool, q, new)
        check_chunk(pool, q, new, out, lse, some=6)


def test_one_sequence_against_decode_and_prompt(ctx):
    """A chunk of one is decode, a chunk of all is the prompt, to the last roundings."""
    n, heads, dim = 700, 8, 128
    pool = Paged(ctx, torch.bfloat16, 2, dim, 64, [n])
    q = normal(generator(2), (n, heads, dim), torch.bfloat16, 2.0)
    out, lse = run_chunk(pool, q, [n])
    last, lse1 = run_chunk(pool, q[-1:], [1])
    # each within half a unit of the same number, twice (the weights' rounding)
    assert (out[-1].float() - last[0].float()).abs().max() <= 4 * EPS[torch.bfloat16] * last.float().abs().max()
    assert (lse[-1] - lse1[0]).abs().max() < 1e-4
    check_chunk(pool, q, [n], out, lse)


def test_captured_calls(ctx):
    """Two graphs with workspaces of their own, replayed after the lengths and offsets changed;
    bounds stay."""
    lens = [1000, 1200]
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, lens, max_pages=100)
    q = normal(generator(2), (8, 8, 64), torch.bfloat16, 2.0)
    o, side = ints([0, 3, 8]), torch.cuda.Stream()
    results, graphs, keep = [], [], []
    need = pool.cache.chunk_workspace(8, 2, 8, 1600)
    assert need > 0
    for layer in (0, 1):
        out = torch.zeros_like(q)
        lse = torch.zeros(8, 8, device="cuda")
        work = torch.empty(need, dtype=torch.uint8, device="cuda")
        keep.append(work)
        results.append((out, lse))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            pool.cache.chunk_attention(layer=layer, heads=8, q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
                                       offsets=o.data_ptr(), n=2, tokens=8, max_length=1600,
                                       workspace=work.data_ptr(), workspace_bytes=need, stream=side.cuda_stream)
        graphs.append(g)
    for new, shorter in (([3, 5], 0), ([1, 2], 7), ([0, 8], 0), ([4, 0], 100)):
        pool.lens = [n - shorter for n in lens]
        pool.lengths.copy_(ints(pool.lens))
        o.copy_(ints(offsets(new)))
        for out, lse in results:
            out.fill_(float("nan"))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for layer, (out, lse) in enumerate(results):
            check_chunk(pool, q, new, out, lse, layer=layer)


def test_two_streams(ctx):
    """Calls side by side, each with its own workspace, give what they give alone."""
    pool = Paged(ctx, torch.bfloat16, 2, 128, 32, [3000, 2000])
    q = [normal(generator(i), (5, 8, 128), torch.bfloat16, 2.0) for i in range(2)]
    alone = [run_chunk(pool, x, [2, 3])[0] for x in q]
    streams = [torch.cuda.Stream() for _ in q]
    need = pool.cache.chunk_workspace(8, 2, 5, 3000)
    work = [torch.empty(max(16, need), dtype=torch.uint8, device="cuda") for _ in q]
    outs = [torch.empty_like(x) for x in q]
    o = ints([0, 2, 5])
    torch.cuda.synchronize()
    for _ in range(20):
        for x, out, w, s in zip(q, outs, work, streams):
            pool.cache.chunk_attention(layer=1, heads=8, q=x.data_ptr(), out=out.data_ptr(), offsets=o.data_ptr(), n=2,
                                       tokens=5, max_length=3000, workspace=w.data_ptr(), workspace_bytes=need,
                                       stream=s.cuda_stream)
    torch.cuda.synchronize()
    for a, b in zip(alone, outs):
        assert torch.equal(a, b)


def test_empty_calls_and_refusals(ctx):
    # a bound on the lengths that no block walks alone, so that there is a workspace
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, [500], max_pages=4000)
    q = normal(generator(2), (4, 4, 64), torch.bfloat16)
    o = ints([0, 4])
    good = dict(layer=0, heads=4, q=q.data_ptr(), out=q.data_ptr(), offsets=o.data_ptr(), n=1, tokens=4, max_length=60000)
    size = pool.cache.chunk_workspace(4, 1, 4, 60000)
    work = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
    good.update(workspace=work.data_ptr(), workspace_bytes=size)
    pool.cache.chunk_attention(**dict(good, n=0))
    pool.cache.chunk_attention(**dict(good, tokens=0))
    assert size > 0
    for change, status in [
            (dict(layer=2), N.ERR_INVALID_LAYER), (dict(layer=-1), N.ERR_INVALID_LAYER),
            (dict(heads=3), N.ERR_ELEMENT_COUNT), (dict(heads=0), N.ERR_ELEMENT_COUNT),
            (dict(heads=2 * 129), N.ERR_ELEMENT_COUNT), (dict(n=-1), N.ERR_ELEMENT_COUNT),
            (dict(n=(1 << 20) + 1), N.ERR_ELEMENT_COUNT), (dict(tokens=-1), N.ERR_ELEMENT_COUNT),
            (dict(tokens=1 << 31), N.ERR_ELEMENT_COUNT), (dict(tokens=1 << 30), N.ERR_OVERFLOW),
            (dict(max_length=-1), N.ERR_ELEMENT_COUNT), (dict(window=-1), N.ERR_ELEMENT_COUNT),
            (dict(sinks=-1), N.ERR_ELEMENT_COUNT), (dict(scale=float("nan")), N.ERR_POSITIVE_PARAMETER),
            (dict(scale=-1.0), N.ERR_POSITIVE_PARAMETER), (dict(q=0), N.ERR_INVALID_ARGUMENT),
            (dict(out=0), N.ERR_INVALID_ARGUMENT), (dict(offsets=0), N.ERR_INVALID_ARGUMENT),
            (dict(q=q.data_ptr() + 2), N.ERR_INVALID_ARGUMENT), (dict(q_stride=(256, 4)), N.ERR_INVALID_ARGUMENT),
            (dict(out_stride=(-256, 64)), N.ERR_INVALID_ARGUMENT), (dict(workspace=0), N.ERR_INVALID_ARGUMENT),
            (dict(workspace=work.data_ptr() + 4), N.ERR_INVALID_ARGUMENT),
            (dict(workspace_bytes=size - 1), N.ERR_BYTE_LENGTH)]:
        with pytest.raises(DmError) as e:
            pool.cache.chunk_attention(**dict(good, **change))
        assert e.value.status == status, change
    torch.cuda.synchronize()
    assert pool.cache.status() == 0
