"""Calls whose number of entries is a bound, few of which have rows."""
import numpy as np
import pytest
import torch

from diskmule_b200 import CudaContext, _native as N
from diskmule_b200.attention import attention_status, offsets
from paged import Paged, generator, ints, normal
from test_gpu_chunk import check_chunk, run_chunk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = CudaContext(0)
    yield c
    c.close()


def idle(n, busy):
    """n entries, of which busy = {place: (table row, rows)} have rows."""
    new, rows = np.zeros(n, int), np.zeros(n, int)
    for at, (row, count) in busy.items():
        new[at], rows[at] = count, row
    return new, rows


def milliseconds(run):
    """The shortest of five calls."""
    took = []
    run()
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        run()
        b.record()
        b.synchronize()
        took.append(a.elapsed_time(b))
    return min(took)


@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("n", [1000, 40000, 1 << 20])
def test_few_rows_among_idle_entries(ctx, n, dim):
    """Single tokens and drafts (blocks of 16 rows): what has no rows costs next to nothing."""
    lens = [700, 300, 90]
    pool = Paged(ctx, torch.bfloat16, 2, dim, 16, lens)
    new, rows = idle(n, {0: (1, 1), n // 3: (0, 3), n - 2: (2, 2)})
    q = normal(generator(n), (6, 8, dim), torch.bfloat16, 2.0)
    busy = [i for i in range(n) if new[i]] if n < 5000 else [0, n // 3, n - 2]
    out, lse = run_chunk(pool, q, new, rows=rows)
    check_chunk(pool, q, [int(new[i]) for i in busy], out, lse, rows=[int(rows[i]) for i in busy])
    if n == 40000:
        took = milliseconds(lambda: run_chunk(pool, q, new, rows=rows))
        # lists are made and copied within it; a search through all entries takes every block ms: 1450 in all
        assert took < 100, took


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1000, 1 << 18])
def test_pieces_of_prompts_among_idle_entries(ctx, n, dim):
    """Tiles: looking through the entries is no reason to give up, however long (a look at each of
    2^18 four times takes 20 ms)."""
    lens = [700, 900, 90]
    pool = Paged(ctx, torch.bfloat16, 2, dim, 16, lens)
    new, rows = idle(n, {0: (1, 300), n // 3: (0, 260), n - 2: (2, 2)})
    q = normal(generator(n), (562, 8, dim), torch.bfloat16, 2.0)
    try:
        N.check(N.lib().dm_selftest_attention_wait(ctx.handle, 2000000))  # 1 ms
        out, lse = run_chunk(pool, q, new, rows=rows)
        attention_status(ctx)
    finally:
        N.check(N.lib().dm_selftest_attention_wait(ctx.handle, 0))
    check_chunk(pool, q, [300, 260, 2], out, lse, rows=[1, 0, 2], some=4)


@pytest.mark.parametrize("dim,heads,kv", [(64, 8, 2), (256, 4, 1)])
def test_hundreds_of_drafts(ctx, dim, heads, kv):
    """Items are found whatever the order in which a block takes them, in all steps of the lengths."""
    r = np.random.RandomState(dim)
    new = [int(x) for x in r.choice([0, 1, 5, 40, 70, 200], 300)]
    lens = [n + int(x) for n, x in zip(new, r.choice([0, 10, 300, 900], 300))]
    pool = Paged(ctx, torch.bfloat16, kv, dim, 16, lens)
    q = normal(generator(4), (sum(new), heads, dim), torch.bfloat16, 2.0)
    for max_length in (max(lens), 5000):
        out, lse = run_chunk(pool, q, new, max_length=max_length)
        check_chunk(pool, q, new, out, lse, some=1)


@pytest.mark.parametrize("dim", [64, 256])
def test_idle_entries_are_passed_over_at_once(ctx, dim):
    """Pieces of prompts on tiles; offsets beyond the bound of tokens, too."""
    n, lens = 1 << 20, [700, 900, 90]
    pool = Paged(ctx, torch.bfloat16, 2, dim, 16, lens)
    new, rows = idle(n, {5: (1, 300), n // 3: (0, 260), n - 40: (2, 2)})
    q = normal(generator(n), (562, 8, dim), torch.bfloat16, 2.0)
    o, r, out = ints(offsets(new)), ints(rows), torch.zeros_like(q)

    def run(tokens=562):
        need = pool.cache.chunk_workspace(8, n, tokens, 900)
        work = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
        pool.cache.chunk_attention(layer=1, heads=8, q=q.data_ptr(), out=out.data_ptr(), sequences=r.data_ptr(),
                                   offsets=o.data_ptr(), n=n, tokens=tokens, max_length=900, workspace=work.data_ptr(),
                                   workspace_bytes=need)

    # a look at each of 2^20 entries takes a block some 20 ms
    assert milliseconds(run) < 5
    want = out.clone()
    out.zero_()
    run(tokens=560)  # the last entry's rows are not there
    torch.cuda.synchronize()
    attention_status(ctx)
    assert torch.equal(out[:560], want[:560]) and (out[560:] == 0).all()
