"""Calls whose number of entries is a bound, few of which have rows."""
import numpy as np
import pytest
import torch

from diskmule_b200 import CudaContext
from diskmule_b200.attention import attention_status
from paged import Paged, generator, normal
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
    run()
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    a.record()
    run()
    b.record()
    b.synchronize()
    return a.elapsed_time(b)


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
        assert took < 25, took
