"""Waits of chunks and of received weight that must run out: caches far larger than L2, read by all
SMs at once, where no copy lands within a clock."""
import pytest
import torch

from diskmule_b200 import CudaContext
from paged import Paged, generator, normal
from test_gpu_chunk import run_chunk
from test_gpu_evict import run_weights
from test_gpu_paged_edges import out_of_time

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = CudaContext(0)
    yield c
    c.close()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new,length", [([1] * 300, 2000), ([300] * 40, 6000)])
def test_chunks_run_out(ctx, dim, new, length):
    """Blocks of 16 rows, and tiles."""
    pool = Paged(ctx, torch.bfloat16, 4, dim, 64, [length] * len(new), layers=1)
    q = normal(generator(dim), (sum(new), 8, dim), torch.bfloat16, 2.0)
    run = lambda: run_chunk(pool, q, new, layer=0)
    assert out_of_time(ctx, run, run()) > 0


@pytest.mark.parametrize("dim,broadcast", [(64, False), (128, False), (256, False), (256, True)])
def test_weights_run_out(ctx, dim, broadcast):
    """Tiles, and the kernel for queries that no tensor map holds. (Up to dim 128 that one has copied
    its queries before it asks for its keys, which are there by then.)"""
    new = [3 if broadcast else 1] * 400
    pool = Paged(ctx, torch.float16, 4, dim, 64, [2000] * len(new), layers=1)
    q = normal(generator(dim), (sum(new), 8, dim), torch.float16, 2.0)
    if broadcast:
        q = q[:1].expand(sum(new), 8, dim)
    lse = torch.full((sum(new), 8), 9.0, device="cuda")

    def run():
        weights = torch.zeros(len(new), 2000, device="cuda")
        run_weights(pool, q, lse, new, weights, layer=0)
        return (weights,)

    assert out_of_time(ctx, run, run()) > 0
