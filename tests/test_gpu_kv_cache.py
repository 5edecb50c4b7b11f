"""The paged cache (dm_kv_cache_*) against its bookkeeping written out one page at a time."""
import numpy as np
import pytest
import torch

from attention_plain import PlainCache
from diskmule_b200 import CudaContext, DmError, _native as N
from diskmule_b200.attention import KvCache, offsets

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = CudaContext(0)
    yield c
    c.close()


def ints(values):
    return torch.tensor(np.asarray(values, np.int64), dtype=torch.int32, device="cuda")


class Pair:
    """A cache on the device and the same one in plain Python, driven side by side."""

    def __init__(self, ctx, layers=2, kv=2, dim=64, page=16, pages=40, seqs=8, max_pages=12, seed=0):
        self.shape = (pages, layers, 2, kv, page, dim)
        r = np.random.RandomState(seed)
        pool = r.randint(0, 1 << 16, self.shape).astype(np.uint16)  # any bits, NaN among them
        self.memory = torch.tensor(pool.astype(np.int32), device="cuda").to(torch.int16)
        self.memory.copy_(torch.tensor(pool.view(np.int16)))
        self.plain = PlainCache(pool.copy(), page, seqs, max_pages)
        self.table = torch.full((seqs, max_pages), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.cache = KvCache(ctx, type=N.BF16, layers=layers, kv_heads=kv, head_dim=dim,
                             page_tokens=page, pages=pages, max_sequences=seqs, max_pages=max_pages,
                             memory=self.memory.data_ptr(), page_table=self.table.data_ptr(),
                             lengths=self.lengths.data_ptr(), references=self.refs.data_ptr())
        self.r = r

    def check(self, status=0):
        assert self.cache.status() == status
        assert np.array_equal(self.lengths.cpu().numpy(), self.plain.lengths)
        assert np.array_equal(self.table.cpu().numpy(), self.plain.table)
        assert np.array_equal(self.refs.cpu().numpy(), self.plain.refs)
        assert np.array_equal(self.memory.cpu().numpy().view(np.uint16), self.plain.pool)

    def extend(self, seqs, counts):
        s, c = ints(seqs), ints(counts)
        self.cache.extend(s.data_ptr(), c.data_ptr(), len(seqs))
        return self.plain.extend(seqs, counts)

    def fork(self, parents, children):
        p, c = ints(parents), ints(children)
        self.cache.fork(p.data_ptr(), c.data_ptr(), len(parents))
        return self.plain.fork(parents, children)

    def compact(self, seqs, keeps):
        s, o, k = ints(seqs), ints(offsets([len(x) for x in keeps])), ints(np.concatenate(keeps + [[0]]))
        self.cache.compact(s.data_ptr(), o.data_ptr(), k.data_ptr(), len(seqs), k.numel() - 1)
        return self.plain.compact(seqs, keeps)

    def free(self, seqs):
        s = ints(seqs)
        self.cache.free(s.data_ptr(), len(seqs))
        self.plain.free(seqs)

    def write(self, layer, seqs, counts):
        kv, dim = self.shape[3], self.shape[5]
        rows = [self.r.randint(0, 1 << 16, (sum(counts), kv, dim)).astype(np.uint16) for _ in range(2)]
        dev = [torch.tensor(x.view(np.int16), device="cuda") for x in rows]
        s, o = ints(seqs), ints(offsets(counts))
        self.cache.write(layer, dev[0].data_ptr(), dev[1].data_ptr(), s.data_ptr(), o.data_ptr(),
                         len(seqs), sum(counts))
        self.plain.write(layer, *rows, seqs, offsets(counts))


@pytest.mark.parametrize("page,dim,kv,layers", [(16, 64, 2, 2), (32, 8, 1, 1), (64, 80, 3, 2), (16, 256, 1, 3)])
def test_every_call_in_turn(ctx, page, dim, kv, layers):
    t = Pair(ctx, page=page, dim=dim, kv=kv, layers=layers)
    P = page
    assert t.extend([3, 0, 5], [2 * P + 1, 1, P])
    t.check()
    t.write(layers - 1, [0, 3, 5], [1, P + 3, P])
    t.write(0, [3], [2 * P + 1])
    t.check()
    assert t.fork([3, 3, 0, 5], [1, 2, 4, 6])
    t.check()
    assert t.extend([1, 2, 6], [P, 3, 1])
    t.write(0, [2, 1, 6], [3, P, 1])
    t.check()
    # a tail that goes, a hole, a first token that goes, all of it
    n1, n2 = 3 * P + 1, 2 * P + 4
    assert t.compact([1], [list(range(n1 - 5))])
    t.check()
    assert t.compact([2, 1], [list(range(0, P)) + list(range(P + 2, n2)), list(range(1, n1 - 5, 2))])
    t.check()
    assert t.compact([6, 3], [[], list(range(2 * P + 1))])
    t.check()
    t.free([3, 1, 6])
    t.check()
    assert t.extend([3], [3 * P])
    t.check()
    t.free([0, 2, 3, 4, 5])
    t.check()
    assert t.refs.sum().item() == 0


def test_truncation_into_a_shared_page_takes_a_copy(ctx):
    """Both holders of a full page cut it short: each gets its own, the old one goes."""
    t = Pair(ctx)
    assert t.extend([0], [32]) and t.fork([0], [1])
    t.check()
    assert t.compact([1], [list(range(20))])
    t.check()
    assert t.fork([0], [2])
    assert t.compact([0, 2], [list(range(17)), list(range(31))])
    t.check()
    t.write(1, [0, 2], [3, 3])
    t.check()


def test_many_sequences_and_pages(ctx):
    """More list entries than a block has threads, more pages than one step of the search."""
    seqs, pages = 2600, 20000
    t = Pair(ctx, layers=1, kv=1, dim=8, page=16, pages=pages, seqs=seqs, max_pages=6)
    order = list(np.random.RandomState(1).permutation(1300))
    assert t.extend(order, [int(x) for x in t.r.randint(0, 90, 1300)])
    t.check()
    t.free(order[::3])
    assert t.fork(order[1:1200], list(range(1300, 2499)))
    t.check()
    keeps = []
    for s in range(1300, 2499):
        n = int(t.plain.lengths[s])
        keeps.append(sorted(t.r.permutation(n)[:t.r.randint(0, n + 1)].tolist()))
    assert t.compact(list(range(1300, 2499)), keeps)
    t.check()


def test_leading_part_of_every_length(ctx):
    """The first moved token at every place of a long keep list."""
    n, P = 190, 16
    for hole in list(range(0, n, 7)) + [n - 1, 31, 32, 33, 64]:
        t = Pair(ctx, layers=1, kv=1, dim=8, pages=30, seqs=2, max_pages=12, seed=hole)
        assert t.extend([1], [n])
        assert t.compact([1], [[j for j in range(n) if j != hole]])
        t.check()


def test_copy_pages(ctx):
    t = Pair(ctx, dim=128, layers=3)
    src, dst = [3, 7, 3, 0], [1, 39, 20, 2]
    s, d = ints(src), ints(dst)
    t.cache.copy_pages(s.data_ptr(), d.data_ptr(), 4)
    t.plain.pool[dst] = t.plain.pool[src]
    t.check()
    bad = ints([40])
    t.cache.copy_pages(bad.data_ptr(), d.data_ptr(), 1)
    t.check(status=N.KV_BAD_TOKEN)


def test_calls_that_cannot_be_done_change_nothing(ctx):
    t = Pair(ctx, pages=5, seqs=4, max_pages=6)
    assert t.extend([0, 1], [33, 10])
    t.check()
    assert not t.extend([2, 3], [16, 1])          # one page is left
    t.check(status=N.KV_OUT_OF_PAGES)
    assert t.fork([0], [2])
    t.check()
    assert not t.fork([1], [3])
    t.check(status=N.KV_OUT_OF_PAGES)
    assert not t.compact([0], [list(range(1, 33))])
    t.check(status=N.KV_OUT_OF_PAGES)

    def refused(call, *lists, bits):
        arrays = [ints(x) for x in lists]
        call(*[a.data_ptr() for a in arrays], len(lists[0]))
        t.check(status=bits)

    refused(t.cache.extend, [0, 4], [0, 0], bits=N.KV_BAD_SEQUENCE)
    refused(t.cache.extend, [-1], [0], bits=N.KV_BAD_SEQUENCE)
    refused(t.cache.extend, [1, 1], [1, 1], bits=N.KV_BAD_SEQUENCE)
    refused(t.cache.extend, [1], [-1], bits=N.KV_BAD_TOKEN)
    refused(t.cache.extend, [1], [6 * 16], bits=N.KV_TOO_LONG)
    refused(t.cache.extend, [1], [2 ** 31 - 1], bits=N.KV_TOO_LONG)
    refused(t.cache.fork, [0], [1], bits=N.KV_BAD_SEQUENCE)       # not empty
    refused(t.cache.fork, [9], [3], bits=N.KV_BAD_SEQUENCE)
    refused(t.cache.fork, [3], [3], bits=N.KV_BAD_SEQUENCE)       # its own parent
    s, o, k = ints([1]), ints([0, 11]), ints(range(11))
    t.cache.compact(s.data_ptr(), o.data_ptr(), k.data_ptr(), 1, 11)   # longer than it is
    t.check(status=N.KV_BAD_TOKEN)
    t.cache.compact(s.data_ptr(), o.data_ptr(), k.data_ptr(), 1, 10)   # beyond the list
    t.check(status=N.KV_BAD_TOKEN)
    w = torch.zeros(16, 2, 64, dtype=torch.int16, device="cuda")
    o = ints([0, 11])
    t.cache.write(0, w.data_ptr(), w.data_ptr(), s.data_ptr(), o.data_ptr(), 1, 1)  # 11 rows of 10
    t.check(status=N.KV_BAD_TOKEN)
    s = ints([7, 1, 1])
    t.cache.free(s.data_ptr(), 3)                 # the good one is freed once
    t.plain.free([1])
    t.check(status=N.KV_BAD_SEQUENCE)
    t.check()


def test_write_strides(ctx):
    t = Pair(ctx, dim=64, kv=2)
    assert t.extend([1], [20])
    fused = torch.randint(-30000, 30000, (20, 5 * 64 + 8), dtype=torch.int16, device="cuda")
    k, v = fused[:, 8:8 + 128], fused[:, 136:136 + 128]
    s, o = ints([1]), ints([0, 20])
    t.cache.write(1, k.data_ptr(), v.data_ptr(), s.data_ptr(), o.data_ptr(), 1, 20,
                  k_stride=(328, 64), v_stride=(328, 64))
    rows = [x.cpu().numpy().view(np.uint16).reshape(20, 2, 64) for x in (k.contiguous(), v.contiguous())]
    t.plain.write(1, *rows, [1], [0, 20])
    t.check()


def test_pages_beyond_32_bits_of_bytes(ctx):
    """A pool of more than 4 GB: rows in its last pages."""
    pages, layers, kv, page, dim = 2200, 8, 4, 128, 128   # 2 MB a page
    cache = KvCache(ctx, type=N.F16, layers=layers, kv_heads=kv, head_dim=dim, page_tokens=page,
                    pages=pages, max_sequences=2, max_pages=pages)
    d = cache.describe()
    refs = torch.ones(pages, dtype=torch.int32)
    refs[-3:] = 0
    s, c = ints([0]), ints([130])
    N.lib()
    view = _device_ints(d.references, pages)
    view.copy_(refs)
    cache.extend(s.data_ptr(), c.data_ptr(), 1)
    k = torch.randn(130, kv, dim, dtype=torch.float16, device="cuda")
    v = torch.randn(130, kv, dim, dtype=torch.float16, device="cuda")
    o = ints([0, 130])
    cache.write(7, k.data_ptr(), v.data_ptr(), s.data_ptr(), o.data_ptr(), 1, 130)
    child = ints([1])
    cache.fork(s.data_ptr(), child.data_ptr(), 1)
    assert cache.status() == 0
    q = torch.randn(2, kv, dim, dtype=torch.float16, device="cuda")
    out = torch.empty_like(q)
    n = cache.decode_workspace(kv, 2, 128, 130)
    work = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    cache.decode_attention(layer=7, heads=kv, q=q.data_ptr(), out=out.data_ptr(), batch=2,
                           max_length=130, shared_tokens=128, workspace=work.data_ptr(),
                           workspace_bytes=n)
    torch.cuda.synchronize()
    p = torch.softmax(torch.einsum("bhd,thd->bht", q.double(), k.double()) / dim ** 0.5, -1)
    want = torch.einsum("bht,thd->bhd", p, v.double())
    # one rounding of the weights and one of the result: 2^-11 of each value's spread
    assert (out.double() - want).abs().max() <= 2.0 ** -11 * 2.1 * v.double().abs().max()
    cache.close()


def _device_ints(pointer, n):
    """A torch view of n int32 on the device."""
    class Holder:
        __cuda_array_interface__ = {"shape": (n,), "typestr": "<i4", "data": (pointer, False),
                                    "version": 3}
    return torch.as_tensor(Holder(), device="cuda")


def test_own_buffers_start_empty(ctx):
    cache = KvCache(ctx, type=N.BF16, layers=1, kv_heads=1, head_dim=64, page_tokens=16, pages=4,
                    max_sequences=3, max_pages=2)
    d = cache.describe()
    assert (_device_ints(d.lengths, 3) == 0).all() and (_device_ints(d.references, 4) == 0).all()
    assert (_device_ints(d.page_table, 6) == -1).all()
    cache.close()


def test_refusals(ctx):
    good = dict(type=N.BF16, layers=1, kv_heads=1, head_dim=64, page_tokens=16, pages=4,
                max_sequences=2, max_pages=2)

    def status(**change):
        with pytest.raises(DmError) as e:
            KvCache(ctx, **{**good, **change})
        return e.value.status

    assert status(type=N.F32) == N.ERR_UNSUPPORTED_TENSOR_TYPE
    for name in ("layers", "kv_heads", "pages", "max_sequences", "max_pages"):
        assert status(**{name: 0}) == N.ERR_EMPTY_INPUT
    for dim in (0, 60, 264):
        assert status(head_dim=dim) == N.ERR_ELEMENT_COUNT
    for page in (8, 48, 512, 0):
        assert status(page_tokens=page) == N.ERR_ELEMENT_COUNT
    assert status(layers=1 << 20, kv_heads=64) == N.ERR_OVERFLOW
    assert status(max_pages=1 << 28) == N.ERR_OVERFLOW
    assert status(memory=8) == N.ERR_INVALID_ARGUMENT
    cache = KvCache(ctx, **good)
    one = ints([0, 0, 0])
    p = one.data_ptr()

    def refused(code, call, *args):
        with pytest.raises(DmError) as e:
            call(*args)
        assert e.value.status == code

    refused(N.ERR_ELEMENT_COUNT, cache.extend, p, p, 3)
    refused(N.ERR_ELEMENT_COUNT, cache.free, p, -1)
    refused(N.ERR_INVALID_ARGUMENT, cache.free, 0, 1)
    refused(N.ERR_INVALID_ARGUMENT, cache.extend, p, 0, 1)
    refused(N.ERR_INVALID_ARGUMENT, cache.fork, 0, p, 1)
    refused(N.ERR_INVALID_ARGUMENT, cache.compact, p, 0, p, 1, 1)
    refused(N.ERR_ELEMENT_COUNT, cache.compact, p, p, p, 1, -1)
    refused(N.ERR_INVALID_LAYER, cache.write, 1, p, p, p, p, 1, 1)
    refused(N.ERR_INVALID_ARGUMENT, cache.write, 0, 0, p, p, p, 1, 1)
    refused(N.ERR_INVALID_ARGUMENT, cache.write, 0, p + 2, p, p, p, 1, 1)
    refused(N.ERR_ELEMENT_COUNT, cache.copy_pages, p, p, 5)
    refused(N.ERR_INVALID_ARGUMENT, cache.copy_pages, p, 0, 1)
    cache.free(p, 0)
    cache.close()
