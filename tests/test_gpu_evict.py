"""dm_attention_weights and dm_kv_cache_evict against their definitions in plain Python."""
import math

import numpy as np
import pytest
import torch

from attention_plain import PlainCache, to64
from diskmule_b200 import CudaContext, DmError, _native as N
from diskmule_b200.attention import attention_status, offsets
from paged import Paged, generator, ints, normal, seen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = CudaContext(0)
    yield c
    c.close()


# ---------------------------------------------------------------------------
# received weight
# ---------------------------------------------------------------------------

def statistics(pool, q, new, layer, window, sinks, scale, rows):
    """lse of every row (f32, on the device) from scores in 64 bits."""
    g = q.shape[1] // pool.kv
    Q, lse, at = to64(q), np.full(q.shape[:2], -math.inf), 0
    for i, a in enumerate(new):
        s = i if rows is None else rows[i]
        n = pool.lens[s] if 0 <= s < len(pool.lens) else 0
        k = pool.tokens(s, layer)[0] if n else None
        for t in range(a):
            keys = seen(n - a + t, n, window, sinks)
            for h in range(q.shape[1]):
                if len(keys):
                    x = k[h // g, keys] @ Q[at + t, h] * scale
                    lse[at + t, h] = x.max() + math.log(np.exp(x - x.max()).sum())
        at += a
    return torch.tensor(lse, dtype=torch.float32, device="cuda")


def received(pool, q, lse, new, layer, window, sinks, scale, rows):
    """Sums of weights of every table row and token, and what they may be off by: each weight by
    its score's f32 products (d + 4 roundings of the largest sum of |q k|), its exponent's
    roundings and the exponential's (2^-21), and the sum's terms times 2^-24."""
    g, d = q.shape[1] // pool.kv, q.shape[2]
    Q, E = to64(q), to64(lse)
    out = np.zeros((pool.table.shape[0], max(pool.lens)))
    bound, terms, at, done = np.zeros_like(out), np.zeros_like(out), 0, set()
    for i, a in enumerate(new):
        s = i if rows is None else rows[i]
        n = pool.lens[s] if 0 <= s < len(pool.lens) else 0
        if n and s not in done:
            k = pool.tokens(s, layer)[0]
            for t in range(a):
                keys = seen(n - a + t, n, window, sinks)
                for h in range(q.shape[1]):
                    if not len(keys) or E[at + t, h] == -math.inf:
                        continue
                    kk = k[h // g, keys]
                    x = kk @ Q[at + t, h] * scale
                    w = np.exp(x - E[at + t, h])
                    size = (np.abs(kk) @ np.abs(Q[at + t, h])) * scale
                    out[s, keys] += w
                    bound[s, keys] += w * ((d + 4) * 2.0 ** -24 * size + (np.abs(x) + abs(E[at + t, h]) + 2) * 2.0 ** -21)
                    terms[s, keys] += 1
        done.add(s)
        at += a
    return out, bound + out * (terms + 2) * 2.0 ** -24


def run_weights(pool, q, lse, new, weights, layer=1, window=0, sinks=0, rows=None, scale=0.0, max_length=None,
                stride=None, stream=0, tokens=None):
    o = ints(offsets(new))
    r = None if rows is None else ints(rows)
    pool.cache.token_weights(layer=layer, heads=q.shape[1], q=q.data_ptr(), lse=lse.data_ptr(),
                             sequences=r.data_ptr() if r is not None else 0, offsets=o.data_ptr(), n=len(new),
                             tokens=q.shape[0] if tokens is None else tokens,
                             max_length=max(pool.lens + [1]) if max_length is None else max_length,
                             weights=weights.data_ptr(), weights_stride=stride or weights.stride(0), window=window,
                             sinks=sinks, scale=scale, q_stride=(q.stride(0), q.stride(1)), stream=stream)
    torch.cuda.synchronize()


WEIGHTS = [
    # new tokens, tokens with them, heads, kv heads, dim, page, window, sinks
    ([1], [1], 1, 1, 64, 16, 0, 0),
    ([1, 1, 1], [7, 300, 64], 8, 2, 64, 16, 0, 0),
    ([5, 3, 0, 5], [305, 80, 47, 905], 8, 2, 64, 16, 0, 0),
    ([1], [3000], 32, 8, 128, 64, 0, 0),                  # few blocks: queries shared in a cluster
    ([2, 40], [601, 40], 2, 1, 256, 32, 0, 0),
    ([17, 1], [90, 333], 6, 2, 80, 16, 0, 0),
    ([9, 30], [5, 0], 4, 2, 128, 16, 0, 0),               # more rows than tokens: some see nothing
    ([100], [500], 7, 1, 96, 128, 0, 0),
    ([130], [700], 4, 4, 128, 64, 0, 0),
    ([20], [300], 128, 1, 64, 16, 0, 0),
    ([1, 33], [200, 60], 2, 2, 8, 16, 0, 0),
    ([1, 1], [2000, 90], 8, 2, 128, 16, 100, 4),
    ([64, 1, 100], [500, 1000, 100], 8, 2, 64, 32, 128, 1),
    ([60], [900], 4, 1, 256, 16, 200, 40),
    ([50, 9], [400, 40], 4, 2, 128, 64, 33, 500),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,lens,heads,kv,dim,page,window,sinks", WEIGHTS)
def test_weights(ctx, new, lens, heads, kv, dim, page, window, sinks, dtype):
    pool = Paged(ctx, dtype, kv, dim, page, lens, seed=sum(lens))
    q = normal(generator(3), (sum(new) + 2, heads, dim), dtype, 2.0)
    scale = 1.0 / math.sqrt(dim)
    lse = statistics(pool, q, new, 1, window, sinks, scale, None)
    width = max(lens) + 5
    start = torch.rand(len(lens), width, generator=generator(4), device="cuda")
    weights = start.clone()
    run_weights(pool, q, lse, new, weights, window=window, sinks=sinks)
    want, bound = received(pool, q, lse, new, 1, window, sinks, scale, None)
    got, first = to64(weights), to64(start)
    n = max(lens)
    err = np.abs(got[:, :n] - (first[:, :n] + want))
    assert np.all(err <= bound + 2.0 ** -24 * (first[:, :n] + want)), (err - bound).max()
    for s, l in enumerate(lens):
        assert torch.equal(weights[s, l:], start[s, l:])
    attention_status(ctx)
    assert pool.cache.status() == 0
    again = start.clone()
    run_weights(pool, q, lse, new, again, window=window, sinks=sinks)
    assert torch.equal(again, weights)  # the order of the sums is fixed
    if not window:  # every row that sees something gives one in all
        seeing = sum(min(a, l) for a, l in zip(new, lens)) * heads
        assert abs(float((got[:, :n] - first[:, :n]).sum()) - seeing) <= bound.sum() + 1e-6 * seeing + 1e-3


def test_weights_of_rows_strides_and_bounds(ctx):
    """Entries in another order, one named twice, one outside the table; strided queries, tokens
    beyond max_length and beyond the row of weights, rows behind the last entry."""
    lens = [300, 80, 700]
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, lens, rows=5, seed=8)
    new, rows = [3, 2, 2, 4], [2, 0, 7, 2]
    fused = normal(generator(9), (sum(new) + 3, 12, 64), torch.bfloat16, 2.0)
    q = fused[:, 2:10]
    lse = statistics(pool, q, new, 1, 0, 0, 0.125, rows)
    weights = torch.zeros(5, 704, device="cuda")
    run_weights(pool, q, lse, new, weights, rows=rows)
    want, bound = received(pool, q, lse, new, 1, 0, 0, 0.125, rows)
    assert np.all(np.abs(to64(weights)[:, :700] - want) <= bound)
    assert weights[:, 700:].abs().sum() == 0 and weights[1].abs().sum() == 0
    assert pool.cache.status() == N.KV_BAD_SEQUENCE  # row 2 counted once
    # a row of weights shorter than the sequences: its places are summed, the next row's are not
    narrow = torch.zeros(5, 100, device="cuda")
    run_weights(pool, q, lse, new[:3], narrow, rows=rows[:3])
    # how many blocks share a token's queries depends on the call's sizes, and so does the order of
    # a sum, so this is held to the definition like the first call, not to its last bits
    assert np.all(np.abs(to64(narrow) - want[:, :100]) <= bound[:, :100])
    assert pool.cache.status() == 0


@pytest.mark.parametrize("heads", [4, 32])
def test_weights_of_hidden_and_wild_keys(ctx, heads):
    """A key that is not finite changes no other token's sum; hidden from all, it gets nothing."""
    n, new = 400, [6]
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, [n])
    q = normal(generator(2), (6, heads, 64), torch.bfloat16, 2.0)
    lse = statistics(pool, q, new, 1, 60, 4, 0.125, None)
    weights, after = torch.zeros(1, n, device="cuda"), torch.zeros(1, n, device="cuda")
    run_weights(pool, q, lse, new, weights, window=60, sinks=4)
    for j in (200, n - 30):
        page, r = pool.at(0, j)
        pool.memory[page, 1, 0, :, r] = float("nan")
    run_weights(pool, q, lse, new, after, window=60, sinks=4)
    assert torch.isnan(after[0, n - 30]) and after[0, 200] == 0
    after[0, n - 30] = weights[0, n - 30]
    assert torch.equal(weights, after)
    # a row without statistics gives nothing
    lse[2] = -math.inf
    without = torch.zeros(1, n, device="cuda")
    run_weights(pool, q, lse, new, without, window=60, sinks=4)
    page, r = pool.at(0, n - 30)
    pool.memory[page, 1, 0, :, r] = 0
    want, bound = received(pool, q, lse, new, 1, 60, 4, 0.125, None)
    without[0, n - 30] = float(want[0, n - 30])
    assert np.all(np.abs(to64(without) - want) <= bound + 1e-12)


def test_weights_bad_page_and_refusals(ctx):
    pool = Paged(ctx, torch.bfloat16, 2, 64, 16, [300])
    q = normal(generator(2), (1, 4, 64), torch.bfloat16, 2.0)
    lse = torch.zeros(1, 4, device="cuda")
    weights = torch.zeros(1, 304, device="cuda")
    pool.table[0, 3] = 10 ** 6
    run_weights(pool, q, lse, [1], weights)
    assert pool.cache.status() == N.KV_BAD_TOKEN
    assert torch.allclose(weights[0, 48:64], torch.full((16,), 4.0, device="cuda"))  # keys of zero: exp(0 - 0)
    o = ints([0, 1])
    good = dict(layer=0, heads=4, q=q.data_ptr(), lse=lse.data_ptr(), offsets=o.data_ptr(), n=1, tokens=1,
                max_length=300, weights=weights.data_ptr(), weights_stride=304)
    pool.cache.token_weights(**dict(good, n=0))
    pool.cache.token_weights(**dict(good, tokens=0))
    pool.cache.token_weights(**dict(good, max_length=0))
    for change, status in [
            (dict(layer=2), N.ERR_INVALID_LAYER), (dict(heads=3), N.ERR_ELEMENT_COUNT),
            (dict(heads=300), N.ERR_ELEMENT_COUNT), (dict(n=-1), N.ERR_ELEMENT_COUNT),
            (dict(n=65536), N.ERR_ELEMENT_COUNT), (dict(tokens=-1), N.ERR_ELEMENT_COUNT),
            (dict(tokens=1 << 30), N.ERR_OVERFLOW), (dict(max_length=-1), N.ERR_ELEMENT_COUNT),
            (dict(window=-1), N.ERR_ELEMENT_COUNT), (dict(sinks=-1), N.ERR_ELEMENT_COUNT),
            (dict(scale=float("inf")), N.ERR_POSITIVE_PARAMETER), (dict(q=0), N.ERR_INVALID_ARGUMENT),
            (dict(lse=0), N.ERR_INVALID_ARGUMENT), (dict(weights=0), N.ERR_INVALID_ARGUMENT),
            (dict(offsets=0), N.ERR_INVALID_ARGUMENT), (dict(q=q.data_ptr() + 2), N.ERR_INVALID_ARGUMENT),
            (dict(weights=weights.data_ptr() + 2), N.ERR_INVALID_ARGUMENT),
            (dict(weights_stride=-1), N.ERR_INVALID_ARGUMENT), (dict(q_stride=(100, 4)), N.ERR_INVALID_ARGUMENT)]:
        with pytest.raises(DmError) as e:
            pool.cache.token_weights(**dict(good, **change))
        assert e.value.status == status, change


# ---------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------

def kept(weights, n, budget, sinks, recent):
    """The definition: always-kept tokens, then by weight, the earlier of equals; NaN last."""
    if n <= budget:
        return list(range(n))
    always = set(range(sinks)) | set(range(n - recent, n))
    rest = [j for j in range(sinks, n - recent)]
    order = sorted(rest, key=lambda j: (math.isnan(weights[j]), -weights[j] if not math.isnan(weights[j]) else 0, j))
    return sorted(always | set(order[:budget - len(always)]))


class Evict:
    """A cache of random bits beside the plain one, and weights."""

    def __init__(self, ctx, lens, page=16, pages=None, layers=2, kv=2, dim=64, max_pages=None, seed=0, stride=None):
        from test_gpu_kv_cache import Pair
        need = sum(-(-n // page) for n in lens)
        max_pages = max_pages or -(-max(lens) // page) + 2
        self.pair = Pair(ctx, layers=layers, kv=kv, dim=dim, page=page, pages=pages or 2 * need + 4,
                         seqs=len(lens) + 2, max_pages=max_pages, seed=seed)
        if any(lens):
            some = [i for i, n in enumerate(lens) if n]
            assert self.pair.extend(some, [lens[i] for i in some])
        stride = stride or max_pages * page + 3
        self.weights = torch.randn(len(lens) + 2, stride, generator=generator(seed), device="cuda").exp()

    def run(self, seqs, budget, sinks=0, recent=0, status=0, stream=0):
        n = len(seqs)
        self.keep = torch.full((max(1, n * budget),), -7, dtype=torch.int32, device="cuda")
        self.off = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda")
        w = self.weights.cpu().numpy().copy()
        plain = self.pair.plain
        lens = [int(plain.lengths[s]) if 0 <= s < len(plain.lengths) else 0 for s in seqs]
        lists = [kept(w[s], l, budget, sinks, recent) if l else [] for s, l in zip(seqs, lens)]
        rows = ints(seqs)
        self.pair.cache.evict(sequences=rows.data_ptr(), n=n, budget=budget, sinks=sinks, recent=recent,
                              weights=self.weights.data_ptr(), weights_stride=self.weights.stride(0),
                              keep_offsets=self.off.data_ptr(), keep=self.keep.data_ptr(), stream=stream)
        torch.cuda.synchronize()
        if status == 0:
            assert plain.compact(seqs, lists)
            for s, l, k in zip(seqs, lens, lists):
                w[s, :len(k)] = w[s, k]
                w[s, len(k):l] = 0
            off = offsets([len(k) for k in lists])
            assert np.array_equal(self.off.cpu().numpy(), off)
            flat = np.concatenate([np.asarray(k, np.int64) for k in lists] + [np.zeros(0, np.int64)])
            assert np.array_equal(self.keep.cpu().numpy()[:off[-1]], flat)
            assert (self.keep[off[-1]:] == -7).all()
        self.pair.check(status)
        assert np.array_equal(self.weights.cpu().numpy(), w, equal_nan=True)


@pytest.mark.parametrize("lens,budget,sinks,recent", [
    ([100], 50, 4, 10), ([301, 160], 128, 4, 32), ([5, 0, 17, 64], 16, 0, 0), ([33], 0, 0, 0), ([33, 40], 10, 3, 7),
    ([64, 65, 63], 64, 1, 63), ([1, 2, 3], 1, 0, 1), ([1, 2, 3], 1, 1, 0), ([700], 699, 0, 0), ([700, 80], 80, 0, 79)])
def test_evict(ctx, lens, budget, sinks, recent):
    for page in (16, 64):
        e = Evict(ctx, lens, page=page, seed=sum(lens))
        e.run(list(range(len(lens))), budget, sinks, recent)
        e.run(list(range(len(lens)))[::-1], budget, sinks, recent)  # nothing more to do
        some = [i for i, n in enumerate(lens) if n]
        assert e.pair.extend(some, [3] * len(some))
        e.run(some, budget, sinks, recent)


@pytest.mark.parametrize("n", [4096, 4097, 9001, 33000, 70001])
def test_evict_long(ctx, n):
    """One block, and clusters of two to eight; places of weights that meet between rounds."""
    for budget in (n // 3, n - 5, 40):
        e = Evict(ctx, [n, 50], layers=1, kv=1, dim=8, page=64, seed=n)
        e.run([0, 1], budget, 4, 20)


@pytest.mark.parametrize("kind", ["equal", "zeros", "signs", "nan", "inf", "few", "close", "falling", "rising"])
@pytest.mark.parametrize("n,budget", [(500, 200), (9001, 3000)])
def test_evict_ties_and_odd_weights(ctx, kind, n, budget):
    """Equal weights go by place; signs, zeros of both signs, infinities and NaN have an order."""
    e = Evict(ctx, [n, n], layers=1, kv=1, dim=8, page=64)
    w = e.weights
    r = generator(5)
    j = torch.arange(w.shape[1], device="cuda")
    if kind == "equal":
        w[:] = 0.25
    elif kind == "zeros":
        w[:] = 0
        w[:, ::7] = -0.0
    elif kind == "signs":
        w.copy_(torch.randn(w.shape, generator=r, device="cuda"))
    elif kind == "nan":
        w[:, ::2] = float("nan")
        w[1] = float("nan")
    elif kind == "inf":
        w[:, ::3], w[:, 1::3], w[:, 2::5] = float("inf"), -float("inf"), 0.0
    elif kind == "few":
        w.copy_(torch.randint(0, 3, w.shape, generator=r, device="cuda").float())
    elif kind == "close":  # differ in the last bits only
        w.copy_((0x3f800000 + torch.randint(0, 9, w.shape, generator=r, device="cuda", dtype=torch.int32)).view(torch.float32))
    else:
        w[:] = j.float() * (1 if kind == "rising" else -1)
    e.run([1, 0], budget, 2, 5)


def test_evict_shared_pages(ctx):
    """A fork's own copy is cut down; the parent keeps every token."""
    e = Evict(ctx, [200, 90], pages=60, max_pages=16)
    assert e.pair.fork([0, 1], [2, 3])
    e.weights[2:] = e.weights[:2]
    e.run([2, 3], 70, 4, 16)
    e.run([0], 70, 4, 16)


def test_evict_refused_on_the_device(ctx):
    """No room, bad and repeated rows, weights too narrow: cache and weights stay."""
    e = Evict(ctx, [200, 90], pages=20, max_pages=16)  # 13 + 6 pages of 20
    assert e.pair.fork([0], [2])                       # a copied last page: none is free
    e.run([0, 1], 100, 0, 3, status=N.KV_OUT_OF_PAGES)
    e = Evict(ctx, [200, 90])
    for rows in ([0, 9], [-1], [1, 1]):
        e.run(rows, 20, 1, 2, status=N.KV_BAD_SEQUENCE)
    e = Evict(ctx, [90, 200], stride=199)
    e.run([0, 1], 20, 1, 2, status=N.KV_BAD_TOKEN)
    e.run([0], 20, 1, 2)


def test_evict_many_sequences(ctx):
    r = np.random.RandomState(1)
    lens = [int(x) for x in r.randint(0, 90, 1500)]
    e = Evict(ctx, lens, layers=1, kv=1, dim=8, page=16)
    e.run(list(r.permutation(1500)), 20, 2, 5)


def test_evict_captured(ctx):
    """A graph that is replayed as sequences grow."""
    e = Evict(ctx, [200, 90], pages=80, max_pages=20)
    rows, side = ints([0, 1]), torch.cuda.Stream()
    keep = torch.zeros(128, dtype=torch.int32, device="cuda")
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        e.pair.cache.evict(sequences=rows.data_ptr(), n=2, budget=64, sinks=2, recent=8, weights=e.weights.data_ptr(),
                           weights_stride=e.weights.stride(0), keep_offsets=off.data_ptr(), keep=keep.data_ptr(),
                           stream=side.cuda_stream)
    for more in (0, 30, 5):
        if more:
            assert e.pair.extend([0, 1], [more, more])
            torch.cuda.synchronize()
        w = e.weights.cpu().numpy()
        lens = [int(x) for x in e.pair.plain.lengths[:2]]
        lists = [kept(w[s], lens[s], 64, 2, 8) for s in (0, 1)]
        g.replay()
        torch.cuda.synchronize()
        assert e.pair.plain.compact([0, 1], lists)
        e.pair.check()
        assert np.array_equal(keep.cpu().numpy()[:off[-1]], np.concatenate(lists))


def test_evict_refusals(ctx):
    e = Evict(ctx, [200])
    rows, keep, off = ints([0]), ints([0] * 50), ints([0, 0])
    good = dict(sequences=rows.data_ptr(), n=1, budget=50, sinks=2, recent=3, weights=e.weights.data_ptr(),
                weights_stride=e.weights.stride(0), keep_offsets=off.data_ptr(), keep=keep.data_ptr())
    e.pair.cache.evict(**dict(good, n=0))
    for change, status in [
            (dict(n=-1), N.ERR_ELEMENT_COUNT), (dict(n=4), N.ERR_ELEMENT_COUNT), (dict(sequences=0), N.ERR_INVALID_ARGUMENT),
            (dict(budget=-1), N.ERR_ELEMENT_COUNT), (dict(budget=4), N.ERR_ELEMENT_COUNT), (dict(sinks=-1), N.ERR_ELEMENT_COUNT),
            (dict(recent=-1), N.ERR_ELEMENT_COUNT), (dict(recent=(1 << 31) - 1), N.ERR_ELEMENT_COUNT),
            (dict(weights=0), N.ERR_INVALID_ARGUMENT), (dict(keep=0), N.ERR_INVALID_ARGUMENT),
            (dict(keep_offsets=0), N.ERR_INVALID_ARGUMENT), (dict(weights=e.weights.data_ptr() + 1), N.ERR_INVALID_ARGUMENT),
            (dict(weights_stride=-1), N.ERR_INVALID_ARGUMENT)]:
        with pytest.raises(DmError) as err:
            e.pair.cache.evict(**dict(good, **change))
        assert err.value.status == status, change
    two = dict(good, n=2, budget=(1 << 31) - 1)
    with pytest.raises(DmError) as err:
        e.pair.cache.evict(**two)
    assert err.value.status == N.ERR_OVERFLOW
    e.pair.check()
