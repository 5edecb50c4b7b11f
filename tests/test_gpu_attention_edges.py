"""Attention and its cache at their edges: what a finished or short sequence leaves in the page
table, bounds and sizes near their limits, values near the types' limits."""
import math

import numpy as np
import pytest
import torch

from attention_plain import EPS, check_rows, row, to64
from diskmule_b200 import CudaContext, DmError, _native as N
from diskmule_b200.attention import KvCache, attention_status, offsets, prompt_attention
from test_gpu_kv_cache import Pair
from test_gpu_attention import Pool, check_decode, check_prompt, generator, ints, normal, run_decode, run_prompt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = CudaContext(0)
    yield c
    c.close()


def as_left_behind(pool):
    """-1 behind every sequence's pages, as extend, fork, compact and free leave a table row."""
    table = pool.table.cpu().numpy()
    for s, n in enumerate(pool.lengths.cpu().numpy()):
        table[s, -(-int(n) // pool.page):] = -1
    pool.table.copy_(ints(table))
    return pool


# Sizes whose shared tokens go to blocks of 16 rows, to tiles, and to each sequence itself.
SHORT_FIRST = [
    # heads, kv heads, dim, page, batch, shared
    (4, 2, 64, 16, 32, 1056),
    (8, 1, 128, 64, 33, 512),
    (16, 2, 256, 16, 5, 480),
    (8, 2, 64, 16, 16, 8192),
    (40, 4, 128, 32, 20, 1056),
    (8, 2, 128, 16, 40, 4096),
    (8, 2, 256, 16, 16, 2048),
    (8, 2, 128, 16, 3, 128),
]


@pytest.mark.parametrize("heads,kv,dim,page,batch,shared", SHORT_FIRST)
@pytest.mark.parametrize("first", ["empty", "short", "outside", "half"])
@pytest.mark.parametrize("window", [0, 100])
def test_decode_first_sequence_without_the_shared_tokens(ctx, heads, kv, dim, page, batch, shared, first, window):
    """The shared pages come from a sequence that has them, whichever row of the batch that is:
    a first sequence that is empty, short or outside the table changes no other row."""
    lens = [shared + 7 * i % 40 for i in range(batch)]
    lens[0] = {"empty": 0, "short": 20, "outside": shared, "half": shared // 2}[first]
    lens[-1] = shared + 90
    pool = as_left_behind(Pool(ctx, torch.bfloat16, kv, dim, page, shared, lens, seed=batch))
    q = normal(generator(3), (batch, heads, dim), torch.bfloat16, 2.0)
    order = list(range(batch))
    if first == "outside":
        order[0] = batch + 5
        out, lse = run_decode(pool, q, 1, shared, max(lens), sequences=order, window=window)
        check_decode(pool, q[1:], 1, out[1:], lse[1:], sequences=order[1:], window=window)
        assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    else:
        out, lse = run_decode(pool, q, 1, shared, max(lens), window=window)
        check_decode(pool, q, 1, out, lse, window=window)


@pytest.mark.parametrize("heads,kv,dim,page,batch,shared", SHORT_FIRST)
def test_decode_shared_tokens_that_no_sequence_has_in_full(ctx, heads, kv, dim, page, batch, shared):
    """Every sequence ends inside the shared tokens, the longest of them in the middle of the
    batch; the last page of none is mapped."""
    lens = [(shared * (i + 1)) // (batch + 3) for i in range(batch)]
    lens[batch // 2] = shared - page - 3
    lens[0] = 0
    pool = as_left_behind(Pool(ctx, torch.bfloat16, kv, dim, page, shared, lens, seed=batch + 1))
    q = normal(generator(5), (batch, heads, dim), torch.bfloat16, 2.0)
    out, lse = run_decode(pool, q, 0, shared, shared)
    check_decode(pool, q, 0, out, lse)


def test_decode_after_a_row_of_the_batch_is_freed(ctx):
    """A finished sample keeps its place in the batch: its freed row gives zeros, the others
    what they gave before."""
    n, kv, dim, batch = 1060, 8, 128, 24
    cache = KvCache(ctx, type=N.BF16, layers=1, kv_heads=kv, head_dim=dim, page_tokens=16, pages=200,
                    max_sequences=batch + 1, max_pages=80)
    gen = generator(47)
    k, v = (normal(gen, (n, kv, dim), torch.bfloat16) for _ in range(2))
    row, count, off = ints([0]), ints([n]), ints(offsets([n]))
    cache.extend(row.data_ptr(), count.data_ptr(), 1)
    cache.write(0, k.data_ptr(), v.data_ptr(), row.data_ptr(), off.data_ptr(), 1, n)
    rows, parents = ints(range(1, batch + 1)), ints([0] * batch)
    cache.fork(parents.data_ptr(), rows.data_ptr(), batch)
    q = normal(gen, (batch, 32, dim), torch.bfloat16, 2.0)
    shared = n // 16 * 16
    size = cache.decode_workspace(32, batch, shared, n)
    work = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    results = []
    for step in range(2):
        out = torch.full_like(q, float("nan"))
        cache.decode_attention(layer=0, heads=32, q=q.data_ptr(), out=out.data_ptr(), batch=batch, max_length=n,
                               shared_tokens=shared, sequences=rows.data_ptr(), workspace=work.data_ptr(),
                               workspace_bytes=size)
        results.append(out)
        cache.free(rows.data_ptr(), 1)  # the first of the batch
    torch.cuda.synchronize()
    assert cache.status() == 0
    assert torch.equal(results[0][1:], results[1][1:]) and (results[1][0] == 0).all()
    cache.close()


def decode(pool, q, layer, shared, longest, **kw):
    """As run_decode, with the cache's status bits beside the results."""
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    n = pool.cache.decode_workspace(q.shape[1], q.shape[0], shared, longest)
    work = torch.full((max(n, 16),), 0xff, dtype=torch.uint8, device="cuda")
    args = dict(layer=layer, heads=q.shape[1], q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
                batch=q.shape[0], max_length=longest, shared_tokens=shared, workspace=work.data_ptr(),
                workspace_bytes=n)
    pool.cache.decode_attention(**{**args, **kw})
    torch.cuda.synchronize()
    return out, lse, pool.cache.status()


@pytest.mark.parametrize("heads,kv,dim,page,batch,shared", SHORT_FIRST)
@pytest.mark.parametrize("number", [-1, 1 << 30])
def test_decode_reports_pages_outside_the_pool(ctx, heads, kv, dim, page, batch, shared, number):
    lens = [shared + 3 + 11 * i % 70 for i in range(batch)]
    pool = as_left_behind(Pool(ctx, torch.float16, kv, dim, page, shared, lens, seed=batch + 2))
    q = normal(generator(7), (batch, heads, dim), torch.float16, 2.0)
    want, want_lse, status = decode(pool, q, 0, shared, max(lens))
    assert status == 0
    # a page of one sequence's own tokens: its row is told of, the others stay
    last = (lens[1] - 1) // page
    mapped = int(pool.table[1, last])
    pool.table[1, last] = number
    out, lse, status = decode(pool, q, 0, shared, max(lens))
    assert status == N.KV_BAD_TOKEN
    rest = [0] + list(range(2, batch))
    assert torch.equal(out[rest], want[rest]) and torch.equal(lse[rest], want_lse[rest])
    assert torch.isfinite(out[1]).all()
    pool.table[1, last] = mapped
    # a page of the shared tokens
    saved = pool.table.clone()
    pool.table[:, shared // page // 2] = number
    out, lse, status = decode(pool, q, 0, shared, max(lens))
    assert status == N.KV_BAD_TOKEN and torch.isfinite(out).all()
    # behind the end of every sequence: nobody asks
    pool.table.copy_(saved)
    pool.table[:, -1] = number
    out, lse, status = decode(pool, q, 0, shared, max(lens))
    assert status == 0 and torch.equal(out, want) and torch.equal(lse, want_lse)


# One key has nearly all the weight and a value of zero (an attention sink): the result is what
# the many others bring, each of a weight that f16 can hold only next to a larger reference.
# Weights are off by half of f16's last subnormal place at most, 2^-25, where the largest is 2^7
# (tiles) or 2^15: 2^-32 of the largest.
def sink_row(q, k, v, dtype):
    out, lse, bound, lse_bound = row(q, k, v, 1.0, EPS[dtype])
    s = k @ q
    places = len(s) * np.abs(v).max() / math.exp(lse - s.max())
    assert np.abs(out).min() > 100 * 2.0 ** -32 * places / len(s)
    return out, lse, bound + (2.0 ** -32 - 2.0 ** -25) * places, lse_bound


def sink_values(gen, n, gap, place, dim, dtype):
    """Keys whose scores under q = (4, 0, ...) are 0 for the sink and -gap to -gap - 1 else."""
    k, v = torch.zeros(n, dim, device="cuda"), 20 + 20 * torch.rand(n, dim, generator=gen, device="cuda")
    k[:, 0] = -(gap + torch.rand(n, generator=gen, device="cuda")) / 4
    k[place, 0], v[place] = 0.0, 0.0
    return k.to(dtype), v.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("gap,place", [(16, 0), (16, 9000), (19, 0), (19, 16383)])
def test_prompt_beside_a_sink(ctx, dtype, dim, gap, place):
    n, lq = 16384, 40
    k, v = sink_values(generator(dim), n, gap, place, dim, dtype)
    q = torch.zeros(lq, 2, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = 4.0
    for heads_stride in (dim, 0):  # tiles, and blocks of 16 rows
        out, lse = run_prompt(ctx, q, k[:, None], v[:, None], [lq], [n], causal=False, scale=1.0,
                              k_stride=(dim, heads_stride), v_stride=(dim, heads_stride))
        want = sink_row(to64(q[0, 0]), to64(k), to64(v), dtype)
        check_rows(out, lse, [((i, h), want) for i in range(lq) for h in range(2)], "sink")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("batch,heads,shared", [(16, 8, 12288), (2, 4, 12288), (1, 4, 0)])
def test_decode_beside_a_sink(ctx, dtype, dim, batch, heads, shared):
    n, page = 16384, 64
    pool = Pool(ctx, dtype, 1, dim, page, shared, [n] * batch, layers=1, seed=51)
    keys = []
    for b in range(batch):
        k, v = sink_values(generator(b), n, 17, 0, dim, dtype)
        if b and shared:
            k[:shared], v[:shared] = keys[0][0][:shared], keys[0][1][:shared]
        keys.append((k, v))
        ids = pool.table[b, :n // page].long()
        pool.memory[ids, 0, 0, 0], pool.memory[ids, 0, 1, 0] = k.view(-1, page, dim), v.view(-1, page, dim)
    q = torch.zeros(batch, heads, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = 4.0
    out, lse = run_decode(pool, q, 0, shared, n, scale=1.0)
    for b, (k, v) in enumerate(keys):
        want = sink_row(to64(q[b, 0]), to64(k), to64(v), dtype)
        check_rows(out, lse, [((b, h), want) for h in range(heads)], "sink")


@pytest.mark.parametrize("heads,kv,dim,page,batch,shared", SHORT_FIRST)
@pytest.mark.parametrize("broadcast", ["rows", "heads", "no"])
def test_decode_broadcast_queries(ctx, heads, kv, dim, page, batch, shared, broadcast):
    """One query row for the whole batch, one for all heads: whatever the sizes, the call runs
    (and gives what it gives for rows and heads apart)."""
    lens = [shared + 1 + 9 * i % 50 for i in range(batch)]
    pool = as_left_behind(Pool(ctx, torch.bfloat16, kv, dim, page, shared, lens, seed=batch + 3))
    gen = generator(9)
    if broadcast == "rows":
        q = normal(gen, (1, heads, dim), torch.bfloat16, 2.0).expand(batch, heads, dim)
        stride = (0, dim)
    elif broadcast == "heads":
        q = normal(gen, (batch, 1, dim), torch.bfloat16, 2.0).expand(batch, heads, dim)
        stride = (dim, 0)
    else:
        q = normal(gen, (batch, heads, dim), torch.bfloat16, 2.0)
        q = torch.empty(batch, heads, 2, dim, dtype=q.dtype, device="cuda")[:, :, 1].copy_(q)
        stride = q.stride()[:2]
    out, lse, status = decode(pool, q, 1, shared, max(lens), q_stride=stride, out_stride=(heads * dim, dim))
    assert status == 0
    check_decode(pool, q, 1, out, lse)


@pytest.mark.parametrize("heads,kv,dim,page,batch,shared", SHORT_FIRST + [(8, 2, 128, 16, 3, 0), (64, 8, 128, 64, 9, 0)])
def test_decode_without_a_bound_on_lengths(ctx, heads, kv, dim, page, batch, shared):
    """A max_length beyond the table is the table's: the same workspace and the same result."""
    lens = [shared + 1 + 9 * i % 50 for i in range(batch)]
    pool = as_left_behind(Pool(ctx, torch.bfloat16, kv, dim, page, shared, lens, seed=batch + 4))
    most = pool.columns * page
    need = pool.cache.decode_workspace(heads, batch, shared, most)
    q = normal(generator(11), (batch, heads, dim), torch.bfloat16, 2.0)
    want, want_lse, status = decode(pool, q, 0, shared, most)
    assert status == 0
    check_decode(pool, q, 0, want, want_lse)
    for bound in (most + 1, 1 << 20, 2 ** 31 - 100, 2 ** 31 - 1):
        assert pool.cache.decode_workspace(heads, batch, shared, bound) == need
        out, lse, status = decode(pool, q, 0, shared, bound)
        assert status == 0 and torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lq,lk", [([300], [20]), ([50, 9], [20, 0]), ([40], [400]), ([129, 1], [129, 1])])
def test_prompt_window_that_hides_nothing(ctx, dim, causal, lq, lk):
    """However wide the window, also where queries stand before the first key."""
    gen = generator(dim)
    q = normal(gen, (sum(lq), 4, dim), torch.bfloat16, 2.0)
    k, v = (normal(gen, (max(1, sum(lk)), 1, dim), torch.bfloat16) for _ in range(2))
    for heads_stride in (dim, 0):  # tiles, and blocks of 16 rows
        strides = dict(k_stride=(dim, heads_stride), v_stride=(dim, heads_stride))
        want, want_lse = run_prompt(ctx, q, k, v, lq, lk, causal, 0, **strides)
        for window in (sum(lk) + sum(lq) + 1, 2 ** 31 - 300, 2 ** 31 - 10, 2 ** 31 - 1):
            out, lse = run_prompt(ctx, q, k, v, lq, lk, causal, window, **strides)
            assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_more_tokens_than_kernels_can_count_are_refused(ctx):
    """Kernels step past the last token in 32 bits; the limit leaves them room."""
    with pytest.raises(DmError) as e:
        KvCache(ctx, type=N.BF16, layers=1, kv_heads=1, head_dim=8, page_tokens=16, pages=4, max_sequences=1,
                max_pages=(1 << 27) - 1)
    assert e.value.status == N.ERR_OVERFLOW
    t, o = torch.zeros(16, 8, dtype=torch.bfloat16, device="cuda"), ints([0, 1])
    p = t.data_ptr()
    with pytest.raises(DmError) as e:
        prompt_attention(ctx, type=N.BF16, heads=1, kv_heads=1, head_dim=8, q=p, k=p, v=p, out=p, q_tokens=16,
                         k_tokens=16, sequences=(1 << 20) + 1, q_offsets=o.data_ptr())
    assert e.value.status == N.ERR_ELEMENT_COUNT
    for q_tokens, k_tokens in ((2 ** 31 - 4096, 16), (16, 2 ** 31 - 1)):
        with pytest.raises(DmError) as e:
            prompt_attention(ctx, type=N.BF16, heads=1, kv_heads=1, head_dim=8, q=p, k=p, v=p, out=p,
                             q_tokens=q_tokens, k_tokens=k_tokens, sequences=1, q_offsets=o.data_ptr())
        assert e.value.status == N.ERR_ELEMENT_COUNT


@pytest.mark.parametrize("lq", [1, 130])
def test_prompt_over_more_keys_than_a_wait_lasts(ctx, lq):
    """40 million keys, a quarter of a second: a role that waits for the whole item is not to
    give up (a limit of 0.1 s holds for a tile). All scores are 0 and values whole numbers that
    16 keys share, so every sum is exact: partial sums are multiples of 16 below 2^28."""
    n, dim = 40_000_000, 8
    k = torch.zeros(n, 1, dim, dtype=torch.bfloat16, device="cuda")
    gen = generator(lq)
    v = torch.randint(0, 4, (n // 16, 1, dim), generator=gen, device="cuda").to(torch.bfloat16)
    v = v.repeat_interleave(16, 0)
    q = normal(gen, (lq, 1, dim), torch.bfloat16)
    out, lse = run_prompt(ctx, q, k, v, [lq], [n], causal=False)
    attention_status(ctx)
    want = v[:, 0].double().mean(0)
    assert ((out[:, 0].double() - want).abs() <= 1.01 * EPS[torch.bfloat16] * want).all()
    assert (lse - math.log(n)).abs().max() <= 2.0 ** -19 * math.log(n)


def test_a_wait_elsewhere_on_the_context_is_not_attentions(ctx):
    """The self-test of bounded waits runs one out: the attention status does not tell of it."""
    assert N.lib().dm_selftest_device_wait(ctx.handle, 100_000) == N.ERR_TIMEOUT
    attention_status(ctx)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (7, 1, 96), (6, 2, 128), (4, 2, 256)])
def test_prompt_heads_first(ctx, heads, kv, dim, dtype):
    """q, k, v and out as [heads, tokens, dim], and with rows that are part of wider ones."""
    gen = generator(61)
    lens, n = [140, 1, 333], 474
    q = normal(gen, (heads, n, dim), dtype, 2.0).transpose(0, 1)
    k, v = (normal(gen, (kv, n, dim + 8), dtype)[:, :, 8:].transpose(0, 1) for _ in range(2))
    out = torch.full((heads, n, dim + 24), float("nan"), dtype=dtype, device="cuda")[:, :, 16:16 + dim].transpose(0, 1)
    for causal, window in ((True, 0), (False, 0), (True, 50)):
        got, lse = run_prompt(ctx, q, k, v, lens, lens, causal, window, out=out)
        check_prompt(q, k, v, lens, lens, got, lse, causal, window, tokens=16)
        flat, flat_lse = run_prompt(ctx, q.contiguous(), k.contiguous(), v.contiguous(), lens, lens, causal, window)
        assert torch.equal(got, flat) and torch.equal(lse, flat_lse)


@pytest.mark.parametrize("at", [0, 30000, 79999])
def test_prompt_among_very_many_empty_sequences(ctx, at):
    """Finding the one sequence that has tokens takes longer than a wait may last."""
    lens = [0] * 80000
    lens[at] = 200
    gen = generator(67)
    q, k, v = (normal(gen, (200, 1, 64), torch.bfloat16) for _ in range(3))
    out, lse = run_prompt(ctx, q, k, v, lens, lens)
    attention_status(ctx)
    check_prompt(q, k, v, [200], [200], out, lse)


# Limits in clocks: from waits that all run out to a few that do.
LIMITS = (1, 300, 1000, 2000, 3000, 5000, 8000, 12000, 20000, 50000, 200000)


def out_of_time(ctx, run, want):
    """`run` at every limit: a call whose waits held gives `want`, another says so, and the one
    after it, with the limit as built, is right again. The calls that ran out of time."""
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
@pytest.mark.parametrize("lens", [[1], [700, 3, 260], [2500] * 12])
def test_prompt_out_of_time(ctx, dim, lens):
    gen = generator(dim)
    q = normal(gen, (sum(lens), 8, dim), torch.bfloat16, 2.0)
    k, v = (normal(gen, (sum(lens), 2, dim), torch.bfloat16) for _ in range(2))
    late = out_of_time(ctx, lambda: run_prompt(ctx, q, k, v, lens, lens), run_prompt(ctx, q, k, v, lens, lens))
    # a warp sleeps before it looks at the clock: shorter calls are done by then
    assert late > 0 or sum(lens) < 10000


@pytest.mark.parametrize("heads,kv,dim,page,batch,shared", SHORT_FIRST)
def test_decode_out_of_time(ctx, heads, kv, dim, page, batch, shared):
    lens = [shared + 1 + 37 * i % 900 for i in range(batch)]
    pool = Pool(ctx, torch.float16, kv, dim, page, shared, lens, seed=batch)
    q = normal(generator(13), (batch, heads, dim), torch.float16, 2.0)
    late = out_of_time(ctx, lambda: run_decode(pool, q, 0, shared, max(lens)), run_decode(pool, q, 0, shared, max(lens)))
    # where a warp has two copies to wait for, both may be there before it asks
    assert late > 0 or shared == 480


def test_limits_of_a_wait_are_checked(ctx):
    assert N.lib().dm_selftest_attention_wait(None, 10) == N.ERR_INVALID_ARGUMENT
    assert N.lib().dm_selftest_attention_wait(ctx.handle, -1) == N.ERR_INVALID_ARGUMENT
    assert N.lib().dm_selftest_attention_wait(ctx.handle, 1 << 40) == N.ERR_INVALID_ARGUMENT


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------

BAD_KEEPS = {
    "behind the end": lambda n: list(range(1, n - 1)) + [n],
    "far behind the end": lambda n: list(range(0, 20)) + [2 ** 31 - 1],
    "negative": lambda n: [-1] + list(range(1, 30)),
    "twice": lambda n: list(range(0, 33)) + [32] + list(range(40, n)),
    "down": lambda n: list(range(0, 17)) + [20, 19] + list(range(25, n)),
    "first two": lambda n: [1, 0] + list(range(2, n)),
    "last two": lambda n: list(range(0, n - 2)) + [n - 1, n - 2],
    "out of range between": lambda n: list(range(0, 17)) + [n + 5] + list(range(18, n)),
    "negative between": lambda n: list(range(0, 17)) + [-7] + list(range(18, n)),
}


@pytest.mark.parametrize("case", BAD_KEEPS)
@pytest.mark.parametrize("others", [0, 1, 2, 40])
def test_compact_refuses_tokens_out_of_range_or_order(ctx, case, others):
    """Nothing of the call is done, whichever of its lists is wrong."""
    t = Pair(ctx, layers=1, kv=1, dim=8, pages=900, seqs=48, max_pages=12)
    n = 150
    assert t.extend(list(range(41)), [n] * 41)
    t.check()
    good = [list(range(3, n, 2)) for _ in range(others)]
    for place in sorted({0, others // 2, others}):
        keeps = good[:place] + [BAD_KEEPS[case](n)] + good[place:]
        s, o, k = ints(range(len(keeps))), ints(offsets([len(x) for x in keeps])), ints(np.concatenate(keeps))
        t.cache.compact(s.data_ptr(), o.data_ptr(), k.data_ptr(), len(keeps), k.numel())
        t.check(status=N.KV_BAD_TOKEN)


def test_compact_of_lists_that_meet_in_any_way(ctx):
    """What one list ends with says nothing about the next: empty lists between, at both ends,
    equal tokens on both sides."""
    t = Pair(ctx, layers=1, kv=1, dim=8, pages=200, seqs=12, max_pages=12)
    assert t.extend(list(range(12)), [100] * 12)
    keeps = [[], [99], [99], [0], [], [], list(range(50, 100)), list(range(50, 100)), [0, 99], [99], list(range(100)), []]
    assert t.compact(list(range(12)), keeps)
    t.check()


def test_compact_long_lists(ctx):
    """More kept tokens than one step of the check takes; a fault in each of its last places."""
    t = Pair(ctx, layers=1, kv=1, dim=8, page=256, pages=300, seqs=3, max_pages=60)
    n = 14000
    assert t.extend([0, 1], [n, n])
    keep = list(range(5, n))
    s, o = ints([0, 1]), ints(offsets([len(keep)] * 2))
    for at in (1, 1023, 4096, 5 * 1024, len(keep) - 2):
        bad = list(keep)
        bad[at] = bad[at - 1]
        k = ints(keep + bad)
        t.cache.compact(s.data_ptr(), o.data_ptr(), k.data_ptr(), 2, k.numel())
        t.check(status=N.KV_BAD_TOKEN)
    assert t.compact([0, 1], [keep, keep])
    t.check()


def test_calls_that_do_what_can_be_done(ctx):
    """Free, write and copy_pages pass over what is out of range."""
    t = Pair(ctx, seqs=6)
    assert t.extend([0, 1, 2], [20, 20, 20])
    rows = [torch.randint(-30000, 30000, (9, 2, 64), dtype=torch.int16, device="cuda") for _ in range(2)]
    s, o = ints([1, 9, 0]), ints([0, 3, 6, 9])
    t.cache.write(1, rows[0].data_ptr(), rows[1].data_ptr(), s.data_ptr(), o.data_ptr(), 3, 9)
    kept = [torch.cat([x[:3], x[6:]]).cpu().numpy().view(np.uint16) for x in rows]
    t.plain.write(1, *kept, [1, 0], [0, 3, 6])
    t.check(status=N.KV_BAD_TOKEN)
    src, dst = ints([0, 40, 1, -1]), ints([30, 31, 32, 33])
    t.cache.copy_pages(src.data_ptr(), dst.data_ptr(), 4)
    t.plain.pool[[30, 32]] = t.plain.pool[[0, 1]]
    t.check(status=N.KV_BAD_TOKEN)
    s = ints([0, 6, 2, 0])
    t.cache.free(s.data_ptr(), 4)
    t.plain.free([0, 2])
    t.check(status=N.KV_BAD_SEQUENCE)


def test_more_pages_asked_for_than_32_bits_count(ctx):
    """Entries that each fit their row of the table and together ask for more than 2^31 pages."""
    rows, most, pages = 17, 134217471, 40
    with pytest.raises(DmError) as e:
        KvCache(ctx, type=N.BF16, layers=1, kv_heads=1, head_dim=8, page_tokens=16, pages=(1 << 30) + 1,
                max_sequences=1, max_pages=1)
    assert e.value.status == N.ERR_OVERFLOW
    cache = KvCache(ctx, type=N.BF16, layers=1, kv_heads=1, head_dim=8, page_tokens=16, pages=pages,
                    max_sequences=rows, max_pages=most)  # a table of 9 GB
    s, c = ints(range(rows)), ints([most * 16] * rows)
    assert rows * most > 2 ** 31
    for n in range(1, rows + 1):
        cache.extend(s.data_ptr(), c.data_ptr(), n)
        assert cache.status() == N.KV_OUT_OF_PAGES
    c = ints([16] * rows)
    cache.extend(s.data_ptr(), c.data_ptr(), rows)
    assert cache.status() == 0
    cache.close()


@pytest.mark.parametrize("n,max_pages,dim", [(1, 16384, 8), (1, 16385, 8), (16, 1024, 8), (16, 1025, 8), (17, 4, 8),
                                             (16, 4, 256), (9, 40, 80), (70, 300, 64)])
def test_forks_on_both_sides_of_the_small_ones(ctx, n, max_pages, dim):
    """Done by the plan's block, or by a kernel behind it: the same tables and rows."""
    t = Pair(ctx, layers=2, kv=1, dim=dim, pages=10 * n + 9, seqs=2 * n, max_pages=max_pages)
    assert t.extend(list(range(n)), [int(x) for x in t.r.randint(0, 49, n)])
    t.write(1, list(range(n)), [int(x) for x in t.plain.lengths[:n]])
    order = [int(x) for x in t.r.randint(0, n, n)]
    assert t.fork(order, list(range(2 * n - 1, n - 1, -1)))
    t.check()
