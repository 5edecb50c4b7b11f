"""dm_attention_prompt and dm_attention_decode against attention written out in 64 bits."""
import math

import numpy as np
import pytest
import torch

from attention_plain import EPS, check_rows, row, to64
from diskmule_b200 import CudaContext, DmError, _native as N
from diskmule_b200.attention import KvCache, offsets, prompt_attention

pytestmark = pytest.mark.gpu

KIND = {torch.bfloat16: N.BF16, torch.float16: N.F16}


@pytest.fixture(scope="module")
def ctx():
    c = CudaContext(0)
    yield c
    c.close()


def ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def sees(i, lq, lk, causal, window):
    place = i + lk - lq
    high = max(0, min(lk, place + 1)) if causal else lk
    low = max(0, place - window + 1) if window else 0
    return low, max(low, high)


def run_prompt(ctx, q, k, v, lq, lk, causal=True, window=0, scale=0.0, out=None, k_offsets=True, **kw):
    heads, dim = q.shape[1], q.shape[2]
    out = torch.full_like(q, float("nan")) if out is None else out
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    qo, ko = ints(offsets(lq)), ints(offsets(lk))
    strides = {n + "_stride": (t.stride(0), t.stride(1)) for n, t in (("q", q), ("k", k), ("v", v), ("out", out))}
    strides.update(kw)
    prompt_attention(ctx, type=KIND[q.dtype], heads=heads, kv_heads=k.shape[1], head_dim=dim,
                     q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
                     lse=lse.data_ptr(), q_tokens=q.shape[0], k_tokens=k.shape[0],
                     sequences=len(lq), q_offsets=qo.data_ptr(),
                     k_offsets=ko.data_ptr() if k_offsets else 0, causal=causal, window=window,
                     scale=scale, **strides)
    torch.cuda.synchronize()
    return out, lse


def check_prompt(q, k, v, lq, lk, out, lse, causal=True, window=0, scale=0.0, tokens=None):
    """Every row, or those of `tokens` tokens of each sequence."""
    heads, g = q.shape[1], q.shape[1] // k.shape[1]
    scale = scale or 1.0 / math.sqrt(q.shape[2])
    Q, K, V = to64(q), to64(k), to64(v)
    rows, q0, k0 = [], 0, 0
    for a, b in zip(lq, lk):
        some = range(a) if tokens is None or a <= tokens else sorted(
            {0, 1, a - 1, a // 2} | {int(x) for x in np.random.RandomState(a).randint(0, a, tokens)})
        for i in some:
            low, high = sees(i, a, b, causal, window)
            for h in range(heads):
                rows.append(((q0 + i, h), row(Q[q0 + i, h], K[k0 + low:k0 + high, h // g],
                                              V[k0 + low:k0 + high, h // g], scale, EPS[q.dtype])))
        q0, k0 = q0 + a, k0 + b
    check_rows(out, lse, rows, "prompt")


PROMPTS = [
    # lengths of queries, of keys, heads, kv heads, dim, causal, window
    ([1], [1], 1, 1, 64, True, 0),
    ([3, 17, 1, 40], None, 8, 2, 64, True, 0),
    ([127, 128, 129], None, 4, 4, 128, True, 0),
    ([255, 0, 257, 0], None, 4, 2, 128, True, 0),          # empty sequences, also at the end
    ([0, 33], None, 6, 2, 80, True, 0),
    ([200], None, 7, 1, 96, True, 0),                      # a group that does not divide a tile
    ([70, 130], None, 5, 1, 128, False, 0),
    ([300], None, 2, 1, 256, True, 0),
    ([140, 10], None, 6, 2, 192, True, 0),
    ([400, 65], None, 4, 1, 64, True, 100),
    ([300], None, 8, 2, 256, True, 64),
    ([300, 20], None, 2, 2, 128, True, 1),                 # a window of the token itself
    ([10, 64, 1], [500, 64, 333], 8, 1, 128, True, 0),     # continued prompts
    ([50, 9], [20, 0], 4, 2, 128, True, 0),                # more queries than keys: empty rows
    ([50, 9], [20, 0], 4, 2, 128, False, 0),
    ([30], [400], 4, 2, 64, True, 37),
    ([30, 20], [400, 15], 4, 2, 128, False, 50),
    ([4] * 70, None, 16, 1, 64, True, 0),                  # more sequences than a warp's lanes
    ([20], [300], 128, 1, 64, True, 0),                    # the widest group
    ([1], [700], 2, 2, 8, True, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lq,lk,heads,kv,dim,causal,window", PROMPTS)
def test_prompt(ctx, lq, lk, heads, kv, dim, causal, window, dtype):
    lk = lk or lq
    gen = generator(sum(lq) + dim)
    q = normal(gen, (sum(lq), heads, dim), dtype, 2.0)
    k, v = normal(gen, (sum(lk), kv, dim), dtype), normal(gen, (sum(lk), kv, dim), dtype)
    out, lse = run_prompt(ctx, q, k, v, lq, lk, causal, window)
    check_prompt(q, k, v, lq, lk, out, lse, causal, window, tokens=24)


@pytest.mark.parametrize("lq,lk,heads,kv,dim,window", [
    ([2500, 1300], None, 8, 2, 128, 0), ([4100], None, 4, 1, 64, 0), ([1900], None, 2, 1, 256, 512),
    ([600], [3000], 14, 2, 128, 0), ([5], [6000], 8, 1, 128, 0)])
def test_prompt_long(ctx, lq, lk, heads, kv, dim, window):
    lk = lk or lq
    gen = generator(7)
    q = normal(gen, (sum(lq), heads, dim), torch.bfloat16, 2.0)
    k, v = (normal(gen, (sum(lk), kv, dim), torch.bfloat16) for _ in range(2))
    out, lse = run_prompt(ctx, q, k, v, lq, lk, True, window)
    check_prompt(q, k, v, lq, lk, out, lse, True, window, tokens=10)


def test_prompt_same_offsets_no_lse_and_scale(ctx):
    gen = generator(3)
    lens = [60, 131]
    q = normal(gen, (191, 4, 64), torch.bfloat16)
    k, v = (normal(gen, (191, 2, 64), torch.bfloat16) for _ in range(2))
    out, lse = run_prompt(ctx, q, k, v, lens, lens, scale=0.5, k_offsets=False)
    check_prompt(q, k, v, lens, lens, out, lse, scale=0.5, tokens=16)
    again = torch.empty_like(q)
    o = ints(offsets(lens))
    prompt_attention(ctx, type=N.BF16, heads=4, kv_heads=2, head_dim=64, q=q.data_ptr(),
                     k=k.data_ptr(), v=v.data_ptr(), out=again.data_ptr(), q_tokens=191,
                     k_tokens=191, sequences=2, q_offsets=o.data_ptr(), scale=0.5)
    torch.cuda.synchronize()
    assert torch.equal(out, again)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_growing_scores(ctx, dim):
    """Scores that rise from key to key, so that the running maximum never settles, and
    some that fall: the sums are rescaled again and again."""
    n = 700
    gen = generator(dim)
    q = torch.zeros(n, 2, dim, dtype=torch.bfloat16, device="cuda")
    q[:, 0, 0], q[:, 1, 0] = 16.0, -16.0
    k = normal(gen, (n, 1, dim), torch.bfloat16)
    k[:, 0, 0] = torch.linspace(-40, 40, n, device="cuda").to(torch.bfloat16)
    v = normal(gen, (n, 1, dim), torch.bfloat16)
    out, lse = run_prompt(ctx, q, k, v, [n], [n], scale=1.0)
    check_prompt(q, k, v, [n], [n], out, lse, scale=1.0, tokens=40)


def test_prompt_strides(ctx):
    """q, k and v as views of one fused projection, out with its heads first."""
    gen = generator(11)
    n, heads, kv, dim = 211, 6, 2, 128
    fused = normal(gen, (n, (heads + 2 * kv) * dim + 24), torch.float16)
    q = fused[:, 8:8 + heads * dim].view(n, heads, dim)
    k = fused[:, 8 + heads * dim:8 + (heads + kv) * dim].view(n, kv, dim)
    v = fused[:, 8 + (heads + kv) * dim:8 + (heads + 2 * kv) * dim].view(n, kv, dim)
    out = torch.full((heads, n, dim), float("nan"), dtype=torch.float16, device="cuda").transpose(0, 1)
    out, lse = run_prompt(ctx, q, k, v, [100, 111], [100, 111], out=out)
    check_prompt(q, k, v, [100, 111], [100, 111], out, lse, tokens=16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("wild", [float("nan"), float("inf"), -float("inf"), None])
def test_prompt_hidden_values_have_no_influence(ctx, dtype, dim, wild):
    """What later tokens, tokens behind the window and other sequences hold does not reach a
    row: its bits stay when those change to NaN, infinities or the type's lowest value."""
    wild = torch.finfo(dtype).min if wild is None else wild
    lens = [150, 90, 200]
    gen = generator(17)
    n = sum(lens)
    q = normal(gen, (n, 4, dim), dtype, 2.0)
    k, v = (normal(gen, (n, 2, dim), dtype) for _ in range(2))
    for causal, window in ((True, 0), (True, 40), (False, 0)):
        out, lse = run_prompt(ctx, q, k, v, lens, lens, causal, window)
        for key in (0, 7, 149, 150, 200, 240, 439):
            k2, v2 = k.clone(), v.clone()
            k2[key], v2[key] = wild, wild
            out2, lse2 = run_prompt(ctx, q, k2, v2, lens, lens, causal, window)
            hidden = []
            for a, q0 in zip(lens, offsets(lens)):
                for i in range(a):
                    low, high = sees(i, a, a, causal, window)
                    if not (q0 + low <= key < q0 + high):
                        hidden.append(int(q0) + i)
            assert torch.equal(out[hidden], out2[hidden]) and torch.equal(lse[hidden], lse2[hidden])


def test_prompt_visible_nan_and_infinity_show(ctx):
    gen = generator(5)
    n = 300
    q = normal(gen, (n, 2, 128), torch.bfloat16)
    k, v = (normal(gen, (n, 1, 128), torch.bfloat16) for _ in range(2))
    v[130, 0, 5], v[7, 0, 9] = float("nan"), float("inf")
    out, lse = run_prompt(ctx, q, k, v, [n], [n])
    assert torch.isnan(out[130:, :, 5]).all() and not torch.isnan(out[:130]).any()
    assert (out[7:, :, 9] == float("inf")).all() and not torch.isinf(out[:7]).any()
    assert torch.isfinite(lse).all()
    k[40, 0, 3] = float("nan")
    out, lse = run_prompt(ctx, q, k, v, [n], [n])
    assert torch.isnan(lse[40:]).all() and torch.isfinite(lse[:40]).all()
    assert torch.isnan(out[40:]).all()


def test_prompt_on_another_stream(ctx):
    gen = generator(23)
    q = normal(gen, (500, 4, 64), torch.bfloat16)
    k, v = (normal(gen, (500, 4, 64), torch.bfloat16) for _ in range(2))
    want, _ = run_prompt(ctx, q, k, v, [500], [500])
    side = torch.cuda.Stream()
    out = torch.zeros_like(q)
    o = ints([0, 500])
    side.wait_stream(torch.cuda.current_stream())
    prompt_attention(ctx, type=N.BF16, heads=4, kv_heads=4, head_dim=64, q=q.data_ptr(),
                     k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), q_tokens=500,
                     k_tokens=500, sequences=1, q_offsets=o.data_ptr(), stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want)


def test_prompt_offsets_beyond_the_tensors_are_clamped(ctx):
    gen = generator(29)
    q = normal(gen, (100, 2, 64), torch.bfloat16)
    k, v = (normal(gen, (100, 2, 64), torch.bfloat16) for _ in range(2))
    want, _ = run_prompt(ctx, q, k, v, [60, 40], [60, 40])
    out = torch.zeros_like(q)
    o = ints([0, 60, 4000])
    prompt_attention(ctx, type=N.BF16, heads=2, kv_heads=2, head_dim=64, q=q.data_ptr(),
                     k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), q_tokens=100,
                     k_tokens=100, sequences=2, q_offsets=o.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(out, want)


# ---------------------------------------------------------------------------
# decode
# ---------------------------------------------------------------------------

class Pool:
    """A cache whose sequences share their first `shared` tokens, pages in random order."""

    def __init__(self, ctx, dtype, kv, dim, page, shared, lens, layers=2, seed=0, junk=None):
        gen = generator(seed)
        r = np.random.RandomState(seed)
        lens = np.asarray(lens)
        need = [max(0, -(-int(n) // page) - shared // page) for n in lens]
        pages = shared // page + sum(need) + 2
        order = r.permutation(pages)
        self.columns = shared // page + max(need) + 1
        table = np.full((len(lens), self.columns), -1)
        at = shared // page
        for i, n in enumerate(need):
            table[i, :shared // page] = order[:shared // page]
            table[i, shared // page:shared // page + n] = order[at:at + n]
            at += n
        self.memory = normal(gen, (pages, layers, 2, kv, page, dim), dtype)
        if junk is not None:  # in every row that no sequence uses
            used = np.zeros((pages, page), bool)
            for i, n in enumerate(lens):
                for j in range(int(n)):
                    used[table[i, j // page], j % page] = True
            mask = torch.tensor(~used, device="cuda")[:, None, None, None, :, None]
            self.memory.masked_fill_(mask, junk)
        self.table, self.lengths = ints(table), ints(lens)
        self.references = ints(np.ones(pages))
        self.page, self.kv, self.dim = page, kv, dim
        self.cache = KvCache(ctx, type=KIND[dtype], layers=layers, kv_heads=kv, head_dim=dim,
                             page_tokens=page, pages=pages, max_sequences=len(lens),
                             max_pages=self.columns, memory=self.memory.data_ptr(),
                             page_table=self.table.data_ptr(), lengths=self.lengths.data_ptr(),
                             references=self.references.data_ptr())

    def tokens(self, layer, s):
        n = int(self.lengths[s])
        ids = self.table[s, :-(-n // self.page)].long()
        flat = to64(self.memory[ids, layer]).transpose(1, 2, 0, 3, 4)
        flat = flat.reshape(2, self.kv, -1, self.dim)[:, :, :n]
        return flat[0], flat[1]


def run_decode(pool, q, layer, shared, longest, sequences=None, window=0, scale=0.0, out=None):
    out = torch.full_like(q, float("nan")) if out is None else out
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    n = pool.cache.decode_workspace(q.shape[1], q.shape[0], shared, longest)
    work = torch.full((max(n, 16),), 0xff, dtype=torch.uint8, device="cuda")  # NaN in every type
    rows = None if sequences is None else ints(sequences)
    pool.cache.decode_attention(
        layer=layer, heads=q.shape[1], q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
        batch=q.shape[0], max_length=longest, shared_tokens=shared,
        sequences=0 if rows is None else rows.data_ptr(), window=window, scale=scale,
        q_stride=(q.stride(0), q.stride(1)), out_stride=(out.stride(0), out.stride(1)),
        workspace=work.data_ptr(), workspace_bytes=n)
    torch.cuda.synchronize()
    assert pool.cache.status() == 0
    return out, lse


def check_decode(pool, q, layer, out, lse, sequences=None, window=0, scale=0.0, cut=None):
    g = q.shape[1] // pool.kv
    scale = scale or 1.0 / math.sqrt(pool.dim)
    Q, rows = to64(q), []
    for b in range(q.shape[0]):
        K, V = pool.tokens(layer, b if sequences is None else sequences[b])
        n = K.shape[1] if cut is None else min(cut, K.shape[1])
        low = max(0, n - window) if window else 0
        for h in range(q.shape[1]):
            rows.append(((b, h), row(Q[b, h], K[h // g, low:n], V[h // g, low:n], scale, EPS[q.dtype])))
    check_rows(out, lse, rows, "decode")


DECODES = [
    # heads, kv heads, dim, page, shared, lengths
    (1, 1, 64, 16, 0, [1]),
    (8, 2, 64, 16, 160, [161, 200]),
    (4, 4, 128, 32, 0, [1, 31, 32, 33, 700, 5]),
    (8, 1, 128, 16, 64, [64, 65, 300, 64]),                # nothing of their own
    (16, 2, 128, 64, 512, [600, 513, 1000, 512, 777]),
    (5, 1, 80, 16, 48, [50, 90]),
    (12, 2, 256, 16, 96, [100, 333, 97]),
    (40, 2, 192, 32, 64, [64, 200]),                       # more than 16 rows per head
    (8, 2, 128, 128, 256, [300] * 9 + [256]),
    (8, 1, 64, 256, 1024, [1025 + 13 * i for i in range(40)]),
    (64, 8, 128, 16, 320, [321 + 7 * i for i in range(11)]),
    (2, 2, 8, 16, 16, [17, 40]),
    (128, 1, 64, 16, 32, [33, 70, 40]),
    (24, 1, 256, 64, 640, [650 + i for i in range(12)]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,dim,page,shared,lens", DECODES)
def test_decode(ctx, heads, kv, dim, page, shared, lens, dtype):
    pool = Pool(ctx, dtype, kv, dim, page, shared, lens, seed=heads + dim, junk=float("nan"))
    q = normal(generator(1), (len(lens), heads, dim), dtype, 2.0)
    for layer in (0, 1):
        out, lse = run_decode(pool, q, layer, shared, max(lens))
        check_decode(pool, q, layer, out, lse)


@pytest.mark.parametrize("shared,lens,kv,heads", [
    (8192, [8192 + 3, 9000, 8300, 8192], 2, 16), (0, [20000], 1, 4),
    (4096, [4097 + 50 * i for i in range(33)], 1, 8), (16384, [16384 + 1], 1, 1)])
def test_decode_long(ctx, shared, lens, kv, heads):
    pool = Pool(ctx, torch.bfloat16, kv, 128, 64, shared, lens, layers=1, seed=3)
    q = normal(generator(2), (len(lens), heads, 128), torch.bfloat16, 2.0)
    out, lse = run_decode(pool, q, 0, shared, max(lens))
    check_decode(pool, q, 0, out, lse)


# Shared parts of more rows and tokens than blocks of 16 rows take: tiles of 128 rows.
DECODES_ON_TILES = [
    # heads, kv heads, dim, page, shared, lengths
    (64, 2, 64, 16, 4224, [4224 + 31 * i for i in range(7)]),
    (40, 4, 128, 32, 1056, [1056 + 9 * i for i in range(20)]),
    (24, 8, 128, 16, 640, [641 + 40 * i for i in range(22)]),
    (5, 1, 80, 16, 4000, [4001 + i for i in range(33)]),
    (12, 2, 200, 16, 1600, [1600 + 3 * i for i in range(20)]),
    (24, 1, 256, 64, 1280, [1281 + 100 * (i % 5) for i in range(12)]),
    (8, 1, 256, 128, 4096, [4100 + i for i in range(16)]),     # one tile's rows
    (128, 1, 64, 256, 8192, [8192, 8200, 8500]),
    (4, 1, 8, 16, 49984, [49984 + 2 * i for i in range(33)]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,dim,page,shared,lens", DECODES_ON_TILES)
def test_decode_on_tiles(ctx, heads, kv, dim, page, shared, lens, dtype):
    pool = Pool(ctx, dtype, kv, dim, page, shared, lens, seed=heads + dim, junk=float("nan"))
    q = normal(generator(1), (len(lens), heads, dim), dtype, 2.0)
    out, lse = run_decode(pool, q, 1, shared, max(lens))
    check_decode(pool, q, 1, out, lse)


@pytest.mark.parametrize("dim,shared", [(64, 8192), (128, 4096), (256, 2048)])
@pytest.mark.parametrize("window", [0, 1, 30, 700, 100000])
def test_decode_on_tiles_empty_short_and_reordered_sequences(ctx, dim, shared, window):
    """Lengths of zero, inside the shared tokens, at their end and behind it, in any order;
    windows that end before, in and behind the shared tokens."""
    lens = [shared + 70, shared, 0, 50, shared + 9, shared + 300, shared - 1, 1] + [shared + 20] * 8
    pool = Pool(ctx, torch.bfloat16, 2, dim, 16, shared, lens, seed=9)
    order = [5, 0, 2, 4, 4, 3, 1, 6, 7, 9, 8, 10, 11, 12, 13, 14]
    q = normal(generator(4), (len(order), 8, dim), torch.bfloat16, 2.0)
    out, lse = run_decode(pool, q, 1, shared, max(lens), sequences=order, window=window)
    check_decode(pool, q, 1, out, lse, sequences=order, window=window)
    assert (out[2] == 0).all() and torch.isinf(lse[2]).all()


@pytest.mark.parametrize("dim,shared", [(64, 8192), (128, 4096), (256, 2048)])
@pytest.mark.parametrize("wild", [float("nan"), float("inf"), None])
def test_decode_on_tiles_hidden_values_have_no_influence(ctx, dim, shared, wild):
    """Shared tokens that a shorter sequence or a window does not see, and what those see
    that do."""
    wild = torch.finfo(torch.bfloat16).min if wild is None else wild
    lens = [shared + 30, 100, shared + 5, shared] + [shared] * 12
    pool = Pool(ctx, torch.bfloat16, 2, dim, 16, shared, lens, seed=18)
    pool.lengths[1] = 100
    q = normal(generator(10), (16, 8, dim), torch.bfloat16, 2.0)
    for window in (0, 150):
        want, want_lse = run_decode(pool, q, 0, shared, max(lens), window=window)
        saved = pool.memory.clone()
        for key in (100, 104, shared - 1):
            page = int(pool.table[0, key // 16])
            pool.memory[page, 0, :, :, key % 16] = wild
        out, lse = run_decode(pool, q, 0, shared, max(lens), window=window)
        assert torch.equal(out[1], want[1]) and torch.equal(lse[1], want_lse[1])
        assert not torch.equal(out[3], want[3])
        if not math.isfinite(wild):
            assert not torch.isfinite(out[3]).any()
        pool.memory.copy_(saved)
        # a value alone, seen by all but the short sequence: its column, no other
        page = int(pool.table[0, (shared - 20) // 16])
        pool.memory[page, 0, 1, 1, (shared - 20) % 16, 5] = float("inf")
        out, lse = run_decode(pool, q, 0, shared, max(lens), window=window)
        assert torch.equal(lse, want_lse) and torch.equal(out[1], want[1])
        other = torch.ones_like(out, dtype=torch.bool)
        other[:, 4:, 5] = False
        assert torch.equal(out[other], want[other])
        assert (out[[0, 2, 3] + list(range(4, 16)), 4:, 5] == float("inf")).all()
        pool.memory.copy_(saved)


# Shared parts on blocks of 16 rows: joined by the blocks of the own part, or behind them.
DECODES_ON_ROWS = [
    # heads, kv heads, dim, page, shared, lengths
    (4, 2, 64, 16, 1056, [1057 + 3 * i for i in range(32)]),
    (8, 2, 80, 32, 512, [512 + i % 9 for i in range(20)]),
    (8, 1, 128, 64, 512, [513 + i for i in range(33)]),
    (16, 4, 128, 128, 512, [560, 513, 530, 540, 512, 520]),
    (40, 1, 128, 16, 640, [641 + 9 * i for i in range(6)]),
    (8, 1, 200, 64, 320, [321 + i % 20 for i in range(24)]),
    (16, 2, 256, 16, 480, [481, 500, 490, 485]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv,dim,page,shared,lens", DECODES_ON_ROWS)
def test_decode_on_rows(ctx, heads, kv, dim, page, shared, lens, dtype):
    pool = Pool(ctx, dtype, kv, dim, page, shared, lens, seed=heads + dim, junk=float("nan"))
    q = normal(generator(1), (len(lens), heads, dim), dtype, 2.0)
    for layer in (0, 1):
        out, lse = run_decode(pool, q, layer, shared, max(lens))
        check_decode(pool, q, layer, out, lse)


ROWS = [(4, 2, 64, 32, 1056, 90), (8, 1, 128, 33, 512, 40), (16, 2, 256, 4, 480, 20)]


@pytest.mark.parametrize("heads,kv,dim,batch,shared,own", ROWS)
@pytest.mark.parametrize("window", [0, 1, 30, 300, 100000])
def test_decode_on_rows_empty_short_and_reordered_sequences(ctx, heads, kv, dim, batch, shared, own, window):
    lens = [shared + own, 0, shared, 50] + [shared - 1, shared + 9, 1, shared + own] * 8
    lens = lens[:batch]
    pool = Pool(ctx, torch.bfloat16, kv, dim, 16, shared, lens, seed=9)
    order = [(i * 5 + 3) % batch if batch % 5 else i for i in range(batch)]
    order[1] = order[0]
    q = normal(generator(4), (batch, heads, dim), torch.bfloat16, 2.0)
    out, lse = run_decode(pool, q, 1, shared, max(lens), sequences=order, window=window)
    check_decode(pool, q, 1, out, lse, sequences=order, window=window)


@pytest.mark.parametrize("heads,kv,dim,batch,shared,own", ROWS)
@pytest.mark.parametrize("wild", [float("nan"), float("inf"), None])
def test_decode_on_rows_hidden_values_have_no_influence(ctx, heads, kv, dim, batch, shared, own, wild):
    wild = torch.finfo(torch.bfloat16).min if wild is None else wild
    lens = [shared + own, 100, shared + 5, shared] + [shared] * (batch - 4)
    pool = Pool(ctx, torch.bfloat16, kv, dim, 16, shared, lens, seed=18)
    pool.lengths[1] = 100
    q = normal(generator(10), (batch, heads, dim), torch.bfloat16, 2.0)
    for window in (0, 150):
        want, want_lse = run_decode(pool, q, 0, shared, max(lens), window=window)
        for key in (100, 104, shared - 1):
            page = int(pool.table[0, key // 16])
            saved = pool.memory[page].clone()
            pool.memory[page, 0, :, :, key % 16] = wild
            out, lse = run_decode(pool, q, 0, shared, max(lens), window=window)
            assert torch.equal(out[1], want[1]) and torch.equal(lse[1], want_lse[1])
            hidden = window > 0 and key < shared - window
            assert torch.equal(out[3], want[3]) == hidden
            pool.memory[page] = saved


def test_decode_empty_short_and_reordered_sequences(ctx):
    """Rows picked out of order, one of them twice; a length of zero and one below the
    shared tokens; a row number outside the table is an empty sequence."""
    lens = [128 + 70, 128, 0, 50, 128 + 9, 128 + 300]
    pool = Pool(ctx, torch.bfloat16, 2, 128, 16, 128, lens, seed=9)
    order = [5, 0, 2, 4, 4, 3, 1]
    q = normal(generator(4), (len(order), 8, 128), torch.bfloat16, 2.0)
    out, lse = run_decode(pool, q, 1, 128, max(lens), sequences=order)
    check_decode(pool, q, 1, out, lse, sequences=order)
    assert (out[2] == 0).all() and torch.isinf(lse[2]).all()
    out, lse = run_decode(pool, q[:2], 0, 0, max(lens), sequences=[4, 77])
    check_decode(pool, q[:1], 0, out, lse, sequences=[4])
    assert (out[1] == 0).all() and torch.isinf(lse[1]).all()


@pytest.mark.parametrize("window", [1, 30, 200, 100000])
@pytest.mark.parametrize("shared", [0, 256])
def test_decode_window_and_scale(ctx, window, shared):
    lens = [256 + 70, 256 + 1, 256 + 333, 256]
    pool = Pool(ctx, torch.float16, 2, 64, 32, 256, lens, seed=12)
    q = normal(generator(6), (4, 8, 64), torch.float16, 2.0)
    out, lse = run_decode(pool, q, 0, shared, max(lens), window=window, scale=0.3)
    check_decode(pool, q, 0, out, lse, window=window, scale=0.3)


def test_decode_reads_nothing_beyond_max_length(ctx):
    pool = Pool(ctx, torch.bfloat16, 1, 64, 16, 0, [300, 20], seed=13)
    q = normal(generator(8), (2, 2, 64), torch.bfloat16)
    out, lse = run_decode(pool, q, 0, 0, 100)
    check_decode(pool, q, 0, out, lse, cut=100)


def test_decode_shared_or_not_is_the_same_attention(ctx):
    lens = [512 + 3, 512 + 90, 512 + 200]
    pool = Pool(ctx, torch.bfloat16, 2, 128, 32, 512, lens, seed=15)
    q = normal(generator(9), (3, 8, 128), torch.bfloat16, 2.0)
    for shared in (0, 32, 256, 512):
        out, lse = run_decode(pool, q, 0, shared, max(lens))
        check_decode(pool, q, 0, out, lse)


@pytest.mark.parametrize("wild", [float("nan"), float("inf")])
def test_decode_hidden_values_have_no_influence(ctx, wild):
    """Shared tokens that a shorter sequence or a window does not see."""
    lens = [256 + 30, 100, 256 + 5, 256]
    pool = Pool(ctx, torch.bfloat16, 1, 128, 16, 256, lens, seed=18)
    pool.lengths[1] = 100
    q = normal(generator(10), (4, 4, 128), torch.bfloat16, 2.0)
    for window in (0, 150):
        want, want_lse = run_decode(pool, q, 0, 256, max(lens), window=window)
        saved = pool.memory.clone()
        for key in (100, 104, 255):
            page = int(pool.table[0, key // 16])
            pool.memory[page, 0, :, :, key % 16] = wild
        out, lse = run_decode(pool, q, 0, 256, max(lens), window=window)
        assert torch.equal(out[1], want[1]) and torch.equal(lse[1], want_lse[1])
        assert not torch.isfinite(out[3]).any()
        pool.memory.copy_(saved)


def test_decode_strides(ctx):
    pool = Pool(ctx, torch.bfloat16, 2, 64, 16, 64, [70, 90, 64], seed=20)
    wide = normal(generator(11), (3, 6, 2 * 64), torch.bfloat16)
    q = wide[:, :, 64:]
    out = torch.full((6, 3, 64), float("nan"), dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    out, lse = run_decode(pool, q, 1, 64, 90, out=out)
    check_decode(pool, q, 1, out, lse)


def test_decode_in_a_graph(ctx):
    """Captured once, replayed after the lengths have grown."""
    pool = Pool(ctx, torch.bfloat16, 2, 128, 16, 64, [90, 100], seed=21)
    q = normal(generator(12), (2, 8, 128), torch.bfloat16, 2.0)
    out, lse = torch.zeros_like(q), torch.zeros(2, 8, device="cuda")
    n = pool.cache.decode_workspace(8, 2, 64, 100)
    work = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")

    def step():
        pool.cache.decode_attention(layer=0, heads=8, q=q.data_ptr(), out=out.data_ptr(),
                                    lse=lse.data_ptr(), batch=2, max_length=100, shared_tokens=64,
                                    workspace=work.data_ptr(), workspace_bytes=n,
                                    stream=torch.cuda.current_stream().cuda_stream)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    pool.lengths.sub_(5)
    graph.replay()
    torch.cuda.synchronize()
    check_decode(pool, q, 0, out, lse)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------

def test_prompt_refusals(ctx):
    t = torch.zeros(64, 4, 64, dtype=torch.bfloat16, device="cuda")
    o = ints([0, 64])
    good = dict(type=N.BF16, heads=4, kv_heads=4, head_dim=64, q=t.data_ptr(), k=t.data_ptr(),
                v=t.data_ptr(), out=t.data_ptr(), q_tokens=64, k_tokens=64, sequences=1,
                q_offsets=o.data_ptr())

    def status(**change):
        with pytest.raises(DmError) as e:
            prompt_attention(ctx, **{**good, **change})
        return e.value.status

    assert status(type=N.F32) == N.ERR_UNSUPPORTED_TENSOR_TYPE
    assert status(heads=6) == N.ERR_ELEMENT_COUNT
    assert status(heads=0) == N.ERR_ELEMENT_COUNT
    assert status(heads=4 * 129) == N.ERR_ELEMENT_COUNT
    for dim in (0, 12, 264, -8):
        assert status(head_dim=dim) == N.ERR_ELEMENT_COUNT
    assert status(sequences=-1) == N.ERR_ELEMENT_COUNT
    assert status(window=-1) == N.ERR_ELEMENT_COUNT
    assert status(q_tokens=-1) == N.ERR_ELEMENT_COUNT
    assert status(q=0) == N.ERR_INVALID_ARGUMENT
    assert status(q_offsets=0) == N.ERR_INVALID_ARGUMENT
    assert status(v=t.data_ptr() + 2) == N.ERR_INVALID_ARGUMENT
    assert status(k_stride=(256, 60)) == N.ERR_INVALID_ARGUMENT
    assert status(out_stride=(-256, 64)) == N.ERR_INVALID_ARGUMENT
    for scale in (-1.0, float("nan"), float("inf")):
        assert status(scale=scale) == N.ERR_POSITIVE_PARAMETER
    # nothing to do
    prompt_attention(ctx, **{**good, "sequences": 0})
    prompt_attention(ctx, **{**good, "q_tokens": 0})


def test_decode_refusals(ctx):
    pool = Pool(ctx, torch.bfloat16, 2, 64, 16, 64, [70, 900], seed=22)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    n = pool.cache.decode_workspace(4, 2, 64, 900)
    assert n > 0
    work = torch.empty(n, dtype=torch.uint8, device="cuda")
    good = dict(layer=0, heads=4, q=q.data_ptr(), out=q.data_ptr(), batch=2, max_length=900,
                shared_tokens=64, workspace=work.data_ptr(), workspace_bytes=n)

    def status(**change):
        with pytest.raises(DmError) as e:
            pool.cache.decode_attention(**{**good, **change})
        return e.value.status

    assert status(layer=2) == N.ERR_INVALID_LAYER
    assert status(heads=3) == N.ERR_ELEMENT_COUNT
    assert status(batch=-1) == N.ERR_ELEMENT_COUNT
    assert status(shared_tokens=8) == N.ERR_ELEMENT_COUNT
    assert status(shared_tokens=1 << 20) == N.ERR_ELEMENT_COUNT
    assert status(max_length=-1) == N.ERR_ELEMENT_COUNT
    assert status(window=-5) == N.ERR_ELEMENT_COUNT
    assert status(q=0) == N.ERR_INVALID_ARGUMENT
    assert status(out=q.data_ptr() + 8) == N.ERR_INVALID_ARGUMENT
    assert status(workspace=0) == N.ERR_INVALID_ARGUMENT
    assert status(workspace=work.data_ptr() + 8) == N.ERR_INVALID_ARGUMENT
    assert status(workspace_bytes=n - 1) == N.ERR_BYTE_LENGTH
    assert status(scale=-1.0) == N.ERR_POSITIVE_PARAMETER
    assert status(q_stride=(60, 64)) == N.ERR_INVALID_ARGUMENT
    pool.cache.decode_attention(**{**good, "batch": 0})


def test_prompt_broadcast_heads(ctx):
    """Keys and values that all heads share as one row (stride 0): no tensor map describes
    that, so these run on the 16-row kernel."""
    gen = generator(31)
    q = normal(gen, (70, 6, 64), torch.float16, 2.0)
    k1, v1 = (normal(gen, (70, 1, 64), torch.float16) for _ in range(2))
    k, v = k1.expand(70, 3, 64), v1.expand(70, 3, 64)
    out, lse = run_prompt(ctx, q, k, v, [40, 30], [40, 30], k_stride=(64, 0), v_stride=(64, 0))
    check_prompt(q, k, v, [40, 30], [40, 30], out, lse, tokens=16)
    for causal, window in ((False, 0), (True, 9)):
        out, lse = run_prompt(ctx, q, k, v, [40, 30], [40, 30], causal, window, k_stride=(64, 0), v_stride=(64, 0))
        check_prompt(q, k, v, [40, 30], [40, 30], out, lse, causal, window, tokens=16)
    k1[20], v1[33] = float("nan"), float("inf")
    bad, _ = run_prompt(ctx, q, k, v, [40, 30], [40, 30], k_stride=(64, 0), v_stride=(64, 0))
    good, _ = run_prompt(ctx, q, k1.nan_to_num(0, 0, 0).expand(70, 3, 64), v1.nan_to_num(0, 0, 0).expand(70, 3, 64),
                         [40, 30], [40, 30], k_stride=(64, 0), v_stride=(64, 0))
    assert torch.equal(bad[:20], good[:20]) and torch.equal(bad[40:], good[40:])


def test_prompt_without_any_keys(ctx):
    q = normal(generator(33), (5, 2, 128), torch.bfloat16)
    k = torch.zeros(0, 2, 128, dtype=torch.bfloat16, device="cuda")
    out, lse = run_prompt(ctx, q, k, k, [2, 3], [0, 0], k_stride=(0, 0), v_stride=(0, 0))
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("dim", [64, 256])
def test_prompt_rows_beyond_32_bits(ctx, dim):
    """Rows that lie more than 2^31 elements into their tensors."""
    n, stride = 300, 1 << 23
    big = torch.empty((n - 1) * stride + 2 * dim, dtype=torch.bfloat16, device="cuda")
    q, k, v = (big.as_strided((n, 1, dim), (stride, dim, 1)) for _ in range(3))
    gen = generator(37)
    q.copy_(normal(gen, (n, 1, dim), torch.bfloat16))
    out = big.as_strided((n, 1, dim), (stride, dim, 1), dim)
    assert (n - 1) * stride > 2 ** 31
    out, lse = run_prompt(ctx, q, k, v, [n], [n], out=out, q_stride=(stride, dim), k_stride=(stride, dim),
                          v_stride=(stride, dim), out_stride=(stride, dim))
    check_prompt(q, k, v, [n], [n], out, lse, tokens=20)


def test_prompts_back_to_back_on_one_stream(ctx):
    """A call may be scheduled before the one in front of it has ended: it must still read what
    that one writes."""
    gen = generator(41)
    n = 700
    x = normal(gen, (n, 2, 64), torch.bfloat16)
    o = ints([0, n])

    def attend(q, out):
        prompt_attention(ctx, type=N.BF16, heads=2, kv_heads=2, head_dim=64, q=q.data_ptr(), k=q.data_ptr(),
                         v=q.data_ptr(), out=out.data_ptr(), q_tokens=n, k_tokens=n, sequences=1,
                         q_offsets=o.data_ptr())
    bufs = [x] + [torch.zeros_like(x) for _ in range(20)]
    for _ in range(5):
        for a, b in zip(bufs, bufs[1:]):
            attend(a, b)
    torch.cuda.synchronize()
    want = x
    for b in bufs[1:]:
        out = torch.zeros_like(x)
        attend(want, out)
        torch.cuda.synchronize()
        assert torch.equal(out, b)
        want = out


def test_decode_right_after_its_cache_calls(ctx):
    """extend, write, fork and decode queued without a wait in between, against the same calls
    with one after each."""
    def play(wait):
        cache = KvCache(ctx, type=N.BF16, layers=1, kv_heads=2, head_dim=64, page_tokens=16, pages=400,
                        max_sequences=9, max_pages=40)
        gen = generator(43)
        k, v = (normal(gen, (500, 2, 64), torch.bfloat16) for _ in range(2))
        rows, count, off = ints([0]), ints([500]), ints([0, 500])
        kids, parents, ones, koff = ints(range(1, 9)), ints([0] * 8), ints([1] * 8), ints(range(9))
        q = normal(gen, (8, 8, 64), torch.bfloat16, 2.0)
        out = torch.zeros_like(q)
        size = cache.decode_workspace(8, 8, 496, 520)
        work = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        calls = [lambda: cache.extend(rows.data_ptr(), count.data_ptr(), 1),
                 lambda: cache.write(0, k.data_ptr(), v.data_ptr(), rows.data_ptr(), off.data_ptr(), 1, 500),
                 lambda: cache.fork(parents.data_ptr(), kids.data_ptr(), 8)]
        for _ in range(10):
            calls += [lambda: cache.extend(kids.data_ptr(), ones.data_ptr(), 8),
                      lambda: cache.write(0, k.data_ptr(), v.data_ptr(), kids.data_ptr(), koff.data_ptr(), 8, 8),
                      lambda: cache.decode_attention(layer=0, heads=8, q=q.data_ptr(), out=out.data_ptr(), batch=8,
                                                     max_length=520, shared_tokens=496, sequences=kids.data_ptr(),
                                                     workspace=work.data_ptr(), workspace_bytes=size)]
        torch.cuda.synchronize()
        for c in calls:
            c()
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        assert cache.status() == 0
        cache.close()
        return out
    want = play(True)
    for _ in range(3):
        assert torch.equal(play(False), want)
