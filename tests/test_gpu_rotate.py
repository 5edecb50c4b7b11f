"""dm_attention_rotate against norms and rotations written out in 64 bits."""
import math

import numpy as np
import pytest
import torch

from attention_plain import EPS, to64
from diskmule_b200 import CudaContext, DmError, _native as N
from diskmule_b200.attention import Rope, offsets, rotate
from paged import KIND, Paged, generator, ints, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = CudaContext(0)
    yield c
    c.close()


def head64(x, weight, epsilon, normed, angles, interleaved):
    """x [.., d], angles [.., pairs] or None -> result, bound of its error before rounding.

    f32 steps: the sum of d squares and the root (d / 2 + 8) 2^-24 relative, products a few
    2^-24 each; the angle is off by 2^-25 of half a turn and 2^-32 of a turn, sines and
    cosines by a few units: all of it (|a| + |b|) (d + 40) 2^-24."""
    d = x.shape[-1]
    y = x.astype(np.float64)
    if normed:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + epsilon)
        if weight is not None:
            y = y * weight
    size = np.abs(y)
    if angles is not None:
        r = 2 * angles.shape[-1]
        a, b = ((np.arange(0, r, 2), np.arange(1, r, 2)) if interleaved
                else (np.arange(r // 2), np.arange(r // 2, r)))
        c, s = np.cos(angles), np.sin(angles)
        z, w = y[..., a] * c - y[..., b] * s, y[..., b] * c + y[..., a] * s
        both = size[..., a] + size[..., b]
        y, size = y.copy(), size.copy()
        y[..., a], y[..., b] = z, w
        size[..., a] = size[..., b] = both
    return y, size * (d + 40) * 2.0 ** -24


def near(got, want, bound, eps, where):
    g = to64(got)
    allowed = bound + eps * (np.abs(want) + bound) + 2.0 ** -25
    worst = np.abs(g - want) - allowed
    assert np.all(worst <= 0), f"{where}: off by {np.abs(g - want).max()}, {worst.max()} beyond what is allowed"


class Call:
    """Random inputs of a call; run() makes it and checks all outputs."""

    def __init__(self, ctx, new, lens, heads, kv, dim, rotary, page=16, dtype=torch.bfloat16, axes=1,
                 interleaved=False, scale=1.0, theta=1e4, norms=7, weights=True, own_positions=True, far=0,
                 rows=None, extra=2, seed=0):
        self.__dict__.update(ctx=ctx, new=new, heads=heads, kv=kv, dim=dim, rotary=rotary, dtype=dtype,
                             interleaved=interleaved, scale=scale, norms=norms, rows=rows)
        gen, r = generator(seed), np.random.RandomState(seed)
        self.tokens = sum(new) + extra
        self.pool = Paged(ctx, dtype, kv, dim, page, lens, seed=seed) if lens else None
        self.qkv = normal(gen, (self.tokens, heads + 2 * kv, dim), dtype, 3.0)
        self.wq, self.wk = (torch.randn(dim, generator=gen, device="cuda") if weights else None for _ in range(2))
        self.f = theta ** (-2.0 * np.arange(rotary // 2) / max(1, rotary)) if theta else r.randn(rotary // 2) * 4
        self.pair_axes = r.randint(0, axes, rotary // 2) if axes > 1 else None
        self.rope = Rope(ctx, rotary, frequencies=self.f, pair_axes=self.pair_axes, axes=axes,
                         interleaved=interleaved, scale=scale) if rotary else None
        self.positions = r.randint(0, far or 5000, (axes, self.tokens)) if own_positions else None
        if far:
            self.positions[0, 0] = far

    def angles(self):
        p = self.positions
        if p is None:
            p = np.zeros((1, self.tokens))
            at = 0
            for i, a in enumerate(self.new):
                s = i if self.rows is None else self.rows[i]
                p[0, at:at + a] = np.maximum(self.pool.lens[s] - a, 0) + np.arange(a)
                at += a
        axis = np.zeros(self.rotary // 2, int) if self.pair_axes is None else self.pair_axes
        return p[axis].T.astype(np.longdouble) * self.f.astype(np.longdouble)

    def run(self, in_place=False, cached=True, outs=("q",), layer=1, epsilon=1e-6, stream=0):
        h, kv = self.heads, self.kv
        x = self.qkv.clone()
        q, k, v = x[:, :h], x[:, h:h + kv], x[:, h + kv:]
        nan = [torch.full((self.tokens, n, self.dim), float("nan"), dtype=self.dtype, device="cuda")
               for n in (h, kv, kv)]
        o = [t if in_place else n for t, n in zip((q, k, v), nan)]
        given = {n + "_out": t.data_ptr() for n, t in zip("qkv", o) if n in outs}
        stride = (x.stride(0), x.stride(1))
        if in_place:
            given.update({n + "_out_stride": stride for n in outs})
        kw = {}
        if cached:
            off = ints(offsets(self.new))
            rows = None if self.rows is None else ints(self.rows)
            kw = dict(cache=self.pool.cache, layer=layer, offsets=off.data_ptr(), n=len(self.new),
                      sequences=rows.data_ptr() if rows is not None else 0)
        p = None if self.positions is None else ints(self.positions)
        before = self.pool.memory.clone() if cached else None
        rotate(self.ctx, self.rope, type=KIND[self.dtype], heads=h, kv_heads=kv, head_dim=self.dim,
               tokens=self.tokens, q=q.data_ptr() if "q" in outs else 0, k=k.data_ptr(), v=v.data_ptr(),
               q_stride=stride, k_stride=stride, v_stride=stride, positions=p.data_ptr() if p is not None else 0,
               norm_q=bool(self.norms & 1), norm_k=bool(self.norms & 2), norm_v=bool(self.norms & 4),
               q_weight=self.wq.data_ptr() if self.wq is not None else 0,
               k_weight=self.wk.data_ptr() if self.wk is not None else 0, epsilon=epsilon, stream=stream, **given, **kw)
        torch.cuda.synchronize()
        # ---- what it should be
        raw = to64(self.qkv)
        angles = np.asarray(np.mod(self.angles(), 2 * np.pi), np.float64)[:, None] if self.rope else None
        eps = EPS[self.dtype]
        w = [None if t is None else to64(t) for t in (self.wq, self.wk)]
        want = [head64(raw[:, :h], w[0], epsilon, self.norms & 1, angles, self.interleaved),
                head64(raw[:, h:h + kv], w[1], epsilon, self.norms & 2, angles, self.interleaved),
                head64(raw[:, h + kv:], None, epsilon, self.norms & 4, None, False)]
        if self.scale != 1.0 and self.rope:
            for y, b in want[:2]:
                y[..., :self.rotary] *= self.scale
                b[..., :self.rotary] *= self.scale
        used = sum(self.new) if cached else self.tokens
        for n, got, (y, b) in zip("qkv", o, want):
            if n in outs:
                near(got[:used], y[:used], b[:used], eps, n)
                rest = got[used:]
                assert torch.equal(rest, self.qkv[used:, {"q": slice(0, h), "k": slice(h, h + kv), "v": slice(h + kv, None)}[n]]) \
                    if in_place else torch.isnan(rest).all()
        if not cached:
            return
        # ---- the cache: the new tokens' rows, and nothing else
        after, expect = self.pool.memory, before.clone()
        at = 0
        for i, a in enumerate(self.new):
            s = i if self.rows is None else self.rows[i]
            n = self.pool.lens[s] if 0 <= s < len(self.pool.lens) else 0
            for t in range(a):
                place = n - a + t
                if place < 0 or n == 0:
                    continue
                page, r = self.pool.at(s, place)
                for which in (0, 1):
                    y, b = want[1 + which]
                    near(after[page, layer, which, :, r], y[at + t], b[at + t], eps, f"cache {which} token {at + t}")
                expect[page, layer, :, :, r] = after[page, layer, :, :, r]
            at += a
        assert torch.equal(after.view(torch.int16), expect.view(torch.int16))


ROTATIONS = [
    # new, lens, heads, kv, dim, rotary, page, options
    ([1], [1], 1, 1, 64, 64, 16, {}),
    ([1, 1, 1, 1], [310, 17, 64, 1200], 8, 2, 64, 64, 16, {}),
    ([5, 0, 40], [70, 3, 40], 8, 2, 128, 128, 32, dict(own_positions=False)),
    ([33, 129], [100, 129], 6, 2, 80, 80, 16, dict(own_positions=False)),
    ([20], [20], 4, 4, 80, 32, 16, {}),
    ([50], [60], 16, 2, 256, 64, 64, dict(axes=3)),
    ([7, 9], [7, 90], 4, 1, 256, 256, 16, dict(axes=4, interleaved=True)),
    ([12], [12], 3, 1, 96, 48, 16, dict(interleaved=True, own_positions=False)),
    ([10], [25], 5, 1, 8, 0, 16, {}),                             # no rotation
    ([10], [25], 5, 1, 24, 16, 16, dict(norms=0)),
    ([600], [700], 32, 8, 128, 128, 64, dict(norms=3)),
    ([600, 1, 300], [600, 5, 900], 8, 2, 64, 32, 16, dict(norms=1, weights=False)),
    ([30], [30], 40, 8, 128, 128, 128, dict(norms=4, scale=1.37)),
    ([20, 3], [30, 30], 4, 2, 64, 64, 16, dict(rows=[1, 0], theta=0)),  # any frequencies, entries in another order
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,lens,heads,kv,dim,rotary,page,options", ROTATIONS)
def test_rotate_into_the_cache(ctx, new, lens, heads, kv, dim, rotary, page, options, dtype):
    call = Call(ctx, new, lens, heads, kv, dim, rotary, page, dtype, **options)
    call.run()
    assert call.pool.cache.status() == 0
    call.run(in_place=True, outs=("q", "k", "v"))
    call.run(outs=())


@pytest.mark.parametrize("dim,rotary,tokens", [(64, 64, 1), (128, 128, 700), (256, 128, 33), (40, 16, 9)])
def test_rotate_without_a_cache(ctx, dim, rotary, tokens):
    for in_place in (False, True):
        Call(ctx, [], None, 6, 2, dim, rotary, extra=tokens).run(cached=False, outs=("q", "k", "v"), in_place=in_place)
        Call(ctx, [], None, 6, 2, dim, rotary, extra=tokens, dtype=torch.float16).run(cached=False, outs=("k",),
                                                                                     in_place=in_place)


@pytest.mark.parametrize("far", [1 << 20, (1 << 31) - 1])
def test_far_positions(ctx, far):
    """The fraction of a turn stays exact where an f32 angle has none of it left."""
    Call(ctx, [40], [50], 4, 2, 128, 128, far=far).run()


def test_negative_positions_and_fast_pairs(ctx):
    call = Call(ctx, [40], [50], 4, 2, 64, 64, theta=0, seed=5)
    call.positions = -call.positions
    call.run()


def test_small_and_large_heads(ctx):
    """Values whose squares leave f16 (not f32), zeros (epsilon alone), and no epsilon."""
    call = Call(ctx, [6], [6], 2, 1, 64, 64, dtype=torch.float16)
    call.qkv[0] = 0
    call.qkv[1] *= 2000
    call.qkv[2] *= 2.0 ** -12
    call.run()
    call.qkv[0] = 1
    call.run(epsilon=0.0)


def test_heads_that_are_not_finite_stay_alone(ctx):
    call = Call(ctx, [6], [6], 2, 1, 64, 64)
    call.run()
    kept = call.pool.memory.clone()
    call.qkv[2, 1, 7] = float("nan")
    call.qkv[2, 2] = float("inf")  # the key
    x, h = call.qkv, 2
    q = torch.zeros(8, 2, 64, dtype=torch.bfloat16, device="cuda")
    off, p = ints(offsets(call.new)), ints(call.positions)
    st = (x.stride(0), x.stride(1))
    rotate(ctx, call.rope, type=N.BF16, heads=2, kv_heads=1, head_dim=64, tokens=8, q=x.data_ptr(),
           k=x[:, 2:].data_ptr(), v=x[:, 3:].data_ptr(), q_out=q.data_ptr(), q_stride=st, k_stride=st, v_stride=st,
           cache=call.pool.cache, layer=1, offsets=off.data_ptr(), n=1, positions=p.data_ptr(), norm_q=True,
           norm_k=True, norm_v=True, q_weight=call.wq.data_ptr(), k_weight=call.wk.data_ptr())
    torch.cuda.synchronize()
    assert torch.isnan(q[2, 1]).all() and torch.isfinite(q[2, 0]).all() and torch.isfinite(q[3]).all()
    page, r = call.pool.at(0, 2)
    assert torch.isnan(call.pool.memory[page, 1, 0, 0, r]).all()
    call.pool.memory[page, 1, 0, 0, r] = kept[page, 1, 0, 0, r]
    assert torch.equal(call.pool.memory.view(torch.int16), kept.view(torch.int16))


def test_rows_outside_the_cache(ctx):
    """Entries outside the table, more rows than tokens, pages that are none: queries come out,
    nothing is cached for them, and the status says so."""
    call = Call(ctx, [3, 4, 2], [40, 2, 30], 4, 2, 64, 64, rows=[0, 9, 2])
    call.run()
    assert call.pool.cache.status() == N.KV_BAD_TOKEN
    call = Call(ctx, [3, 4], [40, 2], 4, 2, 64, 64)
    call.run()
    assert call.pool.cache.status() == N.KV_BAD_TOKEN
    call = Call(ctx, [3], [40], 4, 2, 64, 64, own_positions=False)
    call.pool.table[0, 2] = call.pool.memory.shape[0]
    x, st = call.qkv, (call.qkv.stride(0), call.qkv.stride(1))
    before = call.pool.memory.clone()
    off = ints([0, 3])
    rotate(ctx, call.rope, type=N.BF16, kv_heads=2, head_dim=64, tokens=5, k=x[:, 4:].data_ptr(), v=x[:, 6:].data_ptr(),
           k_stride=st, v_stride=st, cache=call.pool.cache, layer=0, offsets=off.data_ptr(), n=1)
    assert call.pool.cache.status() == N.KV_BAD_TOKEN
    assert torch.equal(before.view(torch.int16), call.pool.memory.view(torch.int16))


@pytest.mark.parametrize("n", [33, 700, 1100])
def test_many_entries(ctx, n):
    """More entries than a search step has lanes, some without rows."""
    r = np.random.RandomState(n)
    new = [int(x) for x in r.randint(0, 3, n)]
    Call(ctx, new, [a + int(b) for a, b in zip(new, r.randint(0, 4, n))], 2, 1, 16, 16, own_positions=False).run()


def test_captured_call(ctx):
    """Bounds stay, lengths, offsets and positions change."""
    call = Call(ctx, [3, 5], [50, 40], 4, 2, 64, 64)
    x, st, side = call.qkv, (call.qkv.stride(0), call.qkv.stride(1)), torch.cuda.Stream()
    q = torch.zeros(call.tokens, 4, 64, dtype=torch.bfloat16, device="cuda")
    off, p = ints([0, 3, 8]), ints(call.positions)
    g = torch.cuda.CUDAGraph()
    def run(stream):
        rotate(ctx, call.rope, type=N.BF16, heads=4, kv_heads=2, head_dim=64, tokens=call.tokens, q=x.data_ptr(),
               k=x[:, 4:].data_ptr(), v=x[:, 6:].data_ptr(), q_out=q.data_ptr(), q_stride=st, k_stride=st, v_stride=st,
               cache=call.pool.cache, layer=0, offsets=off.data_ptr(), n=2, positions=p.data_ptr(), norm_k=True,
               stream=stream)
    with torch.cuda.graph(g, stream=side):
        run(side.cuda_stream)
    for new in ([3, 5], [0, 2], [8, 1]):
        off.copy_(ints(offsets(new)))
        p.copy_(p + 17)
        call.pool.memory.zero_(), q.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = q.clone(), call.pool.memory.clone()
        call.pool.memory.zero_(), q.zero_()
        run(0)
        torch.cuda.synchronize()
        assert torch.equal(got[0], q) and torch.equal(got[1], call.pool.memory) and q[sum(new):].abs().sum() == 0
        assert (q[:sum(new)] != 0).any()


def test_refusals(ctx):
    call = Call(ctx, [4], [30], 4, 2, 64, 64)
    x = call.qkv.data_ptr()
    off = ints([0, 4])
    good = dict(type=N.BF16, heads=4, kv_heads=2, head_dim=64, tokens=4, q=x, k=x, v=x, q_out=x, cache=call.pool.cache,
                offsets=off.data_ptr(), n=1, layer=0, q_stride=(512, 64), k_stride=(512, 64), v_stride=(512, 64))
    before = call.qkv.clone()
    rotate(ctx, call.rope, **dict(good, tokens=0))
    rotate(ctx, call.rope, **dict(good, n=0))
    for change, status in [
            (dict(type=N.F32), N.ERR_UNSUPPORTED_TENSOR_TYPE), (dict(type=N.F16), N.ERR_INVALID_ARGUMENT),
            (dict(head_dim=60), N.ERR_ELEMENT_COUNT), (dict(head_dim=32), N.ERR_ELEMENT_COUNT),
            (dict(head_dim=264), N.ERR_ELEMENT_COUNT), (dict(head_dim=128), N.ERR_INVALID_ARGUMENT),
            (dict(heads=0), N.ERR_ELEMENT_COUNT), (dict(kv_heads=4), N.ERR_ELEMENT_COUNT),
            (dict(tokens=-1), N.ERR_ELEMENT_COUNT), (dict(n=-1), N.ERR_ELEMENT_COUNT), (dict(n=2), N.ERR_ELEMENT_COUNT),
            (dict(layer=2), N.ERR_INVALID_LAYER), (dict(offsets=0), N.ERR_INVALID_ARGUMENT),
            (dict(k=0), N.ERR_INVALID_ARGUMENT), (dict(q=0), N.ERR_INVALID_ARGUMENT), (dict(q=x + 2), N.ERR_INVALID_ARGUMENT),
            (dict(q_stride=(510, 64)), N.ERR_INVALID_ARGUMENT), (dict(k_stride=(-512, 64)), N.ERR_INVALID_ARGUMENT),
            (dict(norm_q=True, epsilon=-1.0), N.ERR_POSITIVE_PARAMETER),
            (dict(norm_q=True, epsilon=float("nan")), N.ERR_POSITIVE_PARAMETER),
            (dict(norm_q=True, q_weight=x + 2), N.ERR_INVALID_ARGUMENT),
            (dict(cache=None), N.ERR_INVALID_ARGUMENT)]:
        with pytest.raises(DmError) as e:
            rotate(ctx, call.rope, **dict(good, **change))
        assert e.value.status == status, change
    other = CudaContext(0)
    try:
        with pytest.raises(DmError):
            rotate(other, call.rope, **good)
    finally:
        other.close()
    for bad in (dict(rotary_dim=0), dict(rotary_dim=24), dict(rotary_dim=272), dict(rotary_dim=64, axes=5),
                dict(rotary_dim=64, theta=-1.0), dict(rotary_dim=64, theta=float("inf")),
                dict(rotary_dim=32, frequencies=[math.nan] * 16), dict(rotary_dim=32, pair_axes=[2] * 16, axes=2),
                dict(rotary_dim=32, pair_axes=[-1] * 16, axes=2), dict(rotary_dim=32, scale=math.inf)):
        with pytest.raises(DmError):
            Rope(ctx, **bad)
    with pytest.raises(ValueError):
        Rope(ctx, 32, frequencies=[1.0] * 15)
    torch.cuda.synchronize()
    assert torch.equal(before, call.qkv) and call.pool.cache.status() == 0


@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_in_place_with_other_strides_is_refused(ctx, which):
    """A result over its input under other strides would overwrite what other warps have yet to
    read. What is alike, or has one token and one head only, is done."""
    fused = normal(generator(1), (9, 12, 64), torch.bfloat16)
    before, at = fused.clone(), ints([[3] * 9])
    given = {which: fused.data_ptr(), f"{which}_out": fused.data_ptr(), "heads" if which == "q" else "kv_heads": 4}
    call = lambda tokens=9, **more: rotate(ctx, None, type=N.BF16, head_dim=64, tokens=tokens, positions=at.data_ptr(),
                                           norm_q=True, norm_k=True, norm_v=True, **{**given, **more})
    for strides in ({f"{which}_stride": (768, 64)}, {f"{which}_out_stride": (768, 64)},
                    {f"{which}_stride": (768, 64), f"{which}_out_stride": (768, 128)}):
        with pytest.raises(DmError) as e:
            call(**strides)
        assert e.value.status == N.ERR_INVALID_ARGUMENT
    torch.cuda.synchronize()
    assert torch.equal(fused, before)
    call(**{f"{which}_stride": (768, 64), f"{which}_out_stride": (768, 64)})
    call(tokens=1, **{f"{which}_stride": (64, 64)})  # one token: its place is the same whatever the stride
    torch.cuda.synchronize()
    assert not torch.equal(fused[:, :4], before[:, :4]) and torch.equal(fused[:, 4:], before[:, 4:])
