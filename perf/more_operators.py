"""Workloads of the operators around the paged cache: norms and position rotation of queries
and keys on their way into it, attention of chunks of new tokens over it (with a window and
sinks), the weight that each cached token has received, and eviction by that weight.

Each case runs one pass the way a serving program does; `run` computes it in elementary
torch operations (32-bit arithmetic, angles in 64, one rounding at the end) or, with `own`
set, through `diskmule_b200.attention`. `exact` is the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPSILON = 1e-6


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _lens(text):
    return [int(v) for v in text.split(",")]


def _text(lens):
    return ",".join(map(str, lens))


def listed():
    return [
        # one new token for each of four chats: launch latency
        dict(name="rotate_step", op="rotate", type="bf16", new="1,1,1,1", cached="310,17,64,1200", heads=8,
             kv_heads=2, dim=64, rotary=64, page=16, layers=2, axes=1, theta=1e4, norm_v=False),
        # an ordinary prefill batch: ragged prompts, some of which continue cached ones
        dict(name="rotate_prompts", op="rotate", type="bf16", new="4100,911,1777,640,763",
             cached="0,0,2048,33,0", heads=32, kv_heads=8, dim=128, rotary=128, page=64, layers=1, axes=1,
             theta=1e6, norm_v=False),
        # text and images in one prompt: positions in time, height and width, a quarter of wide heads rotated
        dict(name="rotate_images", op="rotate", type="f16", new="1501,2301", cached="0,100", heads=16,
             kv_heads=2, dim=256, rotary=64, page=32, layers=1, axes=3, theta=1e4, norm_v=True),
        # drafts of a few tokens checked against four short caches: latency
        dict(name="chunk_drafts", op="chunk", type="bf16", new="5,3,6,5", cached="300,77,641,900", heads=8,
             kv_heads=2, dim=64, page=16, layers=2, window=0, sinks=0),
        # one token of one very long conversation: few rows, a long axis
        dict(name="chunk_token", op="chunk", type="bf16", new="1", cached="98303", heads=32, kv_heads=8,
             dim=128, page=64, layers=1, window=0, sinks=0),
        # continuous batching: a piece of a long prompt beside the next tokens of other chats
        dict(name="chunk_mixed", op="chunk", type="bf16",
             new="2001," + _text([1] * 30), heads=32, kv_heads=8, dim=128,
             cached="6000," + _text([257 * i + 190 for i in range(30)]), page=64, layers=1, window=0, sinks=0),
        # the last piece of a long document
        dict(name="chunk_document", op="chunk", type="bf16", new="4096", cached="28672", heads=16, kv_heads=2,
             dim=128, page=64, layers=1, window=0, sinks=0),
        # a sliding-window layer with wide heads whose first tokens stay visible
        dict(name="chunk_window", op="chunk", type="f16", new="1500,1,700,64", cached="9001,7777,0,4000",
             heads=8, kv_heads=4, dim=256, page=16, layers=1, window=1024, sinks=4),
        # what each token of a batch of chats receives in one step, over two layers
        dict(name="weights_step", op="weights", type="bf16", new=_text([1] * 16),
             cached=_text([3900 - 181 * i for i in range(16)]), heads=32, kv_heads=8, dim=128, page=32,
             layers=2, window=0, sinks=0),
        # what the tokens of long prompts receive from their last queries
        dict(name="weights_prompts", op="weights", type="f16", new="128,128,77,128", cached="8064,12000,3000,5500",
             heads=32, kv_heads=8, dim=128, page=64, layers=1, window=0, sinks=0),
        # two short branches cut down: latency
        dict(name="evict_branches", op="evict", type="f16", cached="301,160", heads=2, dim=64, page=16,
             layers=2, budget=128, sinks=4, recent=32),
        # slim copies of eight long conversations
        dict(name="evict_long", op="evict", type="bf16", cached="6000,8191,4097,7000,5555,6400,7777,3500",
             heads=8, dim=128, page=32, layers=4, budget=2048, sinks=4, recent=256),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotate", "chunk", "weights", "evict"])
    case = dict(op=op, type=rng.choice(["bf16", "f16"]), page=rng.choice([16, 32, 64, 128]))
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 80, 128, 128, 256])
    if op == "evict":
        n = _between(rng, 1, 16)
        most = _between(rng, 40, 8192)
        lens = [rng.randint(1, most) for _ in range(n)]
        layers = _between(rng, 1, 4)
        # no more to hold than the listed conversations
        while 4 * dim * kv * layers * sum(lens) > 8e8:
            lens = [max(1, a // 2) for a in lens]
        sinks, recent = rng.choice([0, 4, 7]), _between(rng, 1, 256)
        return dict(case, cached=_text(lens), heads=kv, dim=dim, layers=layers,
                    budget=sinks + recent + _between(rng, 1, 2048), sinks=sinks, recent=recent)
    heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
    case.update(heads=heads, kv_heads=kv, dim=dim, layers=rng.choice([1, 2]))
    n = _between(rng, 1, 24)
    if op == "rotate":
        new = [_between(rng, 1, 2048) for _ in range(n)] if rng.random() < 0.6 else [1] * n
        # no more rows than the listed prefill batch's
        while sum(new) * (heads + 2 * kv) * dim > 8191 * 48 * 128:
            new = [max(1, a // 2) for a in new]
        axes = rng.choice([1, 1, 2, 3])
        return dict(case, new=_text(new), cached=_text(rng.randint(0, 400) for _ in new),
                    rotary=rng.choice([dim, dim, dim // 32 * 16]), axes=axes,
                    theta=rng.choice([1e4, 5e5, 1e6]), norm_v=rng.random() < 0.3)
    window = rng.choice([0, 0, _between(rng, 16, 2048)])
    case.update(window=window, sinks=rng.choice([0, 1, 4, 40]) if window else 0)
    if op == "chunk":
        kind = rng.choice(["steps", "drafts", "chunks", "mixed"])
        most = _between(rng, 1, 2048)
        new = {"steps": [1] * n, "drafts": [rng.randint(1, 8) for _ in range(n)],
               "chunks": [rng.randint(1, most) for _ in range(n)],
               "mixed": [1 if rng.random() < 0.8 else rng.randint(1, most) for _ in range(n)]}[kind]
        longest = _between(rng, 16, 32768 if n < 8 else 8192)
    else:
        new = [1] * n if rng.random() < 0.5 else [_between(rng, 1, 128) for _ in range(n)]
        longest = _between(rng, 16, 12000 if n < 8 else 4000)
    cached = [rng.randint(0, longest) for _ in new]
    # no more work than the listed document's and prompts'
    while heads * dim * sum(a * (a + b) for a, b in zip(new, cached)) > (2.5e11 if op == "chunk" else 1.5e10):
        new, cached = [max(1, a // 2) for a in new], [b // 2 for b in cached]
    return dict(case, new=_text(new), cached=_text(cached))


def _new(case):
    return _lens(case["new"])


def _all(case):
    """Tokens of each sequence, new ones included."""
    return [a + b for a, b in zip(_new(case), _lens(case["cached"]))]


# ---------------------------------------------------------------------------
# what a pass has to read, write and compute
# ---------------------------------------------------------------------------

def _visible_keys(case):
    """Of each sequence: (query, key) pairs, and keys that some query sees."""
    pairs = keys = 0
    for a, n in zip(_new(case), _all(case)):
        p = np.arange(n - a, n, dtype=np.int64)
        low = np.maximum(0, p - case["window"] + 1) if case["window"] else np.zeros(a, np.int64)
        first = np.minimum(case["sinks"], low)  # keys of the sinks that the window does not hold
        pairs += int((p + 1 - low + first).sum())
        keys += n - int(low[0]) + int(min(case["sinks"], low[0]))
    return pairs, keys


def work(case):
    d = case["dim"]
    if case["op"] == "evict":
        lens = _lens(case["cached"])
        token = 4 * d * case["heads"] * case["layers"]
        kept = [min(n, case["budget"]) for n in lens]
        # the partial pages of the copies, and the rows that are gathered; tables, weights, lists
        moved = sum(n % case["page"] for n in lens) + sum(k for n, k in zip(lens, kept) if k < n)
        table = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * token * moved + 8 * table + 4 * sum(3 * n for n in lens) + 8 * sum(kept), "flops": 0}
    tokens = sum(_new(case))
    if case["op"] == "rotate":
        rows = case["heads"] + 2 * case["kv_heads"]
        return {"bytes": tokens * (4 * d * rows + 4 * case["axes"]), "flops": 0}
    pairs, keys = _visible_keys(case)
    if case["op"] == "chunk":
        return {"bytes": 4 * d * case["kv_heads"] * keys + tokens * case["heads"] * (4 * d + 4),
                "flops": 4 * d * case["heads"] * pairs}
    return {"bytes": case["layers"] * (2 * d * case["kv_heads"] * keys + tokens * case["heads"] * (2 * d + 4))
            + 4 * sum(_all(case)), "flops": case["layers"] * 2 * d * case["heads"] * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device=DEV)


def _offsets(lens):
    return _ints(np.concatenate([[0], np.cumsum(lens)]))


def _paged(s, case, seed, gen, lens, extra_rows=0, extra_pages=3):
    """Pool, table, lengths and references of sequences of these lengths, in shuffled pages."""
    page, kv, dtype = case["page"], case.get("kv_heads", case["heads"]), TYPES[case["type"]]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra_pages
    order = np.random.RandomState(int(seed) % (1 << 31)).permutation(pages)
    table = np.full((len(lens) + extra_rows, max(need) + 1), -1)
    references = np.zeros(pages)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        references[order[at:at + n]] = 1
        at += n
    pool = torch.empty((pages, case["layers"], 2, kv, page, case["dim"]), dtype=dtype, device=DEV)
    for part in pool.split(max(1, (1 << 28) // max(1, pool[0].numel()))):
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV, dtype=torch.float32))
    s.update(pool=pool, table=_ints(table), references=_ints(references),
             lengths=_ints(list(lens) + [0] * extra_rows), rows=_ints(np.arange(len(lens))))


def _handles(s, case):
    """The context and the cache that a program keeps over its buffers."""
    from diskmule_b200 import CudaContext, _native
    from diskmule_b200.attention import KvCache
    s["kind"] = _native.BF16 if case["type"] == "bf16" else _native.F16
    s["context"] = CudaContext(0)
    s["cache"] = KvCache(s["context"], type=s["kind"], layers=case["layers"],
                         kv_heads=case.get("kv_heads", case["heads"]), head_dim=case["dim"],
                         page_tokens=case["page"], pages=s["pool"].shape[0],
                         max_sequences=s["table"].shape[0], max_pages=s["table"].shape[1],
                         memory=s["pool"].data_ptr(), page_table=s["table"].data_ptr(),
                         lengths=s["lengths"].data_ptr(), references=s["references"].data_ptr())


def _frequencies(case):
    return case["theta"] ** (-2.0 * np.arange(case["rotary"] // 2) / case["rotary"])


def _pair_axes(case):
    """Which axis a pair turns with: time, then height and width in equal parts."""
    return np.arange(case["rotary"] // 2) * case["axes"] // (case["rotary"] // 2)


def _positions(case, seed):
    """Text counts on along every axis; an image stands still in time and spans a grid."""
    r = np.random.RandomState(int(seed) % (1 << 31))
    out = []
    for a, cached in zip(_new(case), _lens(case["cached"])):
        p = np.tile(np.arange(cached, cached + a), (case["axes"], 1))
        if case["axes"] > 1 and a > 16:
            begin, size = int(r.randint(0, a // 2)), a // 3
            wide = max(1, int(math.sqrt(size)))
            j = np.arange(size)
            p[:, begin:begin + size] = cached + begin
            p[1, begin:begin + size] += j // wide
            p[-1, begin:begin + size] += j % wide
        out.append(p)
    return np.concatenate(out, 1)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    dtype = TYPES[case["type"]]
    s = {"case": case}
    d = case["dim"]
    if case["op"] == "evict":
        lens = _lens(case["cached"])
        n, page = len(lens), case["page"]
        # copies: a page each for partial last ones, and what the kept tokens are gathered into
        most = sum(-(-min(x, case["budget"]) // page) + 1 for x in lens)
        _paged(s, case, seed, gen, lens, extra_rows=n, extra_pages=most + 3)
        s["children"] = _ints(n + np.arange(n))
        # sums of attention weights: a few tokens have most
        stride = s["table"].shape[1] * page
        s["weights"] = torch.zeros(2 * n, stride, device=DEV)
        for i, x in enumerate(lens):
            s["weights"][i, :x] = torch.randn(x, generator=gen, device=DEV).mul_(2.0).exp_()
        s["keep"] = torch.zeros(n * case["budget"], dtype=torch.int32, device=DEV)
        s["keep_offsets"] = torch.zeros(n + 1, dtype=torch.int32, device=DEV)
        if own:
            _handles(s, case)
        return s
    new, lens = _new(case), _all(case)
    tokens, heads, kv = sum(new), case["heads"], case["kv_heads"]
    _paged(s, case, seed, gen, lens)
    s["offsets"] = _offsets(new)
    s["longest"] = max(lens)
    if case["op"] == "rotate":
        # the fused projection's output: queries, keys and values of a token side by side
        s["qkv"] = _normal(gen, (tokens, heads + 2 * kv, d), dtype, 1.5)
        s["q_weight"] = 1.0 + 0.2 * torch.randn(d, generator=gen, device=DEV)
        s["k_weight"] = 1.0 + 0.2 * torch.randn(d, generator=gen, device=DEV)
        s["positions"] = _ints(_positions(case, seed))
        s["q_out"] = torch.zeros(tokens, heads, d, dtype=dtype, device=DEV)
        if own:
            from diskmule_b200.attention import Rope
            _handles(s, case)
            s["rope"] = Rope(s["context"], case["rotary"], frequencies=_frequencies(case),
                             pair_axes=_pair_axes(case))
        return s
    if case["op"] == "chunk":
        s["q"] = _normal(gen, (tokens, heads, d), dtype, 2.0)
        if own:
            _handles(s, case)
            n = s["cache"].chunk_workspace(heads, len(new), tokens, s["longest"], window=case["window"],
                                           sinks=case["sinks"])
            s["workspace"] = torch.empty(max(16, n), dtype=torch.uint8, device=DEV)
        return s
    s["q"] = _normal(gen, (case["layers"], tokens, heads, d), dtype, 2.0)
    # what attention has returned beside its output
    s["lse"] = torch.stack([_plain_attend(s, s["q"][i], i)[1] for i in range(case["layers"])])
    s["weights"] = torch.zeros(len(new), s["table"].shape[1] * case["page"], device=DEV)
    if own:
        _handles(s, case)
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _plain_rotate(s):
    c = s["case"]
    heads, kv, half = c["heads"], c["kv_heads"], c["rotary"] // 2
    x = s["qkv"].float()
    q, k, v = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]

    def normed(t, weight):
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPSILON)
        return t if weight is None else t * weight

    f = torch.tensor(_frequencies(c), dtype=torch.float64, device=DEV)
    at = s["positions"].double()[torch.tensor(_pair_axes(c), device=DEV)].T  # [tokens, pairs]
    angle = at * f
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(t):
        a, b = t[..., :half], t[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, t[..., 2 * half:]], -1)

    dtype = s["qkv"].dtype
    s["q_out"].copy_(turned(normed(q, s["q_weight"])).to(dtype))
    k = turned(normed(k, s["k_weight"])).to(dtype)
    v = (normed(v, None) if c["norm_v"] else v).to(dtype)
    # into the pages, behind what the sequences had
    offsets, page = s["offsets"].long(), c["page"]
    t = torch.arange(x.shape[0], device=DEV)
    seq = torch.searchsorted(offsets[1:], t, right=True)
    place = s["lengths"].long()[seq] - (offsets[seq + 1] - t)
    ids = s["table"][seq, place // page].long()
    layer = c["layers"] - 1
    s["pool"][ids, layer, 0, :, place % page] = k
    s["pool"][ids, layer, 1, :, place % page] = v
    return {"q": s["q_out"], "pool": s["pool"]}


def _cached(s, i, n, layer):
    """Keys and values of sequence i: [2, kv heads, tokens, dim]."""
    c = s["case"]
    ids = s["table"][i, :-(-n // c["page"])].long()
    x = s["pool"][ids, layer].permute(1, 2, 0, 3, 4)
    return x.reshape(2, c["kv_heads"], -1, c["dim"])[:, :, :n]


def _sees(c, a, n, first, last):
    """Which keys the new tokens first .. last - 1 of a sequence see: [rows, keys]."""
    p = torch.arange(n - a + first, n - a + last, device=DEV)[:, None]
    j = torch.arange(n, device=DEV)
    seen = j <= p
    if c["window"]:
        seen = seen & ((j > p - c["window"]) | (j < c["sinks"]))
    return seen


def _plain_attend(s, q, layer):
    c = s["case"]
    heads, kv, d = c["heads"], c["kv_heads"], c["dim"]
    g = heads // kv
    outs, lses, at = [], [], 0
    for i, (a, n) in enumerate(zip(_new(c), _all(c))):
        both = _cached(s, i, n, layer).float()
        step = max(1, (1 << 29) // (heads * n))  # rows whose scores fit
        for r0 in range(0, a, step):
            r1 = min(a, r0 + step)
            x = q[at + r0:at + r1].float().view(r1 - r0, kv, g, d).permute(1, 2, 0, 3)
            score = torch.matmul(x.reshape(kv, -1, d) * (1.0 / math.sqrt(d)), both[0].transpose(1, 2))
            score = score.view(kv, g, r1 - r0, n).masked_fill_(~_sees(c, a, n, r0, r1), -math.inf)
            top = score.amax(-1, keepdim=True)
            score.sub_(top).exp_()
            total = score.sum(-1, keepdim=True)
            out = torch.matmul(score.view(kv, -1, n), both[1]).view(kv, g, r1 - r0, d) / total
            outs.append(out.permute(2, 0, 1, 3).reshape(r1 - r0, heads, d))
            lses.append((top + torch.log(total)).squeeze(-1).permute(2, 0, 1).reshape(r1 - r0, heads))
        at += a
    return torch.cat(outs).to(q.dtype), torch.cat(lses)


def _plain_weights(s):
    c = s["case"]
    heads, kv, d = c["heads"], c["kv_heads"], c["dim"]
    s["weights"].zero_()
    for layer in range(c["layers"]):
        at = 0
        for i, (a, n) in enumerate(zip(_new(c), _all(c))):
            k = _cached(s, i, n, layer)[0].float()
            x = s["q"][layer, at:at + a].float().view(a, kv, heads // kv, d).permute(1, 2, 0, 3)
            score = torch.matmul(x.reshape(kv, -1, d) * (1.0 / math.sqrt(d)), k.transpose(1, 2))
            score = score.view(kv, heads // kv, a, n)
            lse = s["lse"][layer, at:at + a].view(a, kv, heads // kv).permute(1, 2, 0)[..., None]
            weight = torch.exp(score - lse).masked_fill_(~_sees(c, a, n, 0, a), 0.0)
            s["weights"][i, :n] += weight.sum((0, 1, 2))
            at += a
    return {"weights": s["weights"]}


def _free_pages(s):
    """Page numbers, the free ones first and ascending."""
    return torch.sort((s["references"] > 0).to(torch.uint8), stable=True).indices


def _plain_evict(s):
    c = s["case"]
    page, budget = c["page"], c["budget"]
    table, lengths, references = s["table"], s["lengths"], s["references"]
    col = torch.arange(table.shape[1], device=DEV)
    parents, children = s["rows"].long(), s["children"].long()

    def release(rows, held):
        references.scatter_add_(0, table[rows].long().clamp_min(0).flatten(), -held.flatten().int())

    # the last copies go
    release(children, col < ((lengths[children] + page - 1) // page)[:, None])
    table[children] = -1
    # new ones: full pages shared, a partial last one copied
    lens = lengths[parents].long()
    full, rest = (lens // page)[:, None], lens % page
    taken = _free_pages(s)[torch.cumsum((rest > 0).long(), 0) - 1]
    entries = table[parents].long()
    old = torch.where(rest > 0, entries.gather(1, full).squeeze(1), entries[:, 0])
    new = torch.where(rest > 0, taken, old)
    row = torch.arange(page, device=DEV)[None, None, None, None, :, None]
    used = row < rest[:, None, None, None, None, None]
    s["pool"][new] = torch.where(used, s["pool"][old], s["pool"][new])
    references.scatter_add_(0, entries.clamp_min(0).flatten(), (col < full).flatten().int())
    references.scatter_add_(0, taken.clamp_min(0), (rest > 0).int())
    entries = torch.where(col < full, entries,
                          torch.where((col == full) & (rest > 0)[:, None], new[:, None], -1))
    table[children] = entries.int()
    lengths[children] = lens.int()
    s["weights"][children] = s["weights"][parents]
    # the tokens that stay: first and last ones, then the heaviest, the earlier of equals
    weights = s["weights"][children]
    j = torch.arange(weights.shape[1], device=DEV)
    inside = j < lens[:, None]
    always = inside & ((j < c["sinks"]) | (j >= (lens - c["recent"])[:, None]))
    value = weights.masked_fill(always, math.inf).masked_fill(~inside, -math.inf)
    order = torch.sort(value, dim=1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, j.expand_as(order).contiguous())
    stays = inside & (rank < budget)
    count = torch.minimum(lens, torch.full_like(lens, budget))
    slot = torch.cumsum(stays.long(), 1) - 1
    source = torch.zeros(lens.numel(), budget + 1, dtype=torch.long, device=DEV)
    source.scatter_(1, torch.where(stays, slot, torch.full_like(slot, budget)), j.expand_as(slot))
    source = source[:, :budget]
    k = torch.arange(budget, device=DEV)
    valid = k < count[:, None]
    s["keep_offsets"][1:] = torch.cumsum(count, 0).int()
    s["keep_offsets"][0] = 0
    flat = torch.where(valid, s["keep_offsets"][:-1, None].long() + k, torch.full_like(source, s["keep"].numel()))
    s["keep"].copy_(torch.cat([s["keep"], s["keep"][:1]]).scatter(0, flat.flatten(), source.int().flatten())[:-1])
    # their rows move to fresh pages, but for leading pages that stay as they are
    same = torch.cumprod(((source == k) & valid).long(), 1).sum(1)
    now, before = (count + page - 1) // page, (lens + page - 1) // page
    stay = torch.where(same == count, now, same // page)
    last = entries.gather(1, (now - 1)[:, None]).squeeze(1)
    stay = torch.where((same == count) & (count % page > 0) & (references[last.clamp_min(0)] > 1), now - 1, stay)
    fresh = (col >= stay[:, None]) & (col < now[:, None])
    taken = _free_pages(s)[(torch.cumsum(fresh.flatten().long(), 0).view(fresh.shape) - 1).clamp_min(0)]
    after = torch.where(fresh, taken, torch.where(col < stay[:, None], entries, -1))
    moves = valid & (k >= (stay * page)[:, None])
    from_page = entries.gather(1, source // page).clamp_min(0)
    to_page = torch.where(moves, after.gather(1, (k // page).clamp_max(col.numel() - 1).expand(source.shape)), from_page)
    to_row = torch.where(moves, (k % page).expand(source.shape), source % page)
    s["pool"][to_page.flatten(), :, :, :, to_row.flatten()] = \
        s["pool"][from_page.flatten(), :, :, :, (source % page).flatten()]
    release(children, (col >= stay[:, None]) & (col < before[:, None]))
    references.scatter_add_(0, taken.flatten(), fresh.flatten().int())
    table[children] = after.int()
    lengths[children] = count.int()
    # the weights go along; what is behind them starts anew
    moved = torch.zeros_like(weights)
    wide = min(budget, weights.shape[1])
    moved[:, :wide] = torch.where(valid, weights.gather(1, source), torch.zeros((), device=DEV))[:, :wide]
    s["weights"][children] = moved


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_rotate(s):
    from diskmule_b200.attention import rotate
    c, x = s["case"], s["qkv"]
    heads, kv, d = c["heads"], c["kv_heads"], c["dim"]
    at, step = x.data_ptr(), d * x.element_size()
    strides = (x.stride(0), x.stride(1))
    rotate(s["context"], s["rope"], type=s["kind"], heads=heads, kv_heads=kv, head_dim=d, tokens=x.shape[0],
           q=at, k=at + heads * step, v=at + (heads + kv) * step, q_out=s["q_out"].data_ptr(),
           q_stride=strides, k_stride=strides, v_stride=strides, cache=s["cache"], layer=c["layers"] - 1,
           sequences=s["rows"].data_ptr(), offsets=s["offsets"].data_ptr(), n=s["rows"].numel(),
           positions=s["positions"].data_ptr(), norm_q=True, norm_k=True, norm_v=c["norm_v"],
           q_weight=s["q_weight"].data_ptr(), k_weight=s["k_weight"].data_ptr(), epsilon=EPSILON,
           stream=_stream())
    return {"q": s["q_out"], "pool": s["pool"]}


def _own_chunk(s):
    c, q = s["case"], s["q"]
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=DEV)
    s["cache"].chunk_attention(
        layer=c["layers"] - 1, heads=c["heads"], q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
        sequences=s["rows"].data_ptr(), offsets=s["offsets"].data_ptr(), n=s["rows"].numel(),
        tokens=q.shape[0], max_length=s["longest"], window=c["window"], sinks=c["sinks"],
        workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel(), stream=_stream())
    return {"out": out, "lse": lse}


def _own_weights(s):
    c = s["case"]
    s["weights"].zero_()
    for layer in range(c["layers"]):
        s["cache"].token_weights(
            layer=layer, heads=c["heads"], q=s["q"][layer].data_ptr(), lse=s["lse"][layer].data_ptr(),
            sequences=s["rows"].data_ptr(), offsets=s["offsets"].data_ptr(), n=s["rows"].numel(),
            tokens=s["q"].shape[1], max_length=s["longest"], weights=s["weights"].data_ptr(),
            weights_stride=s["weights"].stride(0), window=c["window"], sinks=c["sinks"], stream=_stream())
    return {"weights": s["weights"]}


def _own_evict(s):
    c, cache, n = s["case"], s["cache"], s["rows"].numel()
    rows, children, stream = s["rows"].data_ptr(), s["children"].data_ptr(), _stream()
    cache.free(children, n, stream=stream)
    cache.fork(rows, children, n, stream=stream)
    s["weights"][n:].copy_(s["weights"][:n])
    cache.evict(sequences=children, n=n, budget=c["budget"], sinks=c["sinks"], recent=c["recent"],
                weights=s["weights"].data_ptr(), weights_stride=s["weights"].stride(0),
                keep_offsets=s["keep_offsets"].data_ptr(), keep=s["keep"].data_ptr(), stream=stream)


def run(state):
    op = state["case"]["op"]
    if op == "rotate":
        return _own_rotate(state) if own else _plain_rotate(state)
    if op == "chunk":
        if own:
            return _own_chunk(state)
        out, lse = _plain_attend(state, state["q"], state["case"]["layers"] - 1)
        return {"out": out, "lse": lse}
    if op == "weights":
        return _own_weights(state) if own else _plain_weights(state)
    if own:
        _own_evict(state)
    else:
        _plain_evict(state)
    return {k: state[k] for k in ("table", "lengths", "references", "pool", "weights", "keep", "keep_offsets")}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _exact_rotate(s):
    c = s["case"]
    d, half, heads, kv = c["dim"], c["rotary"] // 2, c["heads"], c["kv_heads"]
    f, axis = _frequencies(c), _pair_axes(c)
    position = s["positions"].cpu().numpy().astype(np.float64)
    # each pair is a complex number that turns
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                       torch.tensor((position[axis] * f[:, None]).T.copy(), device=DEV))[:, None]
    x = s["qkv"].double()

    def head(t, weight, rotates):
        if weight is not None:
            t = t / (t.pow(2).sum(-1, keepdim=True) / d + EPSILON).sqrt() * weight
        if not rotates:
            return t
        z = torch.complex(t[..., :half].contiguous(), t[..., half:2 * half].contiguous()) * turn
        return torch.cat([z.real, z.imag, t[..., 2 * half:]], -1)

    q = head(x[:, :heads], s["q_weight"].double(), True)
    k = head(x[:, heads:heads + kv], s["k_weight"].double(), True)
    v = head(x[:, heads + kv:], 1.0 if c["norm_v"] else None, False)
    pool = s["pool"].double()
    table = s["table"].cpu().numpy()
    at = 0
    for i, (a, n) in enumerate(zip(_new(c), _all(c))):
        place = np.arange(n - a, n)
        ids = torch.tensor(table[i, place // c["page"]].astype(np.int64), device=DEV)
        inside = torch.tensor(place % c["page"], device=DEV)
        pool[ids, c["layers"] - 1, 0, :, inside] = k[at:at + a]
        pool[ids, c["layers"] - 1, 1, :, inside] = v[at:at + a]
        at += a
    return {"q": q, "pool": pool}


def _exact_scores(s, case, layer, visit):
    """visit(sequence, kv head, rows of q, scores with hidden keys at -inf, values) for pieces of
    each sequence's queries, in 64 bits."""
    kv, d, page = case["kv_heads"], case["dim"], case["page"]
    g = case["heads"] // kv
    q = s["q"] if case["op"] == "chunk" else s["q"][layer]
    at = 0
    for i, (a, n) in enumerate(zip(_new(case), _all(case))):
        ids = s["table"][i, :-(-n // page)].tolist()
        for h in range(kv):
            k = torch.cat([s["pool"][p, layer, 0, h] for p in ids])[:n].double()
            v = torch.cat([s["pool"][p, layer, 1, h] for p in ids])[:n].double()
            for r0 in range(0, a, 1024):
                r1 = min(a, r0 + 1024)
                rows = slice(at + r0, at + r1)
                x = q[rows, h * g:(h + 1) * g].double()  # [rows, g, d]
                score = torch.einsum("rgd,nd->rgn", x, k) / math.sqrt(d)
                place = torch.arange(n - a + r0, n - a + r1, device=DEV)[:, None, None]
                key = torch.arange(n, device=DEV)
                hidden = key > place
                if case["window"]:
                    hidden = hidden | ((place - key >= case["window"]) & (key >= case["sinks"]))
                visit(i, h, rows, score.masked_fill(hidden, -math.inf), v)
        at += a


def exact(case, seed):
    global own
    if case["op"] == "evict":
        return None  # copies and whole numbers
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    if case["op"] == "rotate":
        return _exact_rotate(s)
    g = case["heads"] // case["kv_heads"]
    if case["op"] == "chunk":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)

        def attend(i, h, rows, score, v):
            e = torch.logsumexp(score, -1)
            lse[rows, h * g:(h + 1) * g] = e
            out[rows, h * g:(h + 1) * g] = torch.einsum("rgn,nd->rgd", torch.exp(score - e[..., None]), v)

        _exact_scores(s, case, case["layers"] - 1, attend)
        return {"out": out, "lse": lse}
    weights = torch.zeros(s["weights"].shape, dtype=torch.float64, device=DEV)
    for layer in range(case["layers"]):
        def add(i, h, rows, score, v):
            e = s["lse"][layer][rows, h * g:(h + 1) * g].double()
            weights[i, :score.shape[-1]] += torch.exp(score - e[..., None]).sum((0, 1))

        _exact_scores(s, case, layer, add)
    return {"weights": weights}
