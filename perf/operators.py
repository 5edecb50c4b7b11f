"""Workloads of the attention operators: prompt attention, decode attention over a
shared prefix, and the page operations of the key/value cache.

Each case runs one pass the way a serving program does; `run` computes it in elementary
torch operations (32-bit arithmetic, one rounding at the end) or, with `own` set, through
`diskmule_b200.attention`. `exact` is the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _lens(text):
    return [int(v) for v in text.split(",")]


def listed():
    return [
        # four short chat turns that arrive together: launch latency and mostly empty tiles
        dict(name="prompt_short", op="prompt", type="bf16", q="3,17,1,40", k="3,17,1,40", heads=8,
             kv_heads=2, dim=64, causal=True, window=0),
        # an ordinary prefill batch: ragged prompts packed end to end
        dict(name="prompt_packed", op="prompt", type="bf16", q="1777,129,640,1023,300,911,1500,58",
             k="1777,129,640,1023,300,911,1500,58", heads=32, kv_heads=8, dim=128, causal=True,
             window=0),
        # one long document
        dict(name="prompt_long", op="prompt", type="bf16", q="16384", k="16384", heads=16, kv_heads=2,
             dim=128, causal=True, window=0),
        # a sliding-window layer with wide heads; the first prompt continues a cached one
        dict(name="prompt_window", op="prompt", type="f16", q="2500,1000", k="4099,1000", heads=8,
             kv_heads=4, dim=256, causal=True, window=1024),
        # two continuations of a short system prompt: latency
        dict(name="decode_two", op="decode", type="f16", batch=2, shared=160, own_low=1, own_high=40,
             heads=8, kv_heads=2, dim=64, page=16, layers=2),
        # a batch of chats behind one system prompt
        dict(name="decode_chats", op="decode", type="bf16", batch=16, shared=2048, own_low=0,
             own_high=600, heads=32, kv_heads=8, dim=128, page=32, layers=1),
        # many samples of an answer about one long document
        dict(name="decode_samples", op="decode", type="bf16", batch=64, shared=32768, own_low=1,
             own_high=1500, heads=64, kv_heads=8, dim=128, page=64, layers=1),
        # wide heads, small pages
        dict(name="decode_wide", op="decode", type="bf16", batch=24, shared=8192, own_low=100,
             own_high=900, heads=16, kv_heads=2, dim=256, page=16, layers=1),
        # beam search: eight beams taken anew from four
        dict(name="fork_beams", op="fork", type="bf16", parents=4, children=8, low=20, high=120,
             heads=2, dim=64, page=16, layers=4),
        # sixteen prompts, sixteen samples each
        dict(name="fork_samples", op="fork", type="bf16", parents=16, children=256, low=300, high=2500,
             heads=8, dim=128, page=64, layers=16),
        # a draft tree per sequence: append the draft, keep the accepted path
        dict(name="compact_draft", op="compact", type="f16", parents=8, children=8, low=40, high=900,
             heads=4, dim=128, page=16, layers=4, draft=13, keep=1.0),
        # eviction: half of the tokens of long sequences go
        dict(name="compact_evict", op="compact", type="bf16", parents=16, children=16, low=1500,
             high=3000, heads=8, dim=128, page=16, layers=8, draft=1, keep=0.5),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["prompt", "decode", "fork", "compact"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "prompt":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
        n = _between(rng, 1, 12)
        most = _between(rng, 16, 6000)
        q = [rng.randint(1, most) for _ in range(n)]
        if rng.random() < 0.3:  # chunks of prompts whose beginnings are cached
            k = [a + rng.randint(0, most) for a in q]
        else:
            k = list(q)
        # no more work than the long document's
        while n * heads * dim * max(q) * max(k) > 2.5e11:
            q, k = [max(1, a // 2) for a in q], [max(1, a // 2) for a in k]
        window = rng.choice([0, 0, _between(rng, 16, 2048)])
        return dict(op=op, type=dtype, q=",".join(map(str, q)), k=",".join(map(str, k)), heads=heads,
                    kv_heads=kv, dim=dim, causal=rng.random() < 0.85 or window > 0, window=window)
    if op == "decode":
        page = rng.choice([16, 32, 64, 128])
        kv = rng.choice([1, 2, 4, 8])
        high = _between(rng, 2, 1500)
        return dict(op=op, type=dtype, batch=_between(rng, 1, 64),
                    shared=page * (_between(rng, 1, 32768 // page) - 1), own_low=rng.choice([0, 1]),
                    own_high=high, heads=kv * rng.choice([1, 2, 4, 5, 8]), kv_heads=kv,
                    dim=rng.choice([64, 80, 128, 128, 256]), page=page, layers=rng.choice([1, 2]))
    case = dict(op=op, type=dtype, heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 80, 128, 256]),
                page=rng.choice([16, 32, 64]), layers=_between(rng, 1, 8))
    if op == "fork":
        parents = _between(rng, 1, 16)
        return dict(case, parents=parents, children=parents * _between(rng, 1, 16), low=1,
                    high=_between(rng, 8, 2500))
    parents = _between(rng, 1, 16)
    return dict(case, parents=parents, children=parents, low=1, high=_between(rng, 8, 2500),
                draft=_between(rng, 1, 40), keep=rng.choice([1.0, round(rng.uniform(0.2, 0.95), 2)]))


def _own_lens(case):
    """Tokens of each decode sequence behind the shared ones; one at least in the batch."""
    r = np.random.RandomState(case["batch"] * 1009 + case["own_high"])
    own_ = r.randint(case["own_low"], case["own_high"] + 1, case["batch"])
    own_[0] = case["own_high"]
    return own_


def _parent_lens(case):
    r = np.random.RandomState(case["parents"] * 1013 + case["high"])
    n = r.randint(case["low"], case["high"] + 1, case["parents"])
    n[0] = case["high"]
    return n


def _kept(case):
    """The token positions that each child keeps, ascending."""
    r = np.random.RandomState(case["children"] * 1019 + case["draft"])
    kept = []
    for c in range(case["children"]):
        n = int(_parent_lens(case)[c % case["parents"]])
        if case["keep"] < 1.0:
            total = n + case["draft"]
            m = max(1, int(case["keep"] * total))
            kept.append(np.sort(r.permutation(total)[:m]))
        else:  # the whole sequence and a random path of the draft
            path = n + np.nonzero(r.rand(case["draft"]) < 0.4)[0]
            kept.append(np.concatenate([np.arange(n), path]))
    return kept


# ---------------------------------------------------------------------------
# what a pass has to read, write and compute
# ---------------------------------------------------------------------------

def _pairs(case):
    total = 0
    for lq, lk in zip(_lens(case["q"]), _lens(case["k"])):
        i = np.arange(lq, dtype=np.int64) + (lk - lq)
        high = np.minimum(i + 1, lk) if case["causal"] else np.full(lq, lk)
        low = np.maximum(0, i - case["window"] + 1) if case["window"] else np.zeros(lq, np.int64)
        total += int(np.maximum(0, high - low).sum())
    return total


def work(case):
    d = case["dim"]
    if case["op"] == "prompt":
        q, k = sum(_lens(case["q"])), sum(_lens(case["k"]))
        return {"bytes": 2 * d * (2 * q * case["heads"] + 2 * k * case["kv_heads"]) + 4 * q * case["heads"],
                "flops": 4 * d * case["heads"] * _pairs(case)}
    if case["op"] == "decode":
        own_ = int(_own_lens(case).sum())
        rows = case["batch"] * case["heads"]
        return {"bytes": 4 * d * case["kv_heads"] * (case["shared"] + own_) + rows * (4 * d + 4),
                "flops": 4 * d * case["heads"] * (case["batch"] * case["shared"] + own_)}
    token = 4 * d * case["heads"] * case["layers"]  # K and V of one token, all layers
    lens = _parent_lens(case)
    of = [int(lens[c % case["parents"]]) for c in range(case["children"])]
    table = sum(-(-n // case["page"]) for n in of)
    if case["op"] == "fork":
        rows = sum(n % case["page"] for n in of)
        return {"bytes": 2 * token * rows + 8 * table, "flops": 0}
    moved = sum(n % case["page"] for n in of)
    for n, keep in zip(of, _kept(case)):
        same = int((keep == np.arange(len(keep))).sum())  # leading tokens that stay
        moved += 0 if same == len(keep) else len(keep) - same // case["page"] * case["page"]
    new = 4 * d * case["heads"] * case["children"] * case["draft"]
    return {"bytes": 2 * token * moved + 2 * new + 8 * table, "flops": 0}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _ints(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device=DEV)


def _offsets(lens):
    return _ints(np.concatenate([[0], np.cumsum(lens)]))


def _pool(gen, case, kv_heads, pages, dtype):
    shape = (pages, case["layers"], 2, kv_heads, case["page"], case["dim"])
    pool = torch.empty(shape, dtype=dtype, device=DEV)
    for part in pool.split(max(1, (1 << 28) // max(1, pool[0].numel()))):
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV, dtype=torch.float32))
    return pool


def _cache(s, case, kv_heads):
    """The handle that a program keeps over its cache's buffers."""
    if own:
        from diskmule_b200 import CudaContext, _native
        from diskmule_b200.attention import KvCache
        kind = _native.BF16 if case["type"] == "bf16" else _native.F16
        s["context"] = CudaContext(0)
        s["cache"] = KvCache(s["context"], type=kind, layers=case["layers"], kv_heads=kv_heads,
                             head_dim=case["dim"], page_tokens=case["page"], pages=s["pool"].shape[0],
                             max_sequences=s["table"].shape[0], max_pages=s["table"].shape[1],
                             memory=s["pool"].data_ptr(), page_table=s["table"].data_ptr(),
                             lengths=s["lengths"].data_ptr(), references=s["references"].data_ptr())


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    shuffle = np.random.RandomState(int(seed) % (1 << 31))
    dtype = TYPES[case["type"]]
    s = {"case": case}
    d = case["dim"]
    if case["op"] == "prompt":
        lq, lk = _lens(case["q"]), _lens(case["k"])
        # the fused projection's output where every token has its own keys
        s["q"] = _normal(gen, (sum(lq), case["heads"], d), dtype, 2.0)
        s["k"] = _normal(gen, (sum(lk), case["kv_heads"], d), dtype)
        s["v"] = _normal(gen, (sum(lk), case["kv_heads"], d), dtype)
        s["q_offsets"], s["k_offsets"] = _offsets(lq), _offsets(lk)
        if own:
            from diskmule_b200 import CudaContext
            s["context"] = CudaContext(0)
        return s
    if case["op"] == "decode":
        page, b = case["page"], case["batch"]
        own_ = _own_lens(case)
        shared = case["shared"] // page
        need = [-(-int(n) // page) for n in own_]
        pages = shared + sum(need) + 3
        order = shuffle.permutation(pages)
        table = np.full((b, shared + max(need) + 1), -1)
        table[:, :shared] = order[:shared]
        at = shared
        for i, n in enumerate(need):
            table[i, shared:shared + n] = order[at:at + n]
            at += n
        s["pool"] = _pool(gen, case, case["kv_heads"], pages, dtype)
        s["table"], s["lengths"] = _ints(table), _ints(own_ + case["shared"])
        references = np.zeros(pages)
        references[order[:shared]] = b
        references[order[shared:at]] = 1
        s["references"] = _ints(references)
        s["rows"] = _ints(np.arange(b))
        s["longest"] = int(own_.max()) + case["shared"]
        s["q"] = _normal(gen, (b, case["heads"], d), dtype, 2.0)
        _cache(s, case, case["kv_heads"])
        if own:
            n = s["cache"].decode_workspace(case["heads"], b, case["shared"], s["longest"])
            s["workspace"] = torch.empty(max(16, n), dtype=torch.uint8, device=DEV)
        return s
    # fork and compact: parents in the first rows, children behind them
    page, lens, children = case["page"], _parent_lens(case), case["children"]
    need = [-(-int(n) // page) for n in lens]
    draft = case.get("draft", 0)
    longest = int(lens.max()) + draft
    # compaction gathers into fresh pages while the old ones are still held
    pages = sum(need) + children * ((2 * -(-longest // page) if draft else 1) + 1)
    order = shuffle.permutation(pages)
    table = np.full((case["parents"] + children, -(-longest // page) + 1), -1)
    references = np.zeros(pages)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        references[order[at:at + n]] = 1
        at += n
    s["pool"] = _pool(gen, case, case["heads"], pages, dtype)
    s["table"], s["references"] = _ints(table), _ints(references)
    s["lengths"] = _ints(np.concatenate([lens, np.zeros(children, int)]))
    s["from"] = _ints(np.arange(children) % case["parents"])
    s["to"] = _ints(case["parents"] + np.arange(children))
    s["pages_per_row"] = -(-longest // page)
    if draft:
        s["counts"] = _ints(np.full(children, draft))
        s["new_offsets"] = _offsets([draft] * children)
        kept = _kept(case)
        s["keep"], s["keep_offsets"] = _ints(np.concatenate(kept)), _offsets([len(x) for x in kept])
        s["most_kept"] = max(len(x) for x in kept)
        s["k"] = _normal(gen, (children * draft, case["heads"], d), dtype)
        s["v"] = _normal(gen, (children * draft, case["heads"], d), dtype)
    _cache(s, case, case["heads"])
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _softmax_values(score, visible, values):
    """exp-normalised sums of `values` [.., keys, dim] under `score` [.., rows, keys], and
    ln of the sums. A row that sees nothing gives zeros and -inf."""
    score.masked_fill_(~visible, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score, values) / torch.where(total > 0, total, torch.ones_like(total))
    return out, (top + torch.log(total)).squeeze(-1)


def _plain_prompt(s):
    c = s["case"]
    heads, kv, d = c["heads"], c["kv_heads"], c["dim"]
    g = heads // kv
    mq, mk = max(_lens(c["q"])), max(_lens(c["k"]))
    qo, ko = s["q_offsets"].long(), s["k_offsets"].long()
    n = qo.numel() - 1
    lq, lk = (qo[1:] - qo[:-1])[:, None], (ko[1:] - ko[:-1])[:, None]
    iq, ik = torch.arange(mq, device=DEV), torch.arange(mk, device=DEV)
    # padded copies [sequence, kv head, rows, dim]
    at_q = (qo[:-1, None] + iq).clamp_max(s["q"].shape[0] - 1)
    at_k = (ko[:-1, None] + ik).clamp_max(s["k"].shape[0] - 1)
    q = s["q"][at_q].float().view(n, mq, kv, g, d).permute(0, 2, 3, 1, 4).reshape(n, kv, g * mq, d)
    k = s["k"][at_k].float().permute(0, 2, 3, 1)
    v = s["v"][at_k].float().masked_fill((ik >= lk)[:, :, None, None], 0).permute(0, 2, 1, 3)
    score = torch.matmul(q * (1.0 / math.sqrt(d)), k)
    del q, k
    place = (iq + lk - lq)[:, :, None]
    visible = (ik < lk)[:, None, :] & (iq < lq)[:, :, None]
    if c["causal"]:
        visible = visible & (ik <= place)
    if c["window"]:
        visible = visible & (ik > place - c["window"])
    out, lse = _softmax_values(score.view(n, kv, g, mq, mk), visible[:, None, None], v[:, :, None])
    # back to packed rows
    row = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(qo[1:], row, right=True)
    out = out.permute(0, 3, 1, 2, 4)[seq, row - qo[seq]].reshape(-1, heads, d)
    lse = lse.permute(0, 3, 1, 2)[seq, row - qo[seq]].reshape(-1, heads)
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _plain_decode(s):
    c = s["case"]
    b, heads, kv, d, page, shared = (c[x] for x in ("batch", "heads", "kv_heads", "dim", "page", "shared"))
    layer = s["pool"][:, c["layers"] - 1]
    q = s["q"].float().view(b, kv, heads // kv, d) * (1.0 / math.sqrt(d))
    first = shared // page
    last = -(-s["longest"] // page)
    lens = s["lengths"].long()
    # the shared pages once: [kv, tokens, dim]
    pre = layer[s["table"][0, :first].long()].float()
    pk, pv = (pre[:, i].permute(1, 0, 2, 3).reshape(kv, shared, d) for i in (0, 1))
    s_pre = torch.matmul(q.permute(1, 0, 2, 3).reshape(kv, -1, d), pk.transpose(1, 2))
    s_pre = s_pre.view(kv, b, heads // kv, shared).permute(1, 0, 2, 3)
    # each sequence's own pages, padded to the longest: [b, kv, tokens, dim]
    at = s["table"][:, first:last].long().clamp_min(0)
    mine = layer[at].float()
    mk, mv = (mine[:, :, i].permute(0, 2, 1, 3, 4).reshape(b, kv, -1, d) for i in (0, 1))
    place = shared + torch.arange(mk.shape[2], device=DEV)
    visible = (place < lens[:, None])[:, None, None]
    s_own = torch.matmul(q, mk.transpose(2, 3)).masked_fill_(~visible, -math.inf)
    top = torch.cat([s_pre, s_own], -1).amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p_pre, p_own = (s_pre - top).exp(), (s_own - top).exp()
    total = p_pre.sum(-1, keepdim=True) + p_own.sum(-1, keepdim=True)
    o_pre = torch.matmul(p_pre.permute(1, 0, 2, 3).reshape(kv, -1, shared), pv)
    o_pre = o_pre.view(kv, b, heads // kv, d).permute(1, 0, 2, 3)
    out = o_pre + torch.matmul(p_own, mv.masked_fill((place >= lens[:, None])[:, None, :, None], 0))
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    return {"out": out.reshape(b, heads, d).to(s["q"].dtype),
            "lse": (top + torch.log(total)).reshape(b, heads)}


def _release(s, rows, held):
    """One reference less for each page of `held` (a mask over the rows' table entries)."""
    ids = s["table"][rows].long().clamp_min(0)
    s["references"].scatter_add_(0, ids.flatten(), -held.flatten().int())


def _columns(s):
    return torch.arange(s["table"].shape[1], device=DEV)


def _free_pages(s):
    """Page numbers, the free ones first and ascending."""
    return torch.sort((s["references"] > 0).to(torch.uint8), stable=True).indices


def _plain_free(s, rows):
    page = s["case"]["page"]
    held = _columns(s) < ((s["lengths"][rows] + page - 1) // page)[:, None]
    _release(s, rows, held)
    s["table"][rows] = -1
    s["lengths"][rows] = 0


def _plain_fork(s, parents, children):
    page, col = s["case"]["page"], _columns(s)
    lens = s["lengths"][parents].long()
    full, rest = (lens // page)[:, None], lens % page
    taken = _free_pages(s)[torch.cumsum((rest > 0).long(), 0) - 1]
    entries = s["table"][parents].long()
    old = torch.where(rest > 0, entries.gather(1, full.clamp_max(col.numel() - 1)).squeeze(1),
                      entries[:, 0].clamp_min(0))
    new = torch.where(rest > 0, taken, old)
    # used rows of the partial page; a row with none copies a page onto itself
    row = torch.arange(page, device=DEV)[None, None, None, None, :, None]
    used = row < rest[:, None, None, None, None, None]
    s["pool"][new] = torch.where(used, s["pool"][old], s["pool"][new])
    s["references"].scatter_add_(0, entries.clamp_min(0).flatten(), (col < full).flatten().int())
    s["references"].scatter_add_(0, taken.clamp_min(0), (rest > 0).int())
    partial = (col == full) & (rest > 0)[:, None]
    s["table"][children] = torch.where(col < full, entries, torch.where(partial, new[:, None], -1)).int()
    s["lengths"][children] = lens.int()


def _plain_extend(s, rows, counts):
    page, col = s["case"]["page"], _columns(s)
    old = (s["lengths"][rows].long() + page - 1) // page
    lens = s["lengths"][rows].long() + counts
    new = (lens + page - 1) // page
    fresh = (col >= old[:, None]) & (col < new[:, None])
    rank = torch.cumsum(fresh.flatten().long(), 0).view(fresh.shape) - 1
    taken = _free_pages(s)[rank.clamp_min(0)]
    s["table"][rows] = torch.where(fresh, taken, s["table"][rows].long()).int()
    s["references"].scatter_add_(0, taken.flatten(), fresh.flatten().int())
    s["lengths"][rows] = lens.int()


def _plain_write(s, layer, k, v, rows, offsets):
    page = s["case"]["page"]
    at = torch.arange(k.shape[0], device=DEV)
    seq = torch.searchsorted(offsets[1:].long(), at, right=True)
    place = s["lengths"][rows].long()[seq] - (offsets.long()[seq + 1] - at)
    ids = s["table"][rows.long()[seq], place // page].long()
    s["pool"][ids, layer, 0, :, place % page] = k
    s["pool"][ids, layer, 1, :, place % page] = v


def _plain_compact(s, rows, keep_offsets, keep, most):
    page, col = s["case"]["page"], _columns(s)
    off = keep_offsets.long()
    count = off[1:] - off[:-1]
    j = torch.arange(most, device=DEV)
    inside = j < count[:, None]
    source = keep.long()[(off[:-1, None] + j).clamp_max(keep.numel() - 1)]
    same = torch.cumprod(((source == j) & inside).long(), 1).sum(1)
    new = (count + page - 1) // page
    old = (s["lengths"][rows].long() + page - 1) // page
    entries = s["table"][rows].long()
    # a sequence that only loses its tail keeps its pages, unless the last one is partial and shared
    last = entries.gather(1, (new - 1).clamp_min(0)[:, None]).squeeze(1).clamp_min(0)
    split = (count % page > 0) & (s["references"][last] > 1)
    stay = torch.where((same == count) & ~split, new, same // page)
    fresh = (col >= stay[:, None]) & (col < new[:, None])
    rank = torch.cumsum(fresh.flatten().long(), 0).view(fresh.shape) - 1
    taken = _free_pages(s)[rank.clamp_min(0)]
    after = torch.where(fresh, taken, torch.where(col < stay[:, None], entries, -1))
    held = (col >= stay[:, None]) & (col < old[:, None])
    # gather the kept tokens; what does not move is written onto itself
    from_page = entries.gather(1, source // page).clamp_min(0)
    moves = inside & (j >= (stay * page)[:, None])
    to_page = torch.where(moves, after.gather(1, (j // page).expand(source.shape)), from_page)
    to_row = torch.where(moves, j.expand(source.shape) % page, source % page)
    s["pool"][to_page.flatten(), :, :, :, to_row.flatten()] = \
        s["pool"][from_page.flatten(), :, :, :, (source % page).flatten()]
    _release(s, rows, held)
    s["references"].scatter_add_(0, taken.flatten(), fresh.flatten().int())
    s["table"][rows] = after.int()
    s["lengths"][rows] = count.int()


def _plain_pages(s):
    c = s["case"]
    _plain_free(s, s["to"])
    _plain_fork(s, s["from"], s["to"])
    if c["op"] == "compact":
        _plain_extend(s, s["to"], s["counts"])
        _plain_write(s, c["layers"] - 1, s["k"], s["v"], s["to"], s["new_offsets"])
        _plain_compact(s, s["to"], s["keep_offsets"], s["keep"], s["most_kept"])


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------

def _own_prompt(s):
    from diskmule_b200 import _native, attention
    c, q, k = s["case"], s["q"], s["k"]
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=DEV)
    attention.prompt_attention(
        s["context"], type=_native.BF16 if c["type"] == "bf16" else _native.F16, heads=c["heads"],
        kv_heads=c["kv_heads"], head_dim=c["dim"], q=q.data_ptr(), k=k.data_ptr(),
        v=s["v"].data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), q_tokens=q.shape[0],
        k_tokens=k.shape[0], sequences=s["q_offsets"].numel() - 1,
        q_offsets=s["q_offsets"].data_ptr(), k_offsets=s["k_offsets"].data_ptr(),
        causal=c["causal"], window=c["window"], stream=torch.cuda.current_stream().cuda_stream)
    return {"out": out, "lse": lse}


def _own_decode(s):
    c, q = s["case"], s["q"]
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=DEV)
    s["cache"].decode_attention(
        layer=c["layers"] - 1, heads=c["heads"], q=q.data_ptr(), out=out.data_ptr(),
        lse=lse.data_ptr(), sequences=s["rows"].data_ptr(), batch=c["batch"],
        shared_tokens=c["shared"], max_length=s["longest"], workspace=s["workspace"].data_ptr(),
        workspace_bytes=s["workspace"].numel(), stream=torch.cuda.current_stream().cuda_stream)
    return {"out": out, "lse": lse}


def _own_pages(s):
    c, cache, n = s["case"], s["cache"], s["case"]["children"]
    stream = torch.cuda.current_stream().cuda_stream
    cache.free(s["to"].data_ptr(), n, stream=stream)
    cache.fork(s["from"].data_ptr(), s["to"].data_ptr(), n, stream=stream)
    if c["op"] == "compact":
        cache.extend(s["to"].data_ptr(), s["counts"].data_ptr(), n, stream=stream)
        cache.write(c["layers"] - 1, s["k"].data_ptr(), s["v"].data_ptr(), s["to"].data_ptr(),
                    s["new_offsets"].data_ptr(), n, s["k"].shape[0], stream=stream)
        cache.compact(s["to"].data_ptr(), s["keep_offsets"].data_ptr(), s["keep"].data_ptr(), n,
                      s["keep"].numel(), stream=stream)


def run(state):
    op = state["case"]["op"]
    if op == "prompt":
        return _own_prompt(state) if own else _plain_prompt(state)
    if op == "decode":
        return _own_decode(state) if own else _plain_decode(state)
    if own:
        _own_pages(state)
    else:
        _plain_pages(state)
    return {"table": state["table"], "lengths": state["lengths"], "references": state["references"],
            "pool": state["pool"]}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _attend64(q, k, v, low, high):
    """q [rows, d], k and v [keys, d] in 64 bits; row i sees the keys low[i] <= j < high[i]."""
    j = torch.arange(k.shape[0], device=q.device)
    seen = (j >= low[:, None]) & (j < high[:, None])
    x = (q @ k.T) / math.sqrt(q.shape[1])
    x = torch.where(seen, x, torch.full_like(x, -math.inf))
    lse = torch.logsumexp(x, 1)
    w = torch.where(seen, torch.exp(x - lse[:, None]), torch.zeros_like(x))
    return w @ v, lse


def exact(case, seed):
    global own
    if case["op"] in ("fork", "compact"):
        return None  # copies and whole numbers
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    heads, d = case["heads"], case["dim"]
    g = heads // case["kv_heads"]
    if case["op"] == "prompt":
        out = torch.zeros((s["q"].shape[0], heads, d), dtype=torch.float64, device=DEV)
        lse = torch.zeros((s["q"].shape[0], heads), dtype=torch.float64, device=DEV)
        q0 = k0 = 0
        for lq, lk in zip(_lens(case["q"]), _lens(case["k"])):
            for r0 in range(0, lq, 4096):
                r1 = min(lq, r0 + 4096)
                i = torch.arange(r0, r1, device=DEV) + lk - lq
                high = i + 1 if case["causal"] else torch.full_like(i, lk)
                low = i - case["window"] + 1 if case["window"] else torch.zeros_like(i)
                for h in range(heads):
                    o, e = _attend64(s["q"][q0 + r0:q0 + r1, h].double(),
                                     s["k"][k0:k0 + lk, h // g].double(),
                                     s["v"][k0:k0 + lk, h // g].double(), low, high)
                    out[q0 + r0:q0 + r1, h], lse[q0 + r0:q0 + r1, h] = o, e
            q0, k0 = q0 + lq, k0 + lk
        return {"out": out, "lse": lse}
    b, page = case["batch"], case["page"]
    out = torch.zeros((b, heads, d), dtype=torch.float64, device=DEV)
    lse = torch.zeros((b, heads), dtype=torch.float64, device=DEV)
    lens = s["lengths"].tolist()
    pool = s["pool"][:, case["layers"] - 1]
    for i in range(b):
        n = lens[i]
        pages = pool[s["table"][i, :-(-n // page)].long()]  # [pages, 2, kv, page, d]
        flat = pages.permute(1, 2, 0, 3, 4).reshape(2, case["kv_heads"], -1, d)[:, :, :n].double()
        every = torch.full((g,), n, device=DEV)
        for h in range(case["kv_heads"]):
            o, e = _attend64(s["q"][i, h * g:(h + 1) * g].double(), flat[0, h], flat[1, h],
                             torch.zeros_like(every), every)
            out[i, h * g:(h + 1) * g], lse[i, h * g:(h + 1) * g] = o, e
    return {"out": out, "lse": lse}
