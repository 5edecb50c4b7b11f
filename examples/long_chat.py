"""A chat whose cache stays small: prompts in pieces, positions of their own, and eviction of the
tokens that receive least attention.

The stack of shared_prompt_decode.py with norms and rotation of queries and keys: each piece of
a prompt, and each later token, is rotated into the paged cache (rotate), attends over all that
its sequence holds (KvCache.chunk_attention) and adds to what every cached token has received
(KvCache.token_weights). Whenever a sequence has outgrown its budget it is cut down to its first
tokens, its last ones and the heaviest between (KvCache.evict); positions go on counting, so what
is left keeps its distances.

    python examples/long_chat.py --prompt 3000 --piece 512 --budget 1024 --steps 64
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from diskmule_b200 import CudaContext, _native as N  # noqa: E402
from diskmule_b200.attention import Rope, attention_status, offsets, rotate  # noqa: E402
from shared_prompt_decode import Stack, ints  # noqa: E402


class Chat(Stack):
    """Sequences in cache rows 0 .. chats - 1; `seen` counts the tokens of each, `held` those that
    its cache row still has."""

    def __init__(self, ctx: CudaContext, chats: int, budget: int, sinks: int = 4, recent: int = 64, **stack):
        super().__init__(ctx, max_sequences=chats, **stack)
        self.chats, self.budget, self.sinks, self.recent = chats, budget, sinks, recent
        self.rope = Rope(ctx, self.head_dim, theta=1e4)
        capacity = self.cache.describe().max_pages * self.page_tokens
        self.weights = torch.zeros(chats, capacity, device="cuda")
        self.norm = [torch.ones(self.head_dim, device="cuda") for _ in range(2)]
        self.seen, self.held = np.zeros(chats, int), np.zeros(chats, int)

    def feed(self, rows, tokens: list) -> torch.Tensor:
        """New tokens of some rows, any number of each; the next token of each."""
        lens = [len(t) for t in tokens]
        n, total, longest = len(rows), sum(lens), int(max(self.held[r] + m for r, m in zip(rows, lens)))
        row, off, count = ints(rows), ints(offsets(lens)), ints(lens)
        positions = ints(np.concatenate([self.seen[r] + np.arange(m) for r, m in zip(rows, lens)]))
        self.cache.extend(row.data_ptr(), count.data_ptr(), n, stream=self.stream)
        size = self.cache.chunk_workspace(self.heads, n, total, longest)
        work = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        x = self.embed[torch.cat(tokens)].float()
        for i in range(self.layers):
            def attend(q, k, v, stride, i=i):
                turned, a = (torch.empty(total, self.heads, self.head_dim, dtype=torch.bfloat16, device="cuda")
                             for _ in range(2))
                lse = torch.empty(total, self.heads, device="cuda")
                entries = dict(sequences=row.data_ptr(), offsets=off.data_ptr(), n=n, tokens=total, stream=self.stream)
                rotate(self.ctx, self.rope, type=N.BF16, heads=self.heads, kv_heads=self.kv_heads,
                       head_dim=self.head_dim, q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), q_out=turned.data_ptr(),
                       q_stride=stride, k_stride=stride, v_stride=stride, cache=self.cache, layer=i,
                       positions=positions.data_ptr(), norm_q=True, norm_k=True, q_weight=self.norm[0].data_ptr(),
                       k_weight=self.norm[1].data_ptr(), **entries)
                call = dict(layer=i, heads=self.heads, q=turned.data_ptr(), lse=lse.data_ptr(), max_length=longest,
                            **entries)
                self.cache.chunk_attention(out=a.data_ptr(), workspace=work.data_ptr(), workspace_bytes=size, **call)
                self.cache.token_weights(weights=self.weights.data_ptr(), weights_stride=self.weights.stride(0), **call)
                return a
            x = self._layer(i, x, attend)
        self.seen[rows] += lens
        self.held[rows] += lens
        return self.tokens_of(x[torch.tensor(np.cumsum(lens) - 1, device="cuda")])

    def cut(self, slack: int = 0):
        """Rows of more than budget + slack tokens go down to the budget."""
        rows = [r for r in range(self.chats) if self.held[r] > self.budget + slack]
        if not rows:
            return
        row, off, keep = ints(rows), ints([0] * (len(rows) + 1)), ints([0] * len(rows) * self.budget)
        self.cache.evict(sequences=row.data_ptr(), n=len(rows), budget=self.budget, sinks=self.sinks, recent=self.recent,
                         weights=self.weights.data_ptr(), weights_stride=self.weights.stride(0),
                         keep_offsets=off.data_ptr(), keep=keep.data_ptr(), stream=self.stream)
        self.held[rows] = self.budget

    def close(self):
        self.rope.close()
        super().close()


def run(chats: int = 3, prompt: int = 300, piece: int = 64, budget: int = 160, steps: int = 24, seed: int = 3) -> dict:
    """Prompts of about `prompt` tokens in pieces, then `steps` tokens of every chat."""
    ctx = CudaContext(0)
    st = Chat(ctx, chats, budget, max_pages=(max(prompt, budget) + steps + piece) // 16 + 2)
    r = np.random.RandomState(seed)
    prompts = [torch.tensor(r.randint(0, st.embed.shape[0], prompt - 17 * c), device="cuda") for c in range(chats)]
    now = [None] * chats
    for at in range(0, prompt, piece):
        rows = [c for c in range(chats) if at < prompts[c].numel()]
        after = st.feed(rows, [prompts[c][at:at + piece] for c in rows])
        for i, c in enumerate(rows):
            now[c] = after[i:i + 1]
        st.cut(slack=piece)
    out, every = [], list(range(chats))
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(steps):
        after = st.feed(every, now)
        now = [after[c:c + 1] for c in every]
        out.append(after)
        st.cut(slack=16)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - began
    attention_status(ctx, st.stream)
    result = dict(tokens=torch.stack(out).cpu().numpy(), status=st.cache.status(st.stream), seen=st.seen.copy(),
                  held=st.held.copy(), received=st.weights.sum(1).cpu().numpy(), us_per_step=seconds / steps * 1e6,
                  layers=st.layers, heads=st.heads)
    st.close()
    ctx.close()
    return result


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--chats", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=3000)
    ap.add_argument("--piece", type=int, default=512)
    ap.add_argument("--budget", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=64)
    a = ap.parse_args()
    r = run(a.chats, a.prompt, a.piece, a.budget, a.steps)
    print(f"{a.chats} chats of {r['seen'].tolist()} tokens hold {r['held'].tolist()}, {r['us_per_step']:.0f} us a step, "
          f"cache status {r['status']}")
    print("first chat:", r["tokens"][:, 0].tolist())


if __name__ == "__main__":
    main()
