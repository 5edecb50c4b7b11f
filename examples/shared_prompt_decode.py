"""Several continuations of one prompt, decoded together: the attention calls and the routed
feed-forward layer as a serving loop uses them.

A small stack (synthetic weights): attention -> residual -> RMS norm -> MoeLayer -> residual,
`layers` times, between an embedding and an output head that share one matrix. The prompt runs
once (prompt_attention), its keys and values go into a paged cache, the sequence is forked
into `samples` rows that share its full pages, and every step feeds one token per sample
(KvCache.extend / write / decode_attention with the shared tokens read once). At the end the
even samples are cut back by half of their new tokens (compact) and everything is freed.

    python examples/shared_prompt_decode.py --prompt 1000 --samples 16 --steps 32
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from diskmule_b200 import CudaContext, _native as N  # noqa: E402
from diskmule_b200.attention import KvCache, attention_status, offsets, prompt_attention  # noqa: E402
from diskmule_b200.synthetic import build_layer  # noqa: E402


def ints(values) -> torch.Tensor:
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


class Stack:
    def __init__(self, ctx: CudaContext, config: str = "qwen35-small", layers: int = 2, heads: int = 8,
                 kv_heads: int = 2, head_dim: int = 64, vocab: int = 1024, page_tokens: int = 16,
                 pages: int = 2048, max_sequences: int = 64, max_pages: int = 256, seed: int = 1):
        self.ctx, self.layers = ctx, layers
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.routed = [build_layer(ctx, config, seed=seed + i) for i in range(layers)]
        self.hidden = h = self.routed[0].cfg["hidden"]
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)

        def weight(rows, cols):
            return torch.randn(rows, cols, generator=gen, device="cuda").mul_(cols ** -0.5).bfloat16()

        self.embed = weight(vocab, h)
        self.qkv = [weight((heads + 2 * kv_heads) * head_dim, h) for _ in range(layers)]
        self.out = [weight(h, heads * head_dim) for _ in range(layers)]
        self.cache = KvCache(ctx, type=N.BF16, layers=layers, kv_heads=kv_heads, head_dim=head_dim,
                             page_tokens=page_tokens, pages=pages, max_sequences=max_sequences,
                             max_pages=max_pages)
        self.page_tokens = page_tokens

    def _norm(self, x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def _layer(self, i: int, x: torch.Tensor, attend) -> torch.Tensor:
        """One block on x [tokens, hidden] f32; attend(q, k, v, fused row stride) -> attention."""
        fused = self._norm(x).bfloat16() @ self.qkv[i].T
        d, stride = self.head_dim, fused.stride(0)
        q = fused[:, :self.heads * d]
        k = fused[:, self.heads * d:(self.heads + self.kv_heads) * d]
        v = fused[:, (self.heads + self.kv_heads) * d:]
        a = attend(q, k, v, (stride, d))
        x = x + (a.reshape(x.shape[0], -1) @ self.out[i].T).float()
        y = torch.empty_like(x)
        normed = self._norm(x).contiguous()
        self.routed[i].layer.forward(normed.data_ptr(), y.data_ptr(), x.shape[0], stream=self.stream)
        return x + y

    @property
    def stream(self) -> int:
        return torch.cuda.current_stream().cuda_stream

    def tokens_of(self, x: torch.Tensor) -> torch.Tensor:
        return (self._norm(x).bfloat16() @ self.embed.T).argmax(-1)

    def prompt(self, row: int, tokens: torch.Tensor) -> torch.Tensor:
        """Run a prompt into cache row `row` (empty); the next token."""
        n = tokens.numel()
        rows, off = ints([row]), ints(offsets([n]))
        count = ints([n])
        self.cache.extend(rows.data_ptr(), count.data_ptr(), 1, stream=self.stream)
        x = self.embed[tokens].float()
        for i in range(self.layers):
            def attend(q, k, v, stride, i=i):
                a = torch.empty(n, self.heads, self.head_dim, dtype=torch.bfloat16, device="cuda")
                self.cache.write(i, k.data_ptr(), v.data_ptr(), rows.data_ptr(), off.data_ptr(), 1, n,
                                 k_stride=stride, v_stride=stride, stream=self.stream)
                prompt_attention(self.ctx, type=N.BF16, heads=self.heads, kv_heads=self.kv_heads,
                                 head_dim=self.head_dim, q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(),
                                 out=a.data_ptr(), q_tokens=n, k_tokens=n, sequences=1,
                                 q_offsets=off.data_ptr(), q_stride=stride, k_stride=stride,
                                 v_stride=stride, stream=self.stream)
                return a
            x = self._layer(i, x, attend)
        return self.tokens_of(x[-1:])

    def step(self, rows: torch.Tensor, tokens: torch.Tensor, shared: int, longest: int) -> torch.Tensor:
        """Feed one token to each cache row; the next tokens. `shared` leading tokens lie in
        common pages; `longest` bounds the lengths with the new token."""
        n = rows.numel()
        one, off = ints([1] * n), ints(offsets([1] * n))
        self.cache.extend(rows.data_ptr(), one.data_ptr(), n, stream=self.stream)
        size = self.cache.decode_workspace(self.heads, n, shared, longest)
        work = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        x = self.embed[tokens].float()
        for i in range(self.layers):
            def attend(q, k, v, stride, i=i):
                a = torch.empty(n, self.heads, self.head_dim, dtype=torch.bfloat16, device="cuda")
                self.cache.write(i, k.data_ptr(), v.data_ptr(), rows.data_ptr(), off.data_ptr(), n, n,
                                 k_stride=stride, v_stride=stride, stream=self.stream)
                self.cache.decode_attention(layer=i, heads=self.heads, q=q.data_ptr(), out=a.data_ptr(),
                                            batch=n, max_length=longest, shared_tokens=shared,
                                            sequences=rows.data_ptr(), q_stride=stride,
                                            workspace=work.data_ptr(), workspace_bytes=size,
                                            stream=self.stream)
                return a
            x = self._layer(i, x, attend)
        return self.tokens_of(x)

    def close(self):
        torch.cuda.synchronize()
        self.cache.close()
        for r in self.routed:
            r.close()


def run(prompt: int = 200, samples: int = 4, steps: int = 8, seed: int = 3, share: bool = True,
        stack: Stack | None = None) -> dict:
    """Decode `samples` continuations of a prompt; each starts with a token of its own."""
    ctx = CudaContext(0) if stack is None else stack.ctx
    st = Stack(ctx, max_sequences=samples + 1) if stack is None else stack
    r = np.random.RandomState(seed)
    tokens = torch.tensor(r.randint(0, st.embed.shape[0], prompt), device="cuda")
    st.prompt(0, tokens)
    parents, rows = ints([0] * samples), ints(range(1, samples + 1))
    st.cache.fork(parents.data_ptr(), rows.data_ptr(), samples, stream=st.stream)
    shared = prompt // st.page_tokens * st.page_tokens if share else 0
    now = torch.tensor(r.randint(0, st.embed.shape[0], samples), device="cuda")
    out = []
    torch.cuda.synchronize()
    began = time.perf_counter()
    for i in range(steps):
        now = st.step(rows, now, shared, prompt + i + 1)
        out.append(now)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - began
    # the even samples give back half of what they have decoded
    cut = [s for s in range(samples) if s % 2 == 0]
    keep = prompt + steps // 2
    some, off = ints([1 + s for s in cut]), ints(offsets([keep] * len(cut)))
    kept = ints(np.tile(np.arange(keep), len(cut)))
    st.cache.compact(some.data_ptr(), off.data_ptr(), kept.data_ptr(), len(cut), kept.numel(), stream=st.stream)
    after = st.step(rows, now, shared, prompt + steps + 1)
    every = ints(range(samples + 1))
    st.cache.free(every.data_ptr(), samples + 1, stream=st.stream)
    attention_status(ctx, st.stream)
    status = st.cache.status(st.stream)
    result = dict(tokens=torch.stack(out).cpu().numpy(), after=after.cpu().numpy(), status=status,
                  tokens_per_s=samples * steps / seconds, us_per_step=seconds / steps * 1e6)
    if stack is None:
        st.close()
        ctx.close()
    return result


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompt", type=int, default=1000)
    ap.add_argument("--samples", type=int, default=16)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    ctx = CudaContext(0)
    st = Stack(ctx, max_sequences=a.samples + 1)
    run(a.prompt, a.samples, 3, stack=st)  # warm-up
    r = run(a.prompt, a.samples, a.steps, stack=st)
    print(f"{a.samples} samples of a {a.prompt}-token prompt, {a.steps} steps: "
          f"{r['us_per_step']:.0f} us a step, {r['tokens_per_s']:.0f} tokens/s, cache status {r['status']}")
    print("first sample:", r["tokens"][:, 0].tolist())
    st.close()
    ctx.close()


if __name__ == "__main__":
    main()
