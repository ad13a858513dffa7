"""Attention layers served from the 4-bit KV cache: prompts, forks, decode steps, compaction.

Each layer is a q4nx projection to q, k and v, ``KvCache.append`` (head norms,
rotation, quantisation), ``KvCache.attend``, a q4nx projection back and the
residual with its RMS norm; random weights and inputs.  ::

    python -m raon_npu_b200.examples.attention_stack
"""

from __future__ import annotations

import argparse
import time

import numpy as np
import torch

from ..device import Context, Q4nxWeight, add_rms_bf16
from ..kvcache import KvCache, rope_table


class AttentionStack:
    """``layers`` attention layers over one cache."""

    def __init__(self, ctx: Context, layers: int = 4, hidden: int = 2048, q_heads: int = 32, kv_heads: int = 4,
                 head_dim: int = 128, pages: int = 256, page_size: int = 64, positions: int = 4096, window: int = 0,
                 sinks: int = 0, seed: int = 0):
        self.ctx, self.hidden, self.q_heads, self.window, self.sinks = ctx, hidden, q_heads, window, sinks
        self.width, self.qkv_width = q_heads * head_dim, (q_heads + 2 * kv_heads) * head_dim
        self.cache = KvCache(ctx, layers, kv_heads, head_dim, pages, page_size=page_size)
        dev = torch.device("cuda", ctx.device)
        gen = torch.Generator(dev).manual_seed(seed)

        def weight(n, k):
            w = torch.randn((n, k), generator=gen, device=dev) * k ** -0.5
            packed = torch.empty(n * k * 5 // 8, dtype=torch.uint8, device=dev)
            ctx.quantize_q4nx(w, packed, n, k)
            return Q4nxWeight(ctx, packed, n, k)

        self.qkv = [weight(self.qkv_width, hidden) for _ in range(layers)]
        self.out = [weight(hidden, self.width) for _ in range(layers)]
        norm = lambda: (1 + 0.1 * torch.randn(head_dim, generator=gen, device=dev)).to(torch.bfloat16)  # noqa: E731
        self.norms = [(norm(), norm()) for _ in range(layers)]
        self.rope = torch.from_numpy(rope_table(positions, head_dim)).to(dev)

    def forward(self, x, batch):
        """x bf16 [rows, hidden]: the batch's rows.  Returns the last layer's rows."""
        rows = x.shape[0]
        qkv = x.new_empty((rows, self.qkv_width))
        q, o = x.new_empty((rows, self.width)), x.new_empty((rows, self.width))
        for layer, (q_norm, k_norm) in enumerate(self.norms):
            y, z = torch.empty_like(x), torch.empty_like(x)
            self.qkv[layer].gemv_into(x, qkv, rows)
            self.cache.append(layer, qkv, batch, q, q_heads=self.q_heads, q_norm=q_norm, k_norm=k_norm, rope=self.rope)
            self.cache.attend(layer, q, batch, o, window=self.window, sinks=self.sinks)
            self.out[layer].gemv_into(o, y, rows)
            add_rms_bf16(self.ctx, x, y, z)
            x = z
        return x

    def prefill(self, seqs, xs):
        """Rows of xs[i] appended to sequence seqs[i]; returns the rows' outputs, one tensor a sequence."""
        counts = [int(x.shape[0]) for x in xs]
        self.cache.extend(seqs, counts)
        return torch.split(self.forward(torch.cat(xs), self.cache.batch(seqs, rows=counts)), counts)

    def step(self, seqs, x):
        """One token a sequence: x bf16 [sequences, hidden]."""
        self.cache.extend(seqs, 1)
        return self.forward(x, self.cache.batch(seqs))


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    a = ap.parse_args(argv)
    ctx = Context(0)
    stack = AttentionStack(ctx, layers=a.layers, window=a.window, sinks=a.sinks)
    cache, pool = stack.cache, stack.cache.page_pool
    gen = torch.Generator("cuda").manual_seed(1)
    rows = lambda n: torch.randn((n, stack.hidden), generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731

    prompts = [cache.new() for _ in range(3)]
    ends = [y[-1] for y in stack.prefill(prompts, [rows(n) for n in (517, 1300, 90)])]
    # two continuations of the first prompt share its pages until they grow
    seqs = prompts + [cache.fork(prompts[0])]
    x = torch.stack(ends + ends[:1])
    stack.step(seqs, x)
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(a.steps):
        x = stack.step(seqs, x)
    torch.cuda.synchronize()
    ms = (time.perf_counter() - t0) * 1e3 / a.steps
    print(f"{a.steps} steps of {len(seqs)} sequences, {a.layers} layers: {ms:.3f} ms a step; "
          f"{pool.info()[0]} of {cache.pages} pages free")

    cache.free(prompts[1])
    moved = cache.compact()
    free, high = pool.info()
    print(f"one sequence ended: {moved} pages moved, {free} free, all in use below page {high}")
    rest = [s for s in seqs if s != prompts[1]]
    y = stack.step(rest, x[[0, 2, 3]])
    ctx.sync()
    print("after the compaction:", [cache.page_pool.tokens(s) for s in rest], "tokens; finite:",
          bool(np.isfinite(y.float().cpu().numpy()).all()))


if __name__ == "__main__":
    main()
