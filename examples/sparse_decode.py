"""One sparse-attention layer over a paged cache: prompt chunks, then decode steps.

    python examples/sparse_decode.py [--batch 8] [--prompt 8192] [--chunk 1024] [--steps 16]

The prompt goes through dense attention in chunks (``PagedAppender`` + ``paged_attention``) while
the indexer's keys are encoded next to it.  Each decode step then appends the new token to both
caches, scores every indexer key and keeps the top-k (``scores_topk``), and attends to those
positions only (``selected_attention``).  Weights and hidden states are random.  With ``top-k >=``
the length the selection holds every position, so the step is also compared with dense attention.
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from dsa_b200 import device_status, scores_topk  # noqa: E402
from dsa_b200.paged import (  # noqa: E402
    PagedAppender, PagedBatch, PagedKV, paged_attention, selected_attention)
from dsa_b200.sidecar import KeyAppender, QueryProjector, encode_keys  # noqa: E402


class SparseLayer:
    """Attention with ``heads`` query and ``kv_heads`` key/value heads of ``dim``, its paged cache
    and its indexer (64 heads x 128), for ``batch`` sequences of up to ``max_length`` positions."""

    def __init__(self, batch: int, max_length: int, *, hidden: int = 2048, heads: int = 16,
                 kv_heads: int = 4, dim: int = 128, page_size: int = 64, topk: int = 2048,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed)

        def weight(rows, dt=dtype):
            return (torch.randn(rows, hidden, generator=g, device=device)
                    / math.sqrt(hidden)).to(dt)

        self.batch, self.max_length, self.topk = batch, max_length, topk
        self.heads, self.kv_heads, self.dim, self.page_size = heads, kv_heads, dim, page_size
        self.device, self.dtype, self.length = torch.device(device), dtype, 0
        self.w_qkv = weight((heads + 2 * kv_heads) * dim)
        per = -(-max_length // page_size)
        self.cache = PagedKV.empty(batch * per, page_size, kv_heads, dim, dtype=dtype,
                                   device=device)
        self.appender = PagedAppender(self.cache, rope_dim=dim)
        # pages are handed out as a server would have them: in no order
        pages = torch.randperm(batch * per, generator=g, device=device).to(torch.int32)
        self.table = pages.view(batch, per)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.one_each = torch.arange(batch + 1, dtype=torch.int32, device=device)
        self.step_batch = PagedBatch(self.table, self.one_each, self.lengths, max_new=1)
        # the indexer: its keys are one contiguous cache
        self.index_keys = torch.zeros(batch, max_length, 128, dtype=dtype, device=device)
        self.w_k = weight(128)
        self.ln = torch.ones(128, device=device), torch.zeros(128, device=device)
        self.key_appender = KeyAppender(self.w_k, *self.ln)
        self.projector = QueryProjector(weight(64 * 128), weight(64, torch.float32), batch)

    def _qkv(self, hidden: torch.Tensor):
        """hidden [tokens, hidden] -> q, k, v [tokens, heads, dim], slices of one product."""
        x = torch.matmul(hidden, self.w_qkv.t()).view(-1, self.heads + 2 * self.kv_heads, self.dim)
        a, b = self.heads, self.heads + self.kv_heads
        return x[:, :a], x[:, a:b], x[:, b:]

    def chunk(self, hidden: torch.Tensor) -> torch.Tensor:
        """The next positions of every sequence, hidden [batch, n, hidden]: dense attention."""
        n = hidden.shape[1]
        start, self.length = self.length, self.length + n
        self.lengths.fill_(self.length)
        batch = PagedBatch(self.table, self.one_each * n, self.lengths, max_new=n)
        q, k, v = self._qkv(hidden.flatten(0, 1))
        q = self.appender.append(batch, k, v, q)
        positions = torch.arange(start, self.length, device=self.device).expand(self.batch, n)
        self.index_keys[:, start:self.length] = encode_keys(hidden, self.w_k, *self.ln, positions)
        return paged_attention(q, self.cache, batch).view(self.batch, n, self.heads, self.dim)

    def step(self, hidden: torch.Tensor, dense: bool = False) -> torch.Tensor:
        """One token per sequence, hidden [batch, hidden]: attention to the top-k positions."""
        positions = torch.full((self.batch,), self.length, device=self.device)
        self.length += 1
        self.lengths.add_(1)
        q, k, v = self._qkv(hidden)
        q = self.appender.append(self.step_batch, k, v, q)
        self.key_appender.append(hidden, positions, self.index_keys)
        if dense:
            return paged_attention(q, self.cache, self.step_batch)
        iq, iw = self.projector.project(hidden, positions)
        indices, _ = scores_topk(iq, iw, self.index_keys[:, :self.length],
                                 min(self.topk, self.length), sorted=False)
        return selected_attention(q, self.cache, self.step_batch, indices)


def run(batch: int, prompt: int, chunk: int, steps: int, topk: int, **kw) -> dict:
    hidden = kw.get("hidden", 2048)
    layer = SparseLayer(batch, prompt + steps, topk=topk, **kw)
    g = torch.Generator(device="cuda").manual_seed(1)

    def states(*shape):
        return torch.randn(*shape, hidden, generator=g, device="cuda").to(layer.dtype)

    marks = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
    marks[0].record()
    for at in range(0, prompt, chunk):
        layer.chunk(states(batch, min(chunk, prompt - at)))
    marks[1].record()
    out = None
    for _ in range(steps - 1):
        out = layer.step(states(batch))
    marks[2].record()
    last = states(batch)
    out = layer.step(last)
    layer.length -= 1  # the same step again, over every position
    layer.lengths.sub_(1)
    dense = layer.step(last, dense=True)
    torch.cuda.synchronize()
    if device_status():
        raise RuntimeError("a kernel raised the device status word")
    gap = (out.float() - dense.float()).norm() / dense.float().norm()
    return {"prompt_ms": marks[0].elapsed_time(marks[1]),
            "step_us": marks[1].elapsed_time(marks[2]) * 1e3 / max(1, steps - 1),
            "sparse_vs_dense": float(gap), "out": out, "dense": dense}


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=8192)
    ap.add_argument("--chunk", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--topk", type=int, default=2048)
    args = ap.parse_args()
    run(args.batch, min(args.prompt, 2 * args.chunk), args.chunk, 4, args.topk)  # warm up
    r = run(args.batch, args.prompt, args.chunk, args.steps, args.topk)
    print(f"prompt of {args.prompt} x {args.batch} in chunks of {args.chunk}: "
          f"{r['prompt_ms']:.2f} ms")
    print(f"decode step over the top {args.topk}: {r['step_us']:.1f} us")
    if args.topk >= args.prompt + args.steps:
        print(f"relative difference of the last step from dense attention: "
              f"{r['sparse_vs_dense']:.3g}")


if __name__ == "__main__":
    main()
