"""An attention layer served from quantised state: W8A16 projections, an 8-bit
paged key/value cache, a prompt in two chunks and tokens one at a time.

    python examples/quantized_decode.py [--cache int8|fp8] [--steps N]

Two sequences of different lengths share one pool of pages. Prints, against the
same layer in fp32 without quantisation, the relative error of the outputs, and
the memory of the weights and the cache. Needs a GPU.
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
import torch.nn as nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from cublade_amd.quantization import (QuantizedKVCache, append_kv, attend_kv,  # noqa: E402
                                      quantize_model)


class Attention(nn.Module):
    """Grouped-query attention whose keys and values live in a QuantizedKVCache."""

    def __init__(self, hidden: int, heads: int, kv_heads: int, dtype: torch.dtype):
        super().__init__()
        self.heads, self.kv_heads, self.d = heads, kv_heads, hidden // heads
        self.qkv = nn.Linear(hidden, (heads + 2 * kv_heads) * self.d, bias=False, dtype=dtype)
        self.out = nn.Linear(hidden, hidden, bias=False, dtype=dtype)

    def forward(self, x, cache, page_table, lengths, rope, cu=None):
        qkv = self.qkv(x).view(x.shape[0], -1, self.d)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        q = append_kv(cache, k, v, page_table, lengths, cu_new=cu, rope=rope, q=q)
        o = attend_kv(q, cache, page_table, lengths, cu_q=cu)
        return self.out(o.flatten(1))


class Pages:
    """The simplest allocator of a pool's pages: the next free one."""

    def __init__(self, cache: QuantizedKVCache, batch: int, max_length: int):
        self.page = cache.page_size
        self.free = list(range(cache.num_pages - 1, -1, -1))
        self.table = torch.full((batch, -(-max_length // self.page)), -1, dtype=torch.int32)
        self.lengths = [0] * batch

    def grow(self, new: list[int]):
        """Room for new tokens: (page_table, lengths with them), on the GPU."""
        for b, n in enumerate(new):
            have = -(-self.lengths[b] // self.page)
            self.lengths[b] += n
            for p in range(have, -(-self.lengths[b] // self.page)):
                self.table[b, p] = self.free.pop()
        return self.table.cuda(), torch.tensor(self.lengths, dtype=torch.int32, device="cuda")


def rotation(rows: int, d: int):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(d // 2, dtype=torch.float64) / (d // 2))
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def reference(wqkv, wout, x, heads: int, kv_heads: int, rope):
    """The layer on one whole sequence in fp32, nothing quantised."""
    n, hidden = x.shape
    d = hidden // heads
    qkv = (x.float() @ wqkv.t()).view(n, -1, d)
    cos, sin = rope[0][:n, None], rope[1][:n, None]

    def turn(t):
        a, b = t.chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)

    q, k = turn(qkv[:, :heads]), turn(qkv[:, heads:heads + kv_heads])
    rep = heads // kv_heads
    k = k.repeat_interleave(rep, 1)
    v = qkv[:, heads + kv_heads:].repeat_interleave(rep, 1)
    s = (q.transpose(0, 1) @ k.permute(1, 2, 0)) / math.sqrt(d)
    s.masked_fill_(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -math.inf)
    return (torch.softmax(s, -1) @ v.transpose(0, 1)).transpose(0, 1).reshape(n, hidden) @ wout.t()


@torch.no_grad()
def run(store: torch.dtype = torch.int8, steps: int = 40, hidden: int = 1024, heads: int = 8,
        kv_heads: int = 2, prompts=(150, 61), chunk: int = 100, page: int = 32) -> float:
    """Relative error of all outputs of both sequences."""
    torch.manual_seed(0)
    dtype, total = torch.bfloat16, [p + steps for p in prompts]
    layer = Attention(hidden, heads, kv_heads, dtype).cuda()
    wqkv, wout = layer.qkv.weight.float(), layer.out.weight.float()
    layer = quantize_model(layer)                       # W8A16 projections
    d = hidden // heads
    rope = rotation(max(total), d)
    pool = sum(-(-t // page) for t in total)
    cache = QuantizedKVCache.empty(pool, kv_heads, d, page, dtype=store)
    pages = Pages(cache, len(prompts), max(total))
    x = [torch.randn(t, hidden, device="cuda").to(dtype) for t in total]
    got = [[] for _ in x]

    def step(new: list[int], cu=None):
        first = list(pages.lengths)
        table, lengths = pages.grow(new)
        y = layer(torch.cat([xi[f:f + n] for xi, f, n in zip(x, first, new)]), cache, table,
                  lengths, rope, cu)
        for g, part in zip(got, y.split(new)):
            g.append(part)

    done = [0] * len(x)
    while done != list(prompts):                        # prompts, a chunk at a time
        new = [min(chunk, p - n) for p, n in zip(prompts, done)]
        ends = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
        step(new, ends)
        done = [n + m for n, m in zip(done, new)]
    for _ in range(steps):                              # then one token each
        step([1] * len(x))

    err = ref = 0.0
    for xi, g in zip(x, got):
        want = reference(wqkv, wout, xi, heads, kv_heads, rope)
        err += float((torch.cat(g).float() - want).square().sum())
        ref += float(want.square().sum())
    print(f"weights {sum(m.int8_weights.numel() for m in (layer.qkv, layer.out))} bytes, cache "
          f"{cache.k.numel() + cache.v.numel()} bytes ({cache.num_pages} pages of {page} tokens)")
    return math.sqrt(err / ref)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--cache", choices=["int8", "fp8"], default="int8")
    ap.add_argument("--steps", type=int, default=40)
    args = ap.parse_args()
    e = run(torch.int8 if args.cache == "int8" else torch.float8_e4m3fn, args.steps)
    print(f"relative error against fp32: {e:.4f}")
