"""Serving from paged 16-bit caches: prompts, decoding, drafted tokens, eviction by attention weight.

A few attention layers (random projections, no training) answer a handful of requests.  A layer's step is: norms of q and k
with the rotation, write to the pages, attend, and gather the weights of the cached tokens.  When the requests have grown,
each layer and head keeps the tokens that have gathered the most.

    python musa-aiter_b200/examples/paged_serving.py
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import musa_aiter as ma

PROMPTS = (70, 33, 129)  # tokens of the requests
PARENTS = (-1, 0, 0, 2)  # of the drafted tokens


class Layer:
    """Projections, norms and the cache of one layer."""

    def __init__(self, g, hidden, q_heads, kv_heads, head_dim, pages, block_size, device, dtype):
        self.heads = (q_heads, kv_heads, head_dim)
        width = (q_heads + 2 * kv_heads) * head_dim
        self.qkv = (torch.randn((hidden, width), generator=g) / hidden**0.5).to(device, dtype)
        self.out = (torch.randn((q_heads * head_dim, hidden), generator=g) / (q_heads * head_dim) ** 0.5).to(device, dtype)
        self.norms = [torch.ones(head_dim, device=device, dtype=dtype) for _ in range(2)]
        self.cache = torch.zeros((2, pages, block_size, kv_heads, head_dim), device=device, dtype=dtype)

    def project(self, x, positions, cos, sin):
        nq, nk, d = self.heads
        q, k, v = (x @ self.qkv).view(len(x), nq + 2 * nk, d).split((nq, nk, nk), 1)
        return *ma.apply_qk_norm_rope(q, k, *self.norms, positions, cos, sin), v

    def write(self, k, v, slots):
        planes = self.cache.view(2, -1, *self.cache.shape[3:])
        planes[0][slots] = k
        planes[1][slots] = v


class Requests:
    """Block tables, lengths and reference counts on the device."""

    def __init__(self, pages, block_size, width, device):
        self.block_size, self.device = block_size, device
        self.tables = torch.full((len(PROMPTS), width), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(len(PROMPTS), dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)
        self.rows = torch.arange(len(PROMPTS), dtype=torch.int32, device=device)
        self.seen = torch.zeros(len(PROMPTS), dtype=torch.int64, device=device)  # tokens so far, evicted ones too

    def grow(self, counts):
        """Pages for the next tokens; the packed rows' starts, positions and slots."""
        more = torch.tensor(counts, dtype=torch.int32, device=self.device)
        lens = self.lens.clone()
        ma.kv_pages_grow(self.tables, self.lens, self.rows, more, self.refs, self.block_size)
        starts = torch.cat((torch.zeros_like(more[:1]), more.cumsum(0, dtype=torch.int32)))
        whose = torch.repeat_interleave(torch.arange(len(counts), device=self.device), more.long())
        at = torch.arange(int(sum(counts)), device=self.device) - starts[whose]
        place = lens[whose] + at
        slots = self.tables[whose, place // self.block_size].long() * self.block_size + place % self.block_size
        positions = self.seen[whose] + at
        self.seen += more
        return starts, positions, slots


def serve(layers=2, hidden=256, q_heads=8, kv_heads=2, head_dim=64, block_size=16, window=96, sinks=4, keep=48, decode_steps=4,
          device="cuda", dtype=torch.bfloat16):
    """Runs all steps and returns the lengths of the requests after each, and whether every result was finite."""
    g = torch.Generator().manual_seed(0)
    pages, width, scale = 64, 16, head_dim**-0.5
    model = [Layer(g, hidden, q_heads, kv_heads, head_dim, pages, block_size, device, dtype) for _ in range(layers)]
    requests = Requests(pages, block_size, width, device)
    sums = torch.zeros((layers, len(PROMPTS), kv_heads, width * block_size), device=device)
    angle = torch.arange(512)[:, None] / 10000 ** (torch.arange(head_dim // 2) / (head_dim // 2))
    cos, sin = angle.cos().to(device), angle.sin().to(device)
    lengths, finite = [], True

    def step(counts, parents=None):
        nonlocal finite
        starts, positions, slots = requests.grow(counts)
        x = torch.randn((sum(counts), hidden), generator=g).to(device, dtype)
        for i, layer in enumerate(model):
            q, k, v = layer.project(x, positions, cos, sin)
            layer.write(k, v, slots)
            where = (*layer.cache, requests.tables, requests.lens)
            if parents is None:
                o, lse = ma.paged_attention_window(q, *where, cu_seqlens=starts, window=window, sinks=sinks, scale=scale, return_lse=True)
                ma.paged_attention_weights(q, layer.cache[0], requests.tables, requests.lens, lse, sums[i], starts, window=window,
                                           sinks=sinks, scale=scale)
            else:
                o = ma.paged_attention_tree(q, *where, parents=parents, cu_seqlens=starts, scale=scale)
            x = x + o.flatten(1) @ layer.out
        finite = finite and bool(x.isfinite().all())
        lengths.append(requests.lens.tolist())

    step(PROMPTS)
    for _ in range(decode_steps):
        step((1,) * len(PROMPTS))
    left = ma.kv_pages_evict(requests.tables, requests.lens, requests.rows, requests.refs, [x.cache[0] for x in model],
                             [x.cache[1] for x in model], sums, keep, sinks=sinks, recent=16)
    assert int(left) == 0
    lengths.append(requests.lens.tolist())
    step((1,) * len(PROMPTS))
    step((len(PARENTS),) * len(PROMPTS), torch.tensor(PARENTS * len(PROMPTS), dtype=torch.int32, device=device))
    finite = finite and bool(sums.isfinite().all())
    return lengths, finite


if __name__ == "__main__":
    for lens in serve()[0]:
        print(lens)
