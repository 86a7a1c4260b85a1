"""Serving with a block-scaled 8-bit cache: prompts, forked continuations, decoding, freeing, compacting.

A few attention layers (random projections, no training) answer a handful of requests whose tokens have
three position axes.  The scheduler's steps are page calls on device tensors; a layer's step is
rotate, write, attend.  ``differences`` also keeps every request's keys and values as they were and holds
the cache and the layers' attention against them; ``serve`` returns the attention's largest difference.

    python musa-aiter_b200/examples/block_scaled_serving.py
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import musa_aiter as ma

PROMPTS = (70, 33, 129)  # tokens of the requests
SECTIONS = (16, 24, 24)  # pairs of a head turned by time, height, width


class Layer:
    """Projections and the cache planes of one layer."""

    def __init__(self, g, hidden, q_heads, kv_heads, head_dim, pages, block_size, code, device):
        width = (q_heads + 2 * kv_heads) * head_dim
        self.heads = (q_heads, kv_heads, head_dim)
        self.qkv = (torch.randn((hidden, width), generator=g) / hidden**0.5).to(device, torch.bfloat16)
        self.out = (torch.randn((q_heads * head_dim, hidden), generator=g) / (q_heads * head_dim) ** 0.5).to(device, torch.bfloat16)
        shape = (pages, kv_heads, head_dim, block_size)
        self.codes = [torch.zeros(shape, dtype=code, device=device) for _ in range(2)]
        self.scales = [torch.zeros(shape[:2], device=device) for _ in range(2)]

    def planes(self):
        return [*self.codes, *self.scales]

    def read(self, table, length):
        """Keys and values [length, kv_heads, head_dim] of a row as the cache holds them, and the largest that each block
        and head can hold, [length, kv_heads, 1]."""
        block_size = self.codes[0].shape[3]
        token = torch.arange(length, device=table.device)
        page, at = table[token // block_size].long(), token % block_size
        most = 127.0 if self.codes[0].dtype == torch.int8 else 448.0
        scales = [s[page][..., None] for s in self.scales]
        return [c[page, :, :, at].float() * s for c, s in zip(self.codes, scales)], [s * most for s in scales]

    def step(self, x, positions, cos, sin, tables, lens, starts):
        """One layer on packed rows x; returns the new x, the rotated q and k, v and the attention's result."""
        nq, nk, d = self.heads
        q, k, v = (x @ self.qkv).view(len(x), nq + 2 * nk, d).split((nq, nk, nk), 1)
        q, k = ma.apply_rope_axes(q, k, positions, cos, sin, SECTIONS)
        ma.kv_append_block_scaled(k, v, *self.codes, *self.scales, tables, lens, starts)
        o = ma.paged_attention_block_scaled(q, *self.codes, *self.scales, tables, lens, starts)
        return x + o.flatten(1) @ self.out, q, k, v, o


def plain_attention(q, k, v):
    """Causal attention of the last len(q) positions in 64 bits: q [n, H, d], k / v [t, h, d]."""
    q, k, v = (x.double() for x in (q, k, v))
    group = q.shape[1] // k.shape[1]
    k, v = (x.repeat_interleave(group, 1) for x in (k, v))
    s = torch.einsum("ihd,thd->hit", q, k) / q.shape[2] ** 0.5
    n, t = len(q), len(k)
    hidden = torch.arange(t, device=q.device) > torch.arange(t - n, t, device=q.device)[:, None]
    return torch.einsum("hit,thd->ihd", s.masked_fill(hidden, float("-inf")).softmax(-1), v)


def serve(*args, **kwargs):
    """``differences`` for its first result alone."""
    return differences(*args, **kwargs)["values"]


def differences(code=torch.int8, block_size=16, layers=2, decode_steps=6, seed=0, device="cuda"):
    """Serves the requests and returns the largest differences met: ``values``, of the attention from plain attention over
    the keys and values that were written; ``cache``, from plain attention over what the cache holds of them; ``stored``,
    of a value in the cache from the one written, as a part of the largest its block and head can hold."""
    g = torch.Generator().manual_seed(seed)
    hidden, pages, rows, max_blocks = 256, 160, 6, 24
    stack = [Layer(g, hidden, 8, 2, 128, pages, block_size, code, device) for _ in range(layers)]
    planes = [p for layer in stack for p in layer.planes()]
    angle = torch.arange(1024)[:, None] * 10000.0 ** (-torch.arange(64) / 64)
    cos, sin = angle.cos().to(device), angle.sin().to(device)

    tables = torch.full((rows, max_blocks), -1, dtype=torch.int32, device=device)
    lens = torch.zeros(rows, dtype=torch.int32, device=device)
    refs = torch.zeros(pages, dtype=torch.int32, device=device)
    ids = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    history = {}  # (row, layer) -> its keys and values so far
    worst = dict(values=0.0, cache=0.0, stored=0.0)

    def note(name, x):
        worst[name] = max(worst[name], x.abs().max().item())

    def forward(live, counts):
        """The rows `live` take counts[i] tokens each: pages, then every layer."""
        short = ma.kv_pages_grow(tables, lens, ids(live), ids(counts), refs, block_size)
        at = [0]
        for n in counts:
            at.append(at[-1] + n)
        x = torch.randn((at[-1], hidden), generator=g).to(device, torch.bfloat16)
        # time along the request, an 8-wide picture's rows and columns for height and width
        time = torch.cat([torch.arange(int(lens[r]) - n, int(lens[r])) for r, n in zip(live, counts)])
        positions = torch.stack([time, time // 8, time % 8]).to(device)
        # the calls read one table row per sequence of the batch
        batch_tables, batch_lens, starts = tables[live], lens[live], ids(at)
        for i, layer in enumerate(stack):
            x, q, k, v, o = layer.step(x, positions, cos, sin, batch_tables, batch_lens, starts)
            for j, r in enumerate(live):
                s = slice(at[j], at[j + 1])
                old = history.get((r, i))
                history[r, i] = (k[s], v[s]) if old is None else (torch.cat((old[0], k[s])), torch.cat((old[1], v[s])))
                note("values", o[s].double() - plain_attention(q[s], *history[r, i]))
                held, most = layer.read(tables[r], int(lens[r]))
                note("cache", o[s].double() - plain_attention(q[s], *held))
                for x_held, x_most, x_old in zip(held, most, history[r, i]):
                    note("stored", (x_held - x_old.float()) / x_most)
        assert int(short) == 0

    forward([0, 1, 2], list(PROMPTS))
    # request 0 is continued three ways: full pages shared, the part-filled last one copied
    assert int(ma.kv_pages_fork(tables, lens, ids([0, 0]), ids([3, 4]), refs, planes, block_size)) == 0
    for i in range(layers):
        history[3, i] = history[4, i] = history[0, i]
    for _ in range(decode_steps):
        forward([0, 1, 2, 3, 4], [1] * 5)
    forward([2, 3], [5, 3])  # drafted tokens, checked together
    ma.kv_pages_free(tables, lens, ids([0, 1]), refs)
    live = int(ma.kv_pages_compact(tables, refs, planes))
    used = {int(p) for p in tables.flatten().tolist() if p >= 0}
    assert used == set(range(live)), "compaction left holes"
    for _ in range(decode_steps):
        forward([2, 3, 4], [1] * 3)
    ma.kv_pages_free(tables, lens, ids([2, 3, 4]), refs)
    assert int(refs.abs().sum()) == 0, "a page was lost"
    return worst


if __name__ == "__main__":
    for code in (torch.int8, torch.float8_e4m3fn):
        got = differences(code)
        print(f"{code}: attention differs by {got['values']:.4f} from the values written, by {got['cache']:.4f} from what the cache "
              f"holds of them; a value by {got['stored']:.4f} of its block's largest")
