"""Block-scaled caches in other layouts and sizes than the usual ones: head-major planes, offsets past 32 bits,
softmax scales that are zero or negative, tables without columns.

Bounds as in test_gpu_block_cache: derived there, not fitted.
"""

from __future__ import annotations

import math

import pytest
import torch

import musa_aiter as ma

from .test_gpu_block_cache import CODES, append_reference, check_attention
from .test_gpu_block_cache_edges import Case, define, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("hd,bs", [(64, 16), (128, 32), (128, 128), (256, 64)])
@pytest.mark.parametrize("new", [(1, 1), (6, 3), (90, 70)])
def test_head_major_caches(new, hd, bs, codes):
    """[NH, NB, HD, BS] planes: the stride of a head is larger than that of a block."""
    c = Case([200, 135], new, 3, 2, hd, bs, codes, "bf16", seed=hd + bs)
    turn = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1).cuda()  # noqa: E731
    dev = [turn(x) for x in (c.kc, c.vc, c.ks, c.vs)]
    assert dev[0].stride(1) > dev[0].stride(0)
    x = torch.randn((c.starts[-1], 3, hd), generator=c.g).to(torch.bfloat16)
    ma.kv_append_block_scaled(x.cuda(), x.cuda(), *dev, c.table.cuda(), i32(c.ctx), i32(c.starts))
    for cache, scale, y, z in ((c.kc, c.ks, dev[0], dev[2]), (c.vc, c.vs, dev[1], dev[3])):
        append_reference(x, cache, scale, c.table, c.ctx, c.starts, codes)
        assert torch.equal(z.cpu(), scale) and torch.equal(y.cpu().float(), cache.float())
    got, lse = ma.paged_attention_block_scaled(c.q.cuda(), *dev, c.table.cuda(), i32(c.ctx), i32(c.starts), scale=c.scale, return_lse=True)
    want, want_lse, mag = c.want()
    check_attention(got, lse, c.q, want, want_lse, mag)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("bs", [16, 64])
def test_offsets_past_32_bits(bs, codes):
    """Pages on both sides of 4 GB: written, read by few and by many rows, copied."""
    nh, hd, grp = 8, 128, 2
    page = nh * hd * bs
    nb = 2**32 // page + 40
    cache = [torch.empty((nb, nh, hd, bs), dtype=CODES[codes], device="cuda") for _ in range(2)]
    scale = [torch.empty((nb, nh), device="cuda") for _ in range(2)]
    far = list(range(nb - 30, nb)) + [3, 0]
    ctx = [300, 170]
    order = [far[i] for i in torch.randperm(len(far), generator=torch.Generator().manual_seed(1)).tolist()]
    width = -(-300 // bs)
    table = torch.full((2, width), -1, dtype=torch.int32)
    table[0] = torch.tensor(order[:width])
    table[1, : -(-170 // bs)] = torch.tensor(order[width: width - (-170 // bs)])
    g = torch.Generator().manual_seed(bs)
    k, v = (torch.randn((sum(ctx), nh, hd), generator=g).half() for _ in range(2))
    ma.kv_append_block_scaled(k.cuda(), v.cuda(), *cache, *scale, table.cuda(), i32(ctx), i32([0, 300, 470]))
    used = table[table >= 0].long()
    small = table.clone()
    small[table >= 0] = torch.arange(len(used), dtype=torch.int32)
    host = []
    for x, c, s in zip((k, v), cache, scale):
        want, most = torch.zeros((len(used), nh, hd, bs)).to(CODES[codes]), torch.zeros((len(used), nh))
        append_reference(x, want, most, small, ctx, [0, 300, 470], codes)
        assert torch.equal(s[used.cuda()].cpu(), most) and torch.equal(c[used.cuda()].cpu().float(), want.float())
        host += [want, most]
    for new in ((1, 1), (120, 60)):
        starts = [0, new[0], sum(new)]
        q = torch.randn((starts[-1], nh * grp, hd), generator=g).half()
        got, lse = ma.paged_attention_block_scaled(q.cuda(), *cache, *scale, table.cuda(), i32(ctx), i32(starts), return_lse=True)
        want, want_lse, mag = define(q, host[0], host[2], host[1], host[3], small, ctx, starts, 1 / math.sqrt(hd))
        check_attention(got, lse, q, want, want_lse, mag)
    ma.kv_pages_copy(cache + scale, i32([order[0], order[1]]), i32([7, nb - 31]))
    for x in cache + scale:
        x = x.view(torch.uint8) if x.element_size() == 1 else x
        assert torch.equal(x[7], x[order[0]]) and torch.equal(x[nb - 31], x[order[1]])


@pytest.mark.parametrize("scale", [0.0, -0.05])
@pytest.mark.parametrize("new", [(1, 2), (60, 50)])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_softmax_scales_of_zero_and_below(codes, new, scale):
    c = Case([150, 77], new, 2, 4, 64, 16, codes, "f16", seed=4)
    c.scale = scale
    c.check()


@pytest.mark.parametrize("new", [(1, 1), (90, 70)])
def test_tables_without_columns_and_caches_without_blocks(new):
    c = Case([100, 90], new, 2, 4, 64, 64, "int8", "bf16", seed=4)
    whole = (c.table, c.kc, c.vc, c.ks, c.vs)
    for cut in (lambda: setattr(c, "table", c.table[:, :0]), lambda: [setattr(c, n, getattr(c, n)[:0]) for n in ("kc", "vc", "ks", "vs")]):
        c.table, c.kc, c.vc, c.ks, c.vs = whole
        cut()
        got, lse = c.call()
        assert bool((got == 0).all()) and bool((lse == -math.inf).all())
