"""What the writer stores and what the attention reads of it, step by step.

Bounds.  Storing a value once is off by half a step of its block's scale (int8: 1 / 254 of the largest the block can
hold; E4M3: 2^-4 of the value, or 2^-10 of the scale below the least normal code), and once more each time the scale
grows.  Against the cache's own values the attention is held to the bounds derived in test_gpu_block_cache.
"""

from __future__ import annotations

import importlib.util
import math

import pytest
import torch

import musa_aiter as ma

from .test_gpu_block_cache import CODES, check_attention, reference
from .test_gpu_block_cache_example import EXAMPLE

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention_reads_what_was_written(codes, dtype):
    """A prompt, 20 single tokens and 5 drafted ones: after every write the attention of its rows."""
    g = torch.Generator().manual_seed(3)
    nh, grp, hd, bs, nb, counts = 2, 4, 128, 16, 9, [37] + [1] * 20 + [5]
    total = sum(counts)
    k, v = (torch.randn((total, nh, hd), generator=g).to(dtype) for _ in range(2))
    q = torch.randn((total, nh * grp, hd), generator=g).to(dtype)
    cache = [torch.zeros((nb, nh, hd, bs), dtype=CODES[codes], device="cuda") for _ in range(2)]
    scale = [torch.zeros((nb, nh), device="cuda") for _ in range(2)]
    table = torch.randperm(nb, generator=g).to(torch.int32)[None]
    grew = [torch.ones((nb, nh)) for _ in range(2)]  # how often a block was rounded
    at = 0
    for n in counts:
        ctx, starts = [at + n], [0, n]
        here = (table.cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(), torch.tensor(starts, dtype=torch.int32).cuda())
        before = [s.cpu() for s in scale]
        ma.kv_append_block_scaled(k[at:at + n].cuda(), v[at:at + n].cuda(), *cache, *scale, *here)
        for count, old, new in zip(grew, before, scale):
            count += (new.cpu() > old) & (old > 0)
        got, lse = ma.paged_attention_block_scaled(q[at:at + n].cuda(), *cache, *scale, *here, return_lse=True)
        host = [x.cpu() for x in cache + scale]
        want = reference(q[at:at + n], *host, table, ctx, starts, 1 / math.sqrt(hd), True, 0)
        check_attention(got, lse, q[at:at + n], *want)
        at += n
        token = torch.arange(at)
        page, off = table[0, token // bs].long(), token % bs
        for x, c, s, count in zip((k, v), host[:2], host[2:], grew):
            step, times = s[page][..., None], count[page][..., None]
            back, x = c[page, :, :, off].float() * step, x[:at].float()
            # one rounding, and 2^-20 for those of the scale and the product
            one = 0.5 * step if codes == "int8" else torch.maximum(2.0 ** -4 * torch.maximum(x.abs(), back.abs()), 2.0 ** -10 * step)
            assert bool(((back - x).abs() <= times * one * (1 + 2.0 ** -20) + 2.0 ** -20 * x.abs()).all())


# At most 3 growths of a block's scale after its first rounding: 4 half steps of int8, 4 times 2^-4.  Outputs lie below
# 6 and come as bfloat16: 2^-8 of them, and the bounds of the weights.  A token or page that is lost or another's is off
# by about 1 in the cache.
@pytest.mark.parametrize("code,stored", [(torch.int8, 4 / 254 * 1.01), (torch.float8_e4m3fn, 4 / 16 * 1.01)])
@pytest.mark.parametrize("block_size", [16, 64])
def test_serving_example_against_its_cache(code, stored, block_size):
    spec = importlib.util.spec_from_file_location("block_scaled_serving", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    got = module.differences(code, block_size=block_size)
    assert got["stored"] <= stored
    assert got["cache"] <= 6 * (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -14)
