"""Block-scaled attention where the way of working changes: numbers of rows around the sizes of a group of
rows, and scores that keep growing or falling along the sequence, so that the maximum moves again and again.

Bounds as in test_gpu_block_cache: derived there, not fitted.
"""

from __future__ import annotations

import math

import pytest
import torch

import musa_aiter as ma

from .test_gpu_block_cache import DT, check_attention, make_cache, make_tables, reference, run_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,codes", [(64, "fp8"), (128, "int8"), (256, "fp8")])
@pytest.mark.parametrize("rows", [1, 3, 4, 5, 8, 9, 16, 17, 24, 25, 32, 33, 48])
def test_rows_around_the_sizes_of_a_group(rows, hd, codes):
    run_case([150, 77, 300], [rows] * 3, 2, 1, hd, 16, codes, "bf16", seed=rows)
    run_case([130, 129], [1, 1], 2, rows, hd, 32, codes, "f16", seed=rows + 1)


@pytest.mark.parametrize("lens", [[1, 1, 1], [127, 128, 129], [16, 1, 255, 256, 257, 3, 90, 17]])
@pytest.mark.parametrize("grp", [2, 8, 12])
def test_units_of_one_and_two_tiles(lens, grp):
    run_case(lens * 40, [1] * (len(lens) * 40), 2, grp, 64, 16, "fp8", "bf16", seed=grp)


@pytest.mark.parametrize("falling", [False, True])
@pytest.mark.parametrize("new", [1, 6, 90])
@pytest.mark.parametrize("hd,bs,codes", [(64, 16, "int8"), (128, 32, "fp8")])
def test_maximum_that_keeps_moving(new, falling, hd, bs, codes):
    g = torch.Generator().manual_seed(new)
    ctx, nh, grp = [700, 333], 2, 4
    table, nb, _ = make_tables(g, ctx, bs)
    kc, ks = make_cache(g, nb, nh, hd, bs, codes)
    vc, vs = make_cache(g, nb, nh, hd, bs, codes)
    kc = kc.float().abs().to(kc.dtype)
    q = torch.randn((2 * new, nh * grp, hd), generator=g).abs().to(DT["bf16"])
    mean = float(kc.float().mean()) * math.sqrt(2 / math.pi) * math.sqrt(hd)  # of a score with scale 1
    for row in table:
        pages = row[row >= 0].long()
        rise = torch.linspace(0.02, 1.0, len(pages)) * 18.0 / mean  # scores from 0 to about 18, below 2^5 in base 2
        ks[pages] = (rise.flip(0) if falling else rise)[:, None]
    starts = [0, new, 2 * new]
    want, want_lse, mag = reference(q, kc, vc, ks, vs, table, ctx, starts, 1 / math.sqrt(hd), True, 0)
    got, lse = ma.paged_attention_block_scaled(
        q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(), torch.tensor(ctx, dtype=torch.int32, device="cuda"),
        torch.tensor(starts, dtype=torch.int32, device="cuda"), return_lse=True)
    check_attention(got, lse, q, want, want_lse, mag)
