"""Lengths past what the table holds, with windows that lie there: rows see the first tokens alone, which are in the table."""

from __future__ import annotations

import pytest
import torch

import musa_aiter as ma

from ._paged import Cache, check

pytestmark = pytest.mark.gpu


def past(ctx, new, more, bs, hd=64, group=4, nh=2, dtype=torch.bfloat16):
    c = Cache(ctx, new, nh=nh, group=group, hd=hd, bs=bs, dtype=dtype)
    for s, n in enumerate(more):
        c.ctx[s] += n
    c.lens = torch.tensor(c.ctx, dtype=torch.int32)
    return c


# Tables of one to three blocks for all: the windows begin past them, in the same tile of 16, 64 or 128 tokens as the first tokens
# or in a later one, and in some sequences among the table's tokens.
@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("new,group", [(None, 4), (None, 20), ([3, 2, 4], 1), ([3, 2, 4], 8), ([30, 20, 60], 4)])
@pytest.mark.parametrize("sinks", [1, 16, 20, 200])
def test_first_tokens_before_windows_past_the_table(sinks, new, group, bs):
    for w in (1, 7, 30):
        for held, more in ((bs, (10, 27, 33)), (bs, (0, 70, 700)), (3 * bs, (31, 60, 90))):
            c = past([held, held - 3, held], new, more, bs, group=group)
            want, want_lse, bound = c.attention(w, sinks)
            got, lse = ma.paged_attention_window(*c.args(), c.on("starts"), window=w, sinks=sinks, return_lse=True)
            check(got, want, lse, want_lse, bound)
            fine = want_lse.float()
            for accumulate in (False, True):
                before = torch.rand((3, 2, 400), generator=torch.Generator().manual_seed(1))
                sums = before.cuda()
                q, keys, _, tables, lens = c.args()
                ma.paged_attention_weights(q, keys, tables, lens, fine.cuda(), sums, c.on("starts"), window=w, sinks=sinks, accumulate=accumulate)
                right = c.weights(fine, before, w, sinks, accumulate)
                assert ((sums.double().cpu() - right).abs() <= 2.0**-13 * right.abs() + 1e-30).all()
