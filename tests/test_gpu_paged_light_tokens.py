"""An infinite value on a token that a row sees with a weight far below the smallest one of the cache's type: the product of a
positive weight and an infinite value is infinite, whichever kernel takes the row and however its tokens are cut."""

from __future__ import annotations

import math

import pytest
import torch

import musa_aiter as ma

from ._paged import Cache, check

pytestmark = pytest.mark.gpu


def with_gap(ctx, new, dtype, nats, at, hd=64, group=2, nh=1):
    """All scores are 0 but those of token `at` of each sequence, -nats, whose value is infinite in column 3 of head 0.  Rows
    behind it see it."""
    c = Cache(ctx, new, nh=nh, group=group, hd=hd, dtype=dtype)
    c.q.fill_(1.0)
    c.layer[0].zero_()
    for s in range(len(ctx)):
        c.layer[0, c.tables[s, at // 16], at % 16] = -nats / math.sqrt(hd)  # hd products of it with scale hd^-0.5
        c.layer[1, c.tables[s, at // 16], at % 16, 0, 3] = math.inf
    return c


def agree(c, at, parents=None, w=0):
    want, want_lse, bound = c.attention(w, parents=parents)
    if parents is None:
        got, lse = ma.paged_attention_window(*c.args(), c.on("starts"), window=w, return_lse=True)
    else:
        got, lse = ma.paged_attention_tree(*c.args(), parents.cuda(), c.on("starts"), return_lse=True)
    seen = torch.cat([c.sees(s, w, parents=parents)[:, at] for s in range(len(c.ctx))])
    assert seen.any() and (want[seen][:, :c.group, 3] == math.inf).all()
    check(got, want, lse, want_lse, bound)


# float16: 25 nats are 36 log2, below 2^-31 of the largest weight; bfloat16 and both kernels' 32-bit weights: 95 nats are 137
# log2, below 2^-126.  In 64 bits a weight is positive up to 745 nats.
@pytest.mark.parametrize("dtype,nats", [(torch.float16, 25.0), (torch.float16, 95.0), (torch.bfloat16, 25.0), (torch.bfloat16, 95.0)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [None, [3, 2], [60, 40], [200, 150]])
def test_an_infinite_value_with_a_light_weight(new, hd, dtype, nats):
    ctx = [400, 330]
    for at in (5, 70):  # tiles that every row sees whole
        agree(with_gap(ctx, new, dtype, nats, at, hd), at)
    if new is not None:
        for at in (ctx[1] - 1, ctx[1] - new[1]):  # among the rows' own tokens
            agree(with_gap(ctx, new, dtype, nats, at, hd), at)
        parents = torch.cat([torch.arange(-1, n - 1) for n in new]).to(torch.int32)
        agree(with_gap(ctx, new, dtype, nats, 70, hd), 70, parents)
        agree(with_gap(ctx, new, dtype, nats, 300, hd), 300, w=max(new) + 60)


@pytest.mark.parametrize("dtype,nats", [(torch.float16, 95.0), (torch.bfloat16, 95.0)])
@pytest.mark.parametrize("new", [None, [20], [130]])
def test_a_light_token_in_a_sequence_that_many_blocks_share(new, dtype, nats):
    """The maximum of the part that holds the token is as low as the token itself: all of that part is light."""
    for low, n in ((5, 1), (64, 128)):
        c = Cache([9000], new, nh=1, group=2, hd=128, dtype=dtype)
        c.q.fill_(1.0)
        c.layer[0].zero_()
        for t in range(max(low - n, 0), low + n):
            c.layer[0, c.tables[0, t // 16], t % 16] = -nats / math.sqrt(128)
        c.layer[1, c.tables[0, low // 16], low % 16, 0, 3] = math.inf
        agree(c, low)
    c = Cache([9000], new, nh=1, group=2, hd=128, dtype=dtype)  # light up to the middle, the last tokens weigh all
    c.q.fill_(1.0)
    c.layer[0].zero_()
    pages = c.tables[0, :4500 // 16].long()
    c.layer[0, pages] = -nats / math.sqrt(128)
    c.layer[1, c.tables[0, 100 // 16], 100 % 16, 0, 3] = math.inf
    agree(c, 100)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [None, [20], [300]])
def test_light_weights_add_next_to_nothing(new, dtype):
    """20000 tokens too light to count leave the result of the one that weighs all within its rounding: a float16 weight is at
    most 2^-24 in units of which the largest is 2^7 at least, so 20000 of them come to 2^-16.7."""
    c = Cache([20001], new, nh=1, group=1, hd=64, dtype=dtype)
    c.q.fill_(1.0)
    c.layer[0].zero_()
    c.layer[1].fill_(1.0)
    c.layer[0, c.tables[0, 0], 0] = 40 / math.sqrt(64)
    c.layer[1, c.tables[0, 0], 0] = 0.25
    agree_all = c.attention()
    got, lse = ma.paged_attention_window(*c.args(), c.on("starts"), return_lse=True)
    check(got, agree_all[0], lse, agree_all[1], agree_all[2])


def test_a_long_line_of_drafted_tokens_and_values_that_are_no_numbers():
    """Every row's line goes back over 600 rows, and what it sees before them is looked through for NaN and infinite values."""
    c = with_gap([9000], [600], torch.float16, 25.0, 70, group=1)
    line = torch.arange(-1, 599, dtype=torch.int32)
    agree(c, 70, line)
    c.layer[1, c.tables[0, 8000 // 16], 8000 % 16, 0, 9] = math.nan
    agree(c, 70, line)
