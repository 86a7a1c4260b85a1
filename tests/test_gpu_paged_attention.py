"""Attention over paged 16-bit caches against its definition in 64 bits: windows with first tokens, trees of drafted tokens."""

from __future__ import annotations

import math
import threading

import pytest
import torch

import musa_aiter as ma

from ._paged import Cache, check

pytestmark = pytest.mark.gpu


def window(c, w=0, sinks=0, scale=None, **kw):
    return ma.paged_attention_window(*c.args(), c.on("starts"), window=w, sinks=sinks, scale=scale, return_lse=True, **kw)


def tree(c, parents, **kw):
    return ma.paged_attention_tree(*c.args(), parents.cuda(), c.on("starts"), return_lse=True, **kw)


def few(c):
    return sum(c.new) * c.group <= 16 * len(c.ctx)


def agree(c, w=0, sinks=0, scale=None):
    want, want_lse, bound = c.attention(w, sinks, scale=scale)
    got, lse = window(c, w, sinks, scale)
    live = slice(c.begin[0], c.begin[-1])
    check(got[live], want[live], lse[live], want_lse[live], bound[live], few(c))
    return got, lse


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_single_tokens(dtype, hd, bs):
    agree(Cache([1, 2, 15, 16, 17, 100, 127, 128, 129, 700], hd=hd, bs=bs, dtype=dtype), 0, 0)


@pytest.mark.parametrize("group,nh", [(1, 1), (1, 3), (2, 5), (3, 1), (5, 2), (7, 2), (8, 1), (16, 1), (17, 2), (40, 1)])
def test_head_layouts(group, nh):
    agree(Cache([5, 70, 33], nh=nh, group=group, hd=128))
    agree(Cache([5, 70, 33], [3, 20, 33], nh=nh, group=group, hd=64, dtype=torch.float16), 11, 2)


@pytest.mark.parametrize("w,sinks", [(1, 0), (1, 1), (5, 0), (16, 4), (17, 1), (33, 16), (64, 31), (100, 100), (4096, 4), (2**31 - 1, 7), (10**12, 10**12)])
@pytest.mark.parametrize("new", [None, [1, 2, 7, 9, 4], [1, 17, 64, 40, 200]])
def test_windows_and_first_tokens(new, w, sinks):
    c = Cache([1, 17, 64, 150, 333], new, hd=128 if new else 64, group=2)
    top = 2**31 - 1
    want, want_lse, bound = c.attention(min(w, top), min(sinks, top))
    got, lse = window(c, w, sinks)
    check(got, want, lse, want_lse, bound, few(c))


@pytest.mark.parametrize("n", [2, 8, 9, 16, 17, 31, 33, 64, 65, 127, 128, 129, 255, 300])
@pytest.mark.parametrize("hd,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_many_rows(n, hd, dtype):
    agree(Cache([n, n + 1, n + 130, 400], [n, 1, n, min(n, 400)], hd=hd, dtype=dtype, group=3))


def test_rows_and_sequences_that_are_empty():
    """No tokens, no rows, more rows than tokens; rows before the first sequence's and behind the last one's stay."""
    c = Cache([0, 20, 5, 3, 0, 40], [2, 0, 9, 3, 0, 30], lead=3)
    out = torch.full(c.q.shape, 7.0, dtype=c.dtype, device="cuda")
    want, want_lse, bound = c.attention(8, 2)
    got, lse = window(c, 8, 2, out=out)
    assert got.data_ptr() == out.data_ptr()
    live = slice(3, c.begin[-1])
    check(got[live], want[live], lse[live], want_lse[live], bound[live])
    assert (got[:3] == 7).all() and (got[c.begin[-1]:] == 7).all()
    assert (got[3:5] == 0).all() and (lse[3:5] == -math.inf).all()
    agree(Cache([0, 1, 0], group=8))
    for seqs, rows in ((0, 0), (2, 0)):
        q = torch.empty((rows, 4, 64), dtype=torch.bfloat16, device="cuda")
        starts = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
        cache = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16, device="cuda")
        index = torch.zeros((seqs, 2), dtype=torch.int32, device="cuda")
        out, lse = ma.paged_attention_window(q, cache, cache, index, index[:, 0].contiguous(), starts, return_lse=True)
        assert out.shape == q.shape and lse.shape == q.shape[:2]


@pytest.mark.parametrize("new", [None, [1, 30, 60]])
def test_pages_that_are_none_and_lengths_past_the_table(new):
    c = Cache([100, 90, 200], new, group=2)
    c.tables[0, 2], c.tables[1, 0], c.tables[2, 5], c.tables[2, 12] = -1, c.layer.shape[1], -2**31, 2**31 - 1
    agree(c)
    agree(c, 40, 20)
    c.ctx[2] += 25
    c.lens[2] += 25
    agree(c)
    c = Cache([40, 30], [2, 30])
    c.tables[:] = -1
    got, lse = window(c)
    assert (got == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("junk", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new", [None, [1, 5, 16], [40, 1, 129]])
def test_what_nobody_sees_may_hold_anything(new, junk):
    agree(Cache([40, 5, 130], new, junk=junk), 0, 0)
    agree(Cache([40, 5, 130], new, junk=junk, dtype=torch.float16, hd=128), 9, 3)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("new", [[3, 8], [40, 150]])
@pytest.mark.parametrize("hd", [64, 128])
def test_what_one_row_sees_reaches_no_other(hd, new, bad):
    """A value, or a key, that is no number: rows before its token, or past its window, stay as they are."""
    for which in (0, 1):
        c = Cache([45, 160], new, hd=hd, group=2)
        for s, t in ((0, c.ctx[0] - 2), (1, c.ctx[1] - 4), (1, 3)):
            c.layer[which, c.tables[s, t // 16], t % 16, 0, 5] = bad if which else math.nan
        for w, sinks in ((0, 0), (7, 2)):
            want, want_lse, bound = c.attention(w, sinks)
            got, lse = window(c, w, sinks)
            seen = torch.zeros(c.q.shape[:2], dtype=torch.bool)
            for s, t in ((0, c.ctx[0] - 2), (1, c.ctx[1] - 4), (1, 3)):
                seen[c.begin[s]:c.begin[s + 1], :2] |= c.sees(s, w, sinks)[:, t:t + 1]
            clean = ~seen
            assert got[clean.cuda()].isfinite().all()
            check(got[clean], want[clean], lse[clean], want_lse[clean], bound[clean])
            if which == 0:
                assert got[seen.cuda()].isnan().all() and lse[seen.cuda()].isnan().all()
            else:
                assert not got[seen.cuda()][:, 5].isfinite().any() and torch.equal(got[seen.cuda()].isnan().cpu()[:, 5], want[seen].isnan()[:, 5])


@pytest.mark.parametrize("new", [None, [2, 60]])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e-30])
def test_scales(scale, new):
    agree(Cache([70, 300], new, hd=128), 0, 0, scale)
    agree(Cache([70, 300], new, dtype=torch.float16), 50, 3, scale)


@pytest.mark.parametrize("new", [None, [1, 90, 30]])
def test_large_and_growing_scores(new):
    """Maxima that keep moving, and rows whose weight is almost all on one token."""
    c = Cache([130, 500, 33], new, hd=128, dtype=torch.float16)
    for s in range(3):
        for t in range(c.ctx[s]):
            c.layer[0, c.tables[s, t // 16], t % 16] *= 1 + t * 6 / c.ctx[s]
    agree(c)
    c.q *= 8
    agree(c, 77, 5)


def test_one_heavy_token_and_many_light_ones():
    """Weights below 2^-24 of the largest count: 3000 of them come to 2^-14 of the result."""
    c = Cache([3001], nh=1, group=1, dtype=torch.float16)
    c.layer[0].zero_()
    c.q.fill_(1.0)
    c.layer[1].fill_(1.0)
    c.layer[0, c.tables[0, 0], 0] = 2.25  # its score is above the others by 18 = 26 log2
    c.layer[1, c.tables[0, 0], 0] = 0.0
    want, want_lse, bound = c.attention()
    got, lse = window(c)
    check(got, want, lse, want_lse, bound, True)
    assert (got > 0).all()


@pytest.mark.parametrize("ctx,new", [([9000], None), ([20000, 3], None), ([5000] * 3, [4, 1, 2]), ([7000, 800], [300, 20]), ([300] * 70, None)])
def test_sequences_cut_over_the_gpu(ctx, new):
    agree(Cache(ctx, new, nh=1, group=2, hd=128, bs=64))
    agree(Cache(ctx, new, nh=2, group=1, bs=32, dtype=torch.float16), 1500, 40)


def test_many_sequences():
    agree(Cache([1 + 7 * i % 50 for i in range(700)], group=1, nh=1))
    agree(Cache([40] * 300, [i % 3 for i in range(300)], group=2, nh=1))


def test_strides():
    """Views of larger tensors: heads and tokens of other layouts, rows of a projection, results into a slice."""
    c = Cache([70, 20], [9, 20], nh=2, group=2)
    want, want_lse, bound = c.attention(30, 3)
    q = torch.zeros((c.rows + 1, 3, 2, 2 * c.hd), dtype=c.dtype, device="cuda")
    q[1:, :2, :, c.hd:] = c.on("q").view(-1, 2, 2, c.hd)
    q = q[1:, :, :, c.hd:].flatten(1, 2)[:, :4]
    layer = c.on("layer")
    head_major = torch.empty((layer.shape[1], c.nh, c.bs, c.hd), dtype=c.dtype, device="cuda")
    head_major.copy_(layer[0].transpose(1, 2))
    wide = torch.zeros((layer.shape[1], c.bs, c.nh, 3 * c.hd), dtype=c.dtype, device="cuda")
    wide[..., c.hd:2 * c.hd] = layer[1]
    out = torch.zeros((c.rows, 4, 2 * c.hd), dtype=c.dtype, device="cuda")
    tables = torch.full((2, 9), -1, dtype=torch.int32, device="cuda")
    tables[:, 2:2 + c.tables.shape[1]] = c.on("tables")
    got, lse = ma.paged_attention_window(q, head_major.transpose(1, 2), wide[..., c.hd:2 * c.hd], tables[:, 2:2 + c.tables.shape[1]],
                                         c.on("lens"), c.on("starts"), window=30, sinks=3, return_lse=True, out=out[..., 1:c.hd + 1])
    check(got, want, lse, want_lse, bound)
    assert (out[..., 0] == 0).all() and (out[..., c.hd + 1:] == 0).all()


def test_offsets_past_32_bits():
    """A pool of 4.5 GB a plane, the pages in use at its far end."""
    bs, nh, hd = 128, 8, 128
    pages = 17000
    c = Cache([300, 4], [2, 1], nh=nh, group=1, hd=hd, bs=bs)
    far = torch.zeros((pages, bs, nh, hd), dtype=c.dtype, device="cuda")
    n = c.layer.shape[1]
    want, want_lse, bound = c.attention()
    tables = c.on("tables").clone()
    tables[tables >= 0] += pages - n
    values = torch.zeros_like(far)
    far[-n:], values[-n:] = c.on("layer")
    got, lse = ma.paged_attention_window(c.on("q"), far, values, tables, c.on("lens"), c.on("starts"), return_lse=True)
    check(got, want, lse, want_lse, bound, True)


@pytest.mark.parametrize("new", [None, [1, 100, 3]])
def test_results_do_not_depend_on_stream_or_time(new):
    """The same bits on another stream, from two threads at once, again, and from a graph replayed among other calls."""
    c = Cache([5000, 900, 3], new, nh=1, group=2, hd=128)
    other = Cache([100, 2000], [40, 1], nh=1, group=2, hd=128, seed=3)
    first = agree(c, 4000, 5)
    args, starts = c.args(), c.on("starts")
    call = lambda: ma.paged_attention_window(*args, starts, window=4000, sinks=5, return_lse=True)  # noqa: E731
    same = lambda x: torch.equal(x[0], first[0]) and torch.equal(x[1], first[1])  # noqa: E731
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        on_side = [call() for _ in range(20)]
    here = [call() for _ in range(20)]
    torch.cuda.synchronize()
    assert all(same(x) for x in on_side + here)
    got = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = [call() for _ in range(10)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(same(x) for i in range(3) for x in got[i])
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for _ in range(3):
        for x in outs:
            x[0].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        window(other)
        torch.cuda.synchronize()
        assert all(same(x) for x in outs)


# ---- trees ----------------------------------------------------------------------------------------------


def random_parents(c, seed=0, lo=-1):
    g = torch.Generator().manual_seed(seed)
    p = torch.full((c.rows,), -1, dtype=torch.int32)
    for s, n in enumerate(c.new):
        for i in range(n):
            p[c.begin[s] + i] = int(torch.randint(lo, i, (1,), generator=g)) if i > lo else -1
    return p


def agree_tree(c, parents):
    want, want_lse, bound = c.attention(parents=parents)
    got, lse = tree(c, parents)
    live = slice(c.begin[0], c.begin[-1])
    check(got[live], want[live], lse[live], want_lse[live], bound[live], few(c))


@pytest.mark.parametrize("hd,dtype,bs", [(64, torch.float16, 16), (128, torch.bfloat16, 16), (128, torch.float16, 64), (64, torch.bfloat16, 128)])
@pytest.mark.parametrize("group", [1, 4, 5])
def test_trees(hd, dtype, bs, group):
    c = Cache([1, 5, 40, 129, 300, 77], [1, 5, 3, 33, 64, 0], group=group, hd=hd, dtype=dtype, bs=bs)
    agree_tree(c, random_parents(c))


def test_tree_shapes():
    """A line is causal, a star has leaves only; large trees; more drafted tokens than the sequence has."""
    c = Cache([50, 200, 330], [20, 130, 300], group=2)
    line = torch.cat([torch.arange(-1, n - 1) for n in c.new]).to(torch.int32)
    agree_tree(c, line)
    want, want_lse, bound = c.attention()
    check(*(x for y in zip(tree(c, line), (want, want_lse)) for x in y), bound)
    agree_tree(c, torch.full_like(line, -1))
    agree_tree(c, random_parents(c, 5))
    c = Cache([3, 0, 10], [7, 2, 10], lead=2)
    agree_tree(c, random_parents(c, 1))


def test_parents_that_are_none():
    """Itself, later rows, and numbers out of range end a row's line."""
    c = Cache([60, 30], [12, 4], group=1)
    p = torch.tensor([0, 5, 1, 2, 2**31 - 1, -2**31, 4, 6, 99, 8, 9, -7, 1, 0, 2, 16], dtype=torch.int32)
    agree_tree(c, p)


def test_trees_without_starts():
    c = Cache([1, 30, 200], group=2)
    p = torch.tensor([-1, 0, 5], dtype=torch.int32)
    assert torch.equal(tree(c, p)[0], window(c)[0])


def test_trees_with_values_that_are_no_numbers():
    """A branch whose value is infinite or NaN reaches the rows that continue it, and no other."""
    for new in ([6], [70]):
        c = Cache([90], new, group=2)
        n = new[0]
        p = torch.tensor([(i - 2 if i >= 2 else -1) for i in range(n)], dtype=torch.int32)  # two lines
        c.layer[1, c.tables[0, (90 - n + 1) // 16], (90 - n + 1) % 16, 1, 3] = math.nan
        want, want_lse, bound = c.attention(parents=p)
        got, lse = tree(c, p)
        check(got, want, lse, want_lse, bound)
        assert got[1::2, 2:, 3].isnan().all() and got[0::2].isfinite().all()


def test_trees_in_graphs_and_on_streams():
    c = Cache([4000, 60], [8, 24], nh=2, group=2, hd=128)
    p = random_parents(c).cuda()
    args, starts = c.args(), c.on("starts")
    first = ma.paged_attention_tree(*args, p, starts)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ma.paged_attention_tree(*args, p, starts)
    for _ in range(3):
        out.zero_()
        g.replay()
        assert torch.equal(out, first)


def test_head_dims_and_types_refused_on_the_gpu():
    c = Cache([4])
    with pytest.raises(ValueError, match="one type"):
        ma.paged_attention_window(c.on("q").half(), *c.on("layer"), c.on("tables"), c.on("lens"))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ma.paged_attention_window(c.on("q"), *c.on("layer"), c.tables, c.on("lens"))


@pytest.mark.parametrize("group,new,ctx", [(2, 20, 300), (4, 32, 900), (3, 100, 450), (1, 300, 500)])
def test_many_units_to_a_block(group, new, ctx):
    """More units than blocks, some of them cut, between calls of other values and of other kernels on the same stream: each
    call's results are its own, from the first to the last."""
    n = 48
    lens = [ctx - 7 * i % 90 for i in range(n)]
    news = [max(1, new - i % 11) for i in range(n)]
    c, other = (Cache(lens, news, nh=8, group=group, hd=128, seed=seed) for seed in (1, 2))
    few_rows = Cache([4000] * 3, nh=8, group=4, hd=128, seed=3)
    want, want_lse, bound = c.attention(200, 3)
    want_few, few_lse, few_bound = few_rows.attention()
    p = random_parents(c)
    want_tree, tree_lse, tree_bound = c.attention(parents=p)
    for _ in range(4):
        window(other, 200, 3)
        got = window(c, 200, 3)
        tree(other, p)
        got_tree = tree(c, p)
        got_few = window(few_rows)
        check(got[0], want, got[1], want_lse, bound)
        check(got_tree[0], want_tree, got_tree[1], tree_lse, tree_bound)
        check(got_few[0], want_few, got_few[1], few_lse, few_bound, True)
