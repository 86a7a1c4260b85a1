"""The weights that cached tokens gather, and the eviction by them, against their definitions."""

from __future__ import annotations

import math

import pytest
import torch

import musa_aiter as ma

from ._paged import Cache

pytestmark = pytest.mark.gpu


def weigh(c, w=0, sinks=0, accumulate=True, width=None, rows=None, n_rows=None, scale=None):
    width = max(c.ctx) if width is None else width
    g = torch.Generator().manual_seed(9)
    sums = torch.rand((n_rows or len(c.ctx), c.nh, width), generator=g)
    _, lse, _ = c.attention(w, sinks, scale=scale)
    lse = lse.float()
    got = sums.cuda()
    args = (c.on("q"), c.on("layer")[0], c.on("tables"), c.on("lens"), lse.cuda(), got, c.on("starts"))
    ma.paged_attention_weights(*args, rows=None if rows is None else rows.cuda(), window=w, sinks=sinks, scale=scale, accumulate=accumulate)
    want = c.weights(lse, sums, w, sinks, accumulate, rows, scale)
    # a weight is off by its exponent's error, below 2^-15 for scores summed in 32 bits, and each sum by its roundings
    off = (got.double().cpu() - want).abs()
    assert (off <= 2.0**-13 * want.abs() + 1e-30).all(), (off / want.abs().clamp(min=1e-30)).max()
    return got


@pytest.mark.parametrize("bs", [16, 32, 64, 128])
@pytest.mark.parametrize("hd,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_weights_of_single_tokens(accumulate, hd, dtype, bs):
    weigh(Cache([1, 15, 16, 17, 0, 129, 700], hd=hd, dtype=dtype, bs=bs), accumulate=accumulate)


@pytest.mark.parametrize("group,nh", [(1, 3), (3, 1), (5, 2), (8, 1), (17, 2), (40, 1)])
def test_weights_of_head_layouts(group, nh):
    weigh(Cache([5, 70, 33], nh=nh, group=group, hd=128))
    weigh(Cache([5, 70, 33], [3, 20, 33], nh=nh, group=group, dtype=torch.float16), 11, 2)


@pytest.mark.parametrize("n", [2, 16, 17, 33, 64, 65, 128, 129, 300])
@pytest.mark.parametrize("hd,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_weights_of_many_rows(n, hd, dtype):
    weigh(Cache([n, n + 1, n + 130, 400], [n, 1, n, min(n, 400)], hd=hd, dtype=dtype, group=3))
    weigh(Cache([n, n + 130], [n, n], hd=hd, dtype=dtype, group=3), accumulate=False)


@pytest.mark.parametrize("w,sinks", [(1, 0), (1, 1), (16, 4), (17, 40), (100, 100), (4096, 4)])
@pytest.mark.parametrize("new", [None, [1, 2, 7, 9, 4], [1, 17, 64, 140, 200]])
@pytest.mark.parametrize("accumulate", [False, True])
def test_weights_of_windows(accumulate, new, w, sinks):
    weigh(Cache([1, 17, 64, 150, 333], new, group=2), w, sinks, accumulate)


def test_weights_sum_to_the_rows():
    """Every row hands out 1 in all."""
    c = Cache([300, 40], [100, 1], group=4, hd=128)
    got = weigh(c, accumulate=False)
    assert torch.allclose(got.sum(-1).cpu(), torch.tensor([[400.0, 400.0], [4.0, 4.0]]), rtol=1e-4)


@pytest.mark.parametrize("new", [None, [1, 90]])
def test_narrow_and_wide_sums_and_other_rows(new):
    for width in (1, 16, 33, 200):
        for accumulate in (False, True):
            weigh(Cache([40, 120], new), accumulate=accumulate, width=width)
    rows = torch.tensor([4, -1, 0, 7], dtype=torch.int32)
    c = Cache([40, 120, 3, 60], None if new is None else [1, 90, 2, 60])
    got = weigh(c, rows=rows, n_rows=6)
    weigh(c, rows=rows, n_rows=6, accumulate=False)
    untouched = torch.rand((6, 2, 120), generator=torch.Generator().manual_seed(9))[[1, 2, 3, 5]]
    assert torch.equal(got.cpu()[[1, 2, 3, 5]], untouched)


@pytest.mark.parametrize("new", [None, [1, 30, 60]])
def test_weights_of_pages_that_are_none_and_of_empty_rows(new):
    c = Cache([100, 90, 200], new, group=2, junk=math.nan)
    c.tables[0, 2], c.tables[1, 0], c.tables[2, 5], c.tables[2, 12] = -1, c.layer.shape[1], -2**31, 2**31 - 1
    weigh(c)
    weigh(c, 40, 20, accumulate=False)
    c.ctx[2] += 25
    c.lens[2] += 25
    weigh(c, width=260)
    weigh(Cache([0, 20, 5, 3], [2, 0, 9, 3], lead=3), 8, 2)
    weigh(Cache([0, 20, 5, 3], [2, 0, 9, 3], lead=3), accumulate=False, width=70)


@pytest.mark.parametrize("new", [None, [100]])
def test_weights_are_the_same_every_time(new):
    c = Cache([3000] if new else [3000, 5, 80], new, nh=1, hd=128)
    first = weigh(c)
    _, lse, _ = c.attention()
    args = [c.on("q"), c.on("layer")[0], c.on("tables"), c.on("lens"), lse.float().cuda()]
    starts = c.on("starts")
    before = torch.rand(first.shape, generator=torch.Generator().manual_seed(9)).cuda()
    sums = before.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ma.paged_attention_weights(*args, sums, starts)
    for _ in range(3):
        sums.copy_(before)
        g.replay()
        assert torch.equal(sums, first)


# ---- eviction -----------------------------------------------------------------------------------------------


class Pool:
    def __init__(self, lens, layers=2, nh=2, hd=64, bs=16, dtype=torch.bfloat16, seed=0, spare=4, width=None, sums="random"):
        g = torch.Generator().manual_seed(seed)
        counts = [-(-n // bs) for n in lens]
        self.pages, self.bs, self.layers, self.nh = sum(counts) + spare, bs, layers, nh
        self.tables = torch.full((len(lens), max(counts + [1])), -1, dtype=torch.int32)
        self.refs = torch.zeros(self.pages, dtype=torch.int32)
        perm = torch.randperm(self.pages, generator=g).to(torch.int32)
        at = 0
        for i, n in enumerate(counts):
            self.tables[i, :n] = perm[at:at + n]
            at += n
        self.refs[perm[:at].long()] = 1
        self.lens = torch.tensor(lens, dtype=torch.int32)
        self.keys, self.values = (torch.randn((layers, self.pages, bs, nh, hd), generator=g).to(dtype) for _ in range(2))
        self.sums = torch.rand((layers, len(lens), nh, width or max(lens + [1])), generator=g)
        if sums == "ties":
            self.sums = (self.sums * 3).floor()

    def state(self):
        return [x.clone() for x in (self.tables, self.lens, self.refs, self.keys, self.values, self.sums)]

    def evicted(self, rows, keep, sinks, recent):
        """The definition, token by token."""
        tables, lens, refs, keys, values, sums = self.state()
        left, done = 0, set()
        before = refs.clone()
        for row in rows:
            if not 0 <= row < len(lens) or row in done or int(lens[row]) <= keep:
                continue
            n = int(lens[row])
            done.add(row)
            held = -(-n // self.bs)
            pages = tables[row, :held].tolist() if held <= tables.shape[1] else None
            if pages is None or n > sums.shape[3] or any(not 0 <= p < self.pages for p in pages) or \
                    any(before[p] > 1 for p in pages[:-(-keep // self.bs)]):
                left += 1
                continue
            for layer in range(self.layers):
                for h in range(self.nh):
                    x = sums[layer, row, h].tolist()
                    rank = sorted(range(sinks, n - recent), key=lambda t: (-x[t] if x[t] == x[t] else math.inf, t))
                    stay = sorted([*range(sinks), *range(n - recent, n), *rank[: keep - sinks - recent]])
                    assert len(stay) == keep
                    for plane in (keys, values):
                        got = [plane[layer, pages[t // self.bs], t % self.bs, h].clone() for t in stay]
                        for j, v in enumerate(got):
                            plane[layer, pages[j // self.bs], j % self.bs, h] = v
                    sums[layer, row, h] = 0
                    sums[layer, row, h, :keep] = torch.tensor([x[t] for t in stay])
            for j in range(-(-keep // self.bs), held):
                refs[pages[j]] -= 1
                tables[row, j] = -1
            lens[row] = keep
        return [tables, lens, refs, keys, values, sums], left

    def call(self, rows, keep, sinks, recent):
        tables, lens, refs, keys, values, sums = (x.cuda() for x in self.state())
        left = ma.kv_pages_evict(tables, lens, torch.tensor(rows, dtype=torch.int32, device="cuda"), refs, list(keys), list(values), sums, keep,
                                 sinks=sinks, recent=recent)
        return [tables, lens, refs, keys, values, sums], left

    def check(self, rows, keep, sinks=0, recent=0):
        want, want_left = self.evicted(rows, keep, sinks, recent)
        got, left = self.call(rows, keep, sinks, recent)
        assert left.shape == (1,) and left.dtype == torch.int32 and int(left) == want_left
        for name, a, b in zip(("tables", "lens", "refs", "keys", "values", "sums"), got, want):
            if b.dtype.itemsize == 2:
                a, b = a.view(torch.int16), b.view(torch.int16)
            same = torch.equal(a.cpu(), b) if b.dtype != torch.float32 else torch.equal(a.cpu().nan_to_num(-7.0), b.nan_to_num(-7.0))
            assert same, name


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bs", [1, 16, 24, 128])
def test_eviction(bs, hd):
    Pool([1, 40, 41, 100, 170, 33], bs=bs, hd=hd, dtype=torch.float16).check([5, 3, 0, 4, 1], 40, 4, 8)


@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (2, 1, 1), (16, 0, 0), (17, 4, 13), (31, 31, 0), (31, 0, 31), (64, 5, 50), (1199, 0, 0)])
def test_what_stays(keep, sinks, recent):
    Pool([1200, 64, 65], sums="ties").check([0, 1, 2], keep, sinks, recent)


def test_sums_of_all_kinds():
    """Equal ones, zeros of both signs, infinities, NaN, subnormal and negative ones."""
    p = Pool([900, 2500], layers=1, nh=4)
    p.sums[0, :, 0] = 1.0
    p.sums[0, :, 1, ::2], p.sums[0, :, 1, 1::2] = 0.0, -0.0
    odd = torch.tensor([math.inf, -math.inf, math.nan, 1e-40, -1e-40, -2.0, 3e38, 0.0])
    p.sums[0, :, 2] = odd[torch.randint(0, 8, (2, 2500), generator=torch.Generator().manual_seed(1))]
    p.sums[0, :, 3] = torch.arange(2500.0).flip(0)
    p.check([0, 1], 300, 2, 3)
    p.check([0, 1], 880)


def test_rows_left_alone():
    """Shared pages that would be written, pages out of range, lengths past the table or the sums; others shrink all the same."""
    p = Pool([100, 100, 100, 100, 100, 100, 90], width=100)
    p.tables[1, 0] = p.tables[0, 0]
    p.refs[p.tables[0, 0]] = 2
    p.tables[2, 6] = -1
    p.tables[3, 1] = p.pages
    p.lens[4] = 5000
    p.refs[p.tables[5, 4]] = 2  # is given back, not written
    p.check([0, 1, 2, 3, 4, 5, 6], 30, 1, 1)
    p = Pool([100, 60], width=70)
    p.check([0, 1], 30)


def test_rows_out_of_range_twice_and_none():
    p = Pool([100, 90, 80])
    p.check([2, -1, 0, 3, 2, 2**31 - 1, 0, 2], 20, 0, 5)
    p.check([], 20)
    p.check([1], 2**31 - 1)


def test_many_layers_and_strided_planes():
    p = Pool([60, 50], layers=130, nh=1)
    p.check([0, 1], 20, 1, 1)
    p = Pool([200, 150], layers=2)
    tables, lens, refs, keys, values, sums = (x.cuda() for x in p.state())
    layers = torch.stack((keys, values), 1)  # LMCache layers: keys and values in one tensor
    wide = torch.zeros((2, 2, 2, 300), device="cuda")
    wide[..., 50:250] = sums
    left = ma.kv_pages_evict(tables, lens, torch.arange(2, dtype=torch.int32, device="cuda"), refs, [x[0] for x in layers], [x[1] for x in layers],
                             wide[..., 50:250], 64, recent=9)
    want, _ = p.evicted([0, 1], 64, 0, 9)
    assert int(left) == 0 and torch.equal(layers[:, 0].cpu(), want[3]) and torch.equal(layers[:, 1].cpu(), want[4])
    assert torch.equal(wide[..., 50:250].cpu(), want[5]) and (wide[..., :50] == 0).all() and (wide[..., 250:] == 0).all()


def test_eviction_in_a_graph():
    p = Pool([3000, 500], hd=128)
    want, _ = p.evicted([0, 1], 400, 4, 32)
    start = [x.cuda() for x in p.state()]
    tables, lens, refs, keys, values, sums = (x.clone() for x in start)
    rows = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        left = ma.kv_pages_evict(tables, lens, rows, refs, list(keys), list(values), sums, 400, sinks=4, recent=32)
    for _ in range(2):
        for x, y in zip((tables, lens, refs, keys, values, sums), start):
            x.copy_(y)
        g.replay()
        torch.cuda.synchronize()
        assert int(left) == 0
        for x, y in zip((tables, lens, refs, keys, values, sums), want):
            assert torch.equal(x.cpu(), y)


def test_attend_weigh_evict_and_go_on():
    """Together: the attention of a prompt, its weights, the eviction, and the next token over what is left."""
    c = Cache([150, 90], [150, 90], nh=2, group=2, hd=64, bs=16)
    q, k, v, tables, lens = c.args()
    starts = c.on("starts")
    _, lse = ma.paged_attention_window(q, k, v, tables, lens, starts, return_lse=True)
    sums = torch.full((1, 2, 2, 160), 5.0, device="cuda")
    ma.paged_attention_weights(q, k, tables, lens, lse, sums[0], starts, accumulate=False)
    refs = torch.zeros(k.shape[0], dtype=torch.int32, device="cuda")
    refs[tables[tables >= 0].long()] = 1
    held = [[(x[tables[s].long()[torch.arange(n) // 16], torch.arange(n) % 16]).double().cpu() for x in (k, v)] for s, n in enumerate(c.ctx)]
    rank = sums.cpu()
    left = ma.kv_pages_evict(tables, lens, torch.arange(2, dtype=torch.int32, device="cuda"), refs, [k], [v], sums, 48, sinks=2, recent=10)
    assert int(left) == 0 and lens.tolist() == [48, 48] and int((refs > 0).sum()) == 6
    one = torch.randn((2, 4, 64), generator=torch.Generator().manual_seed(4)).to(c.dtype)
    got = ma.paged_attention_window(one.cuda(), k, v, tables, lens).double().cpu()
    for s, n in enumerate(c.ctx):
        for h in range(2):
            x = rank[0, s, h].tolist()
            best = sorted(range(2, n - 10), key=lambda t: (-x[t], t))[:36]
            stay = sorted([0, 1, *range(n - 10, n), *best])
            key, value = (y[stay, h] for y in held[s])
            for j in (2 * h, 2 * h + 1):
                p = torch.softmax(key @ one[s, j].double() / 8, 0)
                off = 2.0**-8 * (p @ value).abs() + 2.0**-13 * (p @ value.abs())
                assert ((got[s, j] - p @ value).abs() <= off).all()
