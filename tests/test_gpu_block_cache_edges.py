"""Block-scaled caches at the edges of what a call may hold: rows that do not start at the packed tensors'
first, lengths past the table, windows of any size, scales and codes that are no numbers or hardly any.

Bounds as in test_gpu_block_cache: derived there, not fitted.
"""

from __future__ import annotations

import math
import threading

import pytest
import torch

import musa_aiter as ma

from .test_gpu_block_cache import DT, append_reference, check_attention, make_cache, make_tables

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def define(q, kc, vc, ks, vs, table, ctx, starts, scale, window=0):
    """Causal attention from its definition in 64 bits: a row's result takes the tokens it sees and no others.
    Output, lse, and the sum of weights times magnitudes that check_attention's bound is made of."""
    hq, hd = q.shape[1:]
    nb, nh, _, bs = kc.shape
    grp, room = hq // nh, table.shape[1] * bs
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    t = torch.arange(room)
    for s in range(len(ctx)):
        n = starts[s + 1] - starts[s]
        page = table[s, t // bs].long()
        there = (page >= 0) & (page < nb)
        page = torch.where(there, page, 0)
        k = kc[page, :, :, t % bs].float().double() * ks[page].double()[..., None]  # [tokens, NH, HD]
        v = vc[page, :, :, t % bs].float().double() * vs[page].double()[..., None]
        for i in range(n):
            pos = ctx[s] - n + i
            seen = there & (t <= pos) & (t > pos - window if window else t >= 0)
            if not bool(seen.any()):
                continue
            row = starts[s] + i
            x = torch.einsum("hgd,thd->hgt", q[row].double().view(nh, grp, hd), k[seen]) * scale
            lse[row] = torch.logsumexp(x, -1).reshape(-1)
            p = torch.softmax(x, -1)
            out[row] = torch.einsum("hgt,thd->hgd", p, v[seen]).reshape(hq, hd)
            mag[row] = torch.einsum("hgt,thd->hgd", p, v[seen].abs()).reshape(hq, hd)
    return out, lse, mag


class Case:
    """Sequences of ctx[i] tokens whose last new[i] are rows of this call, on the CPU."""

    def __init__(self, ctx, new, nh, grp, hd, bs, codes, dtype, seed=0, skip=0, after=0):
        g = self.g = torch.Generator().manual_seed(seed)
        self.ctx, self.codes, self.scale = list(ctx), codes, 1 / math.sqrt(hd)
        self.table, nb, _ = make_tables(g, [max(c, 0) for c in ctx], bs)
        self.kc, self.ks = make_cache(g, nb, nh, hd, bs, codes)
        self.vc, self.vs = make_cache(g, nb, nh, hd, bs, codes)
        self.starts = [skip]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.q = torch.randn((self.starts[-1] + after, nh * grp, hd), generator=g).to(DT[dtype])

    def call(self, window=0, out=None):
        args = (self.q, self.kc, self.vc, self.ks, self.vs, self.table)
        return ma.paged_attention_block_scaled(*(x.cuda() for x in args), i32(self.ctx), i32(self.starts), window=window, scale=self.scale,
                                               return_lse=True, out=out)

    def want(self, window=0):
        return define(self.q, self.kc, self.vc, self.ks, self.vs, self.table, self.ctx, self.starts, self.scale, window)

    def check(self, window=0):
        got, lse = self.call(window)
        out, want_lse, mag = self.want(window)
        check_attention(got, lse, self.q, out, want_lse, mag)

    def check_odd(self, window=0):
        """Where the definition gives no finite number neither may the call; everywhere else the bounds hold."""
        got, lse = (x.cpu() for x in self.call(window))
        out, want_lse, mag = self.want(window)
        odd = ~torch.isfinite(out)
        assert odd.any() and not odd.all()
        assert torch.equal(~torch.isfinite(got), odd)
        zero = torch.zeros((), dtype=torch.float64)
        check_attention(torch.where(odd, zero.to(got.dtype), got), lse, self.q, torch.where(odd, zero, out), want_lse, torch.where(odd, zero, mag))


# ---- rows that do not start at the packed tensors' first ---------------------------------------------


@pytest.mark.parametrize("skip,after", [(1, 0), (130, 7), (1000, 300)])
@pytest.mark.parametrize("new,nh,grp,hd", [((1, 1, 1), 2, 4, 64), ((3, 1, 6), 2, 1, 128), ((100, 40, 77), 2, 4, 128), ((90, 130, 300), 1, 1, 64)])
def test_rows_of_a_slice_of_a_batch(new, nh, grp, hd, skip, after):
    """cu_seqlens that start above 0 and end before the last row: rows of no sequence stay as they are."""
    c = Case([40, 300, 310], new, nh, grp, hd, 16, "int8", "bf16", seed=skip, skip=skip, after=after)
    out = torch.full_like(c.q, 7.0, device="cuda")
    _, lse = c.call(out=out)
    want, want_lse, mag = c.want()
    mine = slice(c.starts[0], c.starts[-1])
    check_attention(out[mine], lse[mine], c.q, want[mine], want_lse[mine], mag[mine])
    assert bool((out[: mine.start] == 7).all()) and bool((out[mine.stop:] == 7).all())


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("skip,new", [(1, (1, 1, 2)), (40, (5, 1, 33)), (500, (64, 17, 3)), (333, (0, 20, 0))])
def test_writer_of_a_slice_of_a_batch(codes, skip, new):
    c = Case([70, 21, 40], new, 2, 1, 64, 16, codes, "bf16", seed=skip, skip=skip, after=9)
    c.vs[c.table[0, 1]] = 0  # a scale of zero of a block that the call does not write, or begins
    dev = [x.cuda() for x in (c.kc, c.vc, c.ks, c.vs)]
    ma.kv_append_block_scaled(c.q.cuda(), c.q.cuda(), *dev, c.table.cuda(), i32(c.ctx), i32(c.starts))
    for cache, scale, x, y in ((c.kc, c.ks, dev[0], dev[2]), (c.vc, c.vs, dev[1], dev[3])):
        append_reference(c.q, cache, scale, c.table, c.ctx, c.starts, codes)
        assert torch.equal(y.cpu(), scale) and torch.equal(x.cpu().float(), cache.float())


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("prompt,singles,grp,hd", [(300, 12, 4, 64), (200, 60, 1, 128), (70, 40, 8, 128), (90, 30, 4, 256)])
def test_a_prompt_and_single_tokens_in_one_call(prompt, singles, grp, hd, codes, window):
    """One kernel takes them all, by their average: a prompt among groups of few rows, single tokens among many."""
    g = torch.Generator().manual_seed(prompt)
    ctx = torch.randint(1, 300, (singles,), generator=g).tolist()
    at = singles // 2
    ctx.insert(at, prompt + 150)
    new = [1] * at + [prompt] + [1] * (singles - at)
    Case(ctx, new, 1, grp, hd, 16, codes, "bf16", seed=prompt).check(window)


# ---- positions ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("window", [0, 9, 200])
@pytest.mark.parametrize("over,new", [(5, (8, 3)), (1, (1, 2)), (40, (16, 50)), (5, (120, 90)), (70, (120, 60))])
def test_lengths_past_the_table_shift_no_position(over, new, window):
    """A length past what the table holds: rows keep the positions that the writer gave them."""
    c = Case([160, 96], new, 2, 4, 64, 16, "int8", "f16", seed=over)
    c.ctx = [160 + over, 160 + over]
    c.check(window)


def test_writer_and_attention_agree_past_the_table():
    g = torch.Generator().manual_seed(1)
    nh, hd, bs, new, ctx = 2, 64, 16, 12, 53  # 48 tokens have a place
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    k, v = (torch.randn((new, nh, hd), generator=g).half() for _ in range(2))
    kc, ks = make_cache(g, 4, nh, hd, bs, "int8")
    vc, vs = make_cache(g, 4, nh, hd, bs, "int8")
    dev = [x.cuda() for x in (kc, vc, ks, vs)]
    ma.kv_append_block_scaled(k.cuda(), v.cuda(), *dev, table.cuda(), i32([ctx]), i32([0, new]))
    kc, vc, ks, vs = (x.cpu() for x in dev)
    q = torch.randn((new, 4, hd), generator=g).half()
    # row i sits where the writer put token i: position ctx - new + i
    got, lse = ma.paged_attention_block_scaled(q.cuda(), *dev, table.cuda(), i32([ctx]), i32([0, new]), window=1, return_lse=True)
    want, want_lse, mag = define(q, kc, vc, ks, vs, table, [ctx], [0, new], 1 / math.sqrt(hd), 1)
    check_attention(got, lse, q, want, want_lse, mag)
    assert torch.isfinite(want_lse).sum() == 7 * 4  # the tokens at 41 to 47
    own = v.double().repeat_interleave(2, 1)[:7]  # a window of one token gives that token's value back
    assert float((got[:7].double().cpu() - own).abs().max()) <= 2 * float(v.abs().max()) / 127


@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 2, 2**31, 2**40, 2**31 - 200])
@pytest.mark.parametrize("ctx,new", [((400, 3), (5, 6)), ((300, 290, 1), (310, 300, 40)), ((500, 129), (500, 135))])
def test_windows_of_any_size(ctx, new, window):
    """More rows than tokens and a window near the largest 32-bit number: as without a window."""
    c = Case(ctx, new, 2, 2, 64, 16, "int8", "bf16", seed=3)
    got, lse = c.call(window)
    out, want_lse, mag = c.want(0)
    check_attention(got, lse, c.q, out, want_lse, mag)


# ---- scales and codes that are no numbers, or hardly any ------------------------------------------------


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("new", [(1, 1), (6, 3), (100, 70)])
@pytest.mark.parametrize("codes,grp", [("int8", 4), ("fp8", 2), ("fp8", 1)])
def test_value_scales_that_are_no_numbers(codes, grp, new, window, value):
    """Rows that see such a block give no finite number, the others are as if it were not there."""
    c = Case([195, 135], new, 2, grp, 64, 16, codes, "f16", seed=5)
    c.vs[c.table[0, (200 - new[0] // 2) // 16], 1] = value  # later rows see it, head 1 alone
    if new[0] == 1:
        c.vs[c.table[0, 11], 1] = value
    c.check_odd(window)


@pytest.mark.parametrize("window", [0, 20, 150])
@pytest.mark.parametrize("hd,bs", [(64, 16), (128, 32), (128, 128), (256, 64)])
@pytest.mark.parametrize("new,grp", [((1, 1), 4), ((6, 3), 2), ((9, 8), 1), ((100, 70), 4), ((140, 130), 1)])
def test_codes_that_are_no_numbers(new, grp, hd, bs, window):
    """E4M3 codes 0x7f and 0xff: a value's reaches its own dimension of the rows that see its token, a key's the whole
    row."""
    c = Case([310, 205], new, 2, grp, hd, bs, "fp8", "bf16", seed=6)
    kraw, vraw = c.kc.view(torch.uint8), c.vc.view(torch.uint8)
    at = lambda s, t: (int(c.table[s, t // bs]), t % bs)  # noqa: E731
    for t, head, d, code in ((309, 0, 3, 0x7F), (307, 0, hd - 1, 0xFF), (310 - new[0] // 2 - 1, 0, 17, 0x7F), (306, 0, 18, 0x7F)):
        page, off = at(0, t)
        vraw[page, head, d, off] = code
    page, off = at(1, 205 - (new[1] + 1) // 2)
    kraw[page, 1, 5, off] = 0x7F
    vraw[page, 1, :, off] = 0xFF
    got, lse = (x.cpu() for x in c.call(window))
    out, want_lse, mag = c.want(window)
    odd = ~torch.isfinite(out)
    assert odd.any() and not odd.all()
    assert torch.equal(torch.isnan(got), odd) and torch.equal(torch.isnan(lse), torch.isnan(want_lse))
    zero = torch.zeros((), dtype=torch.float64)
    clean = lambda x: torch.where(odd, zero.to(x.dtype), x)  # noqa: E731
    check_attention(clean(got), torch.nan_to_num(lse, nan=1.0, neginf=-math.inf), c.q, clean(out),
                    torch.nan_to_num(want_lse, nan=1.0, neginf=-math.inf), clean(mag))


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("new", [(1, 1), (5, 4), (40, 90)])
@pytest.mark.parametrize("power", [-50, -90, -109])
def test_value_scales_near_the_smallest(power, new, codes):
    """Magnitudes down to 2^-100 are stored as what they are: scales down to 2^-109.  Rows of bfloat16 hold such results."""
    c = Case([400, 333], new, 2, 4, 128, 16, codes, "bf16", seed=7)
    c.vs = torch.exp2(torch.rand(c.vs.shape, generator=c.g) * 2 + power)
    got, lse = c.call()
    out, want_lse, mag = c.want()
    big = 2.0 ** -power
    check_attention(got.double() * big, lse, c.q, out * big, want_lse, mag * big)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_long_sequences_of_the_smallest_scales(codes, new):
    """Scores all alike: the sum of the weights is as many as there are tokens."""
    c = Case([40000], [new], 1, 1, 64, 128, codes, "bf16", seed=8)
    c.q.zero_()
    c.vs = torch.full_like(c.vs, 2.0 ** -109)
    got, lse = c.call()
    v = (c.vc[c.table[0].long()].float().double() * 2.0 ** -109).permute(0, 3, 1, 2).reshape(-1, 64)[:40000]
    for i in range(new):
        seen = v[: 40000 - new + i + 1]
        assert abs(float(lse[i]) - math.log(len(seen))) <= 3e-5
        off = (got[i, 0].double().cpu() - seen.mean(0)).abs() * 2.0 ** 109
        # as in check_attention, and sums of so many terms of either sign in 32 bits
        bound = (2.0 ** -11 + 2.0 ** -14) * seen.abs().mean(0) * 2.0 ** 109 + 2.0 ** -8 * 1.01 * seen.mean(0).abs() * 2.0 ** 109
        assert bool((off <= bound).all())


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_weights_of_the_smallest_scales_add_up(codes):
    """Many rows: the first scores of each tile are low and the others are not enough above them to move the maximum."""
    nh, hd, bs, ctx, new = 16, 64, 16, 16384, 40
    g = torch.Generator().manual_seed(11)
    table = torch.randperm(ctx // bs, generator=g).to(torch.int32)[None]
    kc = torch.full((ctx // bs, nh, hd, bs), 8.0).to(torch.int8 if codes == "int8" else torch.float8_e4m3fn)
    vc, _ = make_cache(g, ctx // bs, nh, hd, bs, codes)
    ks, vs = torch.full((ctx // bs, nh), 4.9 * math.log(2) / 8), torch.full((ctx // bs, nh), 2.0 ** -109)
    low = torch.arange(ctx // bs) % 8 < 2  # the first 32 of 128 tokens
    ks[table[0, low].long()] = 1e-6
    q = torch.ones((new, nh, hd), dtype=torch.bfloat16)
    got, lse = ma.paged_attention_block_scaled(*(x.cuda() for x in (q, kc, vc, ks, vs, table)), i32([ctx]), i32([0, new]), scale=1 / hd,
                                               return_lse=True)
    weight = torch.exp(ks[table[0].long(), 0].double() * 8).repeat_interleave(bs)
    v = vc[table[0].long()].float().double().permute(0, 3, 1, 2).reshape(ctx, nh, hd)
    total = weight.cumsum(0)[-new:]
    want = (weight[:, None, None] * v).cumsum(0)[-new:] / total[:, None, None]
    mag = (weight[:, None, None] * v.abs()).cumsum(0)[-new:] / total[:, None, None]
    check_attention(got.double() * 2.0 ** 109, lse, q, want, total.log()[:, None].expand(new, nh), mag)


# ---- tensors with a single row, head or block -----------------------------------------------------------


def test_strides_of_axes_with_one_entry():
    """A stride that no element is reached by counts for nothing."""
    g = torch.Generator().manual_seed(9)
    wide = torch.randn((1, 3, 132), generator=g).half().cuda()
    one = wide[:, :1, :128]
    assert one.stride() == (396, 132, 1)
    cos, sin = torch.rand((5, 64), device="cuda"), torch.rand((5, 64), device="cuda")
    pos = i32([[3], [1]])
    plain = one.clone(memory_format=torch.contiguous_format)
    for x, y in zip(ma.apply_rope_axes(one, one, pos, cos, sin, (32, 32)), ma.apply_rope_axes(plain, plain, pos, cos, sin, (32, 32))):
        assert torch.equal(x, y)
    c = Case([20], [1], 1, 1, 128, 16, "int8", "f16", seed=9)
    want, got = ([x.cuda() for x in (c.kc, c.vc, c.ks, c.vs)] for _ in range(2))
    ma.kv_append_block_scaled(plain, plain, *want, c.table.cuda(), i32([20]))
    ma.kv_append_block_scaled(one, one, *got, c.table.cuda(), i32([20]))
    for x, y in zip(want, got):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    a = ma.paged_attention_block_scaled(plain, *want, c.table.cuda(), i32([20]))
    assert torch.equal(a, ma.paged_attention_block_scaled(one, *want, c.table.cuda(), i32([20])))
    # caches of one head whose head stride is odd
    odd = []
    for x in want[:2]:
        room = torch.zeros((x.shape[0], 128 * 16 + 16), dtype=x.dtype, device="cuda")
        room[:, : 128 * 16] = x.view(x.shape[0], -1)
        odd.append(room.as_strided(x.shape, (128 * 16 + 16, 7, 16, 1)))
    assert torch.equal(a, ma.paged_attention_block_scaled(plain, *odd, *want[2:], c.table.cuda(), i32([20])))


# ---- streams ----------------------------------------------------------------------------------------------


def test_the_default_streams_of_two_threads():
    """One handle, another stream in each thread: their partial sums must not meet."""
    cases = [Case([9000], [1], 1, 8, 64, 64, "int8", "f16", seed=s) for s in (12, 13)]
    args, outs, failed = [], [], []
    for c in cases:
        args.append([x.cuda() for x in (c.q, c.kc, c.vc, c.ks, c.vs, c.table)] + [i32(c.ctx)])
        outs.append([torch.empty_like(args[-1][0]) for _ in range(100)])
    want = [ma.paged_attention_block_scaled(*a) for a in args]
    torch.cuda.synchronize()
    start = threading.Barrier(2)

    def work(i):
        try:
            stream = torch.cuda.ExternalStream(2)  # cudaStreamPerThread
            with torch.cuda.stream(stream):
                start.wait(60)
                for out in outs[i]:
                    ma.paged_attention_block_scaled(*args[i], out=out)
                stream.synchronize()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for i in range(2):
        assert all(torch.equal(out, want[i]) for out in outs[i])
