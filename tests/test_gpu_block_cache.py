"""Block-scaled 8-bit caches on the GPU: the attention and the writer against their definitions in 64 bits.

Bounds.  The attention multiplies codes that are exact in f16, rounds each weight once to f16 (relative
2^-11) and the result once to q's type (relative 2^-11 or 2^-8); scores and sums are 32-bit.  So with
A = sum_t p_t |v_t| / l an output may be off by (2^-11 + 2^-14) A plus its own rounding, where 2^-14
covers the 32-bit scores (errors of about 2^-20 in an exponent below 2^5).  The writer's steps are IEEE
operations in 32 bits, so its codes and scales are compared with the same steps in numpy, bit for bit.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import musa_aiter as ma

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


def make_cache(g, nb, nh, hd, bs, codes):
    if codes == "int8":
        c = torch.randint(-127, 128, (nb, nh, hd, bs), generator=g).to(torch.int8)
    else:
        c = (torch.randn((nb, nh, hd, bs), generator=g) * 120).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.exp(torch.randn((nb, nh), generator=g) * 0.5) / 90
    return c, s


def make_tables(g, ctx, bs, extra=3):
    counts = [-(-c // bs) for c in ctx]
    nb = sum(counts) + extra
    perm = torch.randperm(nb, generator=g)
    table = torch.full((len(ctx), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = perm[at:at + n]
        at += n
    return table, nb, perm[at:]


def reference(q, kc, vc, ks, vs, table, ctx, starts, scale, causal, window):
    """Output, lse and A in float64, one row at a time over all heads."""
    hq, hd = q.shape[1:]
    nb, nh, _, bs = kc.shape
    grp = hq // nh
    k64, v64 = kc.float().double() * ks.double()[..., None, None], vc.float().double() * vs.double()[..., None, None]
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    for s in range(len(ctx)):
        a, b = starts[s], starts[s + 1]
        c = min(max(ctx[s], 0), table.shape[1] * bs)
        pages = table[s, : -(-c // bs)].long()
        ok = (pages >= 0) & (pages < nb)
        pages = torch.where(ok, pages, torch.zeros_like(pages))
        k = k64[pages].permute(1, 0, 3, 2).reshape(nh, -1, hd)[:, :c]
        v = v64[pages].permute(1, 0, 3, 2).reshape(nh, -1, hd)[:, :c]
        there = ok.repeat_interleave(bs)[:c]
        t = torch.arange(c)
        for i in range(a, b):
            pos = c - (b - a) + (i - a)
            seen = there.clone()
            if causal:
                seen &= t <= pos
            if window:
                seen &= t > pos - window
            if not bool(seen.any()):
                continue
            kk, vv = k[:, seen], v[:, seen]
            x = torch.einsum("hgd,htd->hgt", q[i].double().view(nh, grp, hd), kk) * scale
            lse[i] = torch.logsumexp(x, -1).reshape(-1)
            p = torch.softmax(x, -1)
            out[i] = torch.einsum("hgt,htd->hgd", p, vv).reshape(hq, hd)
            mag[i] = torch.einsum("hgt,htd->hgd", p, vv.abs()).reshape(hq, hd)
    return out, lse, mag


def check_attention(got, lse, q, want, want_lse, mag):
    u = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    bound = (2.0 ** -11 + 2.0 ** -14) * mag + u * want.abs() * 1.01 + 2.0 ** -24
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - bound
    assert float(over.max()) <= 0, f"off by {float((got - want).abs().max())}, {float(over.max())} over the bound"
    if lse is not None:
        lse = lse.double().cpu()
        empty = torch.isinf(want_lse)
        assert torch.equal(torch.isinf(lse), empty)
        assert float((lse - want_lse)[~empty].abs().max() if (~empty).any() else 0) <= 3e-5


def run_case(ctx, new, nh, grp, hd, bs, codes, dtype, *, causal=True, window=0, scale=None, seed=0, poison=True, strided=False,
             single=None, big_q=1.0):
    g = torch.Generator().manual_seed(seed)
    table, nb, unused = make_tables(g, ctx, bs)
    kc, ks = make_cache(g, nb, nh, hd, bs, codes)
    vc, vs = make_cache(g, nb, nh, hd, bs, codes)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    hq = nh * grp
    q = (torch.randn((starts[-1], hq, hd), generator=g) * big_q).to(DT[dtype])
    want, want_lse, mag = reference(q, kc, vc, ks, vs, table, ctx, starts, scale or 1 / math.sqrt(hd), causal, window)
    dk, dv, dks, dvs = kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda()
    if poison:  # what no row sees may hold anything: pages nobody has, positions behind the last token
        for d, s in ((dk, dks), (dv, dvs)):
            raw = d.view(torch.uint8)
            raw[unused.cuda().long()] = 0x7F
            s[unused.cuda().long()] = math.nan
            for i, c in enumerate(ctx):
                if c % bs and c > 0:
                    raw[int(table[i, c // bs]), :, :, c % bs:] = 0xFF
    dq = q.cuda()
    if strided:
        wide = torch.full((q.shape[0], hq + 3, hd + 8), math.nan, dtype=q.dtype, device="cuda")
        wide[:, 1:1 + hq, :hd] = dq
        dq = wide[:, 1:1 + hq, :hd]
    cu = None if single else torch.tensor(starts, dtype=torch.int32).cuda()
    args = (dk, dv, dks, dvs, table.cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(), cu)
    got, lse = ma.paged_attention_block_scaled(dq, *args, causal=causal, window=window, scale=scale, return_lse=True)
    check_attention(got, lse, q, want, want_lse, mag)
    return dq, args, got, lse


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd,bs", [(64, 16), (128, 16), (128, 64), (256, 32), (64, 128), (128, 128)])
def test_single_token_rows(codes, dtype, hd, bs):
    ctx = [1, 15, 16, 17, 127, 128, 129, 500, 1025, 2]
    run_case(ctx, [1] * len(ctx), 2, 4, hd, bs, codes, dtype, single=True, seed=hd + bs)


@pytest.mark.parametrize("grp", [1, 2, 3, 5, 7, 8, 9, 16, 17])
def test_query_heads_per_cache_head(grp):
    run_case([333, 64, 1], [1, 1, 1], 3, grp, 128, 16, "int8", "bf16", seed=grp)


@pytest.mark.parametrize("window", [0, 1, 5, 16, 100, 1000])
@pytest.mark.parametrize("hd,grp,dtype", [(64, 1, "f16"), (128, 4, "bf16"), (256, 2, "bf16")])
def test_several_rows_causal_and_window(window, hd, grp, dtype):
    run_case([40, 700, 3, 129, 256], [7, 4, 3, 1, 16], 2, grp, hd, 32, "fp8", dtype, window=window, seed=window + hd)


def test_rows_that_see_everything():
    run_case([40, 700, 3], [7, 4, 3], 2, 4, 128, 16, "int8", "f16", causal=False, seed=3)


@pytest.mark.parametrize("n", [31, 64, 130, 333])
@pytest.mark.parametrize("hd,grp,bs,codes,dtype", [(128, 4, 16, "int8", "bf16"), (64, 8, 64, "fp8", "f16"), (128, 1, 128, "fp8", "bf16"),
                                                  (256, 2, 16, "int8", "f16")])
def test_many_rows(n, hd, grp, bs, codes, dtype):
    run_case([n + 200, n, n + 1], [n, n, max(1, n // 2)], 2, grp, hd, bs, codes, dtype, seed=n)


@pytest.mark.parametrize("window", [1, 30, 128, 300])
def test_many_rows_window(window):
    run_case([600, 500], [300, 257], 2, 4, 128, 16, "int8", "bf16", window=window, seed=window)


def test_many_rows_that_see_everything():
    run_case([600, 250], [300, 250], 1, 4, 128, 16, "fp8", "f16", causal=False, seed=5)


def test_empty_rows_and_sequences():
    """Sequences without tokens, without rows, and with more rows than tokens (their first rows see nothing)."""
    run_case([0, 5, 0, 20, 3, 0], [1, 0, 0, 2, 6, 3], 2, 4, 64, 16, "int8", "bf16", seed=9)
    run_case([90, 0, 7], [200, 100, 150], 2, 4, 128, 16, "fp8", "bf16", seed=10)


def test_many_sequences():
    g = torch.Generator().manual_seed(1)
    ctx = torch.randint(0, 400, (700,), generator=g).tolist()
    run_case(ctx, [1] * 700, 1, 2, 64, 16, "int8", "f16", single=True, seed=11)


@pytest.mark.parametrize("ctx", [[20000], [9001, 33]])
def test_long_sequences_are_split(ctx):
    run_case(ctx, [1] * len(ctx), 1, 8, 64, 64, "fp8", "f16", single=True, seed=12)


def test_pages_out_of_range_are_skipped():
    g = torch.Generator().manual_seed(4)
    ctx, bs, nh, hd = [100, 77], 16, 2, 64
    table, nb, _ = make_tables(g, ctx, bs)
    table[0, 2], table[1, 0], table[0, 5] = -1, nb, 1 << 30
    kc, ks = make_cache(g, nb, nh, hd, bs, "int8")
    vc, vs = make_cache(g, nb, nh, hd, bs, "int8")
    q = torch.randn((2, 8, hd), generator=g).to(torch.float16)
    want, want_lse, mag = reference(q, kc, vc, ks, vs, table, ctx, [0, 1, 2], 1 / 8, True, 0)
    got, lse = ma.paged_attention_block_scaled(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(),
                                               torch.tensor(ctx, dtype=torch.int32).cuda(), return_lse=True)
    check_attention(got, lse, q, want, want_lse, mag)


def test_lengths_past_the_table_are_cut():
    g = torch.Generator().manual_seed(4)
    table, nb, _ = make_tables(g, [64, 64], 16)
    kc, ks = make_cache(g, nb, 1, 64, 16, "fp8")
    vc, vs = make_cache(g, nb, 1, 64, 16, "fp8")
    q = torch.randn((2, 4, 64), generator=g).to(torch.bfloat16)
    want, want_lse, mag = reference(q, kc, vc, ks, vs, table, [1 << 30, -5], [0, 1, 2], 1 / 8, True, 0)
    got, lse = ma.paged_attention_block_scaled(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(),
                                               torch.tensor([1 << 30, -5], dtype=torch.int32).cuda(), return_lse=True)
    check_attention(got, lse, q, want, want_lse, mag)


@pytest.mark.parametrize("dtype,big", [("bf16", 1e-20), ("bf16", 3e4), ("f16", 60.0)])
@pytest.mark.parametrize("new", [1, 100])
def test_magnitudes_of_q(dtype, big, new):
    run_case([300], [new], 2, 4, 128, 16, "int8", dtype, scale=1 / (math.sqrt(128) * max(big, 1.0)), big_q=big, seed=2)


@pytest.mark.parametrize("new", [1, 90])
def test_scales_of_any_size(new):
    """Blocks whose value scales differ by 2^20, scales of zero, and a sequence of zero scales."""
    g = torch.Generator().manual_seed(6)
    ctx, bs, nh, hd = [400, 200], 16, 2, 128
    table, nb, _ = make_tables(g, ctx, bs)
    kc, ks = make_cache(g, nb, nh, hd, bs, "int8")
    vc, vs = make_cache(g, nb, nh, hd, bs, "int8")
    vs = vs * torch.exp2(torch.randint(-10, 11, vs.shape, generator=g).float())
    vs[table[0, 3]] = 0
    ks[table[0, 7]] = 0
    vs[table[1, :13].long()] = 0
    q = torch.randn((2 * new, 8, hd), generator=g).to(torch.float16)
    starts = [0, new, 2 * new]
    want, want_lse, mag = reference(q, kc, vc, ks, vs, table, ctx, starts, 0.05, True, 0)
    # the weight of a block is rounded after its scale: the bound's A is per head then, not per dim
    mag = torch.maximum(mag, torch.zeros(()))
    big = (vc.float().double() * vs.double()[..., None, None]).abs().amax() * 2.0 ** -26
    got, lse = ma.paged_attention_block_scaled(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), table.cuda(),
                                               torch.tensor(ctx, dtype=torch.int32).cuda(),
                                               torch.tensor(starts, dtype=torch.int32).cuda(), scale=0.05, return_lse=True)
    check_attention(got, lse, q, want, want_lse, mag + float(big) * 2.0 ** 11)


def test_strided_tensors():
    run_case([50, 200, 16], [2, 1, 5], 2, 4, 128, 16, "int8", "bf16", strided=True, seed=8)
    run_case([150, 200, 16], [120, 90, 5], 2, 4, 128, 16, "int8", "bf16", strided=True, seed=8)
    # caches that are slices of one allocation: [NB, 2, NH, HD, BS], scales [NB, NH, 2]
    g = torch.Generator().manual_seed(8)
    ctx, bs, nh, hd = [99, 45], 32, 3, 64
    table, nb, _ = make_tables(g, ctx, bs)
    kc, ks = make_cache(g, nb, nh, hd, bs, "int8")
    vc, vs = make_cache(g, nb, nh, hd, bs, "int8")
    both = torch.stack((kc, vc), 1).cuda()
    scales = torch.stack((ks, vs), -1).cuda()
    wide = torch.full((2, 40), -7, dtype=torch.int32)
    wide[:, : table.shape[1]] = table
    q = torch.randn((2, 6, hd), generator=g).to(torch.float16)
    want, want_lse, mag = reference(q, kc, vc, ks, vs, table, ctx, [0, 1, 2], 1 / 8, True, 0)
    out = torch.full((2, 8, hd + 4), 7.0, dtype=torch.float16, device="cuda")
    got = ma.paged_attention_block_scaled(q.cuda(), both[:, 0], both[:, 1], scales[..., 0], scales[..., 1],
                                          wide.cuda()[:, : table.shape[1]], torch.tensor(ctx, dtype=torch.int32).cuda(),
                                          out=out[:, 1:7, :hd])
    check_attention(got, None, q, want, want_lse, mag)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 7] == 7).all()) and bool((out[:, :, hd:] == 7).all())


def test_same_result_on_other_streams_and_in_a_graph():
    dq, args, got, lse = run_case([3000, 100, 2049], [1, 1, 1], 2, 4, 128, 16, "int8", "bf16", single=True, seed=13)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [ma.paged_attention_block_scaled(dq, *args) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(t, got) for t in there)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = ma.paged_attention_block_scaled(dq, *args)
    for _ in range(3):
        cap.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(cap, got)


def test_calls_of_other_sizes_share_a_workspace():
    for seed, ctx in enumerate(([5000], [17, 900], [5000, 1], [40] * 30)):
        run_case(ctx, [1] * len(ctx), 2, 4, 128, 16, "int8", "bf16", single=True, seed=seed)
        run_case(ctx, [2] * len(ctx), 1, 8, 64, 16, "fp8", "f16", seed=seed)


# ---- the writer -----------------------------------------------------------------------------------


def f8_round(x):
    """float32 numpy -> nearest E4M3 value (torch's conversion on the CPU)."""
    return torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn)


def append_reference(x, cache, scale, table, ctx, starts, codes):
    """The writer's steps in float32 on numpy, in place on the CPU tensors."""
    most = np.float32(127 if codes == "int8" else 448)
    bs = cache.shape[3]
    for s in range(len(ctx)):
        a, b = starts[s], starts[s + 1]
        n, c = b - a, ctx[s]
        if n <= 0 or c < n:
            continue
        for blk in range((c - n) // bs, -(-c // bs)):
            if blk >= table.shape[1]:
                continue
            page = int(table[s, blk])
            if not 0 <= page < cache.shape[0]:
                continue
            lo, hi = max(blk * bs, c - n), min((blk + 1) * bs, c)
            v = x[a + lo - (c - n): a + hi - (c - n)].float().numpy().transpose(1, 2, 0)  # [NH, HD, n]
            v = np.where(np.isfinite(v), v, np.float32(0))
            top = np.abs(v).max((1, 2))
            mine = np.where(top < np.float32(2.0 ** -100), np.float32(0), top / most).astype(np.float32)
            begun = lo == blk * bs
            old = scale[page].numpy()
            old = np.where((old > 0) & np.isfinite(old) & (not begun), old, np.float32(0)).astype(np.float32)
            now = np.maximum(old, mine)
            safe = np.where(now > 0, now, np.float32(1))
            ratio = np.where(now > old, old / safe, np.float32(1)).astype(np.float32)
            kept = cache[page].float().numpy() * ratio[:, None, None]
            if begun:
                kept = np.zeros_like(kept)
            tile = kept.astype(np.float32)
            tile[..., lo - blk * bs: hi - blk * bs] = (v / safe[:, None, None]).astype(np.float32)
            if codes == "int8":
                cache[page] = torch.from_numpy(np.clip(np.rint(tile), -127, 127).astype(np.int8))
            else:
                cache[page] = f8_round(tile)
            scale[page] = torch.from_numpy(now)


def append_case(ctx, new, nh, hd, bs, codes, dtype, seed, values=None, strided=False):
    g = torch.Generator().manual_seed(seed)
    table, nb, _ = make_tables(g, ctx, bs)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    made = []
    for _ in range(2):
        cache, scale = make_cache(g, nb, nh, hd, bs, codes)
        x = torch.randn((starts[-1], nh, hd), generator=g) * torch.exp(torch.randn((starts[-1], 1, 1), generator=g))
        x = x.to(DT[dtype])
        if values is not None:
            values(x, g)
        made.append((x, cache, scale, cache.cuda(), scale.cuda()))
    cu = torch.tensor(starts, dtype=torch.int32).cuda()
    (k, kc, ks, dkc, dks), (v, vc, vs, dvc, dvs) = made
    dk, dv = k.cuda(), v.cuda()
    if strided:
        both = torch.zeros((k.shape[0], 2, nh, hd), dtype=k.dtype, device="cuda")
        both[:, 0], both[:, 1] = dk, dv
        dk, dv = both[:, 0], both[:, 1]
    dt, dc = table.cuda(), torch.tensor(ctx, dtype=torch.int32).cuda()
    assert ma.kv_append_block_scaled(dk, dv, dkc, dvc, dks, dvs, dt, dc, cu) is None
    for x, cache, scale, dcache, dscale in made:
        append_reference(x, cache, scale, table, ctx, starts, codes)
        assert torch.equal(dscale.cpu(), scale), "scales"
        got, want = dcache.cpu().float(), cache.float()
        assert torch.equal(got, want), f"{int((got != want).sum())} codes differ"
    return made, table, starts


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("hd,bs", [(64, 16), (128, 16), (128, 64), (256, 32), (64, 128)])
def test_writer(codes, dtype, hd, bs):
    ctx = [1, bs, bs + 1, 3 * bs - 1, 2 * bs, 5 * bs + 3, bs - 1, 200]
    new = [1, 1, 2, 2 * bs, 2 * bs, 1, bs - 1, 33]
    append_case(ctx, new, 3, hd, bs, codes, dtype, seed=hd + bs)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
def test_writer_one_token_at_a_time(codes):
    """Every offset of a block, its scale growing now and then; some sequences without rows."""
    for n in range(1, 36):
        append_case([n, 0, 40 - n], [1, 0, 1], 2, 64, 16, codes, "bf16", seed=n)


@pytest.mark.parametrize("codes", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_writer_values(codes, dtype):
    def odd(x, g):
        x[0] = 0
        x[1, 0] = math.nan
        x[2, :, 3] = math.inf
        x[3, :, 5] = -math.inf
        x[4:20] *= 1e-30 if dtype != "f16" else 1e-7
        x[40:60] = 0
        x[60:70] *= 1e4

    append_case([20, 64, 70], [20, 40, 30], 2, 128, 16, codes, dtype, seed=1, values=odd)
    append_case([20, 64, 70], [20, 40, 30], 2, 128, 64, codes, dtype, seed=2, values=odd, strided=True)


def test_writer_tiny_values():
    def tiny(x, g):
        x.mul_(2.0 ** -95)
        x[5:] *= 2.0 ** -20

    append_case([20, 40], [20, 30], 1, 64, 16, "int8", "f32", seed=3, values=tiny)
    append_case([20, 40], [20, 30], 1, 64, 16, "fp8", "bf16", seed=3, values=tiny)


def test_writer_scales_that_are_no_scales():
    """An old scale that is zero, negative, infinite or NaN counts as none."""
    g = torch.Generator().manual_seed(2)
    table, nb, _ = make_tables(g, [10, 10, 10, 10], 16)
    kc, ks = make_cache(g, nb, 1, 64, 16, "int8")
    for i, s in enumerate((0.0, -1.0, math.inf, math.nan)):
        ks[table[i, 0]] = s
    vc, vs = kc.clone(), ks.clone()
    x = torch.randn((4, 1, 64), generator=g).to(torch.bfloat16)
    dkc, dvc, dks, dvs = kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda()
    ma.kv_append_block_scaled(x.cuda(), x.cuda(), dkc, dvc, dks, dvs, table.cuda(), torch.full((4,), 10, dtype=torch.int32).cuda())
    append_reference(x, kc, ks, table, [10] * 4, [0, 1, 2, 3, 4], "int8")
    assert torch.equal(dks.cpu()[table[:, 0].long()], ks[table[:, 0].long()]) and torch.equal(dkc.cpu(), kc)
    assert torch.equal(dvc.cpu(), kc)


def test_writer_many_sequences():
    g = torch.Generator().manual_seed(5)
    new = torch.randint(0, 4, (1500,), generator=g).tolist()
    ctx = [n + int(x) for n, x in zip(new, torch.randint(0, 60, (1500,), generator=g))]
    append_case(ctx, new, 1, 64, 16, "int8", "f16", seed=6)


def test_writer_skips_what_has_no_place():
    g = torch.Generator().manual_seed(7)
    table = torch.tensor([[0, -1], [9, 1], [2, 3]], dtype=torch.int32)
    kc, ks = make_cache(g, 5, 2, 64, 16, "fp8")
    x = torch.randn((60, 2, 64), generator=g).to(torch.float16)
    ctx, starts = [30, 20, 50], [0, 30, 40, 60]  # no second page; no page 9; a length past the table
    dkc, dks, dvc, dvs = kc.cuda(), ks.cuda(), kc.cuda(), ks.cuda()
    ma.kv_append_block_scaled(x.cuda(), x.cuda(), dkc, dvc, dks, dvs, table.cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(),
                              torch.tensor(starts, dtype=torch.int32).cuda())
    append_reference(x, kc, ks, table, ctx, starts, "fp8")
    assert torch.equal(dkc.cpu().float(), kc.float()) and torch.equal(dks.cpu(), ks)


@pytest.mark.parametrize("codes,step", [("int8", 1 / 127), ("fp8", 2.0 ** -3)])
def test_write_then_attend(codes, step):
    """A prompt and 40 decoded tokens written step by step; attention reads them as the values they were.

    A value is stored within half a step of its block's scale when written and again whenever the scale
    grows: at most 2 blocks' worth of growth steps happen in 16 writes, so codes are held to 5 steps."""
    g = torch.Generator().manual_seed(3)
    nh, hd, bs, prompt, steps = 2, 128, 16, 37, 40
    k = torch.randn((prompt + steps, nh, hd), generator=g).to(torch.bfloat16).cuda()
    v = torch.randn((prompt + steps, nh, hd), generator=g).to(torch.bfloat16).cuda()
    nb = 8
    kc = torch.zeros((nb, nh, hd, bs), dtype=CODES[codes], device="cuda")
    vc, ks = torch.zeros_like(kc), torch.zeros((nb, nh), device="cuda")
    vs = torch.zeros_like(ks)
    table = torch.randperm(nb, generator=g).to(torch.int32)[None].cuda()
    at = 0
    for n in [prompt] + [1] * steps:
        ctx = torch.tensor([at + n], dtype=torch.int32).cuda()
        cu = torch.tensor([0, n], dtype=torch.int32).cuda()
        ma.kv_append_block_scaled(k[at:at + n], v[at:at + n], kc, vc, ks, vs, table, ctx, cu)
        at += n
    for x, cache, scale in ((k, kc, ks), (v, vc, vs)):
        pages = table[0, : -(-at // bs)].long()
        back = (cache[pages].float() * scale[pages][..., None, None]).permute(0, 3, 1, 2).reshape(-1, nh, hd)[:at]
        tops = torch.stack([x[i:i + bs].float().abs().amax((0, 2)) for i in range(0, at, bs)]).repeat_interleave(bs, 0)[:at]
        off = (back - x.float()).abs()
        lim = 5 * 0.5 * step * (tops[..., None] if codes == "int8" else torch.maximum(x.float().abs(), tops[..., None] / 448))
        assert bool((off <= lim).all())


def test_errors_come_from_the_library_too():
    from musa_aiter import _native

    lib = _native.load()
    assert lib.mak_block_attention(None, None) == -1
    assert b"null descriptor" in lib.mak_last_error()
    assert lib.mak_block_append(None, None, None, 0, 0, 0, 0, 2, None) == -1
