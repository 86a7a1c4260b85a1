"""The work that the block-scaled cache operators are timed on, with their plain forms.

The operators are a paged cache held in 8 bits with one scale per page and head (its writer and
the attention that reads it), the page bookkeeping of such caches, and rotary positions with
several axes.  ``run`` makes a user's call of ``musa_aiter`` where ``own`` is true and computes the
same results with elementary torch operations in 32 bits where it is false.

Cases keep their ragged lengths in the case itself (``lens_seed``), so ``work`` is exact; the
values come from the seed given to ``prepare``.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_CODE_MAX = {"int8": 127.0, "fp8": 448.0}
_TINY = 2.0 ** -100  # magnitudes below this count as zero in the writer


def _package():
    path = os.path.join(_ROOT, "musa-aiter_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import musa_aiter

    return musa_aiter


# --------------------------------------------------------------------------------------------
# cases


def listed():
    return [
        # one user asks, one token is decoded: the latency of a single call
        _attend("attend-decode-1", 1, 777, 777, 1, 1, 8, 4, 128, 16, "int8", "bf16", 0, 1),
        # a decode step of 64 requests of 256 to 4096 tokens (this repository's LMCache request mix)
        _attend("attend-decode-64", 64, 256, 4096, 1, 1, 8, 4, 128, 16, "fp8", "bf16", 0, 2),
        # four long conversations in 64-token pages: the work of one row is split over the GPU
        _attend("attend-decode-long", 4, 100000, 131072, 1, 1, 8, 8, 128, 64, "fp8", "f16", 0, 3),
        # 16 requests checking 1 to 8 drafted tokens each, one query head per cache head, sliding window
        _attend("attend-verify-window", 16, 300, 4500, 1, 8, 16, 1, 64, 32, "int8", "f16", 1024, 4),
        # two prompts' chunks of up to 2048 tokens against a cache of up to 8192
        _attend("attend-prompt-chunk", 2, 5000, 8192, 1500, 2048, 8, 4, 128, 16, "int8", "bf16", 0, 5),
        # the decode step's write: one token per request into part-filled pages
        _append("append-decode-64", 64, 256, 4096, 1, 1, 8, 128, 16, "fp8", "bf16", 6),
        # prompts' writes: whole pages with ragged ends
        _append("append-prompts", 8, 900, 4096, 900, 4096, 8, 128, 16, "fp8", "bf16", 7),
        # 16 requests sampled 4 times each: prompts' pages shared, part-filled last pages copied, 8 layers
        _pages("pages-fork", "fork", 4096, 8, 8, 128, 16, 16, 4, 3000, 0.5, 8),
        # 64 requests end: their pages return to a pool of 32768
        _pages("pages-free", "free", 32768, 1, 1, 64, 16, 64, 0, 4096, 0.9, 9),
        # a pool with holes is made dense, 8 layers
        _pages("pages-compact", "compact", 4096, 8, 8, 128, 16, 48, 0, 1000, 0.55, 10),
        # rotary positions of a decode step: q and k as views of one projection
        _rope("rope-decode-64", 64, 32, 8, 128, 128, 3, False, False, "bf16", False, 11),
        # gradient through the rotation of a prompt of images and text
        _rope("rope-prompt-backward", 16411, 32, 8, 128, 128, 3, True, False, "bf16", True, 12),
    ]


def _attend(name, seqs, lo, hi, q_lo, q_hi, kv_heads, group, head_dim, block, codes, dtype, window, lens_seed):
    return dict(name=name, op="attend", seqs=seqs, ctx_lo=lo, ctx_hi=hi, q_lo=q_lo, q_hi=q_hi, kv_heads=kv_heads, group=group,
                head_dim=head_dim, block=block, codes=codes, dtype=dtype, window=window, lens_seed=lens_seed)


def _append(name, seqs, lo, hi, n_lo, n_hi, kv_heads, head_dim, block, codes, dtype, lens_seed):
    return dict(name=name, op="append", seqs=seqs, ctx_lo=lo, ctx_hi=hi, q_lo=n_lo, q_hi=n_hi, kv_heads=kv_heads, head_dim=head_dim,
                block=block, codes=codes, dtype=dtype, lens_seed=lens_seed)


def _pages(name, what, pages, layers, kv_heads, head_dim, block, rows, copies, max_len, live, lens_seed):
    return dict(name=name, op="pages", what=what, pages=pages, layers=layers, kv_heads=kv_heads, head_dim=head_dim, block=block,
                rows=rows, copies=copies, max_len=max_len, live=live, lens_seed=lens_seed)


def _rope(name, tokens, q_heads, kv_heads, head_dim, rot_dim, axes, interleaved, interleaved_axes, dtype, backward, seed):
    return dict(name=name, op="rope", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, rot_dim=rot_dim, axes=axes,
                interleaved=interleaved, interleaved_axes=interleaved_axes, dtype=dtype, backward=backward, lens_seed=seed)


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    op = rng.choice(["attend", "attend", "append", "pages", "rope"])
    codes, dtype, seed = rng.choice(["int8", "fp8"]), rng.choice(["bf16", "f16"]), rng.randrange(1 << 30)
    block, head_dim = rng.choice([16, 16, 32, 64, 128]), rng.choice([64, 128, 128])
    if op == "attend":
        kv_heads, group = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 4, 5, 7, 8])
        q_hi = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 32, 2048)])
        seqs = _log_int(rng, 1, 4 if q_hi > 16 else 128)
        most = 1e9 / (2 * seqs * kv_heads * head_dim)  # bytes of the caches read: at most the largest listed case's
        if q_hi > 16:  # and no more multiplications than the listed chunk
            heads = 4 * seqs * kv_heads * group * head_dim
            q_hi = min(q_hi, int(math.sqrt(2.4e11 / heads)))
            most = min(most, 2.4e11 / (heads * q_hi))
        hi = max(q_hi, _log_int(rng, max(q_hi, 33), max(q_hi + 34, min(131072, int(most)))))
        lo = max(q_hi, hi // rng.choice([1, 2, 8]))
        window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
        return {k: v for k, v in _attend("", seqs, min(lo, hi), hi, max(1, q_hi // rng.choice([1, 2, 4])), q_hi, kv_heads, group, head_dim,
                                         block, codes, dtype, window, seed).items() if k != "name"}
    if op == "append":
        q_hi = rng.choice([1, 1, _log_int(rng, 2, 16), _log_int(rng, 32, 4096)])
        seqs = _log_int(rng, 1, 8 if q_hi > 16 else 128)
        hi = _log_int(rng, q_hi + 1, 8192)
        lo = max(q_hi, hi // 4)
        return {k: v for k, v in _append("", seqs, lo, hi, max(1, q_hi // 2), q_hi, rng.choice([1, 2, 4, 8, 16]), head_dim, block, codes,
                                         rng.choice(["bf16", "f16", "f32"]), seed).items() if k != "name"}
    if op == "pages":
        what = rng.choice(["fork", "free", "compact"])
        pages, rows = _log_int(rng, 256, 32768), _log_int(rng, 2, 64)
        copies = rng.choice([1, 2, 4]) if what == "fork" else 0
        layers, kv_heads = (1, 1) if what == "free" else (rng.choice([1, 2, 5, 8]), rng.choice([1, 2, 8]))
        per_page = 2 * layers * kv_heads * head_dim * block
        pages = max(4 * rows, min(pages, int(1.1e9 / per_page)))
        live = rng.uniform(0.3, 0.8)
        max_len = max(1, int(live * pages / rows) * block - rng.randrange(block))
        return {k: v for k, v in _pages("", what, pages, layers, kv_heads, head_dim, block, rows, copies, max_len, live, seed).items()
                if k != "name"}
    kv_heads = rng.choice([1, 2, 4, 8])
    rot_dim = head_dim if rng.random() < 0.7 else head_dim // 2
    return {k: v for k, v in _rope("", _log_int(rng, 1, 16384), kv_heads * rng.choice([1, 2, 4]), kv_heads, head_dim, rot_dim, rng.choice([1, 2, 3]),
                                   rng.random() < 0.5, rng.random() < 0.4, dtype, rng.random() < 0.4, seed).items() if k != "name"}


def _lengths(case):
    """(tokens in the cache after the call, tokens of the call) of each sequence, from the case alone."""
    r = random.Random(case["lens_seed"])
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    new = [min(c, r.randint(case["q_lo"], case["q_hi"])) for c in ctx]
    return ctx, new


def _row_lengths(case):
    """Token counts of the pages cases' sequences: `live` of the pool in all, none over max_len."""
    r = random.Random(case["lens_seed"])
    room = int(case["live"] * case["pages"])
    got = []
    for left in range(case["rows"], 0, -1):
        want = r.randint(1, case["max_len"])
        want = max(1, min(want, (room // left) * case["block"]))
        got.append(want)
        room -= -(-want // case["block"])
    return got


def _sections(case):
    """Pairs of each axis: an odd first section, the rest shared out."""
    half, axes = case["rot_dim"] // 2, case["axes"]
    if axes == 1:
        return [half]
    first = half // 4
    rest = half - first
    return [first] + [rest // (axes - 1) + (1 if i < rest % (axes - 1) else 0) for i in range(axes - 1)]


def _pair_axes(sections, interleaved_axes):
    """Axis of each pair: sections one after another, or dealt out in turn while a section has pairs left."""
    if not interleaved_axes:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, got = list(sections), []
    while sum(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                got.append(a)
    return got


# --------------------------------------------------------------------------------------------
# what a user's program has in hand


def prepare(case, seed):
    if own:
        _package()
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"attend": _prepare_attend, "append": _prepare_append, "pages": _prepare_pages, "rope": _prepare_rope}[case["op"]](case, g)


def _codes(shape, kind, g):
    """Codes as a quantised cache holds them: a normal distribution whose tails reach the largest code."""
    if kind == "int8":
        return (torch.randn(shape, device="cuda", generator=g, dtype=torch.float16) * 38).round_().clamp_(-127, 127).to(torch.int8)
    return (torch.randn(shape, device="cuda", generator=g, dtype=torch.float16) * 130).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(shape, kind, g):
    s = torch.randn(shape, device="cuda", generator=g) * 0.3
    return s.exp_() / (38.0 if kind == "int8" else 130.0)


def _tables(ctx, block, pages, g):
    """Block tables over a shuffled pool (the pool's last page belongs to nobody)."""
    counts = [-(-c // block) for c in ctx]
    perm = torch.randperm(pages - 1, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(ctx), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = perm[at:at + n]
        at += n
    return table


def _prepare_attend(case, g):
    ctx, new = _lengths(case)
    nh, hd, bs = case["kv_heads"], case["head_dim"], case["block"]
    pages = sum(-(-c // bs) for c in ctx) + 9
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st = {"case": case, "ctx_host": ctx, "new_host": new}
    st["key_cache"], st["value_cache"] = (_codes((pages, nh, hd, bs), case["codes"], g) for _ in range(2))
    st["key_scale"], st["value_scale"] = (_scales((pages, nh), case["codes"], g) for _ in range(2))
    st["tables"] = _tables(ctx, bs, pages, g)
    st["ctx"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    st["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if case["q_hi"] > 1 else None
    st["q"] = torch.randn((starts[-1], nh * case["group"], hd), device="cuda", generator=g).to(_DTYPES[case["dtype"]])
    return st


def _prepare_append(case, g):
    ctx, new = _lengths(case)
    nh, hd, bs = case["kv_heads"], case["head_dim"], case["block"]
    pages = sum(-(-c // bs) for c in ctx) + 9
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st = {"case": case, "most": max(new)}
    st["key_cache"], st["value_cache"] = (_codes((pages, nh, hd, bs), case["codes"], g) for _ in range(2))
    st["key_scale"], st["value_scale"] = (_scales((pages, nh), case["codes"], g) for _ in range(2))
    st["tables"] = _tables(ctx, bs, pages, g)
    st["ctx"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    st["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if case["q_hi"] > 1 else None
    st["k"], st["v"] = (torch.randn((starts[-1], nh, hd), device="cuda", generator=g).to(_DTYPES[case["dtype"]]) for _ in range(2))
    return st


def _prepare_pages(case, g):
    lens = _row_lengths(case)
    nb, bs = case["pages"], case["block"]
    rows = case["rows"] * (1 + case["copies"])
    width = -(-case["max_len"] // bs) + 1
    counts = [-(-n // bs) for n in lens]
    perm = torch.randperm(nb, device="cuda", generator=g).to(torch.int32)
    # one buffer holds the tables, the lengths and the reference counts, so one copy restores them
    whole = torch.zeros(rows * width + rows + nb, dtype=torch.int32, device="cuda")
    table, length, refs = _index_views(case, whole)
    table.fill_(-1)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = perm[at:at + n]
        at += n
    length[:len(lens)] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    refs[perm[:at].long()] = 1
    st = {"case": case, "pristine": whole, "work": whole.clone()}
    st["views"] = _index_views(case, st["work"])
    order = list(range(case["rows"]))
    random.Random(int(g.initial_seed())).shuffle(order)
    if case["what"] == "fork":
        st["parents"] = torch.tensor([p for p in order for _ in range(case["copies"])], dtype=torch.int32, device="cuda")
        st["children"] = torch.arange(case["rows"], rows, dtype=torch.int32, device="cuda")
    elif case["what"] == "free":
        st["gone"] = torch.tensor(order[: max(1, len(order) // 2)], dtype=torch.int32, device="cuda")
    if case["what"] != "free":
        shape = (case["layers"], nb, case["kv_heads"], case["head_dim"], bs)
        st["stacks"] = [_codes(shape, "fp8", g), _codes(shape, "fp8", g), _scales(shape[:3], "fp8", g), _scales(shape[:3], "fp8", g)]
        st["planes"] = [s[i] for s in st["stacks"] for i in range(case["layers"])]
    return st


def _index_views(case, whole):
    rows, width = case["rows"] * (1 + case["copies"]), -(-case["max_len"] // case["block"]) + 1
    return whole[: rows * width].view(rows, width), whole[rows * width: rows * width + rows], whole[rows * width + rows:]


def _prepare_rope(case, g):
    t, hq, hk, hd, half = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"], case["rot_dim"] // 2
    most = 4096
    st = {"case": case, "sections": _sections(case)}
    st["axes"] = torch.tensor(_pair_axes(st["sections"], case["interleaved_axes"]), device="cuda")
    freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * freq
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    st["positions"] = torch.randint(0, most, (case["axes"], t), device="cuda", generator=g, dtype=torch.int32)
    packed = torch.randn((t, hq + 2 * hk, hd), device="cuda", generator=g).to(_DTYPES[case["dtype"]])
    # the projection's output holds q, k and v next to one another; a gradient comes in tensors of its own
    st["q"], st["k"] = packed[:, :hq], packed[:, hq:hq + hk]
    if case["backward"]:
        st["q"], st["k"] = st["q"].contiguous(), st["k"].contiguous()
    return st


# --------------------------------------------------------------------------------------------
# one pass


def run(state):
    op = state["case"]["op"]
    if op == "pages":
        # the tables and counts as they were before the call: a scheduler's next step has new ones
        state["work"].copy_(state["pristine"])
    return {"attend": _run_attend, "append": _run_append, "pages": _run_pages, "rope": _run_rope}[op](state)


def _run_attend(st):
    case = st["case"]
    if own:
        return _package().paged_attention_block_scaled(
            st["q"], st["key_cache"], st["value_cache"], st["key_scale"], st["value_scale"], st["tables"], st["ctx"], st["starts"],
            window=case["window"], return_lse=True)
    return _attend_plain(st, torch.float32)


def _padded(st):
    """Row of the packed tensor for [sequence, token], clamped, and which of them exist."""
    seqs, most = st["case"]["seqs"], max(st["new_host"]) if "new_host" in st else st["most"]
    i = torch.arange(most, device="cuda")
    starts = st["starts"] if st["starts"] is not None else torch.arange(seqs + 1, dtype=torch.int32, device="cuda")
    count = starts[1:] - starts[:-1]
    return (starts[:-1, None] + torch.minimum(i[None], count[:, None] - 1)).long(), i[None] < count[:, None], count


def _attend_plain(st, kind):
    case = st["case"]
    nh, grp, hd, bs, seqs = case["kv_heads"], case["group"], case["head_dim"], case["block"], case["seqs"]
    at, real, count = _padded(st)
    most = at.shape[1]
    pages = st["tables"].clamp(min=0).long()
    keys = st["key_cache"][pages].to(kind) * st["key_scale"][pages].to(kind)[..., None, None]  # [S, MB, NH, HD, BS]
    tokens = pages.shape[1] * bs
    keys = keys.permute(0, 2, 3, 1, 4).reshape(seqs, nh, hd, tokens)
    q = st["q"][at].to(kind).view(seqs, most, nh, grp, hd).permute(0, 2, 1, 3, 4).reshape(seqs, nh, most * grp, hd)
    scores = torch.matmul(q, keys).mul_(1.0 / math.sqrt(hd)).view(seqs, nh, most, grp, tokens)
    del keys
    where = st["ctx"][:, None] - count[:, None] + torch.arange(most, device="cuda")[None]  # position of each query token
    t = torch.arange(tokens, device="cuda")
    seen = t[None, None] <= where[..., None]
    if case["window"]:
        seen &= t[None, None] > where[..., None] - case["window"]
    scores.masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    values = st["value_cache"][pages].to(kind) * st["value_scale"][pages].to(kind)[..., None, None]
    values = values.permute(0, 2, 1, 4, 3).reshape(seqs, nh, tokens, hd)
    values = torch.where((t[None] < st["ctx"][:, None])[:, None, :, None], values, torch.zeros((), dtype=kind, device="cuda"))
    out = torch.matmul(p.view(seqs, nh, most * grp, tokens), values).view(seqs, nh, most, grp, hd) / total
    lse = (top + total.log()).squeeze(-1)
    # back to the packed order: every row of it is one (sequence, token)
    row, seq = torch.arange(st["q"].shape[0], device="cuda"), None
    if st["starts"] is None:
        seq, tok = row, torch.zeros_like(row)
    else:
        seq = torch.searchsorted(st["starts"][1:].contiguous(), row, right=True)
        tok = row - st["starts"][seq]
    out = out.permute(0, 2, 1, 3, 4)[seq, tok].reshape(-1, nh * grp, hd)
    lse = lse.permute(0, 2, 1, 3)[seq, tok].reshape(-1, nh * grp)
    if kind == torch.float32:
        return out.to(st["q"].dtype), lse
    return out, lse


def _run_append(st):
    if own:
        _package().kv_append_block_scaled(st["k"], st["v"], st["key_cache"], st["value_cache"], st["key_scale"], st["value_scale"],
                                          st["tables"], st["ctx"], st["starts"])
    else:
        _append_plain(st, "k", "key_cache", "key_scale")
        _append_plain(st, "v", "value_cache", "value_scale")
    return _appended(st)


def _appended(st):
    """FP8 codes are the values they stand for in units of their page's scale; int8 codes are multiplied out."""
    got = {n: st[n] for n in ("key_scale", "value_scale")}
    for cache, scale in (("key_cache", "key_scale"), ("value_cache", "value_scale")):
        got[cache] = st[cache] if st["case"]["codes"] == "fp8" else st[cache].float() * st[scale][..., None, None]
    return got


def _touched(st):
    """The pages that the call writes, [S, P]: page (the pool's unused last one where there is none), and the packed row
    of each of its offsets, [S, P, BS], with which of them the call writes; whether the call begins the page."""
    case = st["case"]
    bs, nb = case["block"], st["key_cache"].shape[0]
    seqs = case["seqs"]
    starts = st["starts"] if st["starts"] is not None else torch.arange(seqs + 1, dtype=torch.int32, device="cuda")
    count = (starts[1:] - starts[:-1]).long()
    first = st["ctx"].long() - count
    wide = (st["most"] + bs - 2) // bs + 1
    index = torch.div(first, bs, rounding_mode="floor")[:, None] + torch.arange(wide, device="cuda")[None]
    token = index[..., None] * bs + torch.arange(bs, device="cuda")  # position in the sequence
    new = (token >= first[:, None, None]) & (token < st["ctx"].long()[:, None, None])
    used = new.any(-1)
    page = torch.where(used, st["tables"].long().gather(1, index.clamp(max=st["tables"].shape[1] - 1)), torch.tensor(nb - 1, device="cuda"))
    row = (starts[:-1].long()[:, None, None] + token - first[:, None, None]).clamp(0, st["k"].shape[0] - 1)
    return page, row, new, used, index * bs >= first[:, None]


def _append_plain(st, x, cache, scale):
    case = st["case"]
    most, kind = _CODE_MAX[case["codes"]], st[cache].dtype
    page, row, new, used, begun = _touched(st)
    v = st[x][row].float().permute(0, 1, 3, 4, 2)  # [S, P, NH, HD, BS]
    v = torch.where(torch.isfinite(v) & new[:, :, None, None], v, torch.zeros((), device="cuda"))
    top = v.abs().amax((-1, -2))
    # the divisor is a tensor: a product with a rounded reciprocal of it would be another result
    mine = torch.where(top < _TINY, torch.zeros((), device="cuda"), top / torch.full_like(top, most))
    old = st[scale][page]
    fine = torch.isfinite(old) & (old > 0) & ~begun[..., None]
    old = torch.where(fine, old, torch.zeros((), device="cuda"))
    now = torch.maximum(old, mine)
    safe = torch.where(now > 0, now, torch.ones((), device="cuda"))
    codes = st[cache][page]
    kept = codes.float()
    # offsets the call does not write: codes of a begun page are zero, the others follow the scale
    ratio = torch.where(now > old, old / safe, torch.ones((), device="cuda"))
    kept = torch.where(begun[:, :, None, None, None], torch.zeros((), device="cuda"), kept * ratio[..., None, None])
    fresh = v / safe[..., None, None]
    got = torch.where(new[:, :, None, None], fresh, kept)
    if case["codes"] == "int8":
        got = got.round().clamp(-127, 127).to(torch.int8)
    else:
        got = got.clamp(-448, 448).to(torch.float8_e4m3fn)
    keep = used[..., None, None, None]
    got = torch.where(keep, got.view(torch.uint8), codes.view(torch.uint8)).view(kind)
    st[cache].view(torch.uint8)[page] = got.view(torch.uint8)
    st[scale][page] = torch.where(used[..., None], now, st[scale][page])


def _run_pages(st):
    case = st["case"]
    table, length, refs = st["views"]
    if case["what"] == "fork":
        if own:
            missing = _package().kv_pages_fork(table, length, st["parents"], st["children"], refs, st["planes"], case["block"])
        else:
            missing = _fork_plain(st, table, length, refs)
        return [table, length, refs, missing] + st["stacks"]
    if case["what"] == "free":
        if own:
            _package().kv_pages_free(table, length, st["gone"], refs)
        else:
            _free_plain(st, table, length, refs)
        return [table, length, refs]
    if own:
        live = _package().kv_pages_compact(table, refs, st["planes"])
    else:
        live = _compact_plain(st, table, refs)
    return [table, refs, live] + st["stacks"]


def _fork_plain(st, table, length, refs):
    case = st["case"]
    bs = case["block"]
    parents, children = st["parents"].long(), st["children"].long()
    lens = length[parents]
    full = torch.div(lens, bs, rounding_mode="floor")
    ragged = lens % bs != 0
    rows = table[parents]
    column = torch.arange(table.shape[1], device="cuda")
    shared = column[None] < full[:, None]
    # the i-th child with a part-filled last page takes the i-th free page
    free = torch.nonzero(refs == 0).squeeze(1)
    rank = torch.cumsum(ragged, 0) - 1
    got = ragged & (rank < free.numel())
    new = torch.where(got, free[rank.clamp(0, max(0, free.numel() - 1))], torch.tensor(-1, device="cuda"))
    source = rows.gather(1, full.long().clamp(max=table.shape[1] - 1)[:, None]).squeeze(1)
    refs.index_add_(0, rows.clamp(min=0).reshape(-1), (shared & (rows >= 0)).to(torch.int32).reshape(-1))
    entries = torch.where(shared, rows, torch.tensor(-1, dtype=torch.int32, device="cuda"))
    entries = torch.where((column[None] == full[:, None]) & got[:, None], new[:, None].to(torch.int32), entries)
    table[children] = entries
    length[children] = torch.where(ragged & ~got, full * bs, lens)
    pick = torch.nonzero(got).squeeze(1)
    src, dst = source[pick].long(), new[pick]
    refs[dst] = 1
    for s in st["stacks"]:
        b = s.view(torch.uint8) if s.element_size() == 1 else s
        b[:, dst] = b[:, src]
    return (ragged & ~got).sum(dtype=torch.int32).view(1)


def _free_plain(st, table, length, refs):
    rows = st["gone"].long()
    held = table[rows]
    refs.index_add_(0, held.clamp(min=0).reshape(-1), -(held >= 0).to(torch.int32).reshape(-1))
    table[rows] = -1
    length[rows] = 0


def _compact_plain(st, table, refs):
    live = refs > 0
    count = live.sum()
    index = torch.arange(refs.numel(), device="cuda")
    src = torch.nonzero(live & (index >= count)).squeeze(1)
    dst = torch.nonzero(~live & (index < count)).squeeze(1)
    for s in st["stacks"]:
        b = s.view(torch.uint8) if s.element_size() == 1 else s
        b[:, dst] = b[:, src]
    to = index.to(torch.int32)
    to[src] = dst.to(torch.int32)
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0
    return count.to(torch.int32).view(1)


def _run_rope(st):
    case = st["case"]
    if own:
        f = _package().apply_rope_axes_backward if case["backward"] else _package().apply_rope_axes
        return f(st["q"], st["k"], st["positions"], st["cos"], st["sin"], st["sections"], interleaved=case["interleaved"],
                 interleaved_axes=case["interleaved_axes"])
    half = case["rot_dim"] // 2
    at = st["positions"].long()[st["axes"]].t()  # [T, half]
    pair = torch.arange(half, device="cuda")
    cos, sin = st["cos"][at, pair][:, None], st["sin"][at, pair][:, None]
    if case["backward"]:
        sin = -sin
    return tuple(_rotate(x.float(), cos, sin, case).to(x.dtype) for x in (st["q"], st["k"]))


def _rotate(x, cos, sin, case):
    half, rot = case["rot_dim"] // 2, case["rot_dim"]
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., rot:]), -1)


# --------------------------------------------------------------------------------------------
# what one pass cannot do without


def work(case):
    if case["op"] == "attend":
        ctx, new = _lengths(case)
        nh, hd, grp, bs = case["kv_heads"], case["head_dim"], case["group"], case["block"]
        tokens = pairs = blocks = 0
        for c, n in zip(ctx, new):
            first = max(0, c - n - case["window"] + 1) if case["window"] else 0
            tokens += c - first
            blocks += -(-c // bs) - first // bs
            for i in range(n):
                p = c - n + i
                pairs += min(p + 1, case["window"]) if case["window"] else p + 1
        q = sum(new) * nh * grp
        return {"bytes": 2 * tokens * nh * hd + 8 * blocks * nh + 4 * blocks + q * (4 * hd + 4), "flops": 4 * pairs * nh * grp * hd}
    if case["op"] == "append":
        ctx, new = _lengths(case)
        nh, hd, bs = case["kv_heads"], case["head_dim"], case["block"]
        size = 4 if case["dtype"] == "f32" else 2
        kept = touched = 0
        for c, n in zip(ctx, new):
            kept += (c - n) % bs
            touched += -(-c // bs) - (c - n) // bs
        return {"bytes": 2 * nh * (hd * (sum(new) * (size + 1) + 2 * kept) + 8 * touched), "flops": 4 * nh * hd * sum(new)}
    if case["op"] == "pages":
        lens, bs = _row_lengths(case), case["block"]
        page = 2 * case["layers"] * case["kv_heads"] * (case["head_dim"] * bs + 4)
        used = sum(-(-n // bs) for n in lens)
        if case["what"] == "fork":
            ragged = sum(1 for n in lens if n % bs)
            return {"bytes": case["copies"] * (2 * ragged * page + 12 * used) + 4 * used, "flops": 0}
        if case["what"] == "free":
            gone = lens[: max(1, len(lens) // 2)]
            return {"bytes": 16 * sum(-(-n // bs) for n in gone), "flops": 0}
        moved = used * (1 - used / case["pages"])
        return {"bytes": 2 * moved * page + 8 * case["pages"] + 8 * used, "flops": 0}
    t, heads = case["tokens"], case["q_heads"] + case["kv_heads"]
    return {"bytes": t * (4 * heads * case["head_dim"] + 4 * case["rot_dim"] + 4 * case["axes"]), "flops": 3 * t * heads * case["rot_dim"]}


# --------------------------------------------------------------------------------------------
# the same from the definitions in 64 bits


def exact(case, seed):
    """One sequence, one head, one page at a time, in 64 bits."""
    st = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(st)
    if case["op"] == "append":
        return _exact_append(st)
    if case["op"] == "rope":
        return _exact_rope(st)
    return _exact_pages(st)


def _exact_attend(st):
    case = st["case"]
    nh, grp, hd, bs = case["kv_heads"], case["group"], case["head_dim"], case["block"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["q"].shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for s, (c, n) in enumerate(zip(st["ctx_host"], st["new_host"])):
        page = st["tables"][s, : -(-c // bs)].long()
        pos = torch.arange(c - n, c, device="cuda")
        token = torch.arange(c, device="cuda")
        hidden = token[None] > pos[:, None]
        if case["window"]:
            hidden = hidden | (token[None] <= pos[:, None] - case["window"])
        for h in range(nh):
            k = (st["key_cache"][page, h].double() * st["key_scale"][page, h].double()[:, None, None]).transpose(1, 2).reshape(-1, hd)[:c]
            v = (st["value_cache"][page, h].double() * st["value_scale"][page, h].double()[:, None, None]).transpose(1, 2).reshape(-1, hd)[:c]
            for j in range(h * grp, (h + 1) * grp):
                x = st["q"][at:at + n, j].double() @ k.t() / math.sqrt(hd)
                x = x.masked_fill(hidden, -math.inf)
                lse[at:at + n, j] = torch.logsumexp(x, -1)
                out[at:at + n, j] = torch.softmax(x, -1) @ v
        at += n
    return out, lse


def _exact_append(st):
    case = st["case"]
    bs, most = case["block"], _CODE_MAX[case["codes"]]
    ctx, new = _lengths(case)
    if sum(new) > 4 * 1024:  # a page at a time: too slow for the prompts
        got = {n: None for n in ("key_cache", "value_cache")}
        scales = {"key_scale": st["key_scale"].double(), "value_scale": st["value_scale"].double()}
        at = 0
        tables = st["tables"].cpu().tolist()
        tops = {n: st[n].double().abs().amax(-1).cpu().numpy() for n in ("k", "v")}
        for n in ("key_scale", "value_scale"):
            scales[n] = scales[n].cpu().numpy()
        for s, (c, n) in enumerate(zip(ctx, new)):
            for b in range((c - n) // bs, -(-c // bs)):
                lo, hi = max(b * bs, c - n), min((b + 1) * bs, c)
                for x, y in (("k", "key_scale"), ("v", "value_scale")):
                    mine = tops[x][at + lo - (c - n): at + hi - (c - n)].max(0) / most
                    page = tables[s][b]
                    scales[y][page] = mine if lo == b * bs else np.maximum(scales[y][page], mine)
            at += n
        return {**got, **{n: torch.from_numpy(v) for n, v in scales.items()}}
    got = {"key_cache": st["key_cache"].double(), "value_cache": st["value_cache"].double(),
           "key_scale": st["key_scale"].double(), "value_scale": st["value_scale"].double()}
    at = 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        for b in range((c - n) // bs, -(-c // bs)):
            lo, hi = max(b * bs, c - n), min((b + 1) * bs, c)
            page = int(st["tables"][s, b])
            for x, cache, scale in (("k", "key_cache", "key_scale"), ("v", "value_cache", "value_scale")):
                v = st[x][at + lo - (c - n): at + hi - (c - n)].double().permute(1, 2, 0)
                mine = v.abs().amax((1, 2)) / most
                old = got[scale][page].clone()
                now = mine if lo == b * bs else torch.maximum(old, mine)
                tile = got[cache][page]
                tile = torch.zeros_like(tile) if lo == b * bs else _code(tile * (old / now)[:, None, None], case)
                tile[..., lo - b * bs: hi - b * bs] = _code(v / now[:, None, None], case)
                got[cache][page], got[scale][page] = tile, now
        at += n
    if case["codes"] == "int8":
        for cache, scale in (("key_cache", "key_scale"), ("value_cache", "value_scale")):
            got[cache] *= got[scale][..., None, None]
    return got


def _code(v, case):
    """The nearest code's value: whole numbers, or 3 bits behind the leading one down to steps of 2^-9."""
    if case["codes"] == "int8":
        return v.round().clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return ((v / step).round() * step).clamp(-448, 448)


def _exact_rope(st):
    case = st["case"]
    t, half = case["tokens"], case["rot_dim"] // 2
    axes = _pair_axes(st["sections"], case["interleaved_axes"])
    turn = torch.empty((t, half), dtype=torch.complex128, device="cuda")
    for j in range(half):
        p = st["positions"][axes[j]].long()
        turn[:, j] = torch.complex(st["cos"][p, j].double(), st["sin"][p, j].double())
    if case["backward"]:
        turn = turn.conj()
    got = []
    for x in (st["q"], st["k"]):
        y = x.double().clone()
        first = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
        second = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        got.append(y)
    return tuple(got)


def _exact_pages(st):
    """Whole numbers have no rounding; the scales that move with their pages do have a value in 64 bits."""
    case = st["case"]
    table, length, refs = (x.cpu().tolist() for x in _index_views(case, st["pristine"]))
    if case["what"] == "free":
        return None
    bs = case["block"]
    free = iter([p for p, n in enumerate(refs) if n == 0])
    moves = []
    if case["what"] == "fork":
        for p in st["parents"].cpu().tolist():
            if length[p] % bs:
                to = next(free, None)
                if to is not None:
                    moves.append((table[p][length[p] // bs], to))
    else:
        count = sum(n > 0 for n in refs)
        moves = list(zip([p for p, n in enumerate(refs) if n > 0 and p >= count], [p for p, n in enumerate(refs) if n == 0 and p < count]))
    stacks = [s.clone() for s in st["stacks"]]
    for a, b in zip(st["stacks"], stacks):
        for s, d in moves:
            b[:, d] = a[:, s]
    lead = [None] * (4 if case["what"] == "fork" else 3)
    return lead + [None, None] + [s.double() for s in stacks[2:]]
