"""The work that attention over paged 16-bit caches and what goes with it is timed on, with plain forms.

The operators: attention with a sliding window and first tokens that stay visible, attention for trees
of drafted tokens, the eviction of tokens by accumulated attention weight (the sums and the moving), and
norms of queries and keys for each head with the position rotation in the same pass, with its gradient.
``run`` makes a user's call of ``musa_aiter`` where ``own`` is true and computes the same results with
elementary torch operations in 32 bits where it is false.

Caches are the layers of this package's LMCache and SGLang formats, ``[num_blocks, block_size, num_heads,
head_dim]``.  Cases keep their ragged lengths in the case itself (``lens_seed``), so ``work`` is exact but
for the moves of an eviction; the values come from the seed given to ``prepare``.
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
        # one user's conversation, one token decoded in a window: the latency of a single call
        _attend("window-decode-1", "window", 1, 5000, 5000, 1, 1, 8, 4, 128, 16, "bf16", 4096, 4, 1),
        # a decode step of 64 requests of 256 to 4096 tokens (this repository's LMCache request mix)
        _attend("window-decode-64", "window", 64, 256, 4096, 1, 1, 8, 4, 128, 16, "bf16", 2048, 4, 2),
        # two prompts' chunks of up to 2048 tokens against a cache of up to 8192
        _attend("window-prompt-chunk", "window", 2, 5000, 8192, 1500, 2048, 8, 4, 128, 16, "bf16", 4096, 4, 3),
        # 16 requests checking trees of 8 to 32 drafted tokens
        _attend("tree-verify-16", "tree", 16, 300, 4500, 8, 32, 8, 4, 128, 16, "bf16", 0, 0, 4),
        # three long conversations with small trees, in 64-token pages: the work of few rows is split over the GPU
        _attend("tree-verify-long", "tree", 3, 60000, 100000, 3, 8, 4, 2, 128, 64, "f16", 0, 0, 5),
        # every decode step of 64 requests adds its weights to what each cached token has gathered
        _attend("weights-decode-64", "weights", 64, 256, 4096, 1, 1, 8, 4, 128, 16, "bf16", 0, 0, 6),
        # prompts' weights, all rows, before the first eviction
        _attend("weights-prompts", "weights", 2, 4000, 6000, 1500, 2048, 8, 4, 128, 16, "f16", 0, 0, 7),
        # 16 requests shrink to 1024 tokens, each head its own, 8 layers
        _evict("evict-16", 16, 1500, 4096, 8, 8, 128, 16, 1024, 4, 128, "bf16", 8),
        # one conversation of 30000 tokens shrinks to 2000, one layer
        _evict("evict-1", 1, 30000, 30000, 1, 4, 64, 64, 2000, 4, 256, "f16", 9),
        # queries and keys of a decode step, views of one projection
        _norm("norm-decode-64", 64, 32, 8, 128, 128, False, "bf16", "bf16", False, 10),
        # a training step's forward and backward pass over a packed batch
        _norm("norm-train", 16411, 32, 8, 128, 128, False, "bf16", "bf16", True, 11),
        # smaller heads, half of each turned, pairs next to one another, weights in 32 bits
        _norm("norm-train-half", 4099, 16, 16, 64, 32, True, "f16", "f32", True, 12),
    ]


def _attend(name, op, seqs, lo, hi, q_lo, q_hi, kv_heads, group, head_dim, block, dtype, window, sinks, lens_seed):
    return dict(name=name, op=op, seqs=seqs, ctx_lo=lo, ctx_hi=hi, q_lo=q_lo, q_hi=q_hi, kv_heads=kv_heads, group=group,
                head_dim=head_dim, block=block, dtype=dtype, window=window, sinks=sinks, lens_seed=lens_seed)


def _evict(name, rows, lo, hi, layers, kv_heads, head_dim, block, keep, sinks, recent, dtype, lens_seed):
    return dict(name=name, op="evict", seqs=rows, ctx_lo=lo, ctx_hi=hi, q_lo=1, q_hi=1, layers=layers, kv_heads=kv_heads, head_dim=head_dim,
                block=block, keep=keep, sinks=sinks, recent=recent, dtype=dtype, lens_seed=lens_seed)


def _norm(name, tokens, q_heads, kv_heads, head_dim, rot_dim, interleaved, dtype, weight, backward, seed):
    return dict(name=name, op="norm", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, rot_dim=rot_dim,
                interleaved=interleaved, dtype=dtype, weight=weight, backward=backward, lens_seed=seed)


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    op = rng.choice(["window", "window", "tree", "tree", "weights", "weights", "evict", "norm"])
    dtype, seed = rng.choice(["bf16", "f16"]), rng.randrange(1 << 30)
    block, head_dim = rng.choice([16, 16, 32, 64, 128]), rng.choice([64, 128, 128])
    if op == "evict":
        rows, layers, kv_heads = _log_int(rng, 1, 32), rng.choice([1, 1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
        most = 1.1e9 / (4 * rows * layers * kv_heads * head_dim)  # bytes of the caches: below the largest listed case's
        hi = _log_int(rng, 300, max(301, min(40000, int(most))))
        lo = max(1, hi // rng.choice([1, 2, 3]))
        sinks, recent = rng.choice([0, 1, 4, 17]), rng.choice([0, 1, 32, 100])
        keep = max(sinks + recent, _log_int(rng, 64, max(65, hi)))
        case = _evict("", rows, lo, hi, layers, kv_heads, head_dim, block, keep, sinks, recent, dtype, seed)
    elif op == "norm":
        kv_heads = rng.choice([1, 2, 4, 8])
        rot_dim = head_dim if rng.random() < 0.7 else head_dim // 2
        case = _norm("", _log_int(rng, 1, 16384), kv_heads * rng.choice([1, 2, 4]), kv_heads, head_dim, rot_dim, rng.random() < 0.5, dtype,
                     rng.choice([dtype, "f32"]), rng.random() < 0.6, seed)
    else:
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8])
        many = {"window": [1, 1, _log_int(rng, 2, 16), _log_int(rng, 32, 2048)], "tree": [_log_int(rng, 2, 64), _log_int(rng, 2, 24)],
                "weights": [1, 1, _log_int(rng, 2, 64), _log_int(rng, 64, 2048)]}[op]
        q_hi = rng.choice(many)
        seqs = _log_int(rng, 1, 4 if q_hi > 64 else 16 if q_hi > 16 else 128)
        most = 6e8 / (4 * seqs * kv_heads * head_dim)  # bytes of the caches read: below the largest listed case's
        heads = 4 * seqs * kv_heads * group * head_dim
        if q_hi > 16:  # and no more multiplications than the listed chunk
            q_hi = max(17, min(q_hi, int(math.sqrt(1.6e11 / heads))))
            most = min(most, 1.6e11 / (heads * q_hi))
        hi = max(q_hi, _log_int(rng, max(q_hi, 33), max(q_hi + 34, min(131072, int(most)))))
        lo = max(q_hi, hi // rng.choice([1, 2, 8]))
        window, sinks = (rng.choice([0, _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)]), rng.choice([0, 1, 4, 20, 128])) if op != "tree" else (0, 0)
        case = _attend("", op, seqs, min(lo, hi), hi, max(1, q_hi // rng.choice([1, 2, 4])), q_hi, kv_heads, group, head_dim, block, dtype,
                       window, sinks if window else 0, seed)
    return {k: v for k, v in case.items() if k != "name"}


def _lengths(case):
    """(tokens in the cache, tokens of the call) of each sequence, from the case alone."""
    r = random.Random(case["lens_seed"])
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    new = [min(c, r.randint(case["q_lo"], case["q_hi"])) for c in ctx]
    return ctx, new


# --------------------------------------------------------------------------------------------
# what a user's program has in hand


def prepare(case, seed):
    if own:
        _package()
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"evict": _prepare_evict, "norm": _prepare_norm}.get(case["op"], _prepare_attend)(case, g)


def _randn(shape, dtype, g, scale=1.0):
    """Normal values, filled slice by slice so that no 32-bit copy of a cache exists."""
    x = torch.empty(shape, dtype=_DTYPES[dtype], device="cuda")
    return x.normal_(0.0, scale, generator=g)


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
    # one layer of an LMCache cache: keys and values in one tensor
    st["layer"] = _randn((2, pages, bs, nh, hd), case["dtype"], g)
    st["tables"] = _tables(ctx, bs, pages, g)
    st["ctx"] = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    st["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda") if case["q_hi"] > 1 else None
    st["q"] = _randn((starts[-1], nh * case["group"], hd), case["dtype"], g)
    if case["op"] == "tree":
        # token i continues the last cached one or an earlier drafted one, mostly a recent one
        back = torch.rand(starts[-1], device="cuda", generator=g).square_()
        i = torch.cat([torch.arange(n) for n in new]).to("cuda")
        st["parents"] = (i - 1 - (back * (i + 1)).long()).clamp(min=-1).to(torch.int32)
    if case["op"] == "weights":
        st["layer"] = st["layer"][:1]
        scores, _ = _scores(st, torch.float32)
        st["lse"] = _packed(st, torch.logsumexp(scores, -1).permute(0, 2, 1, 3)).contiguous()
        del scores
        # decoding adds to what the steps before have gathered, a prompt begins
        st["before"] = torch.rand((case["seqs"], nh, max(ctx)), device="cuda", generator=g) if case["q_hi"] == 1 else None
        st["sums"] = torch.empty((case["seqs"], nh, max(ctx)), device="cuda")
    return st


def _prepare_evict(case, g):
    ctx, _ = _lengths(case)
    nh, hd, bs, layers = case["kv_heads"], case["head_dim"], case["block"], case["layers"]
    pages = sum(-(-c // bs) for c in ctx) + 9
    st = {"case": case, "most": max(ctx)}
    st["keys"], st["values"] = (_randn((layers, pages, bs, nh, hd), case["dtype"], g) for _ in range(2))
    table = _tables(ctx, bs, pages, g)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[table[table >= 0].long()] = 1
    length = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    st["shapes"] = [t.shape for t in (table, length, refs)]
    # one buffer holds the tables, the lengths and the reference counts, so one copy restores them
    st["index_before"] = torch.cat([table.reshape(-1), length, refs])
    st["index"] = st["index_before"].clone()
    st["rows"] = torch.arange(case["seqs"], dtype=torch.int32, device="cuda")
    # a few tokens gather most of the weight, some gather none at all
    sums = torch.randn((layers, case["seqs"], nh, max(ctx)), device="cuda", generator=g).mul_(2.5).exp_()
    st["sums_before"] = torch.where(torch.rand(sums.shape, device="cuda", generator=g) < 0.02, 0.0, sums)
    st["sums"] = st["sums_before"].clone()
    return st


def _prepare_norm(case, g):
    t, hq, hk, hd, half = case["tokens"], case["q_heads"], case["kv_heads"], case["head_dim"], case["rot_dim"] // 2
    most = 4096
    st = {"case": case}
    freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * freq
    st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    st["positions"] = torch.randint(0, most, (t,), device="cuda", generator=g, dtype=torch.int32)
    packed = _randn((t, hq + 2 * hk, hd), case["dtype"], g, 1.7)
    # the projection's output holds q, k and v next to one another
    st["q"], st["k"] = packed[:, :hq], packed[:, hq:hq + hk]
    st["wq"], st["wk"] = ((1 + 0.2 * torch.randn(hd, device="cuda", generator=g)).to(_DTYPES[case["weight"]]) for _ in range(2))
    if case["backward"]:
        st["gq"], st["gk"] = _randn((t, hq, hd), case["dtype"], g), _randn((t, hk, hd), case["dtype"], g)
        for n in ("q", "k", "wq", "wk"):
            st[n] = st[n].detach().requires_grad_()
    return st


# --------------------------------------------------------------------------------------------
# one pass


def run(state):
    op = state["case"]["op"]
    return {"window": _run_window, "tree": _run_tree, "weights": _run_weights, "evict": _run_evict, "norm": _run_norm}[op](state)


def _run_window(st):
    case = st["case"]
    if own:
        return _package().paged_attention_window(st["q"], st["layer"][0], st["layer"][1], st["tables"], st["ctx"], st["starts"],
                                                 window=case["window"], sinks=case["sinks"], return_lse=True)
    return _attend_plain(st)


def _run_tree(st):
    if own:
        return _package().paged_attention_tree(st["q"], st["layer"][0], st["layer"][1], st["tables"], st["ctx"], st["parents"], st["starts"],
                                               return_lse=True)
    return _attend_plain(st)


def _starts(st):
    return st["starts"] if st["starts"] is not None else torch.arange(st["case"]["seqs"] + 1, dtype=torch.int32, device="cuda")


def _packed(st, x):
    """[S, tokens, ...] in the packed order of q: every row of it is one (sequence, token)."""
    starts = _starts(st)
    row = torch.arange(st["q"].shape[0], device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
    return x[seq, row - starts[seq]].flatten(1, 2)


def _gathered(st, which):
    """A plane's tokens, [S, NH, T, HD] in 32 bits."""
    pages = st["tables"].clamp(min=0).long()
    x = st["layer"][which][pages]  # [S, MB, BS, NH, HD]
    return x.flatten(1, 2).permute(0, 2, 1, 3).float()


def _scores(st, kind):
    """Scores [S, NH, tokens, group, T] of every query row, -inf where it does not see the token."""
    case = st["case"]
    nh, grp, hd, seqs = case["kv_heads"], case["group"], case["head_dim"], case["seqs"]
    most = max(st["new_host"])
    starts = _starts(st)
    i = torch.arange(most, device="cuda")
    count = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + torch.minimum(i[None], count[:, None] - 1)).long()
    keys = _gathered(st, 0)
    tokens = keys.shape[2]
    q = st["q"][at].to(kind).view(seqs, most, nh, grp, hd).permute(0, 2, 1, 3, 4).reshape(seqs, nh, most * grp, hd)
    scores = torch.matmul(q, keys.transpose(2, 3)).mul_(1.0 / math.sqrt(hd)).view(seqs, nh, most, grp, tokens)
    t = torch.arange(tokens, device="cuda")
    before = (st["ctx"] - count)[:, None, None]
    if case["op"] == "tree":
        # the drafted tokens that each one continues: powers of (one step back, or none) reach them all
        step = torch.eye(most, device="cuda").repeat(seqs, 1, 1)
        up = st["parents"].long()[at]
        step.scatter_add_(2, up.clamp(min=0)[..., None], (up >= 0)[..., None].float())
        line = torch.linalg.matrix_power(step, most) > 0
        drafted = t[None, None] - before  # [S, 1, T]
        mine = line.gather(2, drafted.clamp(0, most - 1).expand(seqs, most, tokens))
        seen = (drafted < 0) | (mine & (drafted >= 0) & (t < st["ctx"][:, None, None]))
    else:
        where = before + i[None, :, None]  # position of each query token
        seen = t <= where
        if case["window"]:
            seen = seen & ((t > where - case["window"]) | (t < case["sinks"]))
    return scores.masked_fill_(~seen[:, None, :, None], -math.inf), seen


def _attend_plain(st):
    case = st["case"]
    nh, grp, hd, seqs = case["kv_heads"], case["group"], case["head_dim"], case["seqs"]
    scores, _ = _scores(st, torch.float32)
    most, tokens = scores.shape[2], scores.shape[4]
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    values = _gathered(st, 1)
    values.masked_fill_((torch.arange(tokens, device="cuda")[None] >= st["ctx"][:, None])[:, None, :, None], 0.0)
    out = torch.matmul(p.view(seqs, nh, most * grp, tokens), values).view(seqs, nh, most, grp, hd) / total
    lse = (top + total.log()).squeeze(-1)
    return _packed(st, out.permute(0, 2, 1, 3, 4)).to(st["q"].dtype), _packed(st, lse.permute(0, 2, 1, 3))


def _run_weights(st):
    case = st["case"]
    adds = st["before"] is not None
    if adds:
        # what was gathered before this step, so that every pass is the same step
        st["sums"].copy_(st["before"])
    if own:
        _package().paged_attention_weights(st["q"], st["layer"][0], st["tables"], st["ctx"], st["lse"], st["sums"], st["starts"],
                                           window=case["window"], sinks=case["sinks"], accumulate=adds)
        return st["sums"]
    scores, seen = _scores(st, torch.float32)
    seqs, most, heads = case["seqs"], scores.shape[2], case["kv_heads"] * case["group"]
    starts = _starts(st)
    count = starts[1:] - starts[:-1]
    at = (starts[:-1, None] + torch.minimum(torch.arange(most, device="cuda")[None], count[:, None] - 1)).long()
    lse = st["lse"][at].view(seqs, most, case["kv_heads"], case["group"]).permute(0, 2, 1, 3)
    real = (torch.arange(most, device="cuda")[None] < count[:, None])[:, None, :, None, None]
    got = scores.sub_(lse[..., None]).exp_().mul_(real).sum((2, 3))[..., : max(st["ctx_host"])]
    return st["sums"].add_(got) if adds else st["sums"].copy_(got)


def _index_views(st):
    a, b, c = (math.prod(s) for s in st["shapes"])
    return [x.view(s) for x, s in zip(st["index"].split((a, b, c)), st["shapes"])]


def _run_evict(st):
    case = st["case"]
    # tables, counts and sums as they were before the call: a later eviction has new ones
    st["index"].copy_(st["index_before"])
    st["sums"].copy_(st["sums_before"])
    table, length, refs = _index_views(st)
    if own:
        left = _package().kv_pages_evict(table, length, st["rows"], refs, list(st["keys"]), list(st["values"]), st["sums"], case["keep"],
                                         sinks=case["sinks"], recent=case["recent"])
    else:
        left = _evict_plain(st, table, length, refs)
    return [table, length, refs, left, st["keys"], st["values"], st["sums"]]


def _evict_plain(st, table, length, refs):
    case = st["case"]
    layers, seqs, nh, keep, bs = case["layers"], case["seqs"], case["kv_heads"], case["keep"], case["block"]
    most = st["most"]
    t = torch.arange(most, device="cuda")
    ctx = length.long()[:, None]
    # the first and the last ones stay, tokens past the end do not; equal sums: the lowest index stays
    rank = torch.where(t >= ctx - case["recent"], math.inf, 0.0)
    rank = torch.where(t < case["sinks"], math.inf, rank)
    rank = torch.where(t >= ctx, -math.inf, rank)
    key = torch.where(torch.isfinite(rank)[None, :, None], st["sums"], rank[None, :, None].expand(layers, seqs, nh, most))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.sort(order, dim=-1).values  # [L, S, NH, keep]
    shrinks = (length > keep)
    width = kept.shape[-1]
    source = torch.where(shrinks[None, :, None, None], kept, t[:width])
    real = (torch.arange(width, device="cuda") < ctx)[None, :, None].expand(source.shape)
    layer, row, head, place = torch.nonzero(real & shrinks[None, :, None, None], as_tuple=True)
    src = source[layer, row, head, place]
    page = lambda x: table[row, x // bs].long()  # noqa: E731
    a, b = (layer, page(src), src % bs, head), (layer, page(place), place % bs, head)
    for x in (st["keys"], st["values"]):
        x[b] = x[a]
    moved = st["sums"].gather(3, source).masked_fill_(~real, 0.0)
    cut = torch.zeros_like(st["sums"])
    cut[..., :width] = moved
    st["sums"].copy_(torch.where(shrinks[None, :, None, None], cut, st["sums"]))
    gone = (torch.arange(table.shape[1], device="cuda") >= -(-keep // bs))[None] & shrinks[:, None] & (table >= 0)
    refs.index_add_(0, table.clamp(min=0).reshape(-1).long(), -gone.to(torch.int32).reshape(-1))
    table.masked_fill_(gone, -1)
    length.clamp_(max=keep)
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def _run_norm(st):
    case = st["case"]
    if own:
        y = _package().apply_qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["positions"], st["cos"], st["sin"],
                                          interleaved=case["interleaved"])
        if not case["backward"]:
            return y
        return (*y, *torch.autograd.grad(y, (st["q"], st["k"], st["wq"], st["wk"]), (st["gq"], st["gk"])))
    with torch.no_grad():
        at = st["positions"].long()
        cos, sin = st["cos"][at][:, None], st["sin"][at][:, None]
        both = [_norm_plain(x, w, cos, sin, case, gy) for x, w, gy in
                ((st["q"], st["wq"], st.get("gq")), (st["k"], st["wk"], st.get("gk")))]
    return tuple(b[i] for i in range(3 if case["backward"] else 1) for b in both)


def _norm_plain(x, w, cos, sin, case, gy):
    v, weight = x.float(), w.float()
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)
    n = v * r
    y = _rotate(n * weight, cos, sin, case).to(x.dtype)
    if gy is None:
        return (y,)
    g = _rotate(gy.float(), cos, -sin, case)
    # sums over many rows lose what matters in 32 bits
    dw = (g * n).sum((0, 1), dtype=torch.float64)
    h = g * weight
    dx = r * (h - n * (h * n).mean(-1, keepdim=True))
    return y, dx.to(x.dtype), dw.to(w.dtype)


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
    if case["op"] == "norm":
        t, heads, hd = case["tokens"], case["q_heads"] + case["kv_heads"], case["head_dim"]
        size = 4 if case["weight"] == "f32" else 2
        table = 4 * case["rot_dim"] + 4
        if not case["backward"]:
            return {"bytes": t * (4 * heads * hd + table) + 2 * hd * size, "flops": t * heads * (4 * hd + 3 * case["rot_dim"])}
        # forward: x in, y out; backward: x and the gradient in, the gradient out
        return {"bytes": t * (10 * heads * hd + 2 * table) + 6 * hd * size, "flops": t * heads * (15 * hd + 6 * case["rot_dim"])}
    ctx, new = _lengths(case)
    nh, hd, bs = case["kv_heads"], case["head_dim"], case["block"]
    if case["op"] == "evict":
        keep = case["keep"]
        kept = sum(keep - min(case["sinks"], keep) for c in ctx if c > keep)  # the first ones stay where they are
        shrinks = [c for c in ctx if c > keep]
        move = 2 * 2 * 2 * hd * kept * nh * case["layers"]
        return {"bytes": move + case["layers"] * nh * 4 * (sum(shrinks) + max(ctx) * len(shrinks)) + 16 * sum(-(-c // bs) for c in shrinks),
                "flops": 0}
    grp, window, sinks = case["group"], case["window"], case["sinks"]
    tokens = pairs = 0
    for c, n in zip(ctx, new):
        first = max(0, c - n - window + 1) if window else 0
        tokens += c - first + min(first, sinks)
        if case["op"] == "tree":
            pairs += n * (c - n) + 2 * n  # itself and one more at least
        else:
            for i in range(n):
                p = c - n + i
                lo = max(0, p - window + 1) if window else 0
                pairs += p + 1 - lo + min(lo, sinks)
    rows = sum(new) * nh * grp
    if case["op"] == "weights":
        adds = case["q_hi"] == 1
        sums = 8 * tokens * nh if adds else 4 * case["seqs"] * nh * max(ctx)
        return {"bytes": 2 * tokens * nh * hd + rows * (2 * hd + 4) + sums + 4 * tokens // bs, "flops": 2 * pairs * nh * grp * hd}
    return {"bytes": 4 * tokens * nh * hd + rows * (4 * hd + 4) + 4 * tokens // bs + (4 * sum(new) if case["op"] == "tree" else 0),
            "flops": 4 * pairs * nh * grp * hd}


# --------------------------------------------------------------------------------------------
# the same from the definitions in 64 bits


def exact(case, seed):
    """One sequence, one head at a time, in 64 bits."""
    st = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(st)
    if case["op"] == "evict":
        return _exact_evict(st)
    return _exact_attend(st)


def _exact_attend(st):
    case = st["case"]
    nh, grp, hd, bs, op = case["kv_heads"], case["group"], case["head_dim"], case["block"], case["op"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["q"].shape[:2], dtype=torch.float64, device="cuda")
    if op == "weights":
        sums = torch.zeros(st["sums"].shape, dtype=torch.float64, device="cuda") if st["before"] is None else st["before"].double()
    at = 0
    for s, (c, n) in enumerate(zip(st["ctx_host"], st["new_host"])):
        page = st["tables"][s, : -(-c // bs)].long()
        pos = torch.arange(c - n, c, device="cuda")
        token = torch.arange(c, device="cuda")
        if op == "tree":
            ups = st["parents"][at:at + n].tolist()
            sees = np.zeros((n, c), dtype=bool)
            sees[:, : c - n] = True
            for i in range(n):
                j = i
                while j >= 0:
                    sees[i, c - n + j] = True
                    j = ups[j]
            hidden = ~torch.from_numpy(sees).to("cuda")
        else:
            hidden = token[None] > pos[:, None]
            if case["window"]:
                hidden = hidden | ((token[None] <= pos[:, None] - case["window"]) & (token[None] >= case["sinks"]))
        for h in range(nh):
            k = st["layer"][0, page, :, h].reshape(-1, hd)[:c].double()
            v = st["layer"][1, page, :, h].reshape(-1, hd)[:c].double() if op != "weights" else None
            for j in range(h * grp, (h + 1) * grp):
                x = st["q"][at:at + n, j].double() @ k.t() / math.sqrt(hd)
                x = x.masked_fill(hidden, -math.inf)
                if op == "weights":
                    sums[s, h, :c] += torch.exp(x - st["lse"][at:at + n, j, None].double()).sum(0)
                else:
                    lse[at:at + n, j] = torch.logsumexp(x, -1)
                    out[at:at + n, j] = torch.softmax(x, -1) @ v
        at += n
    return sums if op == "weights" else (out, lse)


def _exact_evict(st):
    """Tokens that move have no rounding; their sums have a value in 64 bits."""
    case = st["case"]
    ctx, _ = _lengths(case)
    keep = case["keep"]
    sums = st["sums_before"].cpu().numpy().astype(np.float64)
    for s, c in enumerate(ctx):
        if c <= keep:
            continue
        for layer in range(case["layers"]):
            for h in range(case["kv_heads"]):
                x = sums[layer, s, h].copy()
                rank = x[:c].copy()
                rank[max(0, c - case["recent"]):] = np.inf
                rank[: case["sinks"]] = np.inf
                stay = np.sort(np.lexsort((np.arange(c), -rank))[:keep])
                sums[layer, s, h] = 0.0
                sums[layer, s, h, :keep] = x[stay]
    return [None, None, None, None, None, None, torch.from_numpy(sums)]


def _exact_norm(st):
    case = st["case"]
    half, hd = case["rot_dim"] // 2, case["head_dim"]
    at = st["positions"].long()
    turn = torch.complex(st["cos"][at].double(), st["sin"][at].double())[:, None]

    def turned(x, by):
        y = x.clone()
        first = slice(0, 2 * half, 2) if case["interleaved"] else slice(0, half)
        second = slice(1, 2 * half, 2) if case["interleaved"] else slice(half, 2 * half)
        z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * by
        y[..., first], y[..., second] = z.real, z.imag
        return y

    got = [[], [], []]
    for x, w, gy in ((st["q"], st["wq"], st.get("gq")), (st["k"], st["wk"], st.get("gk"))):
        v, w = x.detach().double(), w.detach().double()
        root = torch.sqrt((v * v).sum(-1, keepdim=True) / hd + 1e-6)
        got[0].append(turned(v / root * w, turn))
        if gy is not None:
            back = turned(gy.double(), turn.conj())
            along = (back * w * v).sum(-1, keepdim=True)
            got[1].append(back * w / root - v * along / (hd * root ** 3))
            got[2].append((back * v / root).sum((0, 1)))
    return tuple(x for part in got for x in part)
