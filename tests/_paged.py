"""Paged 16-bit caches for tests, and what the calls over them compute, in 64 bits on the CPU."""

from __future__ import annotations

import math

import torch


class Cache:
    """Sequences of `ctx` tokens in a shuffled pool; rows of `new` tokens each (None: one row, no cu_seqlens)."""

    def __init__(self, ctx, new=None, nh=2, group=4, hd=64, bs=16, dtype=torch.bfloat16, seed=0, lead=0, spare=3, junk=None):
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.new = list(ctx), [1] * len(ctx) if new is None else list(new)
        self.nh, self.group, self.hd, self.bs, self.dtype, self.lead = nh, group, hd, bs, dtype, lead
        counts = [-(-c // bs) for c in ctx]
        pages = sum(counts) + spare
        perm = torch.randperm(pages, generator=g).to(torch.int32)
        self.tables = torch.full((len(ctx), max(counts + [1])), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(counts):
            self.tables[i, :n] = perm[at:at + n]
            at += n
        self.layer = torch.randn((2, pages, bs, nh, hd), generator=g).to(dtype)
        if junk is not None:  # places that belong to no token
            held = torch.zeros((pages, bs), dtype=torch.bool)
            for i, c in enumerate(ctx):
                for t in range(c):
                    held[self.tables[i, t // bs], t % bs] = True
            self.layer[:, ~held] = junk
        starts = [lead]
        for n in self.new:
            starts.append(starts[-1] + n)
        self.starts = None if new is None else torch.tensor(starts, dtype=torch.int32)
        self.begin = starts
        self.rows = starts[-1] + (2 if lead else 0)
        self.q = torch.randn((self.rows, nh * group, hd), generator=g).to(dtype)
        self.lens = torch.tensor(self.ctx, dtype=torch.int32)

    def on(self, name, device="cuda"):
        x = getattr(self, name)
        return None if x is None else x.to(device)

    def args(self):
        return [self.on("q"), *self.on("layer").unbind(0), self.on("tables"), self.on("lens")]

    def tokens(self, which, s):
        """Keys or values [nh, tokens, hd] of a sequence in 64 bits, and which of them have a page."""
        room = min(self.ctx[s], self.tables.shape[1] * self.bs)
        t = torch.arange(room)
        page = self.tables[s].long()[t // self.bs]
        fine = (page >= 0) & (page < self.layer.shape[1])
        x = self.layer[which][page.clamp(0, self.layer.shape[1] - 1), t % self.bs].double()
        return x.transpose(0, 1), fine

    def sees(self, s, window=0, sinks=0, parents=None):
        """[rows of s, tokens]: what each row sees."""
        n, c = self.new[s], self.ctx[s]
        room = min(c, self.tables.shape[1] * self.bs)
        t, pos = torch.arange(room), torch.arange(c - n, c)[:, None]
        if parents is None:
            got = t <= pos
            return got & ((t > pos - window) | (t < sinks)) if window else got
        got = (t < c - n).repeat(n, 1)
        for i in range(n):
            j = i
            while j >= 0:
                if 0 <= c - n + j < room:
                    got[i, c - n + j] = True
                up = int(parents[self.begin[s] + j])
                j = up if up < j else -1
        return got

    def attention(self, window=0, sinks=0, parents=None, scale=None):
        """(out, lse, bound): bound holds the weighted mean of |v|, what an error of each weight grows with."""
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        bound, lse = torch.zeros_like(out), torch.full(self.q.shape[:2], -math.inf, dtype=torch.float64)
        for s in range(len(self.ctx)):
            if self.new[s] == 0:
                continue
            at = slice(self.begin[s], self.begin[s] + self.new[s])
            (k, fine), (v, _) = self.tokens(0, s), self.tokens(1, s)
            seen = self.sees(s, window, sinks, parents) & fine
            q = self.q[at].double().view(self.new[s], self.nh, self.group, self.hd)
            x = torch.einsum("ihgd,htd->ihgt", q, k) * scale
            x = torch.where(seen[:, None, None], x, -math.inf)
            top = x.amax(-1, keepdim=True) if x.shape[-1] else torch.full((*x.shape[:-1], 1), -math.inf, dtype=torch.float64)
            w = torch.where(seen[:, None, None], torch.exp(x - torch.where(top.isfinite() | top.isnan(), top, 0.0)), 0.0)
            total = w.sum(-1, keepdim=True)
            # a token that a row does not see has no product at all
            p = torch.where(total == 0, 0.0, w / total)
            o, b = torch.zeros(self.new[s], self.nh, self.group, self.hd, dtype=torch.float64), None
            b = torch.zeros_like(o)
            for i in range(self.new[s]):
                m = seen[i]
                o[i] = torch.einsum("hgt,htd->hgd", p[i][..., m], v[:, m])
                b[i] = torch.einsum("hgt,htd->hgd", p[i][..., m], v[:, m].abs())
            out[at], bound[at] = o.flatten(1, 2), b.flatten(1, 2)
            lse[at] = (top + total.log()).squeeze(-1).flatten(1)
        return out, lse, bound

    def weights(self, lse, sums, window=0, sinks=0, accumulate=True, rows=None, scale=None):
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        got = sums.double().clone()
        for s in range(len(self.ctx)):
            row = s if rows is None else int(rows[s])
            if not 0 <= row < len(sums):
                continue
            if not accumulate:
                got[row] = 0
            if self.new[s] == 0:
                continue
            at = slice(self.begin[s], self.begin[s] + self.new[s])
            k, fine = self.tokens(0, s)
            seen = self.sees(s, window, sinks) & fine
            q = self.q[at].double().view(self.new[s], self.nh, self.group, self.hd)
            x = torch.einsum("ihgd,htd->ihgt", q, k) * scale - lse[at].double().view(self.new[s], self.nh, self.group, 1)
            w = torch.where(seen[:, None, None], x.exp(), 0.0).sum((0, 2))
            n = min(w.shape[1], sums.shape[2])
            got[row, :, :n] += w[:, :n]
        return got


def check(got, want, lse, want_lse, bound, exact_weights=False):
    """A result is rounded by half a step.  Weights are good to half a step of their type with many rows, to 2^-16 with few
    (`exact_weights`); exponents, of scores summed in 32 bits, to 2^-15."""
    half = torch.finfo(got.dtype).eps / 2
    got, lse = got.double().cpu(), lse.double().cpu()
    off = half * want.abs() + ((0 if exact_weights else half) + 2.0**-14) * bound + 1e-30
    if got.dtype == torch.float16:
        off = off + 2.0**-25
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    fine = want.isfinite()
    bad = (got - want).abs() > off + 2.0**-25
    assert not bad[fine].any(), f"{int(bad[fine].sum())} of {fine.sum()} results off, largest {((got - want).abs() / off)[fine].max():.3g}"
    assert torch.equal(lse.isfinite(), want_lse.isfinite()) and torch.equal(lse.isnan(), want_lse.isnan())
    fine = want_lse.isfinite()
    assert ((lse - want_lse)[fine].abs() <= 2.0**-14 + 2.0**-22 * want_lse[fine].abs()).all()
