"""Norms of q and k with the rotation, forward and gradient, against the formulas in 64 bits and against differences."""

from __future__ import annotations

import pytest
import torch

import musa_aiter as ma

pytestmark = pytest.mark.gpu


def rotate(x, c, s, interleaved):
    half = c.shape[-1]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    u, v = a * c - b * s, a * s + b * c
    y = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((y, x[..., 2 * half:]), -1)


class Case:
    def __init__(self, t=9, hq=4, hk=2, hd=64, pairs=None, dtype=torch.bfloat16, weight=torch.float32, interleaved=False, index=torch.int32,
                 big=1.0, seed=0):
        g = torch.Generator().manual_seed(seed)
        pairs = hd // 2 if pairs is None else pairs
        self.q, self.k, self.gq, self.gk = ((torch.randn((t, h, hd), generator=g) * m).to(dtype) for h, m in
                                            ((hq, big), (hk, big), (hq, 1.0), (hk, 1.0)))
        self.wq, self.wk = ((1 + 0.3 * torch.randn(hd, generator=g)).to(weight) for _ in range(2))
        angle = torch.rand((20, pairs), generator=g) * 6
        self.cos, self.sin = angle.cos(), angle.sin()
        self.pos = torch.randint(0, 20, (t,), generator=g).to(index)
        self.interleaved, self.eps = interleaved, 1e-6

    def inputs(self):
        return [x.cuda() for x in (self.q, self.k, self.wq, self.wk, self.pos, self.cos, self.sin)]

    def turns(self):
        at = self.pos.long()
        fine = ((at >= 0) & (at < len(self.cos)))[:, None]
        at = at.clamp(0, max(len(self.cos) - 1, 0))
        c, s = (torch.where(fine, x[at].double(), y) for x, y in ((self.cos, 1.0), (self.sin, 0.0)))
        return c[:, None], s[:, None]

    def formula(self, x, w, gy=None):
        """(result, its magnitude) or the gradients with theirs: errors in 32 bits grow with the magnitudes of what is added."""
        c, s = self.turns()
        x, w = x.double(), w.double()
        r = (x.square().mean(-1, keepdim=True) + self.eps).rsqrt()
        n = x * r
        if gy is None:
            return rotate(n * w, c, s, self.interleaved), rotate((n * w).abs(), c.abs(), -s.abs(), self.interleaved).abs() + (n * w).abs()
        g = rotate(gy.double(), c, -s, self.interleaved)
        mag = rotate(gy.double().abs(), c.abs(), s.abs(), self.interleaved).abs() + 2 * gy.double().abs().amax(-1, keepdim=True)
        h = g * w
        dx = r * (h - n * (h * n).mean(-1, keepdim=True))
        m = r * (mag * w.abs() + n.abs() * (mag * w.abs() * n.abs()).mean(-1, keepdim=True))
        return dx, m, (g * n).sum((0, 1)), (mag * n.abs()).sum((0, 1))

    def check(self, got, want, mag, bits=2.0**-19):
        half = torch.finfo(got.dtype).eps / 2
        off = (got.double().cpu() - want).abs()
        bad = off > half * want.abs() + bits * mag + (2.0**-25 if got.dtype == torch.float16 else 1e-38)
        assert got.isfinite().all() and not bad.any(), (off / (half * want.abs() + bits * mag + 1e-38)).max()

    def forward(self):
        got = ma.apply_qk_norm_rope(*self.inputs(), eps=self.eps, interleaved=self.interleaved)
        for y, x, w in zip(got, (self.q, self.k), (self.wq, self.wk)):
            assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
            self.check(y, *self.formula(x, w))
        return got

    def backward(self):
        got = ma.apply_qk_norm_rope_backward(self.gq.cuda(), self.gk.cuda(), *self.inputs(), eps=self.eps, interleaved=self.interleaved)
        self.check_gradients(got)
        return got

    def check_gradients(self, got):
        for i, (x, w, g) in enumerate(((self.q, self.wq, self.gq), (self.k, self.wk, self.gk))):
            dx, mx, dw, mw = self.formula(x, w, g)
            self.check(got[i], dx, mx, 2.0**-18)
            self.check(got[2 + i], dw, mw, 2.0**-18)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hd,pairs", [(16, 8), (64, 32), (64, 16), (80, 40), (96, 32), (128, 64), (128, 8), (128, 0), (256, 128), (240, 120)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_both_directions(dtype, hd, pairs, interleaved):
    for weight in (torch.float32, dtype):
        c = Case(hd=hd, pairs=pairs, dtype=dtype, weight=weight, interleaved=interleaved)
        c.forward()
        c.backward()


@pytest.mark.parametrize("t,hq,hk", [(1, 1, 1), (1, 32, 8), (2, 5, 3), (7, 1, 0), (7, 0, 3), (700, 7, 2), (3000, 4, 4), (20000, 1, 1)])
def test_counts(t, hq, hk):
    c = Case(t, hq, hk, hd=128, index=torch.int64)
    c.forward()
    c.backward()


def test_none():
    for t, hq, hk in ((0, 3, 1), (4, 0, 0)):
        c = Case(t, hq, hk)
        q, k = ma.apply_qk_norm_rope(*c.inputs())
        assert q.shape == c.q.shape and k.shape == c.k.shape
        got = ma.apply_qk_norm_rope_backward(c.gq.cuda(), c.gk.cuda(), *c.inputs())
        assert (got[2] == 0).all() and (got[3] == 0).all() and got[0].shape == c.q.shape


@pytest.mark.parametrize("big", [1e-20, 1e-3, 1e4, 1e18])
def test_magnitudes(big):
    """Squares within 32 bits, eps larger and smaller than them; a head of zeros."""
    c = Case(big=big)
    c.q[2, 1] = 0
    c.forward()
    c.backward()
    c.eps = 0.5
    c.forward()
    c.backward()


def test_positions_outside_the_tables():
    c = Case(index=torch.int64)
    c.pos[:4] = torch.tensor([-1, 20, 2**40, -2**40])
    c.forward()
    c.backward()
    c.cos, c.sin = c.cos[:0], c.sin[:0]
    q, _ = ma.apply_qk_norm_rope(*c.inputs())
    plain = ma.apply_qk_norm_rope(*c.inputs()[:5], *(torch.zeros((1, 0), device="cuda"),) * 2)
    assert torch.equal(q, plain[0])


def test_rows_that_are_no_numbers_reach_no_others():
    c = Case(40, 4, 2, hd=128)
    clean = c.forward()
    c.q[3, 1, 7] = float("nan")
    c.k[5, 0, 2] = float("inf")
    got = ma.apply_qk_norm_rope(*c.inputs())
    assert got[0][3, 1].isnan().all() and got[1][5, 0, 2].isnan()
    got[0][3, 1], got[1][5, 0] = clean[0][3, 1], clean[1][5, 0]
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])


def test_strides():
    """Views of one projection, unaligned and transposed tensors, tables that are columns of wider ones."""
    c = Case(33, 4, 2)
    want = c.forward()
    packed = torch.cat((c.q, c.k, c.k), 1).cuda()
    args = c.inputs()
    table = torch.cat((c.cos, c.sin), 1).cuda()
    got = ma.apply_qk_norm_rope(packed[:, :4], packed[:, 4:6], *args[2:5], table[:, :32], table[:, 32:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    odd = torch.zeros((33, 4, 67), dtype=c.dtype if hasattr(c, "dtype") else torch.bfloat16, device="cuda")[..., 3:]
    odd.copy_(args[0])
    across = args[1].transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.stack((args[2], args[2]), 1)[:, 0]
    got = ma.apply_qk_norm_rope(odd, across, wide, args[3], torch.stack((args[4], args[4]), 1)[:, 1], args[5], args[6])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = ma.apply_qk_norm_rope_backward(c.gq.cuda().transpose(0, 1).contiguous().transpose(0, 1), c.gk.cuda(), packed[:, :4], packed[:, 4:6], *args[2:])
    c.check_gradients(g)


@pytest.mark.parametrize("weight", [torch.float32, torch.bfloat16])
def test_autograd(weight):
    c = Case(50, 4, 2, weight=weight)
    args = c.inputs()
    for x in args[:4]:
        x.requires_grad_()
    y = ma.apply_qk_norm_rope(*args)
    with torch.no_grad():
        plain = ma.apply_qk_norm_rope(*args)
    assert all(torch.equal(a, b) and a.requires_grad and not b.requires_grad for a, b in zip(y, plain))
    torch.autograd.backward(y, (c.gq.cuda(), c.gk.cuda()))
    c.check_gradients([x.grad for x in args[:4]])


def test_one_wants_a_gradient_and_one_result_is_used():
    c = Case(20, 3, 3)
    args = c.inputs()
    args[2].requires_grad_()
    _, k = ma.apply_qk_norm_rope(*args)
    q, _ = ma.apply_qk_norm_rope(*args)
    q.sum().backward()  # the gradient that comes in is one number, expanded
    _, _, dw, mw = c.formula(c.q, c.wq, torch.ones_like(c.q))
    c.check(args[2].grad, dw, mw, 2.0**-18)
    shared = torch.ones(64, device="cuda", requires_grad=True)  # one weight for both
    y = ma.apply_qk_norm_rope(args[0], args[1], shared, shared, *args[4:])
    torch.autograd.backward(y, (c.gq.cuda(), c.gk.cuda()))
    one = torch.ones(64)
    parts = [c.formula(x, one, g)[2:] for x, g in ((c.q, c.gq), (c.k, c.gk))]
    c.check(shared.grad, parts[0][0] + parts[1][0], parts[0][1] + parts[1][1], 2.0**-18)


def test_gradient_against_differences():
    """Directional differences of the formula in 64 bits against the gradients of the call."""
    c = Case(6, 2, 1, dtype=torch.float16)
    got = [x.double().cpu() for x in c.backward()]
    g = torch.Generator().manual_seed(3)
    value = lambda q, k, wq, wk: sum((c.formula(x, w)[0] * gy.double()).sum() for x, w, gy in ((q, wq, c.gq), (k, wk, c.gk)))  # noqa: E731
    at = [x.double() for x in (c.q, c.k, c.wq, c.wk)]
    for i in range(4):
        d = torch.randn(at[i].shape, generator=g, dtype=torch.float64)
        up, down = ([x + sign * 1e-5 * d if j == i else x for j, x in enumerate(at)] for sign in (1, -1))
        slope = (value(*up) - value(*down)) / 2e-5
        # float16 gradients are rounded by 2^-11 of themselves each, differences are off by 1e-9 or so
        assert abs((got[i] * d).sum() - slope) <= 2.0**-11 * (got[i] * d).abs().sum() + 1e-6


def test_captured_and_the_same_every_time():
    c = Case(3000, 8, 2, hd=128)
    args = c.inputs()
    grads = (c.gq.cuda(), c.gk.cuda())
    first = ma.apply_qk_norm_rope(*args), ma.apply_qk_norm_rope_backward(*grads, *args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ma.apply_qk_norm_rope(*args), ma.apply_qk_norm_rope_backward(*grads, *args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept = ma.apply_qk_norm_rope(*args), ma.apply_qk_norm_rope_backward(*grads, *args)
    g.replay()
    torch.cuda.synchronize()
    for other in (again, kept):
        assert all(torch.equal(a, b) for x, y in zip(first, other) for a, b in zip(x, y))


def test_the_gradient_has_no_gradient():
    """A graph of the gradient may be asked for; walking it is refused, and the process lives on."""
    c = Case(5, 2, 1)
    args = c.inputs()
    args[0].requires_grad_()
    y = ma.apply_qk_norm_rope(*args)
    (dq,) = torch.autograd.grad(y[0].sum(), args[0], create_graph=True)
    with pytest.raises(RuntimeError, match="no gradient of its own"):
        dq.float().square().sum().backward()
    y = ma.apply_qk_norm_rope(*args)
    with torch.no_grad():
        args[0].zero_()  # what was saved has changed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y[0].sum().backward()


def test_backward_captured():
    """Forward and backward in one graph, as torch captures any: no eager graph of the same leaves lives meanwhile."""
    c = Case(200, 4, 2, hd=128)
    args = c.inputs()
    for x in args[:4]:
        x.requires_grad_()
    grads = (c.gq.cuda(), c.gk.cuda())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = torch.autograd.grad(ma.apply_qk_norm_rope(*args), args[:4], grads)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        kept = torch.autograd.grad(ma.apply_qk_norm_rope(*args), args[:4], grads)
    for x in kept:
        x.zero_()
    g.replay()
    torch.cuda.synchronize()
    c.check_gradients(kept)
    assert all(torch.equal(a, b) for a, b in zip(first, kept))
