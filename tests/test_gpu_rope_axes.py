"""Rotary positions with several axes against the rotation in 64 bits.

Bound: products and the sum are 32-bit (relative 2^-23 of |x1| + |x2|), the result is rounded once to
q's type (relative 2^-8 or 2^-11)."""

from __future__ import annotations

import pytest
import torch

import musa_aiter as ma

pytestmark = pytest.mark.gpu


def axes_of(sections, dealt):
    if not dealt:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, got = list(sections), []
    while sum(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                got.append(a)
    return got


def reference(x, pos, cos, sin, sections, interleaved, dealt, sign):
    half = sum(sections)
    axes = axes_of(sections, dealt)
    y = x.double().clone()
    for j in range(half):
        i1, i2 = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        p = pos[axes[j]].long()
        ok = (p >= 0) & (p < cos.shape[0])
        p = p.clamp(0, cos.shape[0] - 1)
        c = torch.where(ok, cos[p, j].double(), torch.ones((), dtype=torch.float64))[:, None]
        s = torch.where(ok, sin[p, j].double(), torch.zeros((), dtype=torch.float64))[:, None] * sign
        a, b = x[..., i1].double(), x[..., i2].double()
        y[..., i1], y[..., i2] = a * c - b * s, a * s + b * c
    return y


def tables(n, half, g):
    angle = torch.rand((n, half), generator=g) * 20
    return angle.cos(), angle.sin()


def near(got, want, x):
    u = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -11
    big = x.double().abs().amax(-1, keepdim=True) * 2
    return bool(((got.double().cpu() - want).abs() <= u * want.abs() + 2.0 ** -22 * big + 2.0 ** -25).all())


CASES = [  # tokens, q heads, k heads, head_dim, sections, interleaved, dealt out
    (1, 4, 2, 128, (16, 24, 24), False, False),
    (7, 32, 8, 128, (16, 24, 24), False, True),
    (33, 5, 1, 64, (5, 11), False, False),
    (100, 3, 3, 128, (9, 12, 11), True, False),
    (64, 8, 2, 256, (128,), False, False),
    (19, 2, 2, 80, (8, 8, 8), True, True),
    (2000, 32, 8, 128, (16, 24, 24), False, False),
    (50, 1, 7, 72, (32,), False, False),
    (3000, 16, 16, 64, (1, 2, 29), True, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rotation_and_gradient(case, dtype):
    t, hq, hk, hd, sections, inter, dealt = case
    g = torch.Generator().manual_seed(t)
    q, k = torch.randn((t, hq, hd), generator=g).to(dtype), torch.randn((t, hk, hd), generator=g).to(dtype)
    cos, sin = tables(500, sum(sections), g)
    pos = torch.randint(0, 500, (len(sections), t), generator=g, dtype=torch.int64 if t % 2 else torch.int32)
    for f, sign in ((ma.apply_rope_axes, 1.0), (ma.apply_rope_axes_backward, -1.0)):
        got = f(q.cuda(), k.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), sections, interleaved=inter, interleaved_axes=dealt)
        for x, y in zip((q, k), got):
            assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
            assert near(y, reference(x, pos, cos, sin, sections, inter, dealt, sign), x)


def test_positions_outside_the_table_keep_their_pairs():
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn((5, 2, 64), generator=g).half(), torch.randn((5, 1, 64), generator=g).half()
    cos, sin = tables(10, 32, g)
    pos = torch.tensor([[0, 10, -1, 9, 1 << 30], [3, 3, 3, -(1 << 31), 3]], dtype=torch.int32)
    got = ma.apply_rope_axes(q.cuda(), k.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), (16, 16))
    for x, y in zip((q, k), got):
        assert near(y, reference(x, pos, cos, sin, (16, 16), False, False, 1.0), x)


def test_strides():
    g = torch.Generator().manual_seed(2)
    packed = torch.randn((9, 12, 136), generator=g).to(torch.bfloat16)
    q, k = packed[:, :8, :128], packed[:, 8:10, :128]
    odd = torch.randn((9, 2, 130), generator=g).to(torch.bfloat16)[..., 1:129]  # rows that are not 16-byte aligned
    cos, sin = tables(40, 64, g)
    pos = torch.randint(0, 40, (9, 3), generator=g).t()
    wide = torch.cat((cos, sin), 1).cuda()
    dev = packed.cuda()
    got = ma.apply_rope_axes(dev[:, :8, :128], dev[:, 8:10, :128], pos.cuda(), wide[:, :64], wide[:, 64:], (16, 24, 24))
    for x, y in zip((q, k), got):
        assert near(y, reference(x, pos, cos, sin, (16, 24, 24), False, False, 1.0), x)
    got = ma.apply_rope_axes(dev[:, :8, :128], odd.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), (16, 24, 24))
    assert near(got[1], reference(odd, pos, cos, sin, (16, 24, 24), False, False, 1.0), odd)


def test_one_position_for_all_axes_is_plain_rope():
    """With the same position along every axis the call is apply_rope up to that one's roundings."""
    g = torch.Generator().manual_seed(3)
    q = torch.randn((12, 4, 64), generator=g).half().cuda()
    cos, sin = (x.cuda() for x in tables(30, 32, g))
    pos = torch.randint(0, 30, (12,), generator=g).cuda()
    got, _ = ma.apply_rope_axes(q, q, pos[None].expand(3, 12), cos, sin, (10, 11, 11))
    want = ma.apply_rope(q, cos[pos][:, None], sin[pos][:, None])
    assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -10 * float(q.abs().max()) * 2


def test_gradient_against_differences():
    """d/dx of sum(w * rope(x)) by central differences of the reference rotation in 64 bits."""
    g = torch.Generator().manual_seed(4)
    sections, inter = (3, 2, 3), True
    x = torch.randn((2, 1, 16), generator=g).half()
    w = torch.randn((2, 1, 16), generator=g).half()
    cos, sin = tables(8, 8, g)
    pos = torch.randint(0, 8, (3, 2), generator=g)
    grad, _ = ma.apply_rope_axes_backward(w.cuda(), w.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), sections, interleaved=inter)
    eps = 1e-3
    for i in range(x.numel()):
        d = torch.zeros(x.numel(), dtype=torch.float64)
        d[i] = eps
        up = reference(x.double() + d.view_as(x), pos, cos, sin, sections, inter, False, 1.0)
        down = reference(x.double() - d.view_as(x), pos, cos, sin, sections, inter, False, 1.0)
        want = float((w.double() * (up - down)).sum()) / (2 * eps)
        assert abs(float(grad.reshape(-1)[i]) - want) <= 2.0 ** -11 * abs(want) + 1e-6


def test_no_tokens():
    e = torch.empty((0, 4, 64), dtype=torch.float16, device="cuda")
    cos = torch.ones((4, 32), device="cuda")
    a, b = ma.apply_rope_axes(e, e, torch.zeros((2, 0), dtype=torch.int32, device="cuda"), cos, cos, (16, 16))
    assert a.shape == e.shape and b.shape == e.shape
