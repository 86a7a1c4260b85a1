"""Gradients of the rotation with several axes as a model takes them, through autograd."""

from __future__ import annotations

import pytest
import torch

import musa_aiter as ma

from .test_gpu_rope_axes import near, reference, tables

pytestmark = pytest.mark.gpu


def inputs(dtype, t=9, hq=4, hk=2, hd=64):
    g = torch.Generator().manual_seed(t)
    q, k, gq, gk = (torch.randn((t, h, hd), generator=g).to(dtype) for h in (hq, hk, hq, hk))
    cos, sin = tables(20, hd // 2, g)
    pos = torch.randint(0, 20, (2, t), generator=g)
    return q, k, gq, gk, pos, cos, sin, (hd // 4, hd // 4)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_reach_q_and_k(dtype, interleaved):
    q, k, gq, gk, pos, cos, sin, sections = inputs(dtype)
    dq, dk = (x.cuda().requires_grad_() for x in (q, k))
    oq, ok = ma.apply_rope_axes(dq, dk, pos.cuda(), cos.cuda(), sin.cuda(), sections, interleaved=interleaved)
    with torch.no_grad():
        pq, pk = ma.apply_rope_axes(dq, dk, pos.cuda(), cos.cuda(), sin.cuda(), sections, interleaved=interleaved)
    assert torch.equal(oq, pq) and torch.equal(ok, pk) and not pq.requires_grad
    torch.autograd.backward((oq, ok), (gq.cuda(), gk.cuda()))
    for got, x in ((dq.grad, gq), (dk.grad, gk)):
        assert near(got, reference(x, pos, cos, sin, sections, interleaved, False, -1.0), x)


def test_one_of_the_two_alone_and_a_broadcast_gradient():
    q, k, _, _, pos, cos, sin, sections = inputs(torch.float16)
    dq = q.cuda().requires_grad_()
    oq, ok = ma.apply_rope_axes(dq, k.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), sections)
    oq.sum().backward()  # the gradient that comes in is one number, expanded
    assert near(dq.grad, reference(torch.ones_like(q), pos, cos, sin, sections, False, False, -1.0), torch.ones_like(q))
    dk = k.cuda().requires_grad_()
    _, ok = ma.apply_rope_axes(q.cuda(), dk, pos.cuda(), cos.cuda(), sin.cuda(), sections)
    ok[2:5].sum().backward()  # and none for q's result
    ones = torch.zeros_like(k)
    ones[2:5] = 1
    assert near(dk.grad, reference(ones, pos, cos, sin, sections, False, False, -1.0), ones)


def test_the_gradient_of_a_projection_and_of_a_gradient():
    """Views of one projection, as a layer has them; and the gradient call itself is differentiable."""
    q, k, gq, gk, pos, cos, sin, sections = inputs(torch.bfloat16)
    packed = torch.cat((q, k), 1).cuda().requires_grad_()
    oq, ok = ma.apply_rope_axes(packed[:, :4], packed[:, 4:], pos.cuda(), cos.cuda(), sin.cuda(), sections)
    torch.autograd.backward((oq, ok), (gq.cuda(), gk.cuda()))
    both = torch.cat((gq, gk), 1)
    assert near(packed.grad, reference(both, pos, cos, sin, sections, False, False, -1.0), both)
    dq = gq.cuda().requires_grad_()
    back, _ = ma.apply_rope_axes_backward(dq, gk.cuda(), pos.cuda(), cos.cuda(), sin.cuda(), sections)
    back.backward(q.cuda())
    assert near(dq.grad, reference(q, pos, cos, sin, sections, False, False, 1.0), q)


def test_tables_that_require_a_gradient_are_refused():
    q, k, _, _, pos, cos, sin, sections = inputs(torch.float16)
    with pytest.raises(ValueError, match="cos and sin are tables"):
        ma.apply_rope_axes(q.cuda(), k.cuda(), pos.cuda(), cos.cuda().requires_grad_(), sin.cuda(), sections)
