"""Gradients that carry a tangent (forward over reverse) are refused by the backward pass, in which the tangent would be lost."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import musa_aiter as ma

pytestmark = pytest.mark.gpu


def test_norms_refuse_gradients_with_tangents():
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn((5, h, 64), generator=g).to(torch.bfloat16).cuda() for h in (4, 2))
    weight = torch.ones(64, device="cuda")
    cos = sin = torch.full((9, 32), 0.5**0.5, device="cuda")
    at = torch.arange(5, dtype=torch.int32, device="cuda")
    q.requires_grad_()
    out, _ = ma.apply_qk_norm_rope(q, k, weight, weight, at, cos, sin)
    grad = torch.ones_like(out)
    plain, = torch.autograd.grad(out, q, grad, retain_graph=True)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            torch.autograd.grad(out, q, forward_ad.make_dual(grad, grad), retain_graph=True)
        with pytest.raises(ValueError, match="tangent"):
            ma.apply_qk_norm_rope(forward_ad.make_dual(q.detach(), grad), k, weight, weight, at, cos, sin)
        again, = torch.autograd.grad(out, q, grad)
    assert torch.equal(plain, again)


def test_rotations_refuse_gradients_with_tangents():
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn((5, h, 64), generator=g).to(torch.bfloat16).cuda() for h in (4, 2))
    where = (torch.arange(5, dtype=torch.int32, device="cuda")[None], *(torch.full((9, 32), 0.5**0.5, device="cuda"),) * 2, (32,))
    q.requires_grad_()
    out, _ = ma.apply_rope_axes(q, k, *where)
    grad = torch.ones_like(out)
    plain, = torch.autograd.grad(out, q, grad, retain_graph=True)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            torch.autograd.grad(out, q, forward_ad.make_dual(grad, grad), retain_graph=True)
        again, = torch.autograd.grad(out, q, grad)
    assert torch.equal(plain, again)
