"""A tensor that carries a tangent (forward-mode differentiation) is refused where a gradient is otherwise taken: the tangent would
be lost in silence.  On CPU tensors: the refusal comes before the device is asked."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import musa_aiter as ma

NAMES = ("q", "k", "q_weight", "k_weight", "cos", "sin")


def norm(change):
    a = dict(q=torch.zeros((3, 2, 64), dtype=torch.float16), k=torch.zeros((3, 1, 64), dtype=torch.float16), q_weight=torch.ones(64),
             k_weight=torch.ones(64), positions=torch.zeros(3, dtype=torch.int32), cos=torch.zeros((5, 32)), sin=torch.zeros((5, 32)))
    for name, f in change.items():
        a[name] = f(a[name])
    return ma.apply_qk_norm_rope(**a)


def dual(x):
    return forward_ad.make_dual(x, torch.ones_like(x))


@pytest.mark.parametrize("name", NAMES)
def test_norms(name):
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="apply_qk_norm_rope: .*tangent"):
            norm({name: dual})
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):  # switches off the other mode alone
            norm({name: dual})
        with pytest.raises(ValueError, match="tangent"):
            norm({name: dual, "k": lambda k: k.clone().requires_grad_()} if name != "k" else {name: dual})
        with pytest.raises(RuntimeError, match="no CPU fallback"):  # a level without tangents changes nothing
            norm({})
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="no CPU fallback"):
            norm({name: dual})


@pytest.mark.parametrize("name", ("q", "k", "cos", "sin"))
@pytest.mark.parametrize("backward", [False, True])
def test_rotations(backward, name):
    a = dict(q=torch.zeros((3, 2, 64), dtype=torch.float16), k=torch.zeros((3, 1, 64), dtype=torch.float16), cos=torch.zeros((5, 32)),
             sin=torch.zeros((5, 32)))

    def call():
        where = (torch.zeros((1, 3), dtype=torch.int32), a["cos"], a["sin"], (32,))
        return (ma.apply_rope_axes_backward if backward else ma.apply_rope_axes)(a["q"], a["k"], *where)

    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
        a[name] = dual(a[name])
        with pytest.raises(ValueError, match="apply_rope_axes.*tangent"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
            call()
