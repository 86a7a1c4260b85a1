"""Rotary positions with several axes (time, height and width of images and video) for q and k.

A token has one position per axis; ``sections`` says how many of a head's pairs each axis turns.  Serving
applies it before ``kv_append_block_scaled`` or ``copy_to_kv_cache``; ``apply_rope_axes_backward`` is its
gradient, which autograd also takes where q or k requires one.  Angles come as cos / sin tables indexed by position, as in ``apply_rope_to_key_cache``.
"""

from __future__ import annotations

from typing import Sequence

import torch

from .. import _native

__all__ = ["apply_rope_axes", "apply_rope_axes_backward"]


class _Rotation(torch.autograd.Function):
    """The rotation is linear in q and k: its gradient is the rotation by the negative angles, and so on.

    The native call answers None where q or k wants a gradient; here it is made again with gradients off."""

    @staticmethod
    def forward(ctx, q, k, positions, cos, sin, sections, interleaved, interleaved_axes, inverse):
        ctx.save_for_backward(positions, cos, sin)
        ctx.how = (tuple(sections), interleaved, interleaved_axes)
        ctx.inverse = inverse
        return _native.front().rope(q, k, positions, cos, sin, sections, interleaved, interleaved_axes, inverse)

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        args = (grad_q, grad_k, *ctx.saved_tensors, *ctx.how, not ctx.inverse)
        return (*(_native.front().rope(*args) or _Rotation.apply(*args)), *(None,) * 7)


def apply_rope_axes(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    sections: Sequence[int],
    *,
    interleaved: bool = False,
    interleaved_axes: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotate ``q`` / ``k`` ``[tokens, heads, head_dim]`` by ``positions`` ``[axes, tokens]``.

    Pair j is (j, j + rot / 2), or (2 j, 2 j + 1) with ``interleaved``, of the first rot = 2 * sum(sections)
    columns; the others are copied.  Its angle is row positions[axis(j), t], column j of the tables; axes
    take their pairs one section after another, or in turn with ``interleaved_axes``.  Computed in 32 bits
    and rounded once.  A pair whose position lies outside the tables stays as it is.  Returns new tensors,
    through which q and k get their gradients; cos and sin get none and may not require one.  There is no
    forward-mode derivative: a tensor that carries a tangent is refused."""
    args = (q, k, positions, cos, sin, sections, interleaved, interleaved_axes, False)
    return _native.front().rope(*args) or _Rotation.apply(*args)


def apply_rope_axes_backward(
    grad_q: torch.Tensor,
    grad_k: torch.Tensor,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    sections: Sequence[int],
    *,
    interleaved: bool = False,
    interleaved_axes: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The gradient of ``apply_rope_axes`` in q and k from that of its outputs: the rotation by the negative
    angles."""
    args = (grad_q, grad_k, positions, cos, sin, sections, interleaved, interleaved_axes, True)
    return _native.front().rope(*args) or _Rotation.apply(*args)
