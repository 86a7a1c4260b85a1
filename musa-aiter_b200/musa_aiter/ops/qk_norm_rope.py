"""Norms of queries and keys for each head, with the position rotation in the same pass, and their gradient.

Between the projection and the cache of a layer that normalises q and k: one pass over both instead of two norms and a
rotation.  Angles come as cos / sin tables indexed by position, as in ``apply_rope_axes``.
"""

from __future__ import annotations

import torch

from .. import _native

__all__ = ["apply_qk_norm_rope", "apply_qk_norm_rope_backward"]


def apply_qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Each head of ``q`` / ``k`` ``[tokens, heads, head_dim]``: x / sqrt(mean(x^2) + eps) * weight, then rotated.

    Weights are ``[head_dim]``, float32 or of q's type; ``positions`` int32 or int64 ``[tokens]``; the tables float32
    ``[max_positions, pairs]``.  Pair j is (j, j + pairs), or (2 j, 2 j + 1) with ``interleaved``, of the first 2 * pairs
    columns; the others are normalised alone, and so is a token whose position lies outside the tables.  head_dim is a
    multiple of 16 up to 256, pairs a multiple of 8.  Computed in 32 bits (a head whose sum of squares is past their range
    gives zeros) and rounded once.  Returns new tensors, through which q, k and the weights get their gradients (these
    have none of their own); cos and sin get none and may not require one.  There is no forward-mode derivative: a tensor
    that carries a tangent is refused.  A backward pass is captured into a CUDA graph like any of torch's: no eager graph
    of the same leaves may live meanwhile."""
    return _native.front().norm(q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved)


def apply_qk_norm_rope_backward(
    grad_q: torch.Tensor,
    grad_k: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients of ``apply_qk_norm_rope`` in q, k and the two weights from those of its outputs (no gradient
    flows through this call).  The weights' are summed in 32 bits in a fixed order."""
    return _native.front().norm_back(grad_q, grad_k, q, k, q_weight, k_weight, positions, cos, sin, eps, interleaved)
