"""Rotary positions with several axes (time, height and width of images and video) for q and k.

A token has one position per axis; ``sections`` says how many of a head's pairs each axis turns.  Serving
applies it before ``kv_append_block_scaled`` or ``copy_to_kv_cache``; ``apply_rope_axes_backward`` is its
gradient.  Angles come as cos / sin tables indexed by position, as in ``apply_rope_to_key_cache``.
"""

from __future__ import annotations

import struct
from typing import Sequence

import torch

from .. import _native
from ..dispatch import emit_native
from ._common import require_cuda

__all__ = ["apply_rope_axes", "apply_rope_axes_backward"]

_HALF_CODES = {torch.float16: _native.MAK_DT_F16, torch.bfloat16: _native.MAK_DT_BF16}
_POS_CODES = {torch.int32: _native.MAK_DT_I32, torch.int64: _native.MAK_DT_I64}
_DESC = struct.Struct("7Q13q10i256s")  # mak_rope_axes_desc
_PAIR_AXES: dict = {}


def _pair_axes(sections: tuple, interleaved_axes: bool) -> bytes:
    """Axis of each pair: the sections one after another, or dealt out in turn (axis 0, 1, 2, 0, ...) while
    a section has pairs left."""
    key = (sections, interleaved_axes)
    got = _PAIR_AXES.get(key)
    if got is None:
        if not interleaved_axes:
            order = [a for a, n in enumerate(sections) for _ in range(n)]
        else:
            left, order = list(sections), []
            while sum(left):
                for a in range(len(left)):
                    if left[a]:
                        left[a] -= 1
                        order.append(a)
        if len(_PAIR_AXES) > 64:
            _PAIR_AXES.clear()
        got = _PAIR_AXES[key] = bytes(order)
    return got


def _rows(x: torch.Tensor) -> torch.Tensor:
    st = x.stride()
    if st[2] == 1 and st[0] % 8 == 0 and st[1] % 8 == 0 and x.data_ptr() % 16 == 0:
        return x
    return x.contiguous() if not x.is_contiguous() else x.clone()


def _run(name, q, k, positions, cos, sin, sections, interleaved, interleaved_axes, inverse):
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"{name}: q and k must be [tokens, heads, head_dim] with the same tokens and head_dim")
    dt = _HALF_CODES.get(q.dtype)
    if dt is None or k.dtype != q.dtype:
        raise ValueError(f"{name}: q and k must both be float16 or both bfloat16")
    tokens, hq, hd = q.shape
    hk = k.shape[1]
    sections = tuple(int(n) for n in sections)
    if not sections or min(sections) < 0:
        raise ValueError(f"{name}: sections must be counts of pairs, one per axis")
    half = sum(sections)
    unit = 4 if interleaved else 8
    if half == 0 or 2 * half > hd or half > 256 or half % unit or hd % 8:
        raise ValueError(f"{name}: sections must add up to a multiple of {unit} pairs, at most head_dim / 2 and 256, got {half} "
                         f"with head_dim {hd} (a multiple of 8)")
    pcode = _POS_CODES.get(positions.dtype)
    if positions.dim() != 2 or positions.shape != (len(sections), tokens) or pcode is None:
        raise ValueError(f"{name}: positions must be int32 or int64 [{len(sections)}, {tokens}]")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != half:
        raise ValueError(f"{name}: cos and sin must both be [max_positions, {half}]")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError(f"{name}: cos and sin must be float32")
    require_cuda(name, q, k, positions, cos, sin)
    q, k = _rows(q), _rows(k)
    if positions.stride(1) != 1 and tokens > 1:
        positions = positions.contiguous()
    if cos.stride(1) != 1 or sin.stride(1) != 1:
        cos, sin = cos.contiguous(), sin.contiguous()
    q_out = torch.empty((tokens, hq, hd), dtype=q.dtype, device=q.device)
    k_out = torch.empty((tokens, hk, hd), dtype=q.dtype, device=q.device)
    qs, ks = q.stride(), k.stride()
    desc = _DESC.pack(q.data_ptr(), k.data_ptr() if hk else 0, q_out.data_ptr(), k_out.data_ptr(), positions.data_ptr(),
                      cos.data_ptr(), sin.data_ptr(), tokens, cos.shape[0], qs[0], qs[1], ks[0], ks[1], hq * hd, hd, hk * hd, hd,
                      positions.stride(0), cos.stride(0), sin.stride(0), hq, hk, hd, 2 * half, dt, pcode, len(sections),
                      1 if interleaved else 0, 1 if inverse else 0, 0, _pair_axes(sections, bool(interleaved_axes)))
    _native.check(_native.load().mak_rope_axes(desc, _native.stream_ptr(q.device)), name)
    emit_native(name, q, "sm100a rotary positions with several axes")
    return q_out, k_out


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
    and rounded once.  A pair whose position lies outside the tables stays as it is.  Returns new tensors."""
    return _run("apply_rope_axes", q, k, positions, cos, sin, sections, interleaved, interleaved_axes, False)


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
    return _run("apply_rope_axes_backward", grad_q, grad_k, positions, cos, sin, sections, interleaved, interleaved_axes, True)
