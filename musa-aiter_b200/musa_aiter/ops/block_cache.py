"""Block-scaled 8-bit KV caches: the quantising writer and the attention that reads them.

A block-scaled cache keeps keys and values as 8-bit codes in the framework's tile layout,
``[num_blocks, num_heads, head_dim, block_size]`` in ``torch.int8`` or ``torch.float8_e4m3fn``, with
one float32 scale per (block, head) in ``[num_blocks, num_heads]``; a code stands for code * scale.
Unlike the FP8 caches of ``kv_linear_to_paged_fp8`` the scale is not an argument: the writer takes it
from the data, block by block.

Both calls take a sequence's pages from ``block_tables`` (int32 ``[num_seqs, max_blocks]``) and its
length from ``context_lens`` (int32, the tokens of this call included); ``cu_seqlens`` (int32
``[num_seqs + 1]``) says which rows of the packed tensors are whose, None means one row per sequence.
Nothing is read back: block ids outside the cache are skipped by the kernels, as are tokens past
``max_blocks * block_size``.
"""

from __future__ import annotations

import math
import struct
import threading

import torch

from .. import _native
from ..dispatch import emit_native
from ._common import require_cuda

__all__ = ["kv_append_block_scaled", "paged_attention_block_scaled"]

_CODE_TYPES = {torch.int8: 0}
if hasattr(torch, "float8_e4m3fn"):
    _CODE_TYPES[torch.float8_e4m3fn] = 1
_FLOAT_CODES = {torch.float16: _native.MAK_DT_F16, torch.bfloat16: _native.MAK_DT_BF16, torch.float32: _native.MAK_DT_F32}
_HEAD_DIMS = (64, 128, 256)
_BLOCK_SIZES = (16, 32, 64, 128)
_CACHE_DESC = struct.Struct("4Q8q3Q5q4i")  # mak_block_cache_desc
_ATTN_DESC = struct.Struct("4Q8q3Q5q4i4Q5q4ifi")  # mak_block_attn_desc

# Attention workspaces, one per (device, stream): the kernels leave its counters at zero, so calls
# that follow one another on a stream share it.
_WORKSPACES: dict = {}
_WORKSPACE_LOCK = threading.Lock()
_WORKSPACE_BYTES = 0


def _workspace(device: torch.device, stream: int) -> tuple[int, int]:
    global _WORKSPACE_BYTES
    if torch.cuda.is_current_stream_capturing():
        # a graph may be replayed on any stream: it gets a workspace of its own
        ws = torch.empty(_WORKSPACE_BYTES or _workspace_bytes(), dtype=torch.uint8, device=device)
        ws[: 1 << 16].zero_()
        return ws, ws.numel()
    key = (device.index, stream)
    ent = _WORKSPACES.get(key)
    if ent is None:
        with _WORKSPACE_LOCK:
            ent = _WORKSPACES.get(key)
            if ent is None:
                ws = torch.zeros(_workspace_bytes(), dtype=torch.uint8, device=device)
                ent = _WORKSPACES[key] = (ws, ws.numel())
    return ent


def _workspace_bytes() -> int:
    global _WORKSPACE_BYTES
    if not _WORKSPACE_BYTES:
        _WORKSPACE_BYTES = int(_native.load().mak_block_attention_workspace_bytes())
    return _WORKSPACE_BYTES


def _cache_fields(name, rows, num_heads, head_dim, key_cache, value_cache, key_scale, value_scale, block_tables, context_lens, cu_seqlens):
    """Checks of the arguments both calls share; returns mak_block_cache_desc's fields."""
    shape = key_cache.shape
    if len(shape) != 4 or value_cache.shape != shape:
        raise ValueError(f"{name}: key_cache and value_cache must both be [num_blocks, num_heads, head_dim, block_size]")
    nb, nh, hd, bs = shape
    code = _CODE_TYPES.get(key_cache.dtype)
    if code is None or value_cache.dtype != key_cache.dtype:
        raise ValueError(f"{name}: caches must both be int8 or both float8_e4m3fn")
    if hd not in _HEAD_DIMS:
        raise ValueError(f"{name}: head_dim must be one of {_HEAD_DIMS}, got {hd}")
    if bs not in _BLOCK_SIZES:
        raise ValueError(f"{name}: block_size must be one of {_BLOCK_SIZES}, got {bs}")
    if head_dim != hd:
        raise ValueError(f"{name}: rows have head_dim {head_dim}, the cache {hd}")
    ks, vs = key_cache.stride(), value_cache.stride()
    if ks[3] != 1 or ks[2] != bs or vs[3] != 1 or vs[2] != bs:
        raise ValueError(f"{name}: the head_dim and block_size axes of the caches must be contiguous")
    if key_scale.shape != (nb, nh) or value_scale.shape != (nb, nh):
        raise ValueError(f"{name}: scales must be [num_blocks, num_heads]")
    if key_scale.dtype != torch.float32 or value_scale.dtype != torch.float32:
        raise ValueError(f"{name}: scales must be float32")
    if block_tables.dim() != 2 or context_lens.dim() != 1 or block_tables.shape[0] != context_lens.shape[0]:
        raise ValueError(f"{name}: block_tables must be [num_seqs, max_blocks] and context_lens [num_seqs]")
    if block_tables.dtype != torch.int32 or context_lens.dtype != torch.int32:
        raise ValueError(f"{name}: block_tables and context_lens must be int32")
    seqs, width = block_tables.shape
    if width > 1 and block_tables.stride(1) != 1:
        raise ValueError(f"{name}: a block table's row must be contiguous")
    if seqs > 1 and context_lens.stride(0) != 1:
        raise ValueError(f"{name}: context_lens must be contiguous")
    if cu_seqlens is None:
        if rows != seqs:
            raise ValueError(f"{name}: without cu_seqlens every sequence has one row: {rows} rows for {seqs} sequences")
        starts = 0
    else:
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] != seqs + 1 or cu_seqlens.dtype != torch.int32:
            raise ValueError(f"{name}: cu_seqlens must be int32 [num_seqs + 1]")
        if not cu_seqlens.is_contiguous():
            raise ValueError(f"{name}: cu_seqlens must be contiguous")
        starts = cu_seqlens.data_ptr()
    require_cuda(name, key_cache, value_cache, key_scale, value_scale, block_tables, context_lens, cu_seqlens)
    kss, vss = key_scale.stride(), value_scale.stride()
    return (key_cache.data_ptr(), value_cache.data_ptr(), key_scale.data_ptr(), value_scale.data_ptr(),
            ks[0], ks[1], vs[0], vs[1], kss[0], kss[1], vss[0], vss[1],
            block_tables.data_ptr(), context_lens.data_ptr(), starts,
            block_tables.stride(0), nb, seqs, width, rows, nh, hd, bs, code)


def _aligned_rows(x: torch.Tensor) -> torch.Tensor:
    """x [rows, heads, head_dim] with contiguous, 16-byte aligned rows (copied where it has none)."""
    st = x.stride()
    per = 16 // x.element_size()
    if st[2] == 1 and st[0] % per == 0 and st[1] % per == 0 and x.data_ptr() % 16 == 0:
        return x
    return x.contiguous() if not x.is_contiguous() else x.clone()


def kv_append_block_scaled(
    k: torch.Tensor,
    v: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scale: torch.Tensor,
    value_scale: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
) -> None:
    """Quantise ``k`` / ``v`` ``[rows, num_heads, head_dim]`` (float16, bfloat16 or float32) into the last
    positions of their sequences.

    For each block and head that a call writes, and for keys and values apart, m is the largest finite
    magnitude among the values written there (0 when below 2**-100).  A block whose first position the
    call writes gets the scale m / 127 (int8) or m / 448 (float8_e4m3fn), and zeros behind its last
    token; a block that held tokens gets the larger of that and its old scale, and where the scale grows
    its codes are rounded again.  Non-finite values are stored as 0.  A block must belong to one sequence
    of the call only.  In place; returns None."""
    name = "kv_append_block_scaled"
    if k.dim() != 3 or k.shape != v.shape:
        raise ValueError(f"{name}: k and v must both be [rows, num_heads, head_dim]")
    dt = _FLOAT_CODES.get(k.dtype)
    if dt is None or v.dtype != k.dtype:
        raise ValueError(f"{name}: k and v must both be float16, bfloat16 or float32")
    rows, nh, hd = k.shape
    fields = _cache_fields(name, rows, nh, hd, key_cache, value_cache, key_scale, value_scale, block_tables, context_lens, cu_seqlens)
    if fields[20] != nh:
        raise ValueError(f"{name}: rows have {nh} heads, the cache {fields[20]}")
    require_cuda(name, key_cache, k, v)
    k, v = _aligned_rows(k), _aligned_rows(v)
    ks, vs = k.stride(), v.stride()
    rc = _native.load().mak_block_append(_CACHE_DESC.pack(*fields), k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], dt,
                                         _native.stream_ptr(k.device))
    _native.check(rc, name)
    emit_native(name, k, "sm100a block-scaled cache writer")


def paged_attention_block_scaled(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scale: torch.Tensor,
    value_scale: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    causal: bool = True,
    window: int = 0,
    return_lse: bool = False,
    out: torch.Tensor | None = None,
):
    """Attention of ``q`` ``[rows, num_q_heads, head_dim]`` (float16 or bfloat16) over a block-scaled cache.

    Query head h reads cache head h // (num_q_heads // num_heads).  The last rows of a sequence sit at its
    last positions: with ``causal`` a row sees the tokens up to its own, otherwise all of its sequence; a
    ``window`` > 0 (causal only) keeps the last ``window`` of those.  ``scale`` defaults to
    1 / sqrt(head_dim).  Sums and softmax statistics are held in 32 bits.  Returns ``out`` (q's dtype), or
    ``(out, lse)`` with the log of each row's sum of exponentials, float32 ``[rows, num_q_heads]``.  A row
    that sees no token gives zeros and an lse of -inf."""
    name = "paged_attention_block_scaled"
    if q.dim() != 3:
        raise ValueError(f"{name}: q must be [rows, num_q_heads, head_dim]")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{name}: q must be float16 or bfloat16, got {q.dtype}")
    rows, hq, hd = q.shape
    nh = key_cache.shape[1] if key_cache.dim() == 4 else 0
    if nh and hq % nh:
        raise ValueError(f"{name}: {hq} query heads do not divide over {nh} cache heads")
    if window < 0 or (window and not causal):
        raise ValueError(f"{name}: window must be positive or 0 and needs causal=True")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or (out.numel() and out.stride(2) != 1)):
        raise ValueError(f"{name}: out must have q's shape and dtype and contiguous rows")
    fields = _cache_fields(name, rows, nh, hd, key_cache, value_cache, key_scale, value_scale, block_tables, context_lens, cu_seqlens)
    if out is None:
        out = torch.empty((rows, hq, hd), dtype=q.dtype, device=q.device)
    require_cuda(name, key_cache, q, out)
    q = _aligned_rows(q)
    lse = torch.empty((rows, hq), dtype=torch.float32, device=q.device) if return_lse else None
    stream = _native.stream_ptr(q.device)
    ws, nbytes = _workspace(q.device, stream)
    qs, os_ = q.stride(), out.stride()
    desc = _ATTN_DESC.pack(*fields, q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, ws.data_ptr(), nbytes,
                           qs[0], qs[1], os_[0], os_[1], hq, _FLOAT_CODES[q.dtype], 1 if causal else 0, min(int(window), 0x7FFFFFFF),
                           1.0 / math.sqrt(hd) if scale is None else scale, 0)
    _native.check(_native.load().mak_block_attention(desc, stream), name)
    emit_native(name, q, "sm100a block-scaled cache attention")
    return (out, lse) if return_lse else out
