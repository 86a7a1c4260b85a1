"""Pages of a KV cache: growing, forking, freeing, compacting and copying them on the device.

A pool of pages is described by three int32 tensors that live on the GPU and are changed in place:
``block_tables`` ``[rows, max_blocks]`` (page ids of each sequence in order, -1 = none),
``context_lens`` ``[rows]`` (its tokens) and ``ref_counts`` ``[num_pages]`` (how many rows hold a page,
0 = free).  The page data lives in ``planes``: any tensors whose first axis is the page (codes, scales,
16-bit caches, every layer's), each page contiguous.  New pages are the free ones of lowest index, given
out in the order of the requests, so results do not depend on timing.  No call reads back; rows and page
ids out of range are skipped.
"""

from __future__ import annotations

import ctypes
import struct
from typing import Sequence

import torch

from .. import _native
from ..dispatch import emit_native
from ._common import require_cuda

__all__ = ["kv_pages_compact", "kv_pages_copy", "kv_pages_fork", "kv_pages_free", "kv_pages_grow"]

_PAGES_DESC = struct.Struct("3Q5q")  # mak_pages_desc


def _index(name: str, what: str, x: torch.Tensor, dim: int = 1) -> None:
    if x.dim() != dim or x.dtype != torch.int32:
        raise ValueError(f"{name}: {what} must be an int32 tensor of {dim} dimension{'s' if dim > 1 else ''}")
    if x.numel() > 1 and x.shape[-1] > 1 and x.stride(-1) != 1:
        raise ValueError(f"{name}: {what} must be contiguous")


def _pool(name, block_tables, context_lens, ref_counts, block_size) -> bytes:
    _index(name, "block_tables", block_tables, 2)
    _index(name, "ref_counts", ref_counts)
    if context_lens is not None:
        _index(name, "context_lens", context_lens)
        if context_lens.shape[0] != block_tables.shape[0]:
            raise ValueError(f"{name}: context_lens must have one entry per row of block_tables")
    if block_size <= 0:
        raise ValueError(f"{name}: block_size must be positive")
    rows, width = block_tables.shape
    return _PAGES_DESC.pack(block_tables.data_ptr(), context_lens.data_ptr() if context_lens is not None else 0,
                            ref_counts.data_ptr(), block_tables.stride(0), rows, width, ref_counts.shape[0], block_size)


class _Planes(ctypes.Structure):
    _fields_ = [("ptrs", ctypes.c_void_p), ("strides", ctypes.c_void_p), ("sizes", ctypes.c_void_p), ("num", ctypes.c_int64)]


def _planes(name: str, planes: Sequence[torch.Tensor], pages: int, *others: torch.Tensor):
    """mak_pages_planes of the tensors, and the arrays it points into."""
    n = len(planes)
    ptrs, strides, sizes = [], [], []
    for t in planes:
        shape = t.shape
        if len(shape) == 0 or shape[0] != pages:
            raise ValueError(f"{name}: every plane's first axis must have {pages} pages")
        size = t.element_size()
        per = t.numel() // pages if pages else 0
        st = t.stride()
        if not t.is_contiguous():
            want = 1
            for d in range(len(shape) - 1, 0, -1):
                if shape[d] != 1 and st[d] != want:
                    raise ValueError(f"{name}: a page of a plane must be contiguous")
                want *= shape[d]
            if st[0] < per:
                raise ValueError(f"{name}: pages of a plane must not overlap")
        ptrs.append(t.data_ptr())
        strides.append((st[0] if pages > 1 else per) * size)
        sizes.append(per * size)
    require_cuda(name, *others, *planes)
    words = (ctypes.c_int64 * (3 * n + 1))(*ptrs, *strides, *sizes)
    at = ctypes.addressof(words)
    return _Planes(at, at + 8 * n, at + 16 * n, n), words


def kv_pages_copy(planes: Sequence[torch.Tensor], src_pages: torch.Tensor, dst_pages: torch.Tensor) -> None:
    """Copy page ``src_pages[i]`` to page ``dst_pages[i]`` within every plane, all planes in one launch.

    Pairs with an id out of range are skipped.  Destinations must be distinct and none may be a source."""
    name = "kv_pages_copy"
    _index(name, "src_pages", src_pages)
    _index(name, "dst_pages", dst_pages)
    if src_pages.shape != dst_pages.shape:
        raise ValueError(f"{name}: src_pages and dst_pages must have the same length")
    if not planes:
        return
    pages = planes[0].shape[0] if planes[0].dim() else 0
    desc, keep = _planes(name, planes, pages, src_pages, dst_pages)
    rc = _native.load().mak_pages_copy(ctypes.byref(desc), pages, src_pages.data_ptr(), dst_pages.data_ptr(), src_pages.shape[0],
                                       _native.stream_ptr(src_pages.device))
    _native.check(rc, name)
    emit_native(name, src_pages, "sm100a page copy")


def kv_pages_fork(
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    parents: torch.Tensor,
    children: torch.Tensor,
    ref_counts: torch.Tensor,
    planes: Sequence[torch.Tensor],
    block_size: int,
) -> torch.Tensor:
    """Make row ``children[i]`` a continuation of row ``parents[i]``: full pages are shared (their counts
    grow), a part-filled last page is copied into a new one.

    Children must be empty rows (freed or never used), distinct, and no parents.  Returns an int32 ``[1]``
    tensor on the device: how many children found no free page; those end at their last full page."""
    name = "kv_pages_fork"
    pool = _pool(name, block_tables, context_lens, ref_counts, block_size)
    _index(name, "parents", parents)
    _index(name, "children", children)
    n = parents.shape[0]
    if children.shape[0] != n:
        raise ValueError(f"{name}: parents and children must have the same length")
    desc, keep = _planes(name, planes, ref_counts.shape[0], block_tables, context_lens, parents, children, ref_counts)
    scratch = torch.empty(2 * n + 3, dtype=torch.int32, device=block_tables.device)
    missing = torch.empty(1, dtype=torch.int32, device=block_tables.device)
    rc = _native.load().mak_pages_fork(pool, ctypes.byref(desc), parents.data_ptr(), children.data_ptr(), n, missing.data_ptr(),
                                       scratch.data_ptr(), _native.stream_ptr(block_tables.device))
    _native.check(rc, name)
    emit_native(name, block_tables, "sm100a page fork")
    return missing


def kv_pages_grow(
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    rows: torch.Tensor,
    new_tokens: torch.Tensor,
    ref_counts: torch.Tensor,
    block_size: int,
) -> torch.Tensor:
    """Make room for ``new_tokens[i]`` more tokens in row ``rows[i]`` (distinct rows): pages are added to
    its table and its length grows.

    Returns an int32 ``[1]`` tensor on the device: how many tokens found no place (the pool or the row's
    table was full); their rows end where their pages do."""
    name = "kv_pages_grow"
    pool = _pool(name, block_tables, context_lens, ref_counts, block_size)
    _index(name, "rows", rows)
    _index(name, "new_tokens", new_tokens)
    if rows.shape != new_tokens.shape:
        raise ValueError(f"{name}: rows and new_tokens must have the same length")
    require_cuda(name, block_tables, context_lens, rows, new_tokens, ref_counts)
    missing = torch.empty(1, dtype=torch.int32, device=block_tables.device)
    rc = _native.load().mak_pages_grow(pool, rows.data_ptr(), new_tokens.data_ptr(), rows.shape[0], missing.data_ptr(),
                                       _native.stream_ptr(block_tables.device))
    _native.check(rc, name)
    emit_native(name, block_tables, "sm100a page growth")
    return missing


def kv_pages_free(block_tables: torch.Tensor, context_lens: torch.Tensor, rows: torch.Tensor, ref_counts: torch.Tensor) -> None:
    """Empty ``rows``: each page they hold loses one reference, their entries become -1, their lengths 0."""
    name = "kv_pages_free"
    pool = _pool(name, block_tables, context_lens, ref_counts, 1)
    _index(name, "rows", rows)
    require_cuda(name, block_tables, context_lens, rows, ref_counts)
    rc = _native.load().mak_pages_free(pool, rows.data_ptr(), rows.shape[0], _native.stream_ptr(block_tables.device))
    _native.check(rc, name)
    emit_native(name, block_tables, "sm100a page release")


def kv_pages_compact(block_tables: torch.Tensor, ref_counts: torch.Tensor, planes: Sequence[torch.Tensor]) -> torch.Tensor:
    """Move the pages in use to the lowest indexes, with tables and counts.

    Pages already among the first ``live`` stay; the others go to the holes there, in index order.  What
    lies behind is left as it was.  Returns ``live`` as an int32 ``[1]`` tensor on the device."""
    name = "kv_pages_compact"
    pool = _pool(name, block_tables, None, ref_counts, 1)
    pages = ref_counts.shape[0]
    desc, keep = _planes(name, planes, pages, block_tables, ref_counts)
    scratch = torch.empty(3 * pages + 2, dtype=torch.int32, device=block_tables.device)
    live = torch.empty(1, dtype=torch.int32, device=block_tables.device)
    rc = _native.load().mak_pages_compact(pool, ctypes.byref(desc), live.data_ptr(), scratch.data_ptr(),
                                          _native.stream_ptr(block_tables.device))
    _native.check(rc, name)
    emit_native(name, block_tables, "sm100a page compaction")
    return live
