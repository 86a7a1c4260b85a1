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

from typing import Sequence

import torch

from .. import _native

__all__ = ["kv_pages_compact", "kv_pages_copy", "kv_pages_fork", "kv_pages_free", "kv_pages_grow"]


def kv_pages_copy(planes: Sequence[torch.Tensor], src_pages: torch.Tensor, dst_pages: torch.Tensor) -> None:
    """Copy page ``src_pages[i]`` to page ``dst_pages[i]`` within every plane, all planes in one launch.

    Pairs with an id out of range are skipped.  Destinations must be distinct and none may be a source."""
    _native.front().copy(planes, src_pages, dst_pages)


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
    return _native.front().fork(block_tables, context_lens, parents, children, ref_counts, planes, block_size)


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
    return _native.front().grow(block_tables, context_lens, rows, new_tokens, ref_counts, block_size)


def kv_pages_free(block_tables: torch.Tensor, context_lens: torch.Tensor, rows: torch.Tensor, ref_counts: torch.Tensor) -> None:
    """Empty ``rows``: each page they hold loses one reference, their entries become -1, their lengths 0."""
    _native.front().free(block_tables, context_lens, rows, ref_counts)


def kv_pages_compact(block_tables: torch.Tensor, ref_counts: torch.Tensor, planes: Sequence[torch.Tensor]) -> torch.Tensor:
    """Move the pages in use to the lowest indexes, with tables and counts.

    Pages already among the first ``live`` stay; the others go to the holes there, in index order.  What
    lies behind is left as it was.  Returns ``live`` as an int32 ``[1]`` tensor on the device."""
    return _native.front().compact(block_tables, ref_counts, planes)
