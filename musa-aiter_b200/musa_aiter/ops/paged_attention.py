"""Attention over paged 16-bit caches: with a sliding window and first tokens that stay visible, for trees of drafted
tokens, and the weight that each cached token gathers.

A cache is a layer of the LMCache or SGLang formats, ``[num_blocks, block_size, num_heads, head_dim]`` in float16 or
bfloat16 with any strides that keep head_dim contiguous and rows on 16 bytes (``cache[0]`` and ``cache[1]`` of an LMCache
layer as they are); head_dim is 64 or 128, block_size 16, 32, 64 or 128.  The calls take a sequence's pages from
``block_tables`` (int32 ``[num_seqs, max_blocks]``) and its length from ``context_lens`` (int32, the tokens of this call
included); ``cu_seqlens`` (int32 ``[num_seqs + 1]``) says which rows of the packed tensors are whose, None means one row per
sequence.  The last rows of a sequence sit at its last positions.  Rows that belong to no sequence are neither read nor
written.  Nothing is read back: block ids outside the cache are skipped by the kernels, as are tokens past
``max_blocks * block_size`` (rows keep the positions that ``context_lens`` gives them).

Query head h reads cache head h // (num_q_heads // num_heads).  ``scale`` defaults to 1 / sqrt(head_dim) and must be
finite.  For inference: no gradient flows through these calls.
"""

from __future__ import annotations

import torch

from .. import _native

__all__ = ["paged_attention_tree", "paged_attention_weights", "paged_attention_window"]


def paged_attention_window(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    *,
    window: int = 0,
    sinks: int = 0,
    scale: float | None = None,
    return_lse: bool = False,
    out: torch.Tensor | None = None,
):
    """Causal attention of ``q`` ``[rows, num_q_heads, head_dim]`` (the cache's type) over a paged cache.

    A row at position p sees the tokens t <= p; with ``window`` > 0 only those with t > p - window, and the first
    ``sinks`` tokens.  Returns ``out`` (q's dtype), or ``(out, lse)`` with the log of each row's sum of exponentials,
    float32 ``[rows, num_q_heads]``.  A row that sees no token gives zeros and an lse of -inf.  Nothing that a row does not
    see reaches its result, NaN among it.  A workspace of 39 MiB is kept per device and stream until the process
    ends; a call captured in a graph has one of its own."""
    return _native.front().paged(q, key_cache, value_cache, block_tables, context_lens, cu_seqlens, None, window, sinks, scale,
                                 return_lse, out)


def paged_attention_tree(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    parents: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    return_lse: bool = False,
    out: torch.Tensor | None = None,
):
    """Attention of trees of drafted tokens, all branches in one call.

    The rows of a sequence are its drafted tokens, in the cache at its last positions in the same order.  ``parents``
    (int32 ``[rows]``) gives the index, within its sequence, of the row that each one continues; it must be an earlier
    row, and anything else means the last token before the tree.  A row sees the tokens before the tree, itself, its parent, that
    one's parent and so on.  The rest is as in ``paged_attention_window``."""
    if parents is None:
        raise ValueError("paged_attention_tree: parents must be a tensor")
    return _native.front().paged(q, key_cache, value_cache, block_tables, context_lens, cu_seqlens, parents, 0, 0, scale, return_lse,
                                 out)


def paged_attention_weights(
    q: torch.Tensor,
    key_cache: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    lse: torch.Tensor,
    sums: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    *,
    rows: torch.Tensor | None = None,
    window: int = 0,
    sinks: int = 0,
    scale: float | None = None,
    accumulate: bool = True,
) -> None:
    """Add the attention weights of a call to what each cached token has gathered, for ``kv_pages_evict``.

    ``sums[row, h, t]`` (float32 ``[rows of sums, num_heads, max_tokens]``, changed in place) gets the sum over the rows of
    the sequence that see token t, and over the query heads of cache head h, of exp(scale * q . k_t - lse), with the
    ``lse`` that ``paged_attention_window`` returned for the same arguments.  ``rows`` (int32 ``[num_seqs]``, distinct)
    says which row of sums is whose, None means each sequence's own number; a number out of range means none.  Without
    ``accumulate`` the rows are written instead, with zeros where no row sees.  Tokens from max_tokens on have no
    place.  Each place has one writer, so results do not depend on timing."""
    _native.front().weights(q, key_cache, block_tables, context_lens, lse, sums, cu_seqlens, rows, window, sinks, scale, accumulate)
