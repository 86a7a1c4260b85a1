"""Block-scaled 8-bit KV caches: the quantising writer and the attention that reads them.

A block-scaled cache keeps keys and values as 8-bit codes in the framework's tile layout,
``[num_blocks, num_heads, head_dim, block_size]`` in ``torch.int8`` or ``torch.float8_e4m3fn``, with
one float32 scale per (block, head) in ``[num_blocks, num_heads]``; a code stands for code * scale.
Unlike the FP8 caches of ``kv_linear_to_paged_fp8`` the scale is not an argument: the writer takes it
from the data, block by block.

Both calls take a sequence's pages from ``block_tables`` (int32 ``[num_seqs, max_blocks]``) and its
length from ``context_lens`` (int32, the tokens of this call included); ``cu_seqlens`` (int32
``[num_seqs + 1]``) says which rows of the packed tensors are whose, None means one row per sequence.
Rows that belong to no sequence are neither read nor written.  Nothing is read back: block ids outside
the cache are skipped by the kernels, as are tokens past ``max_blocks * block_size`` (rows keep the
positions that ``context_lens`` gives them).
"""

from __future__ import annotations

import torch

from .. import _native

__all__ = ["kv_append_block_scaled", "paged_attention_block_scaled"]


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
    of the call only; a sequence with more rows than tokens is left alone.  In place; returns None."""
    _native.front().append(k, v, key_cache, value_cache, key_scale, value_scale, block_tables, context_lens, cu_seqlens)


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
    1 / sqrt(head_dim).  Returns ``out`` (q's dtype), or ``(out, lse)`` with the log of each row's sum of
    exponentials, float32 ``[rows, num_q_heads]``.  A row that sees no token gives zeros and an lse of -inf.
    Nothing that a row does not see reaches its result, NaN among it; a row that sees a value scale that is
    infinite or NaN gives NaN.

    Sums and softmax statistics are held in 32 bits.  The matrix units take less: with many rows to a
    sequence each weight is rounded to float16 (2**-12 of itself; float16 results are off by 2.5e-4 of their
    norm instead of 2.1e-4), with few it is good to 2**-12 of itself or 2**-30 of the largest in its tile,
    and values of q to 2**-22 of their row's largest.

    For inference: no gradient flows through it.  It keeps a workspace of 40 MB per device and stream until
    the process ends; a call captured in a graph has one of its own and zeroes its counters there."""
    return _native.front().attend(q, key_cache, value_cache, key_scale, value_scale, block_tables, context_lens, cu_seqlens, scale,
                                  causal, window, return_lse, out)
