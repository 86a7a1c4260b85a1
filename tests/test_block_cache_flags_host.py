"""Flags of the block-scaled cache and rotary calls that have no truth value: their error is the caller's."""

from __future__ import annotations

import pytest
import torch

import musa_aiter as ma

from .test_block_cache_host import attend


@pytest.mark.parametrize("flag", ["causal", "return_lse"])
def test_attention(flag):
    with pytest.raises(RuntimeError, match="ambiguous"):
        attend(**{flag: torch.ones(2)})


@pytest.mark.parametrize("flag", ["interleaved", "interleaved_axes"])
def test_rotation(flag):
    x = torch.zeros((3, 2, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="ambiguous"):
        ma.apply_rope_axes(x, x, torch.zeros((2, 3), dtype=torch.int32), torch.zeros((5, 32)), torch.zeros((5, 32)), (16, 16),
                           **{flag: torch.ones(2)})
