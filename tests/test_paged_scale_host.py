"""A softmax scale that is no number: the kernels bound it from below, which makes a number of NaN, so it is refused."""

from __future__ import annotations

import ctypes
import math

import pytest

from .test_attention_abi_host import E_INVALID, lib, paged, weights  # noqa: F401
from .test_paged_host import H, I, ma, torch, tree, window

BAD = (math.nan, math.inf, -math.inf, 1e39, 3e38)  # the last one times log2 e is past 32 bits


@pytest.mark.parametrize("scale", BAD)
def test_scales_refused(scale):
    for call in (window, tree):
        with pytest.raises(ValueError, match="scale must be finite"):
            call(scale=scale)
    with pytest.raises(ValueError, match="scale must be finite"):
        ma.paged_attention_weights(H(1, 4, 64), H(4, 16, 2, 64), I(1, 2), I(1), torch.zeros((1, 4)), torch.zeros((1, 2, 32)), scale=scale)


@pytest.mark.parametrize("call", [paged, weights])
@pytest.mark.parametrize("scale", BAD)
def test_scales_refused_at_the_c_entry(lib, call, scale):  # noqa: F811
    assert call(lib, scale=scale) == E_INVALID
    lib.mak_last_error.restype = ctypes.c_char_p
    assert b"scale" in lib.mak_last_error()
