"""The serving example: all block-scaled cache, page and rotary calls together."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "musa-aiter_b200" / "examples" / "block_scaled_serving.py"


# Values lie below 6 or so.  An int8 value is off by half a step m / 127 of its block, 0.024, each time its block is
# rounded (three times at the most here, its scale growing); an E4M3 one by 2^-4 of itself, 0.375.  Attention averages
# that and its weights shift by less.  A lost token or page is off by 1.
@pytest.mark.parametrize("code,bound", [(torch.int8, 0.15), (torch.float8_e4m3fn, 0.4)])
@pytest.mark.parametrize("block_size", [16, 64])
def test_serving_example(code, bound, block_size):
    spec = importlib.util.spec_from_file_location("block_scaled_serving", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert module.serve(code, block_size=block_size) < bound
