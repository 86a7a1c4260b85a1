"""The serving example over paged 16-bit caches: norms, attention, weights, eviction and trees in one run."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "musa-aiter_b200" / "examples" / "paged_serving.py"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("block_size", [16, 64])
def test_serving_example(dtype, block_size):
    spec = importlib.util.spec_from_file_location("paged_serving", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    lengths, finite = module.serve(block_size=block_size, dtype=dtype)
    prompts = list(module.PROMPTS)
    assert lengths[0] == prompts and lengths[4] == [n + 4 for n in prompts]
    assert lengths[5] == [min(n + 4, 48) for n in prompts]
    assert lengths[7] == [n + 1 + len(module.PARENTS) for n in lengths[5]]
    assert finite
