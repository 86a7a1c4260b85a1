"""Arguments that the block-scaled cache, page and rotary calls refuse, on CPU tensors: shapes first, then the device."""

from __future__ import annotations

import pytest
import torch

import musa_aiter as ma
from musa_aiter import registry


def cache(nb=4, nh=2, hd=64, bs=16, dtype=torch.int8):
    return torch.zeros((nb, nh, hd, bs), dtype=dtype), torch.zeros((nb, nh))


def attend(**change):
    kc, ks = cache()
    a = dict(q=torch.zeros((1, 4, 64), dtype=torch.float16), key_cache=kc, value_cache=kc.clone(), key_scale=ks, value_scale=ks.clone(),
             block_tables=torch.zeros((1, 2), dtype=torch.int32), context_lens=torch.ones(1, dtype=torch.int32))
    a.update(change)
    return ma.paged_attention_block_scaled(**a)


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros((4, 64))), "q must be"),
    (dict(q=torch.zeros((1, 4, 64))), "float16 or bfloat16"),
    (dict(q=torch.zeros((1, 3, 64), dtype=torch.float16)), "do not divide"),
    (dict(q=torch.zeros((1, 4, 128), dtype=torch.float16)), "head_dim 128"),
    (dict(q=torch.zeros((2, 4, 64), dtype=torch.float16)), "2 rows for 1 sequences"),
    (dict(key_cache=torch.zeros((4, 2, 64, 16))), "int8 or both float8"),
    (dict(value_cache=torch.zeros((4, 2, 64, 32), dtype=torch.int8)), "must both be"),
    (dict(key_cache=cache(bs=8)[0], value_cache=cache(bs=8)[0]), "block_size"),
    (dict(key_cache=cache(hd=96)[0], value_cache=cache(hd=96)[0], q=torch.zeros((1, 4, 96), dtype=torch.float16)), "head_dim must"),
    (dict(key_cache=torch.zeros((4, 2, 16, 64), dtype=torch.int8).transpose(2, 3)), "contiguous"),
    (dict(key_scale=torch.zeros((4, 3))), "scales must be"),
    (dict(key_scale=torch.zeros((4, 2), dtype=torch.float16)), "float32"),
    (dict(block_tables=torch.zeros((1, 2))), "int32"),
    (dict(block_tables=torch.zeros((2, 2), dtype=torch.int32)), "block_tables must be"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "cu_seqlens"),
    (dict(window=-1), "window"),
    (dict(window=4, causal=False), "window"),
    (dict(out=torch.zeros((1, 4, 64))), "out must"),
    ({}, "no CPU fallback"),
])
def test_attention_refuses(change, text):
    with pytest.raises((ValueError, RuntimeError), match=text):
        attend(**change)


@pytest.mark.parametrize("change,text", [
    (dict(k=torch.zeros((1, 2, 64, 1))), "k and v must both be"),
    (dict(v=torch.zeros((1, 1, 64))), "k and v must both be"),
    (dict(k=torch.zeros((1, 2, 64), dtype=torch.float64), v=torch.zeros((1, 2, 64), dtype=torch.float64)), "float16, bfloat16 or float32"),
    (dict(k=torch.zeros((1, 3, 64)), v=torch.zeros((1, 3, 64))), "3 heads|no CPU fallback"),
    (dict(context_lens=torch.ones(2, dtype=torch.int32)), "context_lens"),
    ({}, "no CPU fallback"),
])
def test_writer_refuses(change, text):
    kc, ks = cache()
    a = dict(k=torch.zeros((1, 2, 64)), v=torch.zeros((1, 2, 64)), key_cache=kc, value_cache=kc.clone(), key_scale=ks,
             value_scale=ks.clone(), block_tables=torch.zeros((1, 2), dtype=torch.int32), context_lens=torch.ones(1, dtype=torch.int32))
    a.update(change)
    with pytest.raises((ValueError, RuntimeError), match=text):
        ma.kv_append_block_scaled(**a)


I = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731


def test_pages_refuse():
    with pytest.raises(ValueError, match="block_tables must be"):
        ma.kv_pages_grow(I(4), I(4), I(1), I(1), I(8), 16)
    with pytest.raises(ValueError, match="one entry per row"):
        ma.kv_pages_grow(I(4, 2), I(3), I(1), I(1), I(8), 16)
    with pytest.raises(ValueError, match="same length"):
        ma.kv_pages_grow(I(4, 2), I(4), I(1), I(2), I(8), 16)
    with pytest.raises(ValueError, match="block_size"):
        ma.kv_pages_grow(I(4, 2), I(4), I(1), I(1), I(8), 0)
    with pytest.raises(ValueError, match="ref_counts must be"):
        ma.kv_pages_free(I(4, 2), I(4), I(1), torch.zeros(8))
    with pytest.raises(ValueError, match="same length"):
        ma.kv_pages_fork(I(4, 2), I(4), I(1), I(2), I(8), [], 16)
    with pytest.raises(ValueError, match="8 pages"):
        ma.kv_pages_fork(I(4, 2), I(4), I(1), I(1), I(8), [torch.zeros((7, 3))], 16)
    with pytest.raises(ValueError, match="contiguous"):
        ma.kv_pages_compact(I(4, 2), I(8), [torch.zeros((8, 3, 4)).transpose(1, 2)])
    with pytest.raises(ValueError, match="overlap"):
        ma.kv_pages_compact(I(4, 2), I(8), [torch.zeros((1, 3)).expand(8, 3)])
    with pytest.raises(ValueError, match="same length"):
        ma.kv_pages_copy([torch.zeros((8, 3))], I(2), I(3))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ma.kv_pages_compact(I(4, 2), I(8), [torch.zeros((8, 3))])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ma.kv_pages_free(I(4, 2), I(4), I(1), I(8))


@pytest.mark.parametrize("change,text", [
    (dict(k=torch.zeros((2, 1, 64), dtype=torch.float16)), "same tokens"),
    (dict(q=torch.zeros((3, 2, 64))), "float16 or both bfloat16"),
    (dict(sections=(30, 3)), "sections must add up"),
    (dict(sections=()), "counts of pairs"),
    (dict(sections=(-8, 40)), "counts of pairs"),
    (dict(sections=(32, 32), cos=torch.zeros((5, 64)), sin=torch.zeros((5, 64))), "sections must add up"),
    (dict(positions=torch.zeros((3, 3), dtype=torch.int32)), "positions must be"),
    (dict(positions=torch.zeros((2, 3))), "positions must be"),
    (dict(cos=torch.zeros((5, 31))), "cos and sin"),
    (dict(cos=torch.zeros((5, 32)).double()), "float32"),
    ({}, "no CPU fallback"),
])
@pytest.mark.parametrize("call", [ma.apply_rope_axes, ma.apply_rope_axes_backward])
def test_rope_axes_refuses(call, change, text):
    a = dict(q=torch.zeros((3, 2, 64), dtype=torch.float16), k=torch.zeros((3, 1, 64), dtype=torch.float16),
             positions=torch.zeros((2, 3), dtype=torch.int32), cos=torch.zeros((5, 32)), sin=torch.zeros((5, 32)), sections=(16, 16))
    a.update(change)
    with pytest.raises((ValueError, RuntimeError), match=text):
        call(a["q"], a["k"], a["positions"], a["cos"], a["sin"], a["sections"])


def test_registered():
    assert {c.name for c in registry.list_capabilities("pages")} == {"kv_pages_copy", "kv_pages_fork", "kv_pages_grow", "kv_pages_free",
                                                                     "kv_pages_compact"}
    for name in ("paged_attention_block_scaled", "kv_append_block_scaled", "apply_rope_axes", "apply_rope_axes_backward"):
        assert registry.get(name).backends == ("cuda-sm100a",) and callable(getattr(ma, name))
