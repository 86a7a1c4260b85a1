"""Arguments that the paged attention, eviction and norm calls refuse, on CPU tensors: shapes first, then the device."""

from __future__ import annotations

import pytest
import torch

import musa_aiter as ma
from musa_aiter import registry

I = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
H = lambda *n: torch.zeros(n, dtype=torch.float16)  # noqa: E731


def window(**change):
    a = dict(q=H(1, 4, 64), key_cache=H(4, 16, 2, 64), value_cache=H(4, 16, 2, 64), block_tables=I(1, 2), context_lens=I(1))
    a.update(change)
    return ma.paged_attention_window(**a)


def tree(**change):
    a = dict(q=H(1, 4, 64), key_cache=H(4, 16, 2, 64), value_cache=H(4, 16, 2, 64), block_tables=I(1, 2), context_lens=I(1), parents=I(1))
    a.update(change)
    return ma.paged_attention_tree(**a)


SHARED = [
    (dict(q=H(4, 64)), "q must be"),
    (dict(q=torch.zeros((1, 4, 64))), "float16 or bfloat16"),
    (dict(q=torch.zeros((1, 4, 64), dtype=torch.bfloat16)), "one type"),
    (dict(q=H(1, 3, 64)), "do not divide"),
    (dict(q=H(1, 4, 128)), "head_dim 128"),
    (dict(q=H(2, 4, 64)), "2 rows for 1 sequences|parents must|lse must"),
    (dict(block_tables=torch.zeros((1, 2))), "int32"),
    (dict(block_tables=I(2, 2)), "block_tables must be"),
    (dict(block_tables=I(2, 2).t()[:1]), "row must be contiguous"),
    (dict(cu_seqlens=I(3)), "cu_seqlens"),
    (dict(scale="x"), "must be real number|float"),
    ({}, "no CPU fallback"),
]


@pytest.mark.parametrize("call", [window, tree])
@pytest.mark.parametrize("change,text", SHARED + [
    (dict(key_cache=H(4, 8, 2, 64), value_cache=H(4, 8, 2, 64)), "block_size"),
    (dict(key_cache=H(4, 16, 2, 96), value_cache=H(4, 16, 2, 96)), "head_dim must"),
    (dict(value_cache=H(4, 16, 1, 64)), "must both be"),
    (dict(value_cache=H(4, 16, 64, 2).transpose(2, 3)), "contiguous"),
    (dict(key_cache=H(4, 16, 2, 65)[..., :64]), "multiples of 8"),
    (dict(key_cache=H(4 * 16 * 2 * 64 + 1)[1:].view(4, 16, 2, 64)), "16 bytes"),
    (dict(out=torch.zeros((1, 4, 64))), "out must"),
    (dict(out=H(1, 64, 4).transpose(1, 2)), "out must"),
])
def test_attention_refuses(call, change, text):
    with pytest.raises((ValueError, RuntimeError, TypeError), match=text):
        call(**change)


@pytest.mark.parametrize("change,text", [
    (dict(window=-1), "window"),
    (dict(sinks=-1, window=3), "sinks"),
    (dict(sinks=2), "sinks need a window"),
    (dict(window=1.5), "window must be an integer"),
])
def test_windows_refused(change, text):
    with pytest.raises(ValueError, match=text):
        window(**change)


@pytest.mark.parametrize("change", [dict(parents=I(2)), dict(parents=torch.zeros(1)), dict(parents=None), dict(parents=I(1, 1))])
def test_trees_refused(change):
    with pytest.raises(ValueError, match="parents must"):
        tree(**change)


@pytest.mark.parametrize("change,text", SHARED + [
    (dict(key_cache=H(4, 8, 2, 64)), "block_size"),
    (dict(lse=torch.zeros((1, 3))), "lse must"),
    (dict(lse=H(1, 4)), "lse must"),
    (dict(sums=torch.zeros((1, 3, 32))), "sums must"),
    (dict(sums=torch.zeros((2, 2, 32))), "2 rows for 1 sequences"),
    (dict(sums=torch.zeros((1, 32, 2)).transpose(1, 2)), "contiguous"),
    (dict(rows=I(2)), "rows must"),
    (dict(sinks=1), "sinks need a window"),
])
def test_weights_refuse(change, text):
    a = dict(q=H(1, 4, 64), key_cache=H(4, 16, 2, 64), block_tables=I(1, 2), context_lens=I(1), lse=torch.zeros((1, 4)),
             sums=torch.zeros((1, 2, 32)))
    a.update(change)
    with pytest.raises((ValueError, RuntimeError, TypeError), match=text):
        ma.paged_attention_weights(**a)


@pytest.mark.parametrize("change,text", [
    (dict(keep=0), "keep must"),
    (dict(keep=4, sinks=3, recent=2), "keep must"),
    (dict(keep=4, sinks=-1), "sinks must not be negative"),
    (dict(key_caches=[]), "same length"),
    (dict(key_caches=[], value_caches=[]), "must have a layer"),
    (dict(key_caches=[torch.zeros((4, 16, 2, 64))], value_caches=[torch.zeros((4, 16, 2, 64))]), "float16 or bfloat16"),
    (dict(key_caches=[H(4, 16, 2, 96)], value_caches=[H(4, 16, 2, 96)]), "head_dim must"),
    (dict(value_caches=[H(4, 32, 2, 64)]), "one shape"),
    (dict(key_caches=[H(4, 16, 2, 64), H(4, 2, 16, 64).transpose(1, 2)], value_caches=[H(4, 16, 2, 64)] * 2), "one layout"),
    (dict(sums=torch.zeros((1, 2, 2, 32))), "sums must"),
    (dict(sums=torch.zeros((1, 3, 32, 2)).transpose(2, 3)), "contiguous"),
    (dict(ref_counts=I(5)), "one entry per page"),
    (dict(context_lens=I(2)), "one entry per row"),
    (dict(rows=torch.zeros(2)), "rows must be"),
    ({}, "no CPU fallback"),
])
def test_eviction_refuses(change, text):
    a = dict(block_tables=I(3, 2), context_lens=I(3), rows=I(2), ref_counts=I(4), key_caches=[H(4, 16, 2, 64)],
             value_caches=[H(4, 16, 2, 64)], sums=torch.zeros((1, 3, 2, 32)), keep=8)
    a.update(change)
    with pytest.raises((ValueError, RuntimeError), match=text):
        ma.kv_pages_evict(**a)


@pytest.mark.parametrize("change,text", [
    (dict(q=H(3, 64)), "q and k must be"),
    (dict(k=H(2, 1, 64)), "q and k must be"),
    (dict(k=torch.zeros((3, 1, 64))), "both be float16"),
    (dict(q=H(3, 2, 24), k=H(3, 1, 24)), "multiple of 16"),
    (dict(q=H(3, 2, 272), k=H(3, 1, 272)), "multiple of 16"),
    (dict(q_weight=torch.ones(32)), "weights must"),
    (dict(q_weight=torch.ones(64, dtype=torch.bfloat16)), "weights must"),
    (dict(q_weight=H(64)), "weights must"),
    (dict(positions=torch.zeros(3)), "positions must"),
    (dict(positions=I(1, 3)), "positions must"),
    (dict(cos=torch.zeros((5, 16))), "cos and sin"),
    (dict(cos=torch.zeros((5, 12)), sin=torch.zeros((5, 12))), "multiple of 8 pairs"),
    (dict(cos=torch.zeros((5, 40)), sin=torch.zeros((5, 40))), "multiple of 8 pairs"),
    (dict(cos=torch.zeros((5, 32)).double()), "float32"),
    (dict(eps=-1e-6), "eps"),
    ({}, "no CPU fallback"),
])
@pytest.mark.parametrize("backward", [False, True])
def test_norms_refuse(backward, change, text):
    a = dict(q=H(3, 2, 64), k=H(3, 1, 64), q_weight=torch.ones(64), k_weight=torch.ones(64), positions=I(3), cos=torch.zeros((5, 32)),
             sin=torch.zeros((5, 32)))
    a.update(change)
    with pytest.raises((ValueError, RuntimeError), match=text):
        if backward:
            ma.apply_qk_norm_rope_backward(a["q"], a["k"], **a)
        else:
            ma.apply_qk_norm_rope(**a)


def test_tables_that_require_a_gradient_are_refused():
    with pytest.raises(ValueError, match="tables without a gradient"):
        ma.apply_qk_norm_rope(H(3, 2, 64), H(3, 1, 64), torch.ones(64), torch.ones(64), I(3), torch.zeros((5, 32), requires_grad=True),
                              torch.zeros((5, 32)))


def test_results_on_top_of_one_another_are_refused():
    with pytest.raises(ValueError, match="out must not be expanded"):
        window(out=H(1, 1, 64).expand(1, 4, 64))
    two = dict(q=H(2, 4, 64), key_cache=H(4, 16, 2, 64), block_tables=I(2, 2), context_lens=I(2), lse=torch.zeros((2, 4)))
    with pytest.raises(ValueError, match="sums must not be expanded"):
        ma.paged_attention_weights(**two, sums=torch.zeros((1, 2, 32)).expand(2, 2, 32))
    plane, other = H(4, 16, 2, 64), H(4, 16, 2, 64)
    evict = dict(block_tables=I(3, 2), context_lens=I(3), rows=I(2), ref_counts=I(4), keep=8)
    for keys, values, text in (
        ([plane, plane], [other, H(4, 16, 2, 64)], "key_caches must not hold a layer twice"),
        ([plane, H(4, 16, 2, 64)], [other, other], "value_caches must not hold a layer twice"),
        ([H(4, 16, 1, 64).expand(4, 16, 2, 64)], [other], "key_caches must not be expanded"),
    ):
        with pytest.raises(ValueError, match=text):
            ma.kv_pages_evict(**evict, key_caches=keys, value_caches=values, sums=torch.zeros((len(keys), 3, 2, 32)))
    with pytest.raises(ValueError, match="sums must not be expanded"):
        ma.kv_pages_evict(**evict, key_caches=[plane], value_caches=[other], sums=torch.zeros((1, 1, 2, 32)).expand(1, 3, 2, 32))


def test_registered():
    for name, family in (("paged_attention_window", "attention"), ("paged_attention_tree", "attention"), ("paged_attention_weights", "eviction"),
                         ("kv_pages_evict", "eviction"), ("apply_qk_norm_rope", "cache"), ("apply_qk_norm_rope_backward", "cache")):
        cap = registry.get(name)
        assert cap.family == family and cap.backends == ("cuda-sm100a",) and callable(getattr(ma, name))
