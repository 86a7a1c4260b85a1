"""What the C entry points of the attention calls refuse before anything reaches a GPU.  CPU-only: descriptors with made-up
addresses, of which none is read."""

from __future__ import annotations

import ctypes
from ctypes import POINTER, Structure, byref, c_float, c_int32, c_int64, c_void_p

import pytest
import torch

from musa_aiter import _build

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses here are made up: a GPU must not get to see them")

E_INVALID, E_WORKSPACE, F16 = -1, -3, 1
ADDRESS = 0x7000000000  # multiple of 256


class Cache(Structure):
    _fields_ = ([("key", c_void_p), ("value", c_void_p)] +
                [(n, c_int64) for n in ("k_sb", "k_st", "k_sh", "v_sb", "v_st", "v_sh")] +
                [(n, c_void_p) for n in ("block_tables", "context_lens", "cu_seqlens")] +
                [(n, c_int64) for n in ("table_stride", "num_blocks", "num_seqs", "max_blocks", "num_rows")] +
                [(n, c_int32) for n in ("num_heads", "head_dim", "block_size", "dtype")])


class Attention(Structure):
    _fields_ = ([("cache", Cache)] + [(n, c_void_p) for n in ("q", "out", "lse", "parents", "workspace")] +
                [(n, c_int64) for n in ("workspace_bytes", "q_sr", "q_sh", "o_sr", "o_sh")] +
                [(n, c_int32) for n in ("num_q_heads", "window", "sinks")] + [("scale", c_float)])


class BlockCache(Structure):
    _fields_ = ([(n, c_void_p) for n in ("key", "value", "key_scale", "value_scale")] +
                [(n, c_int64) for n in ("k_sb", "k_sh", "v_sb", "v_sh", "ks_sb", "ks_sh", "vs_sb", "vs_sh")] +
                [(n, c_void_p) for n in ("block_tables", "context_lens", "cu_seqlens")] +
                [(n, c_int64) for n in ("table_stride", "num_blocks", "num_seqs", "max_blocks", "num_rows")] +
                [(n, c_int32) for n in ("num_heads", "head_dim", "block_size", "code_type")])


class BlockAttention(Structure):
    _fields_ = ([("cache", BlockCache)] + [(n, c_void_p) for n in ("q", "out", "lse", "workspace")] +
                [(n, c_int64) for n in ("workspace_bytes", "q_sr", "q_sh", "o_sr", "o_sh")] +
                [(n, c_int32) for n in ("num_q_heads", "q_dtype", "causal", "window")] + [("scale", c_float), ("reserved", c_int32)])


class Weights(Structure):
    _fields_ = ([("cache", Cache)] + [(n, c_void_p) for n in ("q", "lse", "sums", "rows")] +
                [(n, c_int64) for n in ("q_sr", "q_sh", "lse_sr", "sum_sr", "sum_sh", "sum_rows", "max_tokens")] +
                [(n, c_int32) for n in ("num_q_heads", "window", "sinks", "accumulate")] +
                [("scale", c_float), ("reserved", c_int32), ("workspace", c_void_p), ("workspace_bytes", c_int64)])


@pytest.fixture(scope="module")
def lib():
    result = _build.build()
    assert result.ok, result.message
    lib = ctypes.CDLL(str(_build.LIB_PATH))
    lib.mak_paged_attention_workspace_bytes.restype = c_int64
    lib.mak_block_attention_workspace_bytes.restype = c_int64
    lib.mak_block_attention.argtypes = [POINTER(BlockAttention), c_void_p]
    lib.mak_paged_attention.argtypes = [POINTER(Attention), c_void_p]
    lib.mak_paged_weights.argtypes = [POINTER(Weights), c_void_p]
    return lib


def cache():
    return Cache(key=ADDRESS, value=ADDRESS, k_sb=2048, k_st=128, k_sh=64, v_sb=2048, v_st=128, v_sh=64, block_tables=ADDRESS,
                 context_lens=ADDRESS, table_stride=2, num_blocks=4, num_seqs=1, max_blocks=2, num_rows=1, num_heads=2, head_dim=64,
                 block_size=16, dtype=F16)


def paged(lib, **change):
    d = Attention(cache=cache(), q=ADDRESS, out=ADDRESS, workspace=ADDRESS, workspace_bytes=lib.mak_paged_attention_workspace_bytes(),
                  q_sr=256, q_sh=64, o_sr=256, o_sh=64, num_q_heads=4, scale=0.125)
    for name, x in change.items():
        setattr(d, name, x)
    return lib.mak_paged_attention(byref(d), None)


def weights(lib, **change):
    d = Weights(cache=cache(), q=ADDRESS, lse=ADDRESS, sums=ADDRESS, workspace=ADDRESS,
                workspace_bytes=lib.mak_paged_attention_workspace_bytes(), q_sr=256, q_sh=64, lse_sr=4, sum_sr=64, sum_sh=32, sum_rows=1,
                max_tokens=32, num_q_heads=4, scale=0.125)
    for name, x in change.items():
        setattr(d, name, x)
    return lib.mak_paged_weights(byref(d), None)


def block_scaled(lib, **change):
    c = BlockCache(key=ADDRESS, value=ADDRESS, key_scale=ADDRESS, value_scale=ADDRESS, k_sb=2048, k_sh=1024, v_sb=2048, v_sh=1024, ks_sb=2,
                   ks_sh=1, vs_sb=2, vs_sh=1, block_tables=ADDRESS, context_lens=ADDRESS, table_stride=2, num_blocks=4, num_seqs=1,
                   max_blocks=2, num_rows=1, num_heads=2, head_dim=64, block_size=16)
    d = BlockAttention(cache=c, q=ADDRESS, out=ADDRESS, workspace=ADDRESS, workspace_bytes=lib.mak_block_attention_workspace_bytes(),
                       q_sr=256, q_sh=64, o_sr=256, o_sh=64, num_q_heads=4, q_dtype=F16, causal=1, scale=0.125)
    for name, x in change.items():
        setattr(d, name, x)
    return lib.mak_block_attention(byref(d), None)


@pytest.mark.parametrize("call", [paged, weights, block_scaled])
@pytest.mark.parametrize("change", [dict(workspace=None), dict(workspace_bytes=4096), dict(workspace=ADDRESS + 4),
                                    dict(workspace=ADDRESS + 8), dict(workspace=ADDRESS + 1)])
def test_workspaces_refused(lib, call, change):
    """Missing, too small, or not on 16 bytes: the kernels read partial sums from it 16 bytes at a time."""
    assert call(lib, **change) == E_WORKSPACE
