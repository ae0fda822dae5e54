"""The attention backward's workspace query and its launch accept and refuse the same sizes (host checks only)."""
from __future__ import annotations

import ctypes

import pytest

import _native
from test_training_api import _bwd_params

BIG = 2 ** 31 - 1


def _both(**change):
    need = ctypes.c_size_t(0)
    p = _bwd_params(workspace=None, **change)
    return (_native.lib.fab_attention_bwd_workspace(ctypes.byref(p), ctypes.byref(need)),
            _native.lib.fab_attention_bwd(ctypes.byref(p), None), need.value)


@pytest.mark.parametrize("change", [
    dict(batch=1 << 20, heads_q=4096, heads_kv=4096),                                   # heads
    dict(batch=1 << 20, heads_q=2048, heads_kv=2048),                                   # their tiles: twice 2^31
    dict(batch=1 << 15, heads_q=32, heads_kv=4, seqlen_q=1 << 18, seqlen_k=1 << 18),
    dict(heads_q=256, heads_kv=1, seqlen_q=BIG, seqlen_k=64),
    dict(batch=1 << 24, heads_q=64, heads_kv=64, cu_seqlens_q=4096, cu_seqlens_k=4096, total_q=BIG, total_k=BIG),
], ids=["heads", "tiles", "long", "queries", "packed"])
@pytest.mark.parametrize("dtype", [_native.FAB_DTYPE_BF16, _native.FAB_DTYPE_F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("head_dim", [64, 256])
def test_too_many_pieces_are_refused_by_both(change, dtype, head_dim):
    assert _both(dtype=dtype, head_dim=head_dim, **change) == (_native.FAB_ERR_UNSUPPORTED, _native.FAB_ERR_UNSUPPORTED, 0)


@pytest.mark.parametrize("change", [
    dict(batch=2048, heads_q=32, heads_kv=4),
    dict(batch=65536, heads_q=64, heads_kv=64),
    dict(batch=1 << 20, heads_q=8, heads_kv=8, cu_seqlens_q=4096, cu_seqlens_k=4096, total_q=BIG, total_k=BIG),
])
@pytest.mark.parametrize("dtype", [_native.FAB_DTYPE_BF16, _native.FAB_DTYPE_F16], ids=["bf16", "f16"])
def test_many_heads_are_taken_by_both(change, dtype):
    """More (batch entry, head) pairs than a grid's second dimension holds; the launch asks for the workspace."""
    workspace, launch, need = _both(dtype=dtype, **change)
    assert workspace == _native.FAB_OK and need > 0
    assert launch == _native.FAB_ERR_WORKSPACE
