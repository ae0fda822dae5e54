"""Operands and gradients of the attention backward that lie more than 2^31 elements into their tensors, through the C
ABI: with far heads, far rows and far batch entries, in one piece and joined from several."""
from __future__ import annotations

import ctypes

import pytest
import torch

import _native
from flash_atten import attention_backward, attention_forward
from test_attention_backward_gpu import _inputs, _no_device_errors  # noqa: F401

pytestmark = pytest.mark.gpu

NAMES = ("q", "k", "v", "o", "dout", "dq", "dk", "dv")


def _call(tensors, lse, causal):
    """fab_attention_bwd on [B, H, S, D] views of any strides."""
    p = _native.FabAttentionBwdParams()
    for name, t in (*tensors.items(), ("lse", lse)):
        setattr(p, name, t.data_ptr())
        for d, s in zip("bhs", t.stride()):
            setattr(p, f"{name}_stride_{d}", s)
    q, k = tensors["q"], tensors["k"]
    p.batch, p.heads_q, p.seqlen_q, p.head_dim = q.shape
    p.heads_kv, p.seqlen_k = k.shape[1:3]
    p.dtype, p.sm_scale, p.causal = _native.dtype_code(q.dtype), q.shape[-1] ** -0.5, int(causal)
    need = ctypes.c_size_t(0)
    _native.check(_native.lib.fab_attention_bwd_workspace(ctypes.byref(p), ctypes.byref(need)), "workspace")
    ws = torch.empty(max(need.value, 256), device=q.device, dtype=torch.uint8)
    p.workspace, p.workspace_bytes = ws.data_ptr(), need.value
    _native.check(_native.lib.fab_attention_bwd(ctypes.byref(p), _native.current_stream_handle(q.device)), "backward")


# Whether the sums are cut in slices: a few long tiles are, the workspace then holds more than the statistics.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bfloat16", "float16"])
@pytest.mark.parametrize("B, H, S, strides", [
    (1, 3, 150, (0, 1 << 30, 128)),               # heads
    (1, 1, 140, (0, 0, 1 << 24)),                 # rows
    (3, 1, 150, (1 << 30, 0, 128)),               # batch entries
    (1, 2, 2500, (0, 512, 1 << 20)),              # rows, in slices
    (1, 3, 2100, (0, 1 << 30, 128)),              # heads, in slices
], ids=["heads", "rows", "entries", "rows_sliced", "heads_sliced"])
def test_far_offsets(B, H, S, strides, dtype, cuda_device):
    D = 64
    last = (B - 1) * strides[0] + (H - 1) * strides[1] + (S - 1) * strides[2]
    assert last >= 1 << 31
    dout, q, k, v = _inputs(B, H, H, S, S, D, dtype, cuda_device, S)
    o, lse = attention_forward(q, k, v, causal=True, return_lse=True)
    want = dict(zip(("dq", "dk", "dv"), attention_backward(dout, q, k, v, o, lse, causal=True)))
    given = dict(q=q, k=k, v=v, o=o, dout=dout)
    base = torch.empty(last + 128 + D, device=cuda_device, dtype=dtype)
    for name in NAMES:
        far = base.as_strided((B, H, S, D), (*strides, 1), 0 if name < "k" else 64)
        tensors = dict(given, **{n: torch.full_like(w, float("nan")) for n, w in want.items()})
        if name in given:
            far.copy_(given[name])
        else:
            base.fill_(float("nan"))
        tensors[name] = far
        _call(tensors, lse, True)
        assert all(torch.equal(tensors[n], w) for n, w in want.items()), name
        if name in want:
            far.fill_(float("nan"))
            assert base.isnan().all(), f"{name}: a write beside the gradient"
