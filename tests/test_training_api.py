"""The training entry points refuse bad arguments before they touch a device, and report workspaces without one."""
from __future__ import annotations

import ctypes

import pytest
import torch

import _native
import training
from flash_atten import attention_backward, attention_backward_varlen, attention_backward_workspace_bytes


def _bwd_params(**change):
    p = _native.FabAttentionBwdParams()
    for name in ("q", "k", "v", "o", "dout", "lse", "dq", "dk", "dv"):
        setattr(p, name, 4096)  # never dereferenced: these calls are refused first
        for d, s in zip("bhs", (2 * 64 * 64, 64 * 64, 64)):
            setattr(p, f"{name}_stride_{d}", s)
    p.batch, p.heads_q, p.heads_kv, p.seqlen_q, p.seqlen_k, p.head_dim = 1, 2, 1, 64, 64, 64
    p.dtype, p.sm_scale = _native.FAB_DTYPE_BF16, 0.125
    p.workspace, p.workspace_bytes = 4096, 1 << 20
    for key, value in change.items():
        setattr(p, key, value)
    return p


@pytest.mark.parametrize("change, code", [
    (dict(dtype=_native.FAB_DTYPE_F32), _native.FAB_ERR_UNSUPPORTED),
    (dict(dtype=7), _native.FAB_ERR_INVALID_ARG),
    (dict(head_dim=264), _native.FAB_ERR_UNSUPPORTED),
    (dict(head_dim=0), _native.FAB_ERR_INVALID_ARG),
    (dict(batch=-1), _native.FAB_ERR_INVALID_ARG),
    (dict(heads_kv=0), _native.FAB_ERR_INVALID_ARG),
    (dict(heads_q=3, heads_kv=2), _native.FAB_ERR_INVALID_ARG),
    (dict(sm_scale=float("inf")), _native.FAB_ERR_INVALID_ARG),
    (dict(q=None), _native.FAB_ERR_INVALID_ARG),
    (dict(dv=None), _native.FAB_ERR_INVALID_ARG),
    (dict(lse=None), _native.FAB_ERR_INVALID_ARG),
    (dict(k=4104), _native.FAB_ERR_INVALID_ARG),
    (dict(dq=4098), _native.FAB_ERR_INVALID_ARG),
    (dict(o_stride_s=60), _native.FAB_ERR_INVALID_ARG),
    (dict(dk_stride_s=63), _native.FAB_ERR_INVALID_ARG),
    (dict(cu_seqlens_q=4096), _native.FAB_ERR_INVALID_ARG),
    (dict(cu_seqlens_q=4098, cu_seqlens_k=4096, total_q=64, total_k=64), _native.FAB_ERR_INVALID_ARG),
    (dict(workspace=None), _native.FAB_ERR_WORKSPACE),
    (dict(workspace=4100), _native.FAB_ERR_WORKSPACE),
    (dict(workspace_bytes=16), _native.FAB_ERR_WORKSPACE),
])
def test_attention_backward_refuses_before_any_launch(change, code):
    p = _bwd_params(**change)
    assert _native.lib.fab_attention_bwd(ctypes.byref(p), None) == code


def test_attention_backward_without_work_is_ok():
    assert _native.lib.fab_attention_bwd(None, None) == _native.FAB_ERR_INVALID_ARG
    for change in (dict(batch=0), dict(seqlen_q=0, seqlen_k=0)):
        assert _native.lib.fab_attention_bwd(ctypes.byref(_bwd_params(**change)), None) == _native.FAB_OK


def test_attention_backward_workspace():
    """At least two floats per query row (fp16: three); a multiple of 256 bytes; the same for the same sizes; counted
    in 64 bits; bounded by the statistics where there are tiles enough to fill the GPU."""
    def size(B, H, M, D, dtype, N=77):
        return attention_backward_workspace_bytes((B, H, M, D), (B, 1, N, D), dtype)

    for args, rows, floats in (((2, 3, 129, 128, torch.bfloat16), 2 * 3 * 129, 2), ((2, 3, 129, 256, torch.bfloat16), 2 * 3 * 129, 2),
                               ((2, 3, 129, 64, torch.float16), 2 * 3 * 129, 3)):
        assert size(*args) == size(*args) >= rows * floats * 4 and size(*args) % 256 == 0
    assert size(1, 4, 0, 64, torch.bfloat16) == 0
    assert attention_backward_workspace_bytes((300, 2, 64), (300, 1, 64), torch.bfloat16, packed_batch=3) >= 300 * 2 * 8
    big = size(64, 64, 1 << 20, 128, torch.bfloat16, 1 << 20)
    assert big == 64 * 64 * (1 << 20) * 8


def test_python_entries_refuse_cpu_tensors():
    t = torch.zeros(1, 1, 4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        attention_backward(t, t, t, t, t, torch.zeros(1, 1, 4))
    cu = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        attention_backward_varlen(t[0], t[0], t[0], t[0], t[0], torch.zeros(1, 4), cu, cu, 4, 4)
    with pytest.raises(ValueError, match="CUDA"):
        training.layernorm_forward(t, t[0, 0, 0])
    with pytest.raises(ValueError, match="CUDA"):
        training.rope_multi_axis(t[0], None, cu[None], cu, cu, (4,))
    with pytest.raises(ValueError, match="shape"):
        attention_backward(t[0], t, t, t, t, torch.zeros(1, 1, 4))


def _norm_args(**change):
    a = dict(x=4096, residual=None, w=4096, bias=4096, y=4096, x_out=None, mean=4096, rstd=4096, rows=4, cols=8,
             ld_x=8, ld_res=0, ld_y=8, ld_xo=0, eps=1e-5, dtype=_native.FAB_DTYPE_BF16, w_dtype=_native.FAB_DTYPE_BF16,
             stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change, code", [
    (dict(x=None), _native.FAB_ERR_INVALID_ARG),
    (dict(w=None), _native.FAB_ERR_INVALID_ARG),
    (dict(residual=4096), _native.FAB_ERR_INVALID_ARG),
    (dict(mean=None), _native.FAB_ERR_INVALID_ARG),
    (dict(rows=-1), _native.FAB_ERR_INVALID_ARG),
    (dict(cols=0), _native.FAB_ERR_INVALID_ARG),
    (dict(eps=-1e-5), _native.FAB_ERR_INVALID_ARG),
    (dict(eps=float("nan")), _native.FAB_ERR_INVALID_ARG),
    (dict(x=4097), _native.FAB_ERR_INVALID_ARG),
    (dict(w_dtype=_native.FAB_DTYPE_F16), _native.FAB_ERR_UNSUPPORTED),
    (dict(dtype=_native.FAB_DTYPE_F32), _native.FAB_ERR_UNSUPPORTED),
    (dict(rows=0), _native.FAB_OK),
])
def test_layernorm_refuses_before_any_launch(change, code):
    assert _native.lib.fab_layernorm(*_norm_args(**change)) == code


def test_layernorm_backward_refuses_before_any_launch():
    def call(**change):
        a = dict(dy=4096, x=4096, w=4096, mean=4096, rstd=4096, dres=None, dx=4096, dw=4096, db=4096, ws=4096,
                 ws_bytes=1 << 20, rows=4, cols=8, ld_dy=8, ld_x=8, ld_dres=0, ld_dx=8, dtype=1, w_dtype=1, stream=None)
        a.update(change)
        return _native.lib.fab_layernorm_bwd(*a.values())

    for name in ("dy", "x", "w", "mean", "rstd", "dx"):
        assert call(**{name: None}) == _native.FAB_ERR_INVALID_ARG
    assert call(ws=None) == call(ws_bytes=8) == call(ws=4100) == _native.FAB_ERR_WORKSPACE
    assert call(cols=0) == call(rows=-2) == call(dw=4097) == _native.FAB_ERR_INVALID_ARG
    assert call(dtype=1, w_dtype=0) == _native.FAB_ERR_UNSUPPORTED
    assert call(rows=0, dw=None, db=None) == _native.FAB_OK
    need = ctypes.c_size_t(0)
    assert _native.lib.fab_layernorm_bwd_workspace(1 << 20, 1 << 21, ctypes.byref(need)) == _native.FAB_OK
    assert need.value > 1 << 31  # counted in 64 bits


def test_rope_refuses_before_any_launch():
    def call(**change):
        p = _native.FabRopeAxesParams()
        for name in ("q", "k", "q_out", "k_out", "positions", "cos", "sin"):
            setattr(p, name, 4096)
        p.tokens, p.heads_q, p.heads_k, p.head_dim, p.axes, p.table_rows, p.dtype = 3, 2, 1, 64, 2, 10, 1
        p.sections[0], p.sections[1] = 16, 16
        for key, value in change.items():
            if key == "sections":
                for i, s in enumerate(value):
                    p.sections[i] = s
            else:
                setattr(p, key, value)
        return _native.lib.fab_rope_axes(ctypes.byref(p), None)

    for change in (dict(axes=0), dict(axes=5), dict(sections=(16, 17)), dict(sections=(-1, 16)), dict(sections=(0, 0)),
                   dict(q=None), dict(k_out=None), dict(positions=None), dict(cos=None), dict(sin=4097), dict(q=4097),
                   dict(dtype=9), dict(tokens=-1), dict(head_dim=0), dict(positions=4100, positions_64bit=1)):
        assert call(**change) == _native.FAB_ERR_INVALID_ARG, change
    assert call(tokens=0) == _native.FAB_OK


def test_autograd_attention_refuses_what_has_no_gradient():
    x = torch.zeros(1, 1, 4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        training.attention(x, x, x)


def test_example_positions_and_batches():
    import train_block

    pos = train_block.rope_positions(2, 2, 3)
    assert pos.tolist() == [[0, 1, 2, 2, 2, 2, 2, 2], [0, 1, 2, 2, 2, 3, 3, 3], [0, 1, 2, 3, 4, 2, 3, 4]]
    g = torch.Generator().manual_seed(1)
    words = torch.arange(14).view(2, 7)
    tokens, batch = train_block.make_batch(((3, 2, 2), (1, 1, 4)), words, (2, 1, 1), g, "cpu")
    assert batch["cu"].tolist() == [0, 7, 12] and batch["longest"] == 7 and batch["positions"].shape == (3, 12)
    assert batch["cos"].shape == (int(batch["positions"].max()) + 1, 4)
    assert tokens[0] == tokens[7] % 7 + tokens[0] // 7 * 7
    loss = train_block.next_token_loss(torch.zeros(12, 14), tokens, batch["cu"])
    assert abs(loss.item() - torch.tensor(14.0).log().item()) < 1e-5
