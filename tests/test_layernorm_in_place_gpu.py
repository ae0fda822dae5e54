"""Layer norm in place, as the C ABI allows: x_out over x in the forward pass, dx over dy or over dresidual in the
backward pass.  The results are those of separate tensors of the same layout, bit for bit, on every path."""
from __future__ import annotations

import ctypes

import pytest
import torch

import _native
from test_training_ops_gpu import EPS, _check_backward, _check_forward, _no_device_errors, _norm_inputs  # noqa: F401

pytestmark = pytest.mark.gpu

CASES = [
    # rows, cols, row strides of x and of dy, first element of x, dtype
    (300, 256, 256, 264, 0, torch.bfloat16),        # a warp for each row
    (300, 250, 256, 264, 3, torch.float16),         # the same off the 16-byte grid
    (700, 2048, 2048, 2048, 0, torch.bfloat16),     # a CTA
    (700, 5000, 5008, 5000, 0, torch.bfloat16),
    (700, 2047, 2047, 2055, 0, torch.bfloat16),
    (500, 3000, 3000, 3000, 0, torch.float32),
    (200, 12288, 12288, 12296, 0, torch.bfloat16),  # a cluster
    (200, 12289, 12289, 12289, 5, torch.float16),
    (150, 8001, 8001, 8001, 1, torch.float32),
    (300, 1000, 1000, 1003, 0, torch.bfloat16),     # rows at unlike places of their 16-byte pieces
    (300, 1000, 1001, 1000, 2, torch.float32),
    (9, 66000, 66000, 66000, 0, torch.bfloat16),    # longer than a cluster's share
    (700, 66001, 66001, 66001, 0, torch.float16),
]


def _layout(t, ld, first):
    """A copy of t's rows at row stride ld, `first` elements into its storage."""
    store = torch.zeros(t.shape[0] * ld + 32, device=t.device, dtype=t.dtype)
    view = store.as_strided(t.shape, (ld, 1), first)
    view.copy_(t)
    return view


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0]}x{c[1]}ld{c[2]}-{c[3]}+{c[4]}{str(c[5])[6:]}")
def test_in_place_is_out_of_place(case, cuda_device):
    rows, cols, ld_x, ld_dy, first, dtype = case
    data = _norm_inputs(rows, cols, dtype, dtype, cuda_device, rows + cols)
    dt, stream, ptr = _native.dtype_code(dtype), _native.current_stream_handle(cuda_device), torch.Tensor.data_ptr
    w, b = data[1:3]

    def place():
        return (_layout(data[0], ld_x, first), _layout(data[3], ld_x, first), _layout(data[4], ld_dy, first))

    outs = []
    for in_place in (False, True):
        x, res, dy = place()
        y = _layout(torch.zeros_like(data[0]), ld_x, first)
        xo = x if in_place else _layout(torch.zeros_like(data[0]), ld_x, first)
        mean, rstd = (torch.empty(rows, device=cuda_device) for _ in range(2))
        _native.check(_native.lib.fab_layernorm(
            ptr(x), ptr(res), ptr(w), ptr(b), ptr(y), ptr(xo), ptr(mean), ptr(rstd), rows, cols, ld_x, ld_x, ld_x, ld_x, EPS,
            dt, dt, stream), "fab_layernorm")
        outs.append((y, mean, rstd, xo))
    _check_forward(data[0], w, b, outs[0], data[3])
    assert all(torch.equal(p, q) for p, q in zip(*outs))
    mean, rstd, x = outs[0][1:4]

    need = ctypes.c_size_t(0)
    _native.check(_native.lib.fab_layernorm_bwd_workspace(rows, cols, ctypes.byref(need)), "workspace")

    def backward(over):
        _, res, dy = place()
        # the out-of-place dx lies as the tensor does that the in-place one replaces
        dx = _layout(torch.zeros_like(data[0]), *((ld_x, first) if over.endswith("dres") else (ld_dy, first)))
        dx = {"dy": dy, "dres": res}.get(over, dx)
        ws = torch.full((need.value,), 255, device=cuda_device, dtype=torch.uint8)
        dw, db = torch.empty_like(w), torch.empty_like(w)
        _native.check(_native.lib.fab_layernorm_bwd(
            ptr(dy), ptr(x), ptr(w), ptr(mean), ptr(rstd), ptr(res), ptr(dx), ptr(dw), ptr(db), ptr(ws), need.value, rows,
            cols, ld_dy, ld_x, ld_x, dx.stride(0), dt, dt, stream), "fab_layernorm_bwd")
        return dx, dw, db

    for over in ("dy", "dres"):
        want, got = backward("like " + over), backward(over)
        _check_backward(data[4], x, w, mean, rstd, want, data[3])
        for name, p, q in zip(("dx", "dw", "db"), want, got):
            assert torch.equal(p, q), f"dx over {over}: {name}"
