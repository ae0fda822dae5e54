"""attention_backward for operands whose head dim is not the innermost one in memory, which the forward takes too.

The gradients are the formula's whatever the operands' strides (tolerances as derived in test_attention_backward_gpu),
and those of the same values laid out contiguously, bit for bit.
"""
from __future__ import annotations

import pytest
import torch

import training
from flash_atten import attention_backward, attention_backward_varlen, attention_forward, attention_forward_varlen
from test_attention_backward_gpu import _assert_within, _inputs, _no_device_errors, _packed_inputs, _reference  # noqa: F401

pytestmark = pytest.mark.gpu

WHICH = ["q", "k", "v", "qkv"]


def _rows_innermost(t):
    """The same values with the row (second to last, or first of three) dim innermost."""
    dim = -2 if t.ndim == 4 else 0
    u = t.transpose(dim, -1).contiguous().transpose(dim, -1)
    assert u.stride(dim) == 1 and u.stride(-1) > 1
    return u


@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 72), (torch.bfloat16, 33)])
@pytest.mark.parametrize("which", WHICH)
def test_dense(which, dtype, D, cuda_device):
    dout, *qkv = _inputs(2, 4, 2, 100, 120, D, dtype, cuda_device, D)
    o, lse = attention_forward(*qkv, causal=True, return_lse=True)
    want = attention_backward(dout, *qkv, o, lse, causal=True)
    args = [_rows_innermost(t) if n in which else t for n, t in zip("qkv", qkv)]
    got = attention_backward(dout, *args, o, lse, causal=True)
    _assert_within(got, *_reference(dout, *qkv, o, lse, True, D ** -0.5))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(g.shape == t.shape for g, t in zip(got, qkv))


@pytest.mark.parametrize("which", WHICH)
def test_out_and_its_gradient(which, cuda_device):
    """dout and out in such a layout, one at a time and with q, k and v."""
    dout, *qkv = _inputs(1, 2, 1, 90, 70, 64, torch.float16, cuda_device, 3)
    o, lse = attention_forward(*qkv, return_lse=True)
    want = attention_backward(dout, *qkv, o, lse)
    args = [_rows_innermost(t) if n in which else t for n, t in zip("qkv", qkv)]
    for g, out in ((_rows_innermost(dout), o), (dout, _rows_innermost(o)), (_rows_innermost(dout), _rows_innermost(o))):
        assert all(torch.equal(a, b) for a, b in zip(attention_backward(g, *args, out, lse), want))


@pytest.mark.parametrize("which", WHICH)
def test_packed(which, cuda_device):
    lq, lk = (40, 1, 77), (60, 9, 77)
    dout, *rest = _packed_inputs(lq, lk, 4, 2, 64, torch.bfloat16, cuda_device, 8)
    qkv, cu = rest[:3], (*rest[3:], max(lq), max(lk))
    o, lse = attention_forward_varlen(*qkv, *cu, causal=True, return_lse=True)
    want = attention_backward_varlen(dout, *qkv, o, lse, *cu, causal=True)
    args = [_rows_innermost(t) if n in which else t for n, t in zip("qkv", qkv)]
    got = attention_backward_varlen(dout, *args, o, lse, *cu, causal=True)
    assert all(torch.equal(a, b) and a.shape == b.shape for a, b in zip(got, want))


@pytest.mark.parametrize("which", WHICH)
def test_autograd(which, cuda_device):
    """What the forward pass accepts the backward pass does not refuse."""
    dout, *qkv = _inputs(1, 4, 2, 50, 60, 64, torch.bfloat16, cuda_device, 6)
    o, lse = attention_forward(*qkv, causal=True, return_lse=True)
    want = attention_backward(dout, *qkv, o, lse, causal=True)
    leaves = [_rows_innermost(t).detach().requires_grad_() if n in which else t.clone().requires_grad_()
              for n, t in zip("qkv", qkv)]
    training.attention(*leaves, causal=True).backward(dout)
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))

    dout, *rest = _packed_inputs((30, 70), (30, 70), 2, 1, 64, torch.float16, cuda_device, 10)
    qkv, cu = rest[:3], (*rest[3:], 70, 70)
    o, lse = attention_forward_varlen(*qkv, *cu, return_lse=True)
    want = attention_backward_varlen(dout, *qkv, o, lse, *cu)
    leaves = [_rows_innermost(t).detach().requires_grad_() if n in which else t.clone().requires_grad_()
              for n, t in zip("qkv", qkv)]
    training.attention_varlen(*leaves, *cu).backward(dout)
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
