"""Attention, forward and backward, of a single row, head and batch entry whose head dim is off the 16-byte grid.

No stride of such an output is ever followed, so none may be the reason to refuse it.  Tolerances of the gradients as
derived in test_attention_backward_gpu; o is rounded once from fp32 sums of P rounded to the type: 2 u max|v|.
"""
from __future__ import annotations

import pytest
import torch

import training
from flash_atten import attention_forward, attention_forward_varlen
from test_attention_backward_gpu import U, _assert_within, _inputs, _no_device_errors, _reference  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bfloat16", "float16"])
@pytest.mark.parametrize("D", [1, 7, 33, 100, 255])
@pytest.mark.parametrize("N", [1, 40])
def test_one_query_of_one_head(N, D, dtype, cuda_device):
    dout, q, k, v = _inputs(1, 1, 1, 1, N, D, dtype, cuda_device, N + D)
    o, lse = attention_forward(q, k, v, return_lse=True)
    P = torch.softmax(q.double() @ k.double().transpose(-1, -2) * D ** -0.5, -1)
    assert ((o.double() - P @ v.double()).abs() <= 2 * U[dtype] * v.double().abs().amax()).all()
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    training.attention(*leaves).backward(dout)
    _assert_within([t.grad for t in leaves], *_reference(dout, q, k, v, o, lse, False, D ** -0.5))

    packed = [t[0].transpose(0, 1) for t in (q, k, v)]
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device=cuda_device) for n in (1, N))
    assert torch.equal(attention_forward_varlen(*packed, cu_q, cu_k, 1, N)[:, 0], o[0, 0])
    leaves = [t.clone().requires_grad_() for t in packed]
    training.attention_varlen(*leaves, cu_q, cu_k, 1, N).backward(dout[0].transpose(0, 1))
    _assert_within([t.grad.transpose(0, 1)[None] for t in leaves], *_reference(dout, q, k, v, o, lse, False, D ** -0.5))


def test_an_output_with_an_odd_stride_of_one_element(cuda_device):
    """A caller's `out` whose only odd stride belongs to a dim of one element."""
    _, q, k, v = _inputs(1, 2, 2, 50, 60, 64, torch.bfloat16, cuda_device, 2)
    out = torch.empty(2 * 50 * 64 + 3, device=cuda_device, dtype=q.dtype).as_strided((1, 2, 50, 64), (2 * 50 * 64 + 3, 50 * 64, 64, 1))
    assert torch.equal(attention_forward(q, k, v, out=out), attention_forward(q, k, v)) and out.isfinite().all()
