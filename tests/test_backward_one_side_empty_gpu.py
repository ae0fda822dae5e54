"""attention_backward where one side has no rows and the other many: zero gradients, whatever the length."""
from __future__ import annotations

import pytest
import torch

import training
from flash_atten import attention_backward, attention_backward_varlen, attention_forward, attention_forward_varlen
from test_attention_backward_gpu import _inputs, _no_device_errors, _packed_inputs  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M, N", [(0, 1000), (0, 1200), (0, 9000), (1000, 0), (1200, 0), (9000, 0)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bfloat16", "float16"])
def test_dense(M, N, D, dtype, cuda_device):
    dout, q, k, v = _inputs(1, 4, 2, M, N, D, dtype, cuda_device, 1)
    o, lse = attention_forward(q, k, v, return_lse=True)
    for causal in (False, True):
        grads = attention_backward(dout, q, k, v, o, lse, causal=causal)
        assert all(g.shape == t.shape and (g == 0).all() for g, t in zip(grads, (q, k, v)))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    training.attention(*leaves).backward(dout)
    assert all(t.grad.shape == t.shape and (t.grad == 0).all() for t in leaves)


@pytest.mark.parametrize("lq, lk", [((0, 0), (1500, 3000)), ((1500, 3000), (0, 0)), ((0, 3000), (3000, 0))])
@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 256)])
def test_packed(lq, lk, dtype, D, cuda_device):
    """No sequence has both; with rows outside every sequence, so that no tensor is empty."""
    dout, q, k, v, cu_q, cu_k = _packed_inputs((7, *lq, 5), (3, *lk, 9), 4, 2, D, dtype, cuda_device, 3)
    cu_q, cu_k = cu_q[1:4].contiguous(), cu_k[1:4].contiguous()
    o, lse = attention_forward_varlen(q, k, v, cu_q, cu_k, max(lq), max(lk), return_lse=True)
    grads = attention_backward_varlen(dout, q, k, v, o, lse, cu_q, cu_k, max(lq), max(lk))
    assert all((g == 0).all() for g in grads)
