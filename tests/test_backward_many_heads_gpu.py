"""attention_backward over more (batch entry, head) pairs than one grid dimension of 65535 holds, as the forward takes.

Tolerances as derived in test_attention_backward_gpu.
"""
from __future__ import annotations

import pytest
import torch

import training
from flash_atten import attention_backward, attention_backward_varlen, attention_forward, attention_forward_varlen
from test_attention_backward_gpu import _assert_within, _inputs, _no_device_errors, _reference  # noqa: F401

pytestmark = pytest.mark.gpu

CASES = [
    # batch entries, heads, key/value heads, queries, keys, head dim
    (2049, 32, 4, 3, 5, 64, torch.bfloat16),
    (1500, 32, 16, 5, 3, 64, torch.float16),   # 48000 query heads, 72000 with the key/value heads
    (70001, 1, 1, 2, 2, 64, torch.float16),
    (2100, 32, 32, 2, 3, 128, torch.bfloat16),
    (33000, 2, 2, 2, 1, 256, torch.bfloat16),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"B{c[0]}H{c[1]}/{c[2]}D{c[5]}{str(c[6])[6:]}")
def test_dense(case, cuda_device):
    B, Hq, Hkv, M, N, D, dtype = case
    dout, q, k, v = _inputs(B, Hq, Hkv, M, N, D, dtype, cuda_device, B)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    training.attention(*leaves, causal=True).backward(dout)
    q, k, v = (t.detach() for t in leaves)
    o, lse = attention_forward(q, k, v, causal=True, return_lse=True)
    got = attention_backward(dout, q, k, v, o, lse, causal=True)
    _assert_within(got, *_reference(dout, q, k, v, o, lse, True, D ** -0.5))
    assert all(torch.equal(t.grad, g) for t, g in zip(leaves, got))


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"B{c[0]}H{c[1]}/{c[2]}D{c[5]}{str(c[6])[6:]}")
def test_packed(case, cuda_device):
    """As many documents of one length as the dense batch has entries, with rows before and after all of them."""
    B, Hq, Hkv, M, N, D, dtype = case
    lead_q, lead_k, tail = 3, 130, 5
    g = torch.Generator(device=cuda_device).manual_seed(B)
    q, dout = (torch.randn(lead_q + B * M + tail, Hq, D, generator=g, device=cuda_device).to(dtype) for _ in range(2))
    k, v = (torch.randn(lead_k + B * N + tail, Hkv, D, generator=g, device=cuda_device).to(dtype) for _ in range(2))
    cu_q, cu_k = (torch.arange(B + 1, dtype=torch.int32, device=cuda_device) * n + a for n, a in ((M, lead_q), (N, lead_k)))
    o, lse = attention_forward_varlen(q, k, v, cu_q, cu_k, M, N, causal=True, return_lse=True)
    got = attention_backward_varlen(dout, q, k, v, o, lse, cu_q, cu_k, M, N, causal=True)

    def batch(t, lead, n):  # [batch, heads, rows, D] of the documents
        assert (t[:lead] == 0).all() and (t[lead + B * n:] == 0).all()
        return t[lead:lead + B * n].unflatten(0, (B, n)).transpose(1, 2)

    def inner(t, lead, n):
        return t[lead:lead + B * n].unflatten(0, (B, n)).transpose(1, 2)

    dense = [inner(t, lead_q, M) for t in (dout, q)] + [inner(t, lead_k, N) for t in (k, v)] + [inner(o, lead_q, M)]
    L = lse[:, lead_q:lead_q + B * M].unflatten(1, (B, M)).transpose(0, 1)
    grads = (batch(got[0], lead_q, M), batch(got[1], lead_k, N), batch(got[2], lead_k, N))
    _assert_within(grads, *_reference(*dense, L, True, D ** -0.5))
