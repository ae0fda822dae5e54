"""Calls from a thread that has made no CUDA call yet (autograd runs a backward pass in such threads): the result is the
main thread's, bit for bit.

Every call is made once on the main thread first, so that the allocator has memory of all sizes and the fresh thread's
first CUDA call is the library's own.
"""
from __future__ import annotations

import threading

import pytest
import torch

import _native
import training
from flash_atten import attention_backward, attention_backward_varlen, attention_forward, attention_forward_varlen
from mma import matmul

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    yield
    torch.cuda.synchronize()
    assert _native.device_error() == 0


def _in_a_fresh_thread(call):
    got = []

    def body():
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001 - handed to the main thread
            got.append(e)

    thread = threading.Thread(target=body)
    thread.start()
    thread.join()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


def _data(dev, *shapes):
    g = torch.Generator(device=dev).manual_seed(5)
    return [torch.randn(*s, generator=g, device=dev).to(torch.bfloat16) for s in shapes]


def _dense(dev):
    q, k, v, dout = _data(dev, (1, 4, 150, 64), (1, 2, 130, 64), (1, 2, 130, 64), (1, 4, 150, 64))
    o, lse = attention_forward(q, k, v, causal=True, return_lse=True)
    return (lambda: attention_forward(q, k, v, causal=True, return_lse=True),
            lambda: attention_backward(dout, q, k, v, o, lse, causal=True))


def _packed(dev):
    q, k, v, dout = _data(dev, (150, 4, 64), (150, 2, 64), (150, 2, 64), (150, 4, 64))
    cu = torch.tensor([0, 40, 150], dtype=torch.int32, device=dev)
    o, lse = attention_forward_varlen(q, k, v, cu, cu, 110, 110, causal=True, return_lse=True)
    return (lambda: attention_forward_varlen(q, k, v, cu, cu, 110, 110, causal=True, return_lse=True),
            lambda: attention_backward_varlen(dout, q, k, v, o, lse, cu, cu, 110, 110, causal=True))


def _rest(dev):
    a, b, x, w, q = _data(dev, (256, 192), (192, 320), (50, 640), (640,), (50, 4, 64))
    y, mean, rstd = training.layernorm_forward(x, w)
    table = torch.randn(60, 32, device=dev)
    pos = torch.arange(50, device=dev)[None]
    return (lambda: (matmul(a, b),), lambda: training.layernorm_forward(x, w),
            lambda: training.layernorm_backward(y, x, w, mean, rstd),
            lambda: training.rope_multi_axis(q, None, pos, table, table, (32,))[:1])


@pytest.mark.parametrize("make, which", [(_dense, 0), (_dense, 1), (_packed, 0), (_packed, 1), (_rest, 0), (_rest, 1),
                                         (_rest, 2), (_rest, 3)],
                         ids=["forward", "backward", "packed_forward", "packed_backward", "matmul", "norm", "norm_backward",
                              "rotary"])
def test_same_result(make, which, cuda_device):
    call = make(cuda_device)[which]
    want = call()
    call()
    torch.cuda.synchronize()
    got = _in_a_fresh_thread(call)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
