"""Bounded waits of the attention backward and of layer norm's clusters that run out: an error status, no hang.

As in test_bounded_wait_gpu: with a limit of 2 ms something that a kernel waits for is withheld (the last bytes of its
streamed tiles, a CTA's sums of a row), so that a wait runs out for real; nothing faults or spins without end.  The kernel returns, the host
reads a code and raises, and the next call gives the bits of the call before.
"""
from __future__ import annotations

import pytest
import torch

import _native
import training
from flash_atten import attention_backward, attention_backward_varlen, attention_forward, attention_forward_varlen

pytestmark = pytest.mark.gpu

# The warps that the missing tile stops wait for different things (the tile, its product, a free slot, what the others
# make of it, the next item), from about the same time: any of them may run out first.
PIPELINE_CODES = (1, 2, 3, 4, 5, 6, 7, 8, 12)


def _run_out(call, starve, codes):
    """`call` with something withheld ends with one of `codes`, then works again."""
    want = call()
    torch.cuda.synchronize()
    assert _native.device_error() == 0
    try:
        _native.set_wait_limit_ns(2_000_000)
        starve()
        call()
        torch.cuda.synchronize()  # the kernels returned: no hang
        assert _native.device_error() in codes
        call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="bounded wait"):
            _native.raise_on_device_error()
    finally:
        _native.starve_kv_load(-1)
        _native.starve_row_sums(-1)
        _native.set_wait_limit_ns(0)
    got = call()
    torch.cuda.synchronize()
    assert _native.device_error() == 0
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype, D, S", [(torch.bfloat16, 64, 1000), (torch.float16, 128, 1000), (torch.bfloat16, 256, 500),
                                         (torch.bfloat16, 128, 3500)])
def test_attention_backward(dtype, D, S, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(3)
    q, k, v, dout = (torch.randn(1, 2, S, D, generator=g, device=cuda_device).to(dtype) for _ in range(4))
    o, lse = attention_forward(q, k, v, causal=True, return_lse=True)
    _run_out(lambda: attention_backward(dout, q, k, v, o, lse, causal=True), lambda: _native.starve_kv_load(0),
             PIPELINE_CODES)


def test_packed_attention_backward(cuda_device):
    """With ragged tiles, which their producer itself waits for."""
    g = torch.Generator(device=cuda_device).manual_seed(4)
    q, k, v, dout = (torch.randn(400, 2, 64, generator=g, device=cuda_device).to(torch.bfloat16) for _ in range(4))
    cu = torch.tensor([0, 100, 400], dtype=torch.int32, device=cuda_device)
    o, lse = attention_forward_varlen(q, k, v, cu, cu, 300, 300, return_lse=True)
    _run_out(lambda: attention_backward_varlen(dout, q, k, v, o, lse, cu, cu, 300, 300), lambda: _native.starve_kv_load(0),
             PIPELINE_CODES)


@pytest.mark.parametrize("row", [0, 1, 150])
@pytest.mark.parametrize("cols", [12288, 12289, 60000])
def test_layernorm_clusters(cols, row, cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(5)
    x, dy = (torch.randn(200, cols, generator=g, device=cuda_device).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(cols, device=cuda_device)
    _, mean, rstd = training.layernorm_forward(x, w)
    if cols % 8:  # few rows on the 16-byte grid may run without clusters forward
        _run_out(lambda: training.layernorm_forward(x, w), lambda: _native.starve_row_sums(row), (14,))
    _run_out(lambda: training.layernorm_backward(dy, x, w, mean, rstd), lambda: _native.starve_row_sums(row), (14,))


def test_layernorm_clusters_forward(cuda_device):
    g = torch.Generator(device=cuda_device).manual_seed(6)
    x = torch.randn(2000, 12288, generator=g, device=cuda_device).to(torch.bfloat16)
    w = torch.ones(12288, device=cuda_device)
    _run_out(lambda: training.layernorm_forward(x, w, residual=x), lambda: _native.starve_row_sums(1500), (14,))
