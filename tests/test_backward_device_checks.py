"""Workspaces and offsets that the attention backward's kernels could not use safely are refused on the host.

The tensors are fakes (sizes, strides and devices without memory), so that nothing here can reach a GPU.
"""
from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import training
from flash_atten import attention_backward, attention_backward_varlen, attention_backward_workspace_bytes

NEED = attention_backward_workspace_bytes((1, 2, 64, 64), (1, 2, 64, 64), torch.bfloat16)
NEED_PACKED = attention_backward_workspace_bytes((64, 2, 64), (64, 2, 64), torch.bfloat16, packed_batch=2)


@pytest.fixture
def fakes():
    with FakeTensorMode():
        yield


def _bytes(n, device="cuda:0"):
    return torch.empty(n, dtype=torch.uint8, device=device)


WORKSPACES = {
    "expanded": lambda n: _bytes(1).expand(n),
    "overlapping": lambda n: _bytes(n).as_strided((2, n), (n // 2, 1)),
    "strided": lambda n: _bytes(2 * n)[::2],
    "transposed": lambda n: _bytes(n).view(2, n // 2).t(),
    "another device": lambda n: _bytes(n, "cuda:1"),
    "host": lambda n: _bytes(n, "cpu"),
}


@pytest.mark.parametrize("kind", WORKSPACES)
def test_workspaces(kind, fakes):
    x, lse = torch.empty(1, 2, 64, 64, device="cuda:0", dtype=torch.bfloat16), torch.empty(1, 2, 64, device="cuda:0")
    with pytest.raises(ValueError, match="workspace must be"):
        attention_backward(x, x, x, x, x, lse, workspace=WORKSPACES[kind](NEED))
    cu = torch.empty(3, dtype=torch.int32, device="cuda:0")
    with pytest.raises(ValueError, match="workspace must be"):
        attention_backward_varlen(*[x[0].transpose(0, 1)] * 5, lse[0], cu, cu, 64, 64, workspace=WORKSPACES[kind](NEED_PACKED))


@pytest.mark.parametrize("which", ["q", "k", "qk"])
@pytest.mark.parametrize("device", ["cuda:1", "cpu"])
def test_offsets(which, device, fakes):
    x, lse = torch.empty(64, 2, 64, device="cuda:0", dtype=torch.bfloat16), torch.empty(2, 64, device="cuda:0")
    cu = [torch.empty(3, dtype=torch.int32, device=device if n in which else "cuda:0") for n in "qk"]
    with pytest.raises(ValueError, match=f"cu_seqlens_{which[0]} must be"):
        attention_backward_varlen(x, x, x, x, x, lse, *cu, 64, 64)
    with pytest.raises(ValueError, match=f"cu_seqlens_{which[0]} must be"):
        training.attention_varlen(x, x, x, *cu, 64, 64)
