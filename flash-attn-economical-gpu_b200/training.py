"""Operators for training a transformer block around the attention kernels, and their autograd forms.

Plain calls: `layernorm_forward` / `layernorm_backward` (with the residual add and the weight's and bias's
gradients), `rope_multi_axis` (rotary embedding with several position axes, both directions); the attention's
backward is `flash_atten.attention_backward` / `attention_backward_varlen`.  Differentiable calls: `attention`,
`attention_varlen`, `layernorm`, `rope`, which run the same kernels in both passes.  CUDA tensors only, like the
rest of the package.  No counterpart in the reference, which has no backward pass.
"""
from __future__ import annotations

import ctypes
import functools
import struct

import torch

import _native
from flash_atten import (
    _check_offsets,
    _require_cuda_tensor,
    attention_backward,
    attention_backward_varlen,
    attention_forward,
    attention_forward_varlen,
)


_DTYPES = {torch.float16: _native.FAB_DTYPE_F16, torch.bfloat16: _native.FAB_DTYPE_BF16, torch.float32: _native.FAB_DTYPE_F32}


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """`t` as [rows, cols] with unit column stride (a view where its strides allow it)."""
    if t.ndim != 2:
        t = t.reshape(-1, cols)
    if t.stride(1) != 1 and cols > 1:
        t = t.contiguous()
    return t


def _check_norm_tensor(what: str, name: str, t, like: torch.Tensor) -> None:
    _require_cuda_tensor(name, t)
    if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{what}: {name} must match x's shape, dtype and device")


def _check_norm_weight(what: str, name: str, t, x: torch.Tensor) -> None:
    _require_cuda_tensor(name, t)
    if tuple(t.shape) != (x.shape[-1],) or t.device != x.device:
        raise ValueError(f"{what}: {name} must have shape {(x.shape[-1],)} on x's device")
    if t.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"{what}: {name} must be {x.dtype} or float32, got {t.dtype}")


def _check_norm_input(what: str, x) -> None:
    _require_cuda_tensor("x", x)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: x must have at least one column")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what}: x must be float16, bfloat16 or float32, got {x.dtype}")


def layernorm_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, eps: float = 1e-5,
                      residual: torch.Tensor | None = None):
    """Layer norm over the last dim: (y, mean, rstd), or (y, mean, rstd, x + residual) with a residual.

    The sum x + residual is rounded to x's type and the norm is of the rounded sum.  mean and rstd (float32, one
    per row) are what layernorm_backward needs.  float16, bfloat16 or float32; weight and bias in x's type or
    float32, both the same.
    """
    what = "layernorm_forward"
    _check_norm_input(what, x)
    _check_norm_weight(what, "weight", weight, x)
    if bias is not None:
        _check_norm_weight(what, "bias", bias, x)
        if bias.dtype != weight.dtype:
            raise ValueError(f"{what}: weight and bias must share one dtype")
    if residual is not None:
        _check_norm_tensor(what, "residual", residual, x)
    shape, dev = x.shape, x.device
    cols = shape[-1]
    x2 = _rows(x, cols)
    rows = x2.shape[0]
    y = x.new_empty(shape)
    mean, rstd = x.new_empty(shape[:-1], dtype=torch.float32), x.new_empty(shape[:-1], dtype=torch.float32)
    w, b = weight.contiguous(), bias.contiguous() if bias is not None else None
    if residual is not None:
        r2, total = _rows(residual, cols), x.new_empty(shape)
        r_ptr, r_ld, total_ptr = r2.data_ptr(), r2.stride(0), total.data_ptr()
    else:
        r_ptr, r_ld, total_ptr = None, 0, None
    with _native.on_device(dev):
        rc = _native.lib.fab_layernorm(
            x2.data_ptr(), r_ptr, w.data_ptr(), b.data_ptr() if b is not None else None, y.data_ptr(), total_ptr,
            mean.data_ptr(), rstd.data_ptr(), rows, cols, x2.stride(0), r_ld, cols, cols, eps, _DTYPES[x.dtype],
            _DTYPES[weight.dtype], _native.current_stream_handle(dev))
    _native.check(rc, what)
    return (y, mean, rstd) if residual is None else (y, mean, rstd, total)


def layernorm_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor,
                       rstd: torch.Tensor, *, dresidual: torch.Tensor | None = None):
    """(dx, dweight, dbias) of layernorm_forward.

    x is what was normalised (with a residual, the returned sum); `dresidual` is a gradient that reaches x past
    the norm and is added to dx.  The gradient of a residual input equals dx.  dweight and dbias are summed in
    float32 in a fixed order and returned in the weight's type.
    """
    what = "layernorm_backward"
    _check_norm_input(what, x)
    _check_norm_weight(what, "weight", weight, x)
    _check_norm_tensor(what, "dy", dy, x)
    if dresidual is not None:
        _check_norm_tensor(what, "dresidual", dresidual, x)
    for name, t in (("mean", mean), ("rstd", rstd)):
        _require_cuda_tensor(name, t)
        if t.dtype != torch.float32 or t.shape != x.shape[:-1] or t.device != x.device:
            raise ValueError(f"{what}: {name} must be float32 with shape {tuple(x.shape[:-1])}")
    shape, dev = x.shape, x.device
    cols = shape[-1]
    x2, dy2 = _rows(x, cols), _rows(dy, cols)
    rows = x2.shape[0]
    dx, dw, db = x.new_empty(shape), weight.new_empty(cols), weight.new_empty(cols)
    w, mean, rstd = weight.contiguous(), mean.contiguous(), rstd.contiguous()
    if dresidual is not None:
        r2 = _rows(dresidual, cols)
        r_ptr, r_ld = r2.data_ptr(), r2.stride(0)
    else:
        r_ptr, r_ld = None, 0
    need = _norm_workspace(rows, cols)
    ws = torch.empty(need, device=dev, dtype=torch.uint8)
    with _native.on_device(dev):
        rc = _native.lib.fab_layernorm_bwd(
            dy2.data_ptr(), x2.data_ptr(), w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), r_ptr, dx.data_ptr(),
            dw.data_ptr(), db.data_ptr(), ws.data_ptr(), need, rows, cols, dy2.stride(0), x2.stride(0), r_ld, cols,
            _DTYPES[x.dtype], _DTYPES[weight.dtype], _native.current_stream_handle(dev))
    _native.check(rc, what)
    return dx, dw, db


@functools.lru_cache(maxsize=256)
def _norm_workspace(rows: int, cols: int) -> int:
    need = ctypes.c_size_t(0)
    _native.check(_native.lib.fab_layernorm_bwd_workspace(rows, cols, ctypes.byref(need)), "layernorm_backward")
    return need.value


def rope_multi_axis(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, cos: torch.Tensor,
                    sin: torch.Tensor, sections, *, inverse: bool = False,
                    out: tuple[torch.Tensor, torch.Tensor | None] | None = None):
    """Rotate-half rotary embedding with several position axes: (q', k').

    q [tokens, heads_q, D] and k [tokens, heads_k, D] (or None) may be column views of one packed projection.
    The first 2 * sum(sections) columns of a head are pairs (i, half + i): the first sections[0] pairs turn with
    positions[0] (say time), the next sections[1] with positions[1] (height), and so on; later columns are
    copied.  positions is [axes, tokens] (int32 or int64) and indexes the rows of the float32 tables cos / sin
    [rows, sum(sections)]; a position outside the table gives NaN.  `inverse` turns the other way, which is the
    backward pass.  `out` = (q, k) rotates in place.
    """
    what = "rope_multi_axis"
    tensors = [("q", q), ("positions", positions), ("cos", cos), ("sin", sin)] + ([("k", k)] if k is not None else [])
    for name, t in tensors:
        _require_cuda_tensor(name, t)
    if any(t.device != q.device for _, t in tensors):
        raise ValueError(f"{what}: all tensors must be on one device")
    if q.ndim != 3 or (k is not None and (k.ndim != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2])):
        raise ValueError(f"{what} expects q and k with shape [tokens, heads, head_dim]")
    if k is not None and k.dtype != q.dtype:
        raise ValueError(f"{what}: q and k must share one dtype")
    sections = tuple(int(s) for s in sections)
    T, Hq, D = q.shape
    half = sum(sections)
    if not 1 <= len(sections) <= _native.MAX_ROPE_AXES or min(sections) < 0 or half < 1 or 2 * half > D:
        raise ValueError(f"{what}: sections must be 1 to {_native.MAX_ROPE_AXES} pair counts that sum to at most "
                         f"head_dim / 2, got {sections} for head_dim {D}")
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) != (len(sections), T):
        raise ValueError(f"{what}: positions must be int32 or int64 with shape {(len(sections), T)}")
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.shape != sin.shape or cos.ndim != 2 or \
            cos.shape[1] != half:
        raise ValueError(f"{what}: cos and sin must be float32 tables with {half} columns")
    if q.dtype not in _DTYPES:
        raise ValueError(f"{what}: unsupported dtype {q.dtype}; expected float16, bfloat16 or float32")
    qc = q if q.stride(2) == 1 else q.contiguous()
    kc = k if k is None or k.stride(2) == 1 else k.contiguous()
    if out is None:
        out = (q.new_empty(q.shape), k.new_empty(k.shape) if k is not None else None)
    else:
        for name, t, like in (("out[0]", out[0], q), ("out[1]", out[1], k)):
            if like is None:
                continue
            _require_cuda_tensor(name, t)
            if t.shape != like.shape or t.dtype != like.dtype or t.device != q.device or t.stride(2) != 1:
                raise ValueError(f"{what}: {name} must match its input's shape, dtype and device, with unit stride "
                                 "along the head")
    cos, sin = cos.contiguous(), sin.contiguous()
    qo, ko = out
    if k is not None:
        k_ptrs, heads_k, k_strides = (kc.data_ptr(), ko.data_ptr()), k.shape[1], (*kc.stride()[:2], *ko.stride()[:2])
    else:
        k_ptrs, heads_k, k_strides = (0, 0), 0, (0, 0, 0, 0)
    p = _native.FabRopeAxesParams.from_buffer_copy(_ROPE_RECORD.pack(
        qc.data_ptr(), k_ptrs[0], qo.data_ptr(), k_ptrs[1], positions.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        *qc.stride()[:2], *k_strides[:2], *qo.stride()[:2], *k_strides[2:], *positions.stride(), T, Hq, heads_k, D,
        len(sections), *sections, *(0,) * (_native.MAX_ROPE_AXES - len(sections)), cos.shape[0],
        positions.dtype is torch.int64, bool(inverse), _DTYPES[q.dtype]))
    with _native.on_device(q.device):
        rc = _native.lib.fab_rope_axes(ctypes.byref(p), _native.current_stream_handle(q.device))
    _native.check(rc, what)
    return out


# fab_rope_axes_params as one packed record.
_ROPE_RECORD = struct.Struct("7P10q13i4x")
assert _ROPE_RECORD.size == ctypes.sizeof(_native.FabRopeAxesParams)


# ---------------------------------------------------------------- autograd
class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, causal, sm_scale):
        o, lse = attention_forward(q, k, v, causal=causal, sm_scale=sm_scale, return_lse=True)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.causal, ctx.sm_scale = causal, sm_scale
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, o, lse = ctx.saved_tensors
        grads = attention_backward(dout, q, k, v, o, lse, causal=ctx.causal, sm_scale=ctx.sm_scale)
        return (*grads, None, None)


class _AttentionVarlen(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, max_q, max_k, causal, sm_scale):
        o, lse = attention_forward_varlen(q, k, v, cu_q, cu_k, max_q, max_k, causal=causal, sm_scale=sm_scale,
                                          return_lse=True)
        ctx.save_for_backward(q, k, v, o, lse, cu_q, cu_k)
        ctx.rest = max_q, max_k, causal, sm_scale
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, o, lse, cu_q, cu_k = ctx.saved_tensors
        max_q, max_k, causal, sm_scale = ctx.rest
        grads = attention_backward_varlen(dout, q, k, v, o, lse, cu_q, cu_k, max_q, max_k, causal=causal,
                                          sm_scale=sm_scale)
        return (*grads, None, None, None, None, None, None)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual):
        y, mean, rstd, *total = layernorm_forward(x, weight, bias, eps=eps, residual=residual)
        ctx.save_for_backward(total[0] if total else x, weight, mean, rstd)
        ctx.has_bias, ctx.has_residual = bias is not None, residual is not None
        ctx.set_materialize_grads(False)  # an unused sum costs no pass over zeros
        return (y, total[0]) if total else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dtotal=None):
        x, weight, mean, rstd = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros_like(x)
        dx, dw, db = layernorm_backward(dy, x, weight, mean, rstd, dresidual=dtotal)
        return dx, dw, db if ctx.has_bias else None, None, dx if ctx.has_residual else None


class _Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, cos, sin, sections):
        ctx.save_for_backward(positions, cos, sin)
        ctx.sections = sections
        return rope_multi_axis(q, k, positions, cos, sin, sections)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        dq, dk = rope_multi_axis(dq, dk, *ctx.saved_tensors, ctx.sections, inverse=True)
        return dq, dk, None, None, None, None


def _check_trainable(what: str, q) -> None:
    # The forward pass also takes float32, which the backward pass does not.
    _require_cuda_tensor("q", q)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{what}: q, k and v must be float16 or bfloat16, got {q.dtype}")


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = False,
              sm_scale: float | None = None) -> torch.Tensor:
    """Differentiable flash_atten.attention_forward (float16 or bfloat16)."""
    _check_trainable("attention", q)
    return _Attention.apply(q, k, v, causal, sm_scale)


def attention_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                     cu_seqlens_k: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int, *, causal: bool = False,
                     sm_scale: float | None = None) -> torch.Tensor:
    """Differentiable flash_atten.attention_forward_varlen (float16 or bfloat16)."""
    _check_trainable("attention_varlen", q)
    _check_offsets("attention_varlen", cu_seqlens_q, cu_seqlens_k, q.device)
    return _AttentionVarlen.apply(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, causal, sm_scale)


def layernorm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, eps: float = 1e-5,
              residual: torch.Tensor | None = None):
    """Differentiable layernorm_forward: y, or (y, x + residual) with a residual."""
    return _LayerNorm.apply(x, weight, bias, eps, residual)


def rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
         sections) -> tuple[torch.Tensor, torch.Tensor]:
    """Differentiable rope_multi_axis (in q and k; the tables are constants)."""
    return _Rope.apply(q, k, positions, cos, sin, tuple(sections))


__all__ = [
    "attention",
    "attention_varlen",
    "layernorm",
    "layernorm_forward",
    "layernorm_backward",
    "rope",
    "rope_multi_axis",
]
