"""attention_backward / attention_backward_varlen on the GPU against the formula in 64 bits.

Tolerance, element by element.  P and dS are rounded to the operand type (unit roundoff u: 2^-8 bf16, 2^-11 fp16)
before the products that sum them, and the result is rounded once more, so with exact fp32 arithmetic
    |dv - ref| <= u * (P^T |dout|) + u |ref|
    |dq - ref| <= u * c (|dS| |K|) + u |ref|        (dk likewise)
(each with a factor 1 + u on top).  The fp32 arithmetic of P and dS (an exponential of relative error about 2^-22 of
a score of fp32 error, a difference dP - delta of sums over head_dim) adds at most 2^-16 of the same sums taken over
magnitudes, P (|dout| |V|^T + rowsum |dout o|).  An fp16 result may also be subnormal: 2^-25 absolute.
The 64-bit reference takes the o and lse that the kernel was given, rounded as they are.
"""
from __future__ import annotations

import pytest
import torch

import _native
import training
from flash_atten import (
    attention_backward,
    attention_backward_varlen,
    attention_backward_workspace_bytes,
    attention_forward,
    attention_forward_varlen,
)

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    yield
    torch.cuda.synchronize()
    assert _native.device_error() == 0, "a kernel gave up on a bounded wait"


def _reference(dout, q, k, v, o, lse, causal, scale):
    """Gradients of one dense batch in 64 bits and the tolerances derived above."""
    B, Hq, M, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    g = Hq // Hkv
    u = U[q.dtype]
    Q, dO, O = (t.double() for t in (q, dout, o))
    K, V = (t.double().repeat_interleave(g, 1) for t in (k, v))
    s = Q @ K.transpose(-1, -2) * scale
    mask = torch.ones(M, N, dtype=torch.bool, device=q.device)
    if causal:
        mask = mask.tril()
    P = torch.where(mask, torch.exp(s - lse.double()[..., None]), 0.0)
    dP = dO @ V.transpose(-1, -2)
    delta = (dO * O).sum(-1, keepdim=True)
    dS = torch.where(mask, P * (dP - delta), 0.0)
    size = P * (dO.abs() @ V.abs().transpose(-1, -2) + (dO * O).abs().sum(-1, keepdim=True))

    def shared(t):
        return t.unflatten(1, (Hkv, g)).sum(2)

    c = abs(scale)
    refs = (scale * dS @ K, shared(scale * dS.transpose(-1, -2) @ Q), shared(P.transpose(-1, -2) @ dO))
    rough = (c * dS.abs() @ K.abs(), shared(c * dS.abs().transpose(-1, -2) @ Q.abs()),
             shared(P.transpose(-1, -2) @ dO.abs()))
    fine = (c * size @ K.abs(), shared(c * size.transpose(-1, -2) @ Q.abs()), rough[2])
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 1e-37
    tols = tuple((1 + u) * u * (r + ref.abs()) + 2.0 ** -16 * f + tiny for ref, r, f in zip(refs, rough, fine))
    return refs, tols


def _assert_within(got, refs, tols):
    for name, x, r, t in zip(("dq", "dk", "dv"), got, refs, tols):
        assert x.shape == r.shape, name
        worst = ((x.double() - r).abs() / t).max().item() if x.numel() else 0.0
        assert worst <= 1.0, f"{name}: {worst:.3f} of its tolerance"


def _inputs(B, Hq, Hkv, M, N, D, dtype, dev, seed, dscale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    return ((randn(B, Hq, M, D) * dscale).to(dtype), randn(B, Hq, M, D).to(dtype), randn(B, Hkv, N, D).to(dtype),
            randn(B, Hkv, N, D).to(dtype))


DENSE = [
    # B, Hq, Hkv, M, N, D, dtype, causal
    (1, 1, 1, 1, 1, 64, torch.bfloat16, True),
    (1, 2, 1, 1, 300, 128, torch.bfloat16, False),     # one query against many keys
    (2, 2, 2, 300, 1, 128, torch.float16, True),        # one key
    (2, 4, 2, 127, 127, 128, torch.bfloat16, True),
    (1, 4, 1, 128, 128, 128, torch.bfloat16, False),
    (1, 2, 2, 129, 257, 64, torch.float16, True),       # keys past the last query get zeros
    (1, 6, 2, 257, 129, 64, torch.bfloat16, True),      # queries past the last key
    (2, 7, 1, 200, 640, 128, torch.float16, False),
    (1, 2, 1, 513, 385, 256, torch.bfloat16, True),
    (1, 4, 4, 191, 65, 256, torch.float16, False),
    (1, 2, 2, 100, 90, 80, torch.bfloat16, True),       # padded head dims
    (1, 3, 1, 70, 150, 40, torch.float16, False),
    (1, 2, 1, 66, 130, 72, torch.bfloat16, True),
    (1, 2, 1, 77, 61, 33, torch.bfloat16, False),       # rows off the 16-byte grid
    (1, 1, 1, 33, 45, 1, torch.float16, True),
    (1, 2, 1, 140, 70, 201, torch.bfloat16, True),
    (3, 28, 4, 260, 260, 128, torch.bfloat16, True),
]


@pytest.mark.parametrize("case", DENSE, ids=lambda c: f"B{c[0]}H{c[1]}/{c[2]}M{c[3]}N{c[4]}D{c[5]}{str(c[6])[6:]}{'c' if c[7] else ''}")
def test_dense_matches_the_formula(case, cuda_device):
    B, Hq, Hkv, M, N, D, dtype, causal = case
    dout, q, k, v = _inputs(B, Hq, Hkv, M, N, D, dtype, cuda_device, M * N + D)
    o, lse = attention_forward(q, k, v, causal=causal, return_lse=True)
    got = attention_backward(dout, q, k, v, o, lse, causal=causal)
    refs, tols = _reference(dout, q, k, v, o, lse, causal, D ** -0.5)
    _assert_within(got, refs, tols)
    again = attention_backward(dout, q, k, v, o, lse, causal=causal)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("scale", [0.31, -0.2, 0.0])
def test_any_softmax_scale(scale, cuda_device):
    dout, q, k, v = _inputs(1, 2, 1, 150, 170, 64, torch.bfloat16, cuda_device, 3)
    o, lse = attention_forward(q, k, v, sm_scale=scale, return_lse=True)
    got = attention_backward(dout, q, k, v, o, lse, sm_scale=scale)
    _assert_within(got, *_reference(dout, q, k, v, o, lse, False, scale))


@pytest.mark.parametrize("scale", [-0.2, 0.0])
def test_causal_with_any_softmax_scale(scale, cuda_device):
    """Masked pairs stay out whatever the sign of the scale."""
    dout, q, k, v = _inputs(1, 2, 1, 200, 170, 64, torch.bfloat16, cuda_device, 4)
    o, lse = attention_forward(q, k, v, causal=True, sm_scale=scale, return_lse=True)
    got = attention_backward(dout, q, k, v, o, lse, causal=True, sm_scale=scale)
    _assert_within(got, *_reference(dout, q, k, v, o, lse, True, scale))


SLICED = [
    # few tiles of long sums, in parts that are joined; then many short items for each SM
    (1, 1, 1, 40, 5000, 64, torch.bfloat16, False),
    (1, 1, 1, 5000, 40, 128, torch.float16, False),
    (1, 2, 1, 2500, 2500, 128, torch.bfloat16, True),
    (1, 7, 1, 1100, 1100, 128, torch.bfloat16, True),
    (1, 1, 1, 1700, 1300, 256, torch.float16, True),
    (1, 2, 1, 90, 3333, 256, torch.bfloat16, False),
    (1, 1, 1, 2049, 2049, 96, torch.float16, False),
    (40, 24, 12, 130, 130, 64, torch.bfloat16, True),
    (24, 16, 16, 70, 200, 128, torch.float16, False),
    (17, 9, 3, 150, 129, 256, torch.bfloat16, True),
]


@pytest.mark.parametrize("case", SLICED, ids=lambda c: f"B{c[0]}H{c[1]}/{c[2]}M{c[3]}N{c[4]}D{c[5]}{str(c[6])[6:]}{'c' if c[7] else ''}")
def test_long_sums_and_many_items(case, cuda_device):
    B, Hq, Hkv, M, N, D, dtype, causal = case
    dout, q, k, v = _inputs(B, Hq, Hkv, M, N, D, dtype, cuda_device, M * N + D)
    o, lse = attention_forward(q, k, v, causal=causal, return_lse=True)
    got = attention_backward(dout, q, k, v, o, lse, causal=causal)
    _assert_within(got, *_reference(dout, q, k, v, o, lse, causal, D ** -0.5))
    again = attention_backward(dout, q, k, v, o, lse, causal=causal)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_offsets_past_32_bits(cuda_device):
    """Heads and rows that lie more than 2^31 elements into their tensors, inputs and gradients alike."""
    S, D, step = 150, 64, 1 << 30
    base = torch.zeros(2 * step + S * D + 64, device=cuda_device, dtype=torch.bfloat16)
    dout, q, k, v = _inputs(1, 3, 3, S, S, D, torch.bfloat16, cuda_device, 13)
    far = base.as_strided((1, 3, S, D), (step, step, D, 1))
    o, lse = attention_forward(q, k, v, causal=True, return_lse=True)
    want = attention_backward(dout, q, k, v, o, lse, causal=True)
    ok = dict(dout=dout, q=q, k=k, v=v, out=o)
    for name in ok:
        far.copy_(ok[name])
        got = attention_backward(**{**ok, name: far}, lse=lse, causal=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name


def test_strided_and_broadcast_inputs(cuda_device):
    """Column views of one packed projection, [B, S, H, D] outputs, a key/value head shared by expand, a dout of one
    repeated value."""
    B, S, Hq, Hkv, D = 2, 190, 4, 2, 64
    g = torch.Generator(device=cuda_device).manual_seed(8)
    qkv = torch.randn(B, S, Hq + 2 * Hkv, D, generator=g, device=cuda_device).to(torch.bfloat16)
    q, k, v = (t.transpose(1, 2) for t in qkv.split([Hq, Hkv, Hkv], 2))
    o, lse = attention_forward(q, k, v, causal=True, return_lse=True)
    o = o.transpose(1, 2).contiguous().transpose(1, 2)
    dout = torch.full((), 0.25, device=cuda_device, dtype=torch.bfloat16).expand(B, Hq, S, D)
    got = attention_backward(dout, q, k, v, o, lse, causal=True)
    _assert_within(got, *_reference(dout, q, k, v, o, lse, True, D ** -0.5))
    one_k, one_v = k[:, :1].expand(B, Hq, S, D), v[:, :1].expand(B, Hq, S, D)
    o, lse = attention_forward(q, one_k.contiguous(), one_v.contiguous(), causal=True, return_lse=True)
    got = attention_backward(dout, q, one_k, one_v, o, lse, causal=True)
    _assert_within(got, *_reference(dout, q, one_k, one_v, o, lse, True, D ** -0.5))
    # lse in another layout
    lse_t = lse.transpose(1, 2).contiguous().transpose(1, 2)
    again = attention_backward(dout, q, one_k, one_v, o, lse_t, causal=True)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("M, N", [(0, 40), (40, 0), (0, 0)])
def test_empty_lengths(M, N, cuda_device):
    dout, q, k, v = _inputs(2, 2, 1, M, N, 64, torch.bfloat16, cuda_device, 1)
    o, lse = attention_forward(q, k, v, return_lse=True)
    dq, dk, dv = attention_backward(dout, q, k, v, o, lse)
    for x, like in ((dq, q), (dk, k), (dv, v)):
        assert x.shape == like.shape and (x == 0).all()


@pytest.mark.parametrize("exp", [-14, -6, 8])
def test_fp16_gradients_keep_their_precision_at_any_size(exp, cuda_device):
    """dout times 2^exp gives every gradient times 2^exp, short of the rounding of subnormal results: the operands
    inside are scaled, so small gradients do not vanish before they are summed."""
    B, Hq, Hkv, M, N, D = 1, 2, 1, 256, 4096, 64
    dout, q, k, v = _inputs(B, Hq, Hkv, M, N, D, torch.float16, cuda_device, 11, 2.0 ** -4)
    o, lse = attention_forward(q, k, v, return_lse=True)
    small = (dout.double() * 2.0 ** exp).half()
    got = attention_backward(small, q, k, v, o, lse)
    _assert_within(got, *_reference(small, q, k, v, o, lse, False, D ** -0.5))


@pytest.mark.parametrize("vexp, dexp", [(9, 0), (9, 5), (-12, -8), (3, -12)])
def test_fp16_values_of_any_size(vexp, dexp, cuda_device):
    """Values and gradients times powers of two, among them one key 2^4 larger: nothing overflows inside, and small
    ones keep their precision."""
    dout, q, k, v = _inputs(1, 2, 1, 300, 900, 128, torch.float16, cuda_device, 14, 2.0 ** dexp)
    v = (v.double() * 2.0 ** vexp).half()
    v[:, :, 77] *= 16
    q, k = q * 0.125, k * 0.125  # flat rows, and gradients that stay in range
    o, lse = attention_forward(q, k, v, return_lse=True)
    got = attention_backward(dout, q, k, v, o, lse)
    assert torch.isfinite(torch.cat([t.flatten() for t in got])).all()
    _assert_within(got, *_reference(dout, q, k, v, o, lse, False, 128 ** -0.5))


def test_rows_of_very_different_gradients(cuda_device):
    """Single query rows whose dout is 2^-10 of the others' keep their dq in fp16."""
    dout, q, k, v = _inputs(1, 1, 1, 256, 2048, 64, torch.float16, cuda_device, 12)
    dout[:, :, ::3] *= 2.0 ** -10
    o, lse = attention_forward(q, k, v, return_lse=True)
    dq, _, _ = attention_backward(dout, q, k, v, o, lse)
    refs, tols = _reference(dout, q, k, v, o, lse, False, 64 ** -0.5)
    assert ((dq.double() - refs[0]).abs() <= tols[0]).all()


def test_zero_gradient_in_zero_gradient_out(cuda_device):
    for dtype in U:
        dout, q, k, v = _inputs(1, 2, 1, 140, 140, 128, dtype, cuda_device, 5, 0.0)
        o, lse = attention_forward(q, k, v, causal=True, return_lse=True)
        assert all((g == 0).all() for g in attention_backward(dout, q, k, v, o, lse, causal=True))


def test_directional_differences(cuda_device):
    """<grad, direction> against central differences of <dout, attention> in 64 bits.  o is rounded to the operand
    type, which moves delta by at most u rowsum |dout o|; the gradients are within the derived tolerances otherwise."""
    B, Hq, Hkv, M, N, D = 1, 4, 2, 90, 110, 64
    dout, q, k, v = _inputs(B, Hq, Hkv, M, N, D, torch.float16, cuda_device, 21)
    o, lse = attention_forward(q, k, v, return_lse=True)
    got = attention_backward(dout, q, k, v, o, lse)
    _, tols = _reference(dout, q, k, v, o, lse, False, D ** -0.5)

    def loss(q, k, v):
        k, v = (t.repeat_interleave(Hq // Hkv, 1) for t in (k, v))
        return (dout.double() * (torch.softmax(q @ k.transpose(-1, -2) * D ** -0.5, -1) @ v)).sum()

    base = [t.double() for t in (q, k, v)]
    u = U[torch.float16]
    P = torch.softmax(base[0] @ base[1].repeat_interleave(2, 1).transpose(-1, -2) * D ** -0.5, -1)
    moved = P * (u * (dout.double() * o.double()).abs().sum(-1, keepdim=True))
    moved_q = D ** -0.5 * moved @ base[1].repeat_interleave(2, 1).abs()
    moved_k = (D ** -0.5 * moved.transpose(-1, -2) @ base[0].abs()).unflatten(1, (Hkv, 2)).sum(2)
    g = torch.Generator(device=cuda_device).manual_seed(22)
    h = 1e-5
    for i, extra in enumerate((moved_q, moved_k, 0.0)):
        for _ in range(3):
            d = torch.randn(base[i].shape, generator=g, device=cuda_device, dtype=torch.float64)
            up, down = ([b + s * h * d if j == i else b for j, b in enumerate(base)] for s in (1, -1))
            slope = (loss(*up) - loss(*down)) / (2 * h)
            # errors of the elements are independent in sign: four standard deviations of their sum
            tol = 4 * ((tols[i] + extra) * d).norm() + 1e-6 * slope.abs()
            assert ((got[i].double() * d).sum() - slope).abs() <= tol


PACKED = [
    # q lengths, k lengths, Hq, Hkv, D, dtype, causal
    ((100, 513, 1), (100, 513, 1), 8, 2, 128, torch.bfloat16, True),
    ((5, 300, 0, 257), (700, 20, 9, 257), 4, 4, 64, torch.float16, False),   # cross lengths, an empty query set
    ((129, 64), (129, 64), 2, 1, 256, torch.bfloat16, True),
    ((70, 33, 128), (99, 45, 128), 2, 2, 80, torch.bfloat16, True),
    ((3, 40, 4), (0, 40, 10), 2, 2, 64, torch.bfloat16, False),              # queries with no keys
    ((37, 1), (200, 129), 7, 1, 33, torch.float16, True),
    (tuple(1 + 37 * i % 200 for i in range(60)), tuple(1 + 37 * i % 200 for i in range(60)), 3, 1, 64, torch.bfloat16, True),
    ((1, 2000, 3), (2500, 2, 1), 1, 1, 128, torch.bfloat16, False),          # long sums of one sequence, in parts
    ((1300, 1, 40), (1300, 1, 40), 2, 1, 256, torch.float16, True),
]


def _packed_inputs(lq, lk, Hq, Hkv, D, dtype, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    q, dout = (torch.randn(sum(lq), Hq, D, generator=g, device=dev).to(dtype) for _ in range(2))
    k, v = (torch.randn(sum(lk), Hkv, D, generator=g, device=dev).to(dtype) for _ in range(2))
    cu_q, cu_k = (torch.tensor([0, *torch.tensor(x).cumsum(0).tolist()], dtype=torch.int32, device=dev) for x in (lq, lk))
    return dout, q, k, v, cu_q, cu_k


@pytest.mark.parametrize("case", PACKED, ids=lambda c: f"q{str(c[0])[:20]}k{str(c[1])[:20]}H{c[2]}/{c[3]}D{c[4]}{str(c[5])[6:]}{'c' if c[6] else ''}")
def test_packed_matches_the_formula_per_sequence(case, cuda_device):
    lq, lk, Hq, Hkv, D, dtype, causal = case
    dout, q, k, v, cu_q, cu_k = _packed_inputs(lq, lk, Hq, Hkv, D, dtype, cuda_device, sum(lq))
    o, lse = attention_forward_varlen(q, k, v, cu_q, cu_k, max(lq), max(lk), causal=causal, return_lse=True)
    dq, dk, dv = attention_backward_varlen(dout, q, k, v, o, lse, cu_q, cu_k, max(lq), max(lk), causal=causal)
    a = b = 0
    for m, n in zip(lq, lk):
        qs, ks = slice(a, a + m), slice(b, b + n)
        a, b = a + m, b + n
        got = tuple(t.transpose(0, 1)[None] for t in (dq[qs], dk[ks], dv[ks]))
        if m == 0 or n == 0:
            assert all((t == 0).all() for t in got)
            continue
        one = (t.transpose(0, 1)[None] for t in (dout[qs], q[qs], k[ks], v[ks], o[qs]))
        _assert_within(got, *_reference(*one, lse[None, :, qs], causal, D ** -0.5))


def test_packed_sequences_do_not_reach_each_other(cuda_device):
    """Infinite and NaN values of one sequence leave every other sequence's gradients as they are."""
    lq, lk = (65, 70, 30), (90, 40, 33)
    for dtype, D in ((torch.bfloat16, 128), (torch.float16, 256), (torch.bfloat16, 64)):
        dout, q, k, v, cu_q, cu_k = _packed_inputs(lq, lk, 4, 2, D, dtype, cuda_device, 31)
        args = (cu_q, cu_k, max(lq), max(lk))
        o, lse = attention_forward_varlen(q, k, v, *args, return_lse=True)
        clean = attention_backward_varlen(dout, q, k, v, o, lse, *args)
        bad = [t.clone() for t in (dout, q, k, v, o)]
        for t, (a, b) in zip(bad, ((65, 135), (65, 135), (90, 130), (90, 130), (65, 135))):
            t[a:b:2] = float("nan")
            t[a + 1:b:2] = float("inf")
        got = attention_backward_varlen(*bad, lse, *args)
        for x, y, (a, b) in zip(got, clean, ((65, 135), (90, 130), (90, 130))):
            assert torch.equal(x[:a], y[:a]) and torch.equal(x[b:], y[b:])


def test_rows_outside_every_sequence_get_zeros(cuda_device):
    lq, lk = (50, 60), (70, 30)
    dout, q, k, v, cu_q, cu_k = _packed_inputs((7, *lq, 9), (3, *lk, 140), 2, 1, 64, torch.bfloat16, cuda_device, 4)
    cu_q, cu_k = cu_q[1:4].contiguous(), cu_k[1:4].contiguous()
    o, lse = attention_forward_varlen(q, k, v, cu_q, cu_k, 60, 70, causal=True, return_lse=True)
    o = torch.nan_to_num(o)
    dq, dk, dv = attention_backward_varlen(dout, q, k, v, o, lse, cu_q, cu_k, 60, 70, causal=True)
    for t, (a, b) in ((dq, (7, 117)), (dk, (3, 103)), (dv, (3, 103))):
        assert (t[:a] == 0).all() and (t[b:] == 0).all() and torch.isfinite(t).all()
        assert (t[a:b] != 0).any()


def test_packed_equals_dense_for_equal_lengths(cuda_device):
    B, H, S, D = 3, 4, 300, 128
    g = torch.Generator(device=cuda_device).manual_seed(51)
    dout, q, k, v = (torch.randn(B, S, H, D, generator=g, device=cuda_device).to(torch.bfloat16) for _ in range(4))
    cu = torch.arange(0, (B + 1) * S, S, dtype=torch.int32, device=cuda_device)
    flat = [t.reshape(B * S, H, D) for t in (dout, q, k, v)]
    o, lse = attention_forward_varlen(*flat[1:], cu, cu, S, S, causal=True, return_lse=True)
    packed = attention_backward_varlen(*flat, o, lse, cu, cu, S, S, causal=True)
    tr = [t.transpose(1, 2) for t in (dout, q, k, v)]
    od = o.reshape(B, S, H, D).transpose(1, 2)
    dense = attention_backward(*tr, od, lse.reshape(H, B, S).transpose(0, 1), causal=True)
    for x, y in zip(packed, dense):
        assert torch.equal(x.reshape(B, S, H, D), y.transpose(1, 2))


def test_caller_workspace_and_streams(cuda_device):
    dout, q, k, v = _inputs(1, 4, 2, 200, 200, 64, torch.float16, cuda_device, 6)
    o, lse = attention_forward(q, k, v, causal=True, return_lse=True)
    want = attention_backward(dout, q, k, v, o, lse, causal=True)
    need = attention_backward_workspace_bytes(q.shape, k.shape, q.dtype)
    ws = torch.full((need,), 255, device=cuda_device, dtype=torch.uint8)  # NaN everywhere: nothing may rely on it
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        got = attention_backward(dout, q, k, v, o, lse, causal=True, workspace=ws)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(ValueError, match="workspace"):
        attention_backward(dout, q, k, v, o, lse, workspace=ws[:need - 256])
    with pytest.raises(ValueError, match="workspace"):
        attention_backward(dout, q, k, v, o, lse, workspace=torch.empty(need + 1, device=cuda_device, dtype=torch.uint8)[1:])


def test_backward_in_a_cuda_graph(cuda_device):
    dout, q, k, v = _inputs(1, 4, 2, 300, 300, 128, torch.bfloat16, cuda_device, 7)
    o, lse = attention_forward(q, k, v, causal=True, return_lse=True)
    want = attention_backward(dout, q, k, v, o, lse, causal=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attention_backward(dout, q, k, v, o, lse, causal=True)
    for t in got:
        t.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_autograd_attention(cuda_device):
    _, q, k, v = _inputs(2, 4, 2, 130, 130, 64, torch.bfloat16, cuda_device, 9)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = training.attention(*leaves, causal=True)
    out.float().sum().backward()
    o, lse = attention_forward(q, k, v, causal=True, return_lse=True)
    want = attention_backward(torch.ones_like(o), q, k, v, o, lse, causal=True)
    assert torch.equal(out, o) and all(torch.equal(t.grad, w) for t, w in zip(leaves, want))

    dout, q, k, v, cu_q, cu_k = _packed_inputs((30, 70), (30, 70), 2, 1, 64, torch.float16, cuda_device, 10)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    training.attention_varlen(*leaves, cu_q, cu_k, 70, 70, causal=True).backward(dout)
    o, lse = attention_forward_varlen(q, k, v, cu_q, cu_k, 70, 70, causal=True, return_lse=True)
    want = attention_backward_varlen(dout, q, k, v, o, lse, cu_q, cu_k, 70, 70, causal=True)
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


def test_refusals(cuda_device):
    dout, q, k, v = _inputs(1, 4, 2, 20, 30, 64, torch.bfloat16, cuda_device, 2)
    o, lse = attention_forward(q, k, v, return_lse=True)
    ok = dict(dout=dout, q=q, k=k, v=v, out=o, lse=lse)
    for change, message in (
        (dict(dout=dout[0]), "shape"),
        (dict(q=q[:, :, :10]), "inconsistent shapes"),
        (dict(v=v[:, :, :10]), "inconsistent shapes"),
        (dict(k=k[:, :1].expand(1, 3, 30, 64), v=v[:, :1].expand(1, 3, 30, 64)), "multiple"),
        (dict(dout=dout.half()), "one dtype"),
        (dict(lse=lse.double()), "lse"),
        (dict(lse=lse[:, :2]), "lse"),
        (dict(q=q.cpu()), "CUDA"),
        ({n: t.float() for n, t in ok.items()}, "float16 or bfloat16"),
    ):
        with pytest.raises(ValueError, match=message):
            attention_backward(**{**ok, **change})
    with pytest.raises(ValueError):
        attention_backward(**ok, sm_scale=float("nan"))
    wide = torch.zeros(1, 1, 4, 264, device=cuda_device, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="head_dim"):
        attention_backward(wide, wide, wide, wide, wide, torch.zeros(1, 1, 4, device=cuda_device))
