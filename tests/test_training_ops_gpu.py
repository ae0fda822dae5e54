"""Layer norm (both passes) and multi-axis rotary embedding on the GPU against their formulas in 64 bits.

Tolerances.  Every stored value is rounded once to its type (unit roundoff u: 2^-8 bf16, 2^-11 fp16, 2^-24 fp32);
before that all arithmetic is fp32.  A sum of n terms is formed with at most about 64 additions in a row (registers,
then trees), so its error is below 2^-18 of the sum of magnitudes; column sums over rows add in at most 2^8 steps:
2^-16.  The bounds below carry these through each formula.
"""
from __future__ import annotations

import pytest
import torch

import _native
import training

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
SUBNORMAL = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
EPS = 1e-5


@pytest.fixture(autouse=True)
def _no_device_errors(cuda_device):
    yield
    torch.cuda.synchronize()
    assert _native.device_error() == 0


def _within(name, got, ref, tol):
    tol = tol + U[got.dtype] * ref.abs() + SUBNORMAL[got.dtype] + 1e-37
    worst = ((got.double() - ref).abs() / tol).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3f} of its tolerance"


def _norm_inputs(rows, cols, dtype, wdtype, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    x = (randn(rows, cols) * torch.exp(0.5 * randn(cols)) + 0.3).to(dtype)
    return (x, (1 + 0.2 * randn(cols)).to(wdtype), (0.2 * randn(cols)).to(wdtype), randn(rows, cols).to(dtype),
            (0.25 * randn(rows, cols)).to(dtype))


def _check_forward(x, w, b, got, residual=None, eps=EPS):
    y, mean, rstd = got[:3]
    if residual is not None:
        total = (x.double() + residual.double()).to(x.dtype)
        assert torch.equal(got[3], total)
        x = total
    X = x.double()
    m = X.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((X - m) ** 2).mean(-1, keepdim=True) + eps)
    small = 2.0 ** -18
    size = X.abs().mean(-1, keepdim=True)
    _within("mean", mean, m[..., 0], small * size[..., 0])
    # rstd: the centred squares carry the mean's error once more
    _within("rstd", rstd, r[..., 0], small * (2 + 2 * size * r)[..., 0] * r[..., 0])
    xh = (X - m) * r
    W = w.double()
    ref = xh * W + (b.double() if b is not None else 0)
    _within("y", y, ref, small * (size * r + (3 + 2 * size * r) * xh.abs()) * W.abs() + 2.0 ** -22 * ref.abs())


def _check_backward(dy, x, w, mean, rstd, got, dres=None, with_sums=True):
    X, G, W = x.double(), dy.double(), w.double()
    m, r = mean.double()[..., None], rstd.double()[..., None]
    xh = (X - m) * r
    g = G * W
    a, c = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = r * (g - a - xh * c)
    off = 2.0 ** -22 * (X.abs() + m.abs()) * r  # fp32 error of xhat
    small = 2.0 ** -18
    size_a, size_c = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    err_c = small * size_c + (g.abs() * off).mean(-1, keepdim=True)
    tol = r * (2.0 ** -22 * (g.abs() + a.abs() + (xh * c).abs()) + small * size_a + xh.abs() * err_c + off * c.abs())
    if dres is not None:
        dx = dx + dres.double()
        tol = tol + 2.0 ** -23 * dres.double().abs()
    _within("dx", got[0], dx, tol)
    if with_sums:
        dims = tuple(range(x.ndim - 1))
        _within("dw", got[1], (G * xh).sum(dims), 2.0 ** -16 * (G * xh).abs().sum(dims) + (G.abs() * off).sum(dims))
        _within("db", got[2], G.sum(dims), 2.0 ** -16 * G.abs().sum(dims))


NORMS = [
    # rows, cols, dtype, weight dtype, residual
    (1, 3584, torch.bfloat16, torch.bfloat16, False),
    (3, 3584, torch.bfloat16, torch.float32, True),
    (1000, 896, torch.float16, torch.float16, True),
    (5, 1, torch.float32, torch.float32, False),
    (7, 31, torch.bfloat16, torch.bfloat16, True),
    (700, 333, torch.float32, torch.float32, True),      # more rows than partial sums, odd columns
    (2, 8192, torch.float16, torch.float32, False),
    (3, 8200, torch.bfloat16, torch.bfloat16, True),
    (2, 20000, torch.bfloat16, torch.float32, True),
    (3, 16383, torch.float32, torch.float32, False),
    (2, 40000, torch.float16, torch.float16, True),      # past what a CTA's registers hold
    (603, 33000, torch.bfloat16, torch.bfloat16, False),
    (4099, 64, torch.bfloat16, torch.float32, True),
    # many rows for each worker, every way a row is shared out: by a warp, a CTA, a cluster; rows off the 16-byte grid
    (9001, 136, torch.float16, torch.float16, False),
    (9001, 509, torch.bfloat16, torch.bfloat16, True),
    (9000, 63, torch.float32, torch.float32, True),
    (3100, 1023, torch.bfloat16, torch.float32, True),
    (2777, 4104, torch.bfloat16, torch.bfloat16, True),
    (2500, 4095, torch.float32, torch.float32, False),
    (1501, 6001, torch.float16, torch.float32, True),
    (999, 12288, torch.bfloat16, torch.bfloat16, True),
    (999, 12289, torch.bfloat16, torch.bfloat16, True),
    (777, 16388, torch.float32, torch.float32, True),
    (160, 65528, torch.float16, torch.float16, False),
    (90, 65529, torch.bfloat16, torch.float32, True),
    (40, 32761, torch.float32, torch.float32, True),
]


@pytest.mark.parametrize("case", NORMS, ids=lambda c: f"{c[0]}x{c[1]}{str(c[2])[6:]}w{str(c[3])[6:]}{'r' if c[4] else ''}")
def test_layernorm_matches_the_formula(case, cuda_device):
    rows, cols, dtype, wdtype, with_residual = case
    x, w, b, res, dy = _norm_inputs(rows, cols, dtype, wdtype, cuda_device, rows + cols)
    res = res if with_residual else None
    got = training.layernorm_forward(x, w, b, eps=EPS, residual=res)
    _check_forward(x, w, b, got, res)
    total = got[3] if with_residual else x
    args = (dy, total, w, got[1], got[2])
    grads = training.layernorm_backward(*args, dresidual=res)
    _check_backward(*args, grads, res)
    again = training.layernorm_backward(*args, dresidual=res)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


def test_layernorm_views_strides_and_no_bias(cuda_device):
    """Column slices (16-byte aligned and not), 3-D inputs, transposed inputs, a broadcast gradient, no bias."""
    big, w, b, res, dy = _norm_inputs(40, 1000, torch.bfloat16, torch.bfloat16, cuda_device, 1)
    for lo, hi in ((8, 520), (3, 515), (1, 1000)):
        x, g = big[:, lo:hi], dy[:, lo:hi]
        got = training.layernorm_forward(x, w[lo:hi], None, eps=EPS, residual=res[:, lo:hi])
        _check_forward(x, w[lo:hi], None, got, res[:, lo:hi])
        args = (g, got[3], w[lo:hi], got[1], got[2])
        _check_backward(*args, training.layernorm_backward(*args))
    x3, g3 = big.view(8, 5, 1000), dy.view(8, 5, 1000).transpose(0, 1).contiguous().transpose(0, 1)
    got = training.layernorm_forward(x3, w, b, eps=EPS)
    assert got[0].shape == x3.shape and got[1].shape == (8, 5)
    _check_forward(x3, w, b, got)
    _check_backward(g3, x3, w, got[1], got[2], training.layernorm_backward(g3, x3, w, got[1], got[2]))
    xt = big.t().contiguous().t()  # unit stride along rows
    got_t = training.layernorm_forward(xt, w, b, eps=EPS)
    assert all(torch.equal(p, q.view_as(p)) for p, q in zip(got_t, got))
    one = torch.full((), 0.5, device=cuda_device, dtype=torch.bfloat16).expand(40, 1000)
    _check_backward(one, big, w, got_t[1], got_t[2], training.layernorm_backward(one, big, w, got_t[1], got_t[2]))


def test_layernorm_large_offset_and_flat_rows(cuda_device):
    """A mean far larger than the spread: the variance is not a difference of squares.  A constant row gives the bias."""
    x, w, b, _, _ = _norm_inputs(6, 1024, torch.float32, torch.float32, cuda_device, 2)
    x = x + 1000.0
    x[2] = 7.0
    got = training.layernorm_forward(x, w, b, eps=EPS)
    _check_forward(x, w, b, got)
    assert torch.equal(got[0][2], b)


def test_layernorm_rows_are_independent_of_bad_ones(cuda_device):
    x, w, b, _, dy = _norm_inputs(9, 640, torch.bfloat16, torch.bfloat16, cuda_device, 3)
    clean = training.layernorm_forward(x, w, b)
    bad = x.clone()
    bad[4, 17] = float("nan")
    bad[7] = float("inf")
    got = training.layernorm_forward(bad, w, b)
    keep = [0, 1, 2, 3, 5, 6, 8]
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.isnan(got[0][4]).all() and torch.isnan(got[0][7]).all()


@pytest.mark.parametrize("cols", [640, 641, 83, 9001])
def test_layernorm_gradients_are_independent_of_bad_rows(cols, cuda_device):
    """Where 16-byte pieces reach into the rows before and after, nothing of them gets in."""
    for rows in (9, 700):
        x, w, b, res, dy = _norm_inputs(rows, cols, torch.bfloat16, torch.bfloat16, cuda_device, 3)
        _, mean, rstd = training.layernorm_forward(x, w, b)
        clean = training.layernorm_backward(dy, x, w, mean, rstd, dresidual=res)[0]
        bad_x, bad_dy = x.clone(), dy.clone()
        bad_x[1::2], bad_dy[1::2] = float("nan"), float("inf")
        y, m, r = training.layernorm_forward(bad_x, w, b)
        assert torch.equal(y[::2], training.layernorm_forward(x, w, b)[0][::2])
        got = training.layernorm_backward(bad_dy, bad_x, w, mean, rstd, dresidual=res)[0]
        assert torch.equal(got[::2], clean[::2])


@pytest.mark.parametrize("lead", [0, 1, 5])
def test_layernorm_writes_no_neighbour(lead, cuda_device):
    """Rows with gaps between them and around them, through the C ABI: the gaps keep their bits."""
    rows, cols, ld = 700, 333, 341
    x, w, b, res, dy = _norm_inputs(rows, cols, torch.bfloat16, torch.bfloat16, cuda_device, 9)

    def padded(t=None):
        store = torch.full((rows * ld + 16,), 7.0, device=cuda_device, dtype=torch.bfloat16)
        view = store.as_strided((rows, cols), (ld, 1), lead)
        if t is not None:
            view.copy_(t)
        return store, view

    ins = [padded(t) for t in (x, res, dy)]
    (ys, y), (xos, xo), (dxs, dx) = (padded() for _ in range(3))
    mean, rstd = (torch.empty(rows, device=cuda_device) for _ in range(2))
    stream = _native.current_stream_handle(cuda_device)
    ptr = torch.Tensor.data_ptr
    dt = _native.dtype_code(torch.bfloat16)
    _native.check(_native.lib.fab_layernorm(
        ptr(ins[0][1]), ptr(ins[1][1]), ptr(w), ptr(b), ptr(y), ptr(xo), ptr(mean), ptr(rstd), rows, cols, ld, ld, ld, ld,
        EPS, dt, dt, stream), "fab_layernorm")
    _native.check(_native.lib.fab_layernorm_bwd(
        ptr(ins[2][1]), ptr(xo), ptr(w), ptr(mean), ptr(rstd), ptr(ins[1][1]), ptr(dx), None, None, None, 0, rows, cols, ld,
        ld, ld, ld, dt, dt, stream), "fab_layernorm_bwd")
    _check_forward(x, w, b, (y, mean, rstd, xo), res)
    _check_backward(dy, xo, w, mean, rstd, (dx,), res, with_sums=False)
    for store, view in ((ys, y), (xos, xo), (dxs, dx)):
        view.fill_(7.0)
        assert (store == 7.0).all()


def test_layernorm_without_rows(cuda_device):
    w = torch.ones(16, device=cuda_device, dtype=torch.bfloat16)
    x = torch.empty(0, 16, device=cuda_device, dtype=torch.bfloat16)
    y, mean, rstd = training.layernorm_forward(x, w, w)
    dx, dw, db = training.layernorm_backward(x, x, w, mean, rstd)
    assert y.shape == dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()


def test_layernorm_differences(cuda_device):
    """<gradient, direction> against central differences of <dy, layer norm> in 64 bits (fp32 kernels)."""
    x, w, b, res, dy = _norm_inputs(20, 300, torch.float32, torch.float32, cuda_device, 4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b, res)]
    y, total = training.layernorm(leaves[0], leaves[1], leaves[2], eps=EPS, residual=leaves[3])
    torch.autograd.backward([y, total], [dy, res])

    def loss(x, w, b, r):
        t = x + r
        c = t - t.mean(1, keepdim=True)
        return (dy.double() * (c / torch.sqrt((c * c).mean(1, keepdim=True) + EPS) * w + b)).sum() + (res.double() * t).sum()

    base = [t.double() for t in (x, w, b, res)]
    g = torch.Generator(device=cuda_device).manual_seed(5)
    h = 1e-5
    for i, leaf in enumerate(leaves):
        d = torch.randn(leaf.shape, generator=g, device=cuda_device, dtype=torch.float64)
        up, down = ([t + s * h * d if j == i else t for j, t in enumerate(base)] for s in (1, -1))
        slope = (loss(*up) - loss(*down)) / (2 * h)
        # fp32 gradients: 2^-16 of their size each, four standard deviations of the weighted sum; h^2 of the curvature
        tol = 4 * 2.0 ** -16 * (leaf.grad.double().abs() + 1e-3).mul(d).norm() + 1e-6 * slope.abs()
        assert ((leaf.grad.double() * d).sum() - slope).abs() <= tol


def test_layernorm_refusals(cuda_device):
    x, w, b, res, dy = _norm_inputs(4, 32, torch.bfloat16, torch.bfloat16, cuda_device, 6)
    y, mean, rstd = training.layernorm_forward(x, w, b)
    for args, kw, message in (
        ((x.cpu(), w, b), {}, "CUDA"),
        ((x.double(), w, b), {}, "float"),
        ((x, w[:16], b), {}, "weight"),
        ((x, w.half(), b), {}, "weight"),
        ((x, w, b.float()), {}, "one dtype"),
        ((x, w, b), dict(residual=res.float()), "residual"),
        ((x, w, b), dict(residual=res[:2]), "residual"),
        ((x, w, b), dict(eps=-1.0), "invalid argument"),
        ((x, w, b), dict(eps=float("nan")), "invalid argument"),
    ):
        with pytest.raises(ValueError, match=message):
            training.layernorm_forward(*args, **kw)
    with pytest.raises(ValueError, match="dy"):
        training.layernorm_backward(dy[:2], x, w, mean, rstd)
    with pytest.raises(ValueError, match="mean"):
        training.layernorm_backward(dy, x, w, mean[:2], rstd)
    with pytest.raises(ValueError, match="rstd"):
        training.layernorm_backward(dy, x, w, mean, rstd.double())


ROPES = [
    # tokens, Hq, Hkv, D, sections, dtype, position dtype
    (1, 28, 4, 128, (16, 24, 24), torch.bfloat16, torch.int32),
    (37, 4, 2, 80, (20, 20), torch.float16, torch.int64),
    (300, 3, 1, 64, (32,), torch.bfloat16, torch.int64),
    (65, 2, 2, 64, (3, 5, 1, 2), torch.float32, torch.int32),     # part of the head turns, uneven sections
    (29, 2, 1, 50, (12, 13), torch.bfloat16, torch.int32),         # columns off the 16-byte grid
    (18, 5, 0, 256, (0, 100, 28), torch.float16, torch.int32),     # an axis without pairs, no key heads
    (6, 1, 1, 2, (1,), torch.float32, torch.int64),
    (11, 33, 7, 96, (8, 16, 8), torch.bfloat16, torch.int32),
    (70, 4, 2, 80, (8, 12), torch.float16, torch.int32),           # 20 pairs: 8-byte pieces
    (70, 3, 1, 80, (7, 13), torch.bfloat16, torch.int64),          # and sections that cut them
]


def _rope_inputs(T, Hq, Hkv, D, sections, dtype, pdtype, dev, table=200):
    g = torch.Generator(device=dev).manual_seed(T + D)
    qkv = torch.randn(T, Hq + Hkv + 1, D, generator=g, device=dev).to(dtype)
    pos = torch.randint(0, table, (len(sections), T), generator=g, device=dev).to(pdtype)
    half = sum(sections)
    ang = torch.arange(table, device=dev, dtype=torch.float64)[:, None] * 100.0 ** (
        -torch.arange(half, device=dev, dtype=torch.float64) / half)
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], pos, ang.cos().float(), ang.sin().float()


def _rope_reference(x, pos, cos, sin, sections, inverse):
    half = sum(sections)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=x.device)
    rows = pos.long()[axis]  # [half, tokens]
    col = torch.arange(half, device=x.device)[:, None]
    c, s = cos.double()[rows, col].t()[:, None], sin.double()[rows, col].t()[:, None]
    s = -s if inverse else s
    lo, hi, rest = x[..., :half].double(), x[..., half:2 * half].double(), x[..., 2 * half:].double()
    ref = torch.cat((lo * c - hi * s, hi * c + lo * s, rest), -1)
    tol = 2.0 ** -22 * torch.cat(((lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs(), 0 * rest), -1)
    return ref, tol


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", ROPES, ids=lambda c: f"T{c[0]}H{c[1]}/{c[2]}D{c[3]}s{'-'.join(map(str, c[4]))}{str(c[5])[6:]}")
def test_rope_matches_the_formula(case, inverse, cuda_device):
    T, Hq, Hkv, D, sections, dtype, pdtype = case
    q, k, pos, cos, sin = _rope_inputs(T, Hq, Hkv, D, sections, dtype, pdtype, cuda_device)
    got = training.rope_multi_axis(q, k if Hkv else None, pos, cos, sin, sections, inverse=inverse)
    for x, y in zip((q, k), got):
        if y is not None:
            _within("rope", y, *_rope_reference(x, pos, cos, sin, sections, inverse))
    q2, k2 = q.clone(), k.clone()
    training.rope_multi_axis(q2, k2, pos, cos, sin, sections, inverse=inverse, out=(q2, k2))
    assert torch.equal(q2, got[0]) and (Hkv == 0 or torch.equal(k2, got[1]))


def test_rope_strides_and_views(cuda_device):
    """[heads, tokens, D] storage, strided positions, a column view that starts off the 16-byte grid."""
    sections = (16, 16)
    q, k, pos, cos, sin = _rope_inputs(50, 4, 2, 64, sections, torch.bfloat16, torch.int32, cuda_device)
    want = training.rope_multi_axis(q, k, pos, cos, sin, sections)
    qh = q.transpose(0, 1).contiguous().transpose(0, 1)
    pos_t = pos.t().contiguous().t()
    off = torch.empty(50, 2, 67, device=cuda_device, dtype=torch.bfloat16)[..., 3:]
    off.copy_(k)
    got = training.rope_multi_axis(qh, off, pos_t, cos, sin, sections)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rope_position_outside_the_table_is_nan_and_stays_alone(cuda_device):
    sections = (8, 8, 16)
    q, k, pos, cos, sin = _rope_inputs(20, 2, 1, 64, sections, torch.bfloat16, torch.int64, cuda_device)
    want = training.rope_multi_axis(q, k, pos, cos, sin, sections)[0]
    bad = pos.clone()
    bad[1, 3], bad[1, 5], bad[1, 6] = 200, -1, 1 << 40
    got = training.rope_multi_axis(q, k, bad, cos, sin, sections)[0]
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[[3, 5, 6], :, 8:16] = True
    hit[[3, 5, 6], :, 40:48] = True
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], want[~hit])


def test_rope_gradients(cuda_device):
    """The backward pass is the inverse rotation; against central differences in 64 bits of a linear map (exact up to
    rounding), and turning back restores the input up to rounding."""
    sections = (10, 6)
    q, k, pos, cos, sin = _rope_inputs(40, 2, 1, 40, sections, torch.float32, torch.int32, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(3)
    dq, dk = (torch.randn(t.shape, generator=g, device=cuda_device) for t in (q, k))
    leaves = [t.clone().requires_grad_() for t in (q, k)]
    outs = training.rope(*leaves, pos, cos, sin, sections)
    torch.autograd.backward(outs, [dq, dk])
    for leaf, d, out in zip(leaves, (dq, dk), outs):
        v = torch.randn(leaf.shape, generator=g, device=cuda_device)
        plus, minus = (_rope_reference(leaf.detach() + s * v, pos, cos, sin, sections, False)[0] for s in (1, -1))
        slope = (d.double() * (plus - minus)).sum() / 2
        assert ((leaf.grad.double() * v).sum() - slope).abs() <= 2.0 ** -20 * (leaf.grad * v).double().abs().sum()
    back = training.rope_multi_axis(*(o.detach() for o in outs), pos, cos, sin, sections, inverse=True)
    # cos^2 + sin^2 of the fp32 tables is 1 within 2^-22
    torch.testing.assert_close(back[0], q, rtol=0, atol=2.0 ** -20 * q.abs().max().item())


def test_rope_refusals(cuda_device):
    q, k, pos, cos, sin = _rope_inputs(5, 2, 1, 64, (16, 16), torch.bfloat16, torch.int32, cuda_device)
    ok = dict(q=q, k=k, positions=pos, cos=cos, sin=sin, sections=(16, 16))
    for change, message in (
        (dict(q=q.cpu()), "CUDA"),
        (dict(q=q[0]), "shape"),
        (dict(k=k[:3]), "shape"),
        (dict(k=k.float()), "one dtype"),
        (dict(q=q.double(), k=k.double()), "dtype"),
        (dict(sections=(16, 17)), "sections"),
        (dict(sections=(33,), positions=pos[:1]), "sections"),
        (dict(sections=(1, 1, 1, 1, 1)), "sections"),
        (dict(sections=(40, -8)), "sections"),
        (dict(positions=pos[:1]), "positions"),
        (dict(positions=pos.float()), "positions"),
        (dict(cos=cos.double()), "tables"),
        (dict(cos=cos[:, :8], sin=sin[:, :8]), "tables"),
        (dict(out=(q[:, :1], k)), "out"),
    ):
        with pytest.raises(ValueError, match=message):
            training.rope_multi_axis(**{**ok, **change})


def test_a_pre_norm_block_trains(cuda_device):
    """Norm, packed projection, rotary and attention through autograd: every gradient against the same block in
    64-bit torch operations.  The kernels round activations to fp16 between operators (a handful of roundings of 2^-11
    on the way to each gradient): the 2-norms agree within 2^-6."""
    T, C, H, Hkv, D, sections = 96, 128, 4, 2, 32, (4, 6, 6)
    g = torch.Generator(device=cuda_device).manual_seed(77)
    x = torch.randn(T, C, generator=g, device=cuda_device).half()
    w, b = (1 + 0.1 * torch.randn(C, generator=g, device=cuda_device)), 0.1 * torch.randn(C, generator=g, device=cuda_device)
    proj = (torch.randn(C, (H + 2 * Hkv) * D, generator=g, device=cuda_device) / C ** 0.5).half()
    dout = torch.randn(T, H, D, generator=g, device=cuda_device).half()
    _, _, pos, cos, sin = _rope_inputs(T, H, Hkv, D, sections, torch.float16, torch.int32, cuda_device)

    leaves = [t.clone().requires_grad_() for t in (x, w, b, proj)]
    y = training.layernorm(leaves[0], leaves[1], leaves[2])
    qkv = (y @ leaves[3]).view(T, H + 2 * Hkv, D)
    q, k = training.rope(qkv[:, :H], qkv[:, H:H + Hkv], pos, cos, sin, sections)
    o = training.attention(*(t.transpose(0, 1)[None] for t in (q, k, qkv[:, H + Hkv:])), causal=True)
    o[0].transpose(0, 1).backward(dout)

    ref = [t.double().clone().requires_grad_() for t in (x, w, b, proj)]
    X = ref[0]
    c = X - X.mean(1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * ref[1] + ref[2]
    qkv = (y @ ref[3]).view(T, H + 2 * Hkv, D)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=cuda_device)
    ct, st = (t.double()[pos.long()[axis], torch.arange(16, device=cuda_device)[:, None]].t()[:, None] for t in (cos, sin))

    def turn(z):
        lo, hi = z.split(16, -1)
        return torch.cat((lo * ct - hi * st, hi * ct + lo * st), -1)

    q, k, v = (t.transpose(0, 1) for t in (turn(qkv[:, :H]), turn(qkv[:, H:H + Hkv]), qkv[:, H + Hkv:]))
    k, v = (t.repeat_interleave(H // Hkv, 0) for t in (k, v))
    s = (q @ k.transpose(1, 2) * D ** -0.5).masked_fill(~torch.ones(T, T, device=cuda_device).tril().bool(), float("-inf"))
    (torch.softmax(s, -1) @ v).transpose(0, 1).backward(dout.double())
    for leaf, want in zip(leaves, ref):
        assert (leaf.grad.double() - want.grad).norm() <= 2.0 ** -6 * want.grad.norm()


def test_a_small_decoder_learns(cuda_device):
    """Packed text-and-image sequences of repeated words: the loss starts at chance (log 64 = 4.2) or above and comes
    down to a quarter of it."""
    import train_block

    losses = train_block.train(60, device=cuda_device)
    assert losses[0] > 4.0 and sum(losses[-10:]) / 10 < 1.0, (losses[0], losses[-10:])
