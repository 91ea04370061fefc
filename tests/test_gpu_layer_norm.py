"""Layer norm over block-stack rows against its definition in 64 bits, forward and backward.

Tolerances: half a step of the element type for the one rounding of each output, plus 2^-24 for every fp32
operation on the longest path to it, times the magnitudes that path adds up (computed in 64 bits beside the
expected value)."""
import math

import pytest
import torch

from sbnet_b200 import autograd as sb
from sbnet_b200 import lib, ops

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _inputs(rows, c, dtype, wdtype, seed=0, shift=0.3):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, dy = (r(rows, c) * 1.5 + shift).to(dtype), r(rows, c).to(dtype)
    return x, dy, (r(c) * 0.3 + 1).to(wdtype), (r(c) * 0.3).to(wdtype)


def _steps(c):
    """Longest chain of fp32 operations behind a row statistic: a thread's own channels, the exchange
    between threads, and a handful for the formula."""
    return 16 + c / 1024 + 12 + 8


def _expected(x, w, b, eps, dy=None):
    x64 = x.double()
    w64 = torch.ones(x.shape[-1], device="cuda", dtype=torch.float64) if w is None else w.double()
    b64 = torch.zeros_like(w64) if b is None else b.double()
    mean = x64.mean(-1, keepdim=True)
    d = x64 - mean
    rstd = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    xh = d * rstd
    y = xh * w64 + b64
    n = _steps(x.shape[-1])
    kappa = 1 + x64.abs().mean(-1, keepdim=True) * rstd      # how far the mean's error reaches into xh
    out = dict(y=y, y_mag=U32 * n * kappa * ((1 + xh.abs()) * w64.abs() + b64.abs()), mean=mean, rstd=rstd)
    if dy is not None:
        g = dy.double()
        gw = g * w64
        m0, m1 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
        out["dx"] = rstd * (gw - m0 - xh * m1)
        out["dx_mag"] = 4 * U32 * n * kappa * rstd * (
            gw.abs() + gw.abs().mean(-1, keepdim=True) + (1 + xh.abs()) * (gw.abs() * (1 + xh.abs())).mean(-1, keepdim=True))
        rows = max(1, x64.shape[0])
        parts = max(1, lib.load().sbnet_layer_norm_grad_workspace(rows, x.shape[-1]) // (8 * x.shape[-1]))
        path = rows / parts + 64 + parts / 32 + 8 + n
        out["dw"], out["db"] = (g * xh).sum(0), g.sum(0)
        out["dw_mag"] = U32 * path * (g.abs() * (1 + xh.abs()) * kappa).sum(0)
        out["db_mag"] = U32 * path * g.abs().sum(0)
    return out


def _close(got, e, key, dtype):
    ref, tol = e[key], e[key + "_mag"] + torch.finfo(dtype).eps / 2 * e[key].abs() + torch.finfo(dtype).smallest_normal
    bad = (got.double() - ref).abs() - tol
    assert got.dtype == dtype and torch.isfinite(got).all()
    assert bad.max() <= 0, (key, float(bad.max()), float((got.double() - ref).abs().max()))


# widths around every change of the work split: sub-warp groups, two vectors a thread, whole CTAs, 16 channels a
# thread, the loop kernel; odd ones (one element a vector) and even ones off 16 bytes (two elements a vector)
WIDTHS = [1, 2, 3, 8, 24, 31, 32, 33, 64, 100, 128, 130, 256, 257, 264, 511, 512, 513, 520, 1001, 1024, 2050, 4096, 5001, 8192, 8200, 16384, 16392, 20001]


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES)
def test_forward_and_backward(cuda_ops, dtype, c):
    wdtype = torch.float32 if c % 3 == 0 else dtype
    rows = 1 if c % 5 == 1 else (300 if c <= 1024 else 37)
    x, dy, w, b = _inputs(rows, c, dtype, wdtype, seed=c)
    e = _expected(x, w, b, 1e-5, dy)
    if c == 1:      # a single channel is its own mean: y is the bias, no gradient reaches x or w
        e["dx_mag"] = e["dx_mag"] + 1e-3
    y, stats = ops.layer_norm(x, w, b, 1e-5, stats=True)
    _close(y, e, "y", dtype)
    assert torch.equal(y, ops.layer_norm(x, w, b, 1e-5))
    mean, rstd = stats
    n = _steps(c) * U32
    assert ((mean.double() - e["mean"][:, 0]).abs() <= n * x.double().abs().mean(-1)).all()
    kappa = 1 + x.double().abs().mean(-1) * e["rstd"][:, 0]
    assert ((rstd.double() / e["rstd"][:, 0] - 1).abs() <= 2 * n * kappa).all()
    dx, dw, db = ops.layer_norm_grad(dy, x, stats, w, b)
    _close(dx, e, "dx", dtype)
    _close(dw, e, "dw", wdtype)
    _close(db, e, "db", wdtype)


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 63, 4096, 70001])
@pytest.mark.parametrize("c", [16, 128, 1000])
def test_row_counts(cuda_ops, rows, c):
    x, dy, w, b = _inputs(rows, c, torch.bfloat16, torch.float32, seed=rows)
    e = _expected(x, w, b, 1e-6, dy)
    y, stats = ops.layer_norm(x, w, b, 1e-6, stats=True)
    _close(y, e, "y", x.dtype)
    dx, dw, db = ops.layer_norm_grad(dy, x, stats, w, b)
    _close(dx, e, "dx", x.dtype)
    _close(dw, e, "dw", w.dtype)
    _close(db, e, "db", w.dtype)
    again = ops.layer_norm_grad(dy, x, stats, w, b)
    assert torch.equal(dw, again[1]) and torch.equal(db, again[2])     # a fixed order of additions


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_parameters_are_optional(cuda_ops, which):
    x, dy, w, b = _inputs(50, 72, torch.float16, torch.float16)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    e = _expected(x, w, b, 1e-5, dy)
    y, stats = ops.layer_norm(x, w, b, stats=True)
    _close(y, e, "y", x.dtype)
    dx, dw, db = ops.layer_norm_grad(dy, x, stats, w, b)
    _close(dx, e, "dx", x.dtype)
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    if w is not None:
        _close(dw, e, "dw", w.dtype)
    if b is not None:
        _close(db, e, "db", b.dtype)


def test_constant_rows_and_rows_that_are_not_finite(cuda_ops):
    x, dy, w, b = _inputs(9, 136, torch.float32, torch.float32)
    x[2] = 5.0                       # no variance: rstd = 1 / sqrt(eps), y = b
    x[4, 7] = math.inf
    x[6, 3] = math.nan
    y, stats = ops.layer_norm(x, w, b, 1e-5, stats=True)
    torch.testing.assert_close(y[2], b, rtol=0, atol=16 * 5 * U32 / math.sqrt(1e-5) * 2)
    assert torch.isnan(y[4]).any() and torch.isnan(y[6]).all()
    clean = [0, 1, 3, 5, 7, 8]
    e = _expected(x[clean], w, b, 1e-5, dy[clean])
    dx, _, _ = ops.layer_norm_grad(dy, x, stats, w, b)
    _close(y[clean], e, "y", x.dtype)
    _close(dx[clean], e, "dx", x.dtype)


def test_large_mean(cuda_ops):
    """The variance is taken around the mean, not as a difference of squares."""
    x, dy, w, b = _inputs(20, 512, torch.float32, torch.float32, shift=1000.0)
    e = _expected(x, w, b, 1e-5)
    _close(ops.layer_norm(x, w, b), e, "y", x.dtype)


@pytest.mark.parametrize("off", [1, 2, 4])
def test_tensors_off_a_16_byte_boundary(cuda_ops, off):
    rows, c = 40, 64
    x, dy, w, b = _inputs(rows, c, torch.float16, torch.float16)
    place = lambda t: torch.zeros(t.numel() + 16, dtype=t.dtype, device="cuda")[off:off + t.numel()].view(t.shape).copy_(t)
    buf = torch.full((rows * c + 64,), 7.0, dtype=x.dtype, device="cuda")
    out = buf[16 + off:16 + off + rows * c].view(rows, c)
    e = _expected(x, w, b, 1e-5, dy)
    y, stats = ops.layer_norm(place(x), w, b, out=out, stats=True)
    assert y.data_ptr() == out.data_ptr()
    _close(out, e, "y", x.dtype)
    assert (buf[:16 + off] == 7).all() and (buf[16 + off + rows * c:] == 7).all()
    dx, dw, db = ops.layer_norm_grad(place(dy), place(x), stats, w, b)
    _close(dx, e, "dx", x.dtype)
    _close(dw, e, "dw", x.dtype)


@pytest.mark.parametrize("shape", [(6, 3, 3, 40), (5, 16, 16, 128), (4, 7, 600), (3, 1001)])
@pytest.mark.parametrize("count", [0, 1, 2, 99, -3])
def test_device_count(cuda_ops, shape, count):
    x, _, w, b = _inputs(math.prod(shape[:-1]), shape[-1], torch.float16, torch.float32)
    x = x.view(shape).clone()
    live = min(max(count, 0), shape[0])
    x[live:] = math.nan              # whatever a gather left there
    out = torch.full(shape, -9.0, dtype=x.dtype, device="cuda")
    n = torch.tensor([count], dtype=torch.int32, device="cuda")
    res = ops.layer_norm_dyn(x, n, w, b, out=out)
    assert res.data_ptr() == out.data_ptr() and (out[live:] == -9).all()
    if live:
        assert torch.equal(out[:live], ops.layer_norm(x[:live].contiguous(), w, b))


def test_no_rows(cuda_ops):
    w = torch.ones(24, device="cuda", requires_grad=True)
    x = torch.zeros((0, 4, 4, 24), device="cuda", requires_grad=True)
    y = sb.layer_norm(x, w, None)
    assert y.shape == x.shape
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros_like(y))
    assert gx.shape == x.shape and (gw == 0).all()


def test_more_than_2_31_elements(cuda_ops):
    """Row offsets are 64-bit: the last rows of a tensor past 2^32 bytes and 2^31 elements."""
    rows, c = (1 << 31) // 1024 + 5, 1024
    x = torch.zeros((rows, c), dtype=torch.float16, device="cuda")
    tail = torch.randn((5, c), device="cuda").half()
    x[-5:] = tail
    y = ops.layer_norm(x)
    _close(y[-5:], _expected(tail, None, None, 1e-5), "y", x.dtype)
    assert (y[1000:1005] == 0).all()


def test_autograd_matches_the_formula_and_differences(cuda_ops):
    x, dy, w, b = (t.requires_grad_(True) for t in _inputs(31, 45, torch.float32, torch.float32, shift=0.0))
    y = sb.layer_norm(x, w, b, 1e-5)
    grads = torch.autograd.grad(y, (x, w, b), dy.detach())
    h = 1e-2
    f = lambda xx, ww, bb: (ops.layer_norm(xx, ww, bb, 1e-5).double() * dy.double()).sum().item()
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    for k, g in enumerate(grads):
        args = [x.detach(), w.detach(), b.detach()]
        d = torch.randn(args[k].shape, generator=gen, device="cuda")
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + h * d, args[k] - h * d
        num = (f(*up) - f(*down)) / (2 * h)
        ana = float((g.double() * d.double()).sum())
        # central differences are off by h^2/6 of the third derivative (order of the value itself), and by the
        # rounding of 31*45 outputs over 2h
        assert abs(num - ana) <= 1e-2 * float((g.double().abs() * d.double().abs()).sum()) + 0.01, (k, num, ana)


def test_another_stream_and_a_captured_graph(cuda_ops):
    x, dy, w, b = _inputs(500, 96, torch.bfloat16, torch.float32)
    want, stats = ops.layer_norm(x, w, b, stats=True)
    gwant = ops.layer_norm_grad(dy, x, stats, w, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.layer_norm(x, w, b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    xs = torch.zeros_like(x)
    with torch.cuda.graph(g):
        y, st = ops.layer_norm(xs, w, b, stats=True)
        grads = ops.layer_norm_grad(dy, xs, st, w, b)
    for _ in range(2):
        xs.copy_(x)
        g.replay()
        assert torch.equal(y, want) and all(torch.equal(p, q) for p, q in zip(grads, gwant))
        xs.zero_()
        g.replay()
        assert torch.equal(y, b.to(y.dtype).expand_as(y))
