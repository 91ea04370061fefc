"""The gated feed-forward block against its definition in 64 bits, forward and backward.

Tolerances are carried through the formula.  With u half a step of the element type (relative), every element
that is rounded to that type is off by u of itself: the output, h (the last product's operand), and in the
backward pass dG, dU and h.  A sum of K products on the tensor cores is off by
2^-23 for each of its K/16 instructions and a few more (16), times the sum of the products' magnitudes; the
element-wise steps are off by 2^-19 of their magnitude (the error bound of the fast exponential at |g| <= 16).
Each of these is multiplied with what it meets on its way to the output.  The bounds add magnitudes, so they
are far from what random errors add up to; the second check is on the norm of the error: independent rounding
errors of at most u (variance u^2/3) at the output and at each operand give at most sqrt(2/3) u for y and
the gradients on random data; 1.5u is allowed."""
import math

import pytest
import torch

from sbnet_b200 import autograd as sb
from sbnet_b200 import lib, ops

pytestmark = pytest.mark.gpu

NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down")


def _inputs(rows, c, f, dtype, seed=0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=gen, device="cuda") * scale).to(dtype)
    return (r(rows, c), r(f, c, scale=1 / math.sqrt(c)), r(f, c, scale=1 / math.sqrt(c)), r(c, f, scale=1 / math.sqrt(f)),
            r(rows, c))


def _act64(act, g):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        cdf = torch.special.ndtr(g)
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return g.clamp(min=0), (g > 0).double()


def _expected(act, x, wg, wu, wd, dy=None):
    """name -> (value, tolerance), both in 64 bits."""
    u, dtype = torch.finfo(x.dtype).eps / 2, x.dtype
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps       # one step of the subnormals
    chain = lambda k: (k / 16 + 16) * 2.0 ** -23
    x, wg, wu, wd = x.double(), wg.double(), wu.double(), wd.double()
    c, f, rows = x.shape[1], wg.shape[0], x.shape[0]
    g, up = x @ wg.T, x @ wu.T
    a, s = _act64(act, g)
    h = a * up
    eg, eu = chain(c) * (x.abs() @ wg.abs().T), chain(c) * (x.abs() @ wu.abs().T)
    ea = 2.0 ** -19 * g.abs()
    eh = u * h.abs() + 1.13 * eg * up.abs() + a.abs() * eu + ea * up.abs() + tiny
    y = h @ wd.T
    out = {"y": (y, u * y.abs() + (1.05 * eh + chain(f) * h.abs()) @ wd.abs().T + tiny)}
    if dy is None:
        return out
    dy = dy.double()
    dh = dy @ wd
    edh = chain(c) * (dy.abs() @ wd.abs())
    du, dg = dh * a, dh * up * s
    es = (g.abs() <= eg).double() if act == "relu" else 0.8 * eg + 2.0 ** -19
    edu = u * du.abs() + edh * a.abs() + dh.abs() * (1.13 * eg + ea) + tiny
    edg = u * dg.abs() + edh * (up * s).abs() + dh.abs() * s.abs() * eu + (dh * up).abs() * es + tiny
    dx = dg @ wg + du @ wu
    k2, kr = chain(2 * f), chain(rows)
    out["dx"] = (dx, u * dx.abs() + (1.05 * edg + k2 * dg.abs()) @ wg.abs() + (1.05 * edu + k2 * du.abs()) @ wu.abs() + tiny)
    for name, d, ed, m in (("dw_gate", dg, edg, x), ("dw_up", du, edu, x)):
        v = d.T @ m
        out[name] = (v, u * v.abs() + (1.05 * ed + kr * d.abs()).T @ m.abs() + tiny)
    v = dy.T @ h
    out["dw_down"] = (v, u * v.abs() + dy.abs().T @ (1.05 * eh + kr * h.abs()) + tiny)
    return out


def _check(got, exp, name, dtype, norm=True):
    ref, tol = exp[name]
    assert got.dtype == dtype and got.shape == ref.shape and torch.isfinite(got).all(), name
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), (name, float((err - tol).max()), float(err.max()))
    if norm and ref.numel() >= 1000:
        u = torch.finfo(dtype).eps / 2
        assert float(err.norm() / ref.norm()) <= 1.5 * u, (name, float(err.norm() / ref.norm()) / u)


def _run(act, x, wg, wu, wd, dy):
    return dict(zip(NAMES, (ops.gated_ffn(x, wg, wu, wd, act), *ops.gated_ffn_grad(dy, x, wg, wu, wd, act))))


# rows x C x F: below, at and above tile borders; sizes off 8 (rows that TMA cannot address) in every position; one
# tile and many; few tiles with a long reduction in either direction (split sums)
SIZES = [(1, 8, 8), (1, 64, 128), (2, 1, 1), (3, 16, 40), (37, 33, 31), (5, 24, 257), (64, 72, 100), (127, 128, 128),
         (128, 64, 64), (129, 136, 264), (200, 256, 512), (300, 130, 513), (256, 512, 1024), (777, 333, 1001), (7, 1000, 2048),
         (1000, 16, 1000), (5000, 64, 64), (20001, 40, 24), (1, 2048, 4096), (33, 4096, 128), (130, 264, 4104)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_forward_and_backward(cuda_ops, dtype, size):
    act = ("silu", "gelu", "relu")[sum(size) % 3]
    x, wg, wu, wd, dy = _inputs(*size, dtype, seed=sum(size))
    exp = _expected(act, x, wg, wu, wd, dy)
    _check(ops.gated_ffn(x, wg, wu, wd, act), exp, "y", dtype)
    got = _run(act, x, wg, wu, wd, dy)
    for n in NAMES:
        _check(got[n], exp, n, dtype)
    again = _run(act, x, wg, wu, wd, dy)          # fixed orders of addition
    assert all(torch.equal(got[n], again[n]) for n in NAMES)
    assert lib.wait_timeouts() == 0


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_kept_projections(cuda_ops, dtype, size):
    """The forward pass that keeps G and U, and the backward pass that reads them: the same bounds."""
    act = ("silu", "gelu", "relu")[sum(size) % 3]
    x, wg, wu, wd, dy = _inputs(*size, dtype, seed=sum(size) + 1)
    exp = _expected(act, x, wg, wu, wd, dy)
    y, kept = ops.gated_ffn(x, wg, wu, wd, act, keep=True)
    _check(y, exp, "y", dtype)
    for k, w in enumerate((wg, wu)):
        ref = x.double() @ w.double().T
        tol = (size[1] / 16 + 16) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T)
        assert ((kept[k, :, :size[2]].double() - ref).abs() <= tol).all()
    got = ops.gated_ffn_grad(dy, x, wg, wu, wd, act, kept=kept)
    for n, v in zip(NAMES[1:], got):
        _check(v, exp, n, dtype)
    assert lib.wait_timeouts() == 0


@pytest.mark.parametrize("channels", [1024, 1032])
def test_autograd_on_both_sides_of_the_keeping_limit(cuda_ops, channels):
    args = _inputs(200, channels, 264, torch.bfloat16, seed=channels)
    leaves = [t.requires_grad_(True) for t in args[:4]]
    y = sb.gated_ffn(*leaves, activation="gelu")
    grads = torch.autograd.grad(y, leaves, args[4])
    exp = _expected("gelu", *(t.detach() for t in args))
    for n, v in zip(NAMES, (y.detach(), *grads)):
        _check(v, exp, n, y.dtype)


@pytest.mark.parametrize("delta", [0, 8])
def test_autograd_at_the_keeping_limit(cuda_ops, delta):
    from sbnet_b200 import autograd
    channels = autograd.KEEP_CHANNELS + delta
    args = _inputs(200, channels, 264, torch.bfloat16, seed=channels)
    leaves = [t.requires_grad_(True) for t in args[:4]]
    y = sb.gated_ffn(*leaves, activation="silu")
    assert (y.grad_fn.saved_tensors[-1] is not None) == (delta > 0)
    grads = torch.autograd.grad(y, leaves, args[4])
    exp = _expected("silu", *(t.detach() for t in args))
    for n, v in zip(NAMES, (y.detach(), *grads)):
        _check(v, exp, n, y.dtype)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [4, 40, 260])
def test_activations_over_their_range(cuda_ops, act, dtype, rows):
    """Pre-activations from far below to far above zero, zero among them."""
    x, wg, wu, wd, dy = _inputs(rows, 64, 192, dtype, seed=5)
    wg = wg * 6
    wg[::7] = 0
    exp = _expected(act, x, wg, wu, wd, dy)
    _check(ops.gated_ffn(x, wg, wu, wd, act), exp, "y", dtype, norm=False)
    got = _run(act, x, wg, wu, wd, dy)
    for n in NAMES:
        _check(got[n], exp, n, dtype, norm=False)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 32, 33, 48, 64, 65, 96, 128])
@pytest.mark.parametrize("c,f", [(256, 512), (1032, 776), (45, 70)])
def test_few_rows(cuda_ops, rows, c, f):
    x, wg, wu, wd, _ = _inputs(rows, c, f, torch.bfloat16, seed=rows)
    exp = _expected("silu", x, wg, wu, wd)
    y = ops.gated_ffn(x, wg, wu, wd)
    _check(y, exp, "y", x.dtype)
    # a row's result does not depend on which rows stand beside it
    again = ops.gated_ffn(x.flip(0).contiguous(), wg, wu, wd).flip(0)
    assert torch.equal(y, again)


# many rows and up to 256 channels: both products in one kernel; a last tile of one row and of all but one, channel counts
# around every 64, hidden counts of less than one chunk of 64, of an odd and an even number of chunks
@pytest.mark.parametrize("rows", [9217, 19200, 40191])
@pytest.mark.parametrize("c", [8, 33, 64, 72, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("f", [24, 64, 130, 192, 333])
def test_many_rows_of_few_channels(cuda_ops, rows, c, f):
    act, dtype = ("silu", "gelu", "relu")[(rows + c + f) % 3], (torch.float16, torch.bfloat16)[(c + f) % 2]
    x, wg, wu, wd, _ = _inputs(rows, c, f, dtype, seed=c + f)
    exp = _expected(act, x, wg, wu, wd)
    y = ops.gated_ffn(x, wg, wu, wd, act)
    _check(y, exp, "y", dtype)
    assert torch.equal(y, ops.gated_ffn(x, wg, wu, wd, act)) and lib.wait_timeouts() == 0


def test_many_rows_of_few_channels_stay_alone(cuda_ops):
    x, wg, wu, wd, _ = _inputs(12_000, 128, 256, torch.float16)
    want = ops.gated_ffn(x, wg, wu, wd)
    x[5000, 3], x[11999, 0] = math.nan, math.nan
    y = ops.gated_ffn(x, wg, wu, wd)
    keep = torch.ones(12_000, dtype=torch.bool, device="cuda")
    keep[5000] = keep[11999] = False
    assert torch.equal(y[keep], want[keep]) and torch.isnan(y[~keep]).all()


@pytest.mark.parametrize("rows,block", [(4, 1), (12, 3), (300, 100), (1280, 256), (2048, 64), (12_000, 100)])
@pytest.mark.parametrize("c,f", [(64, 128), (128, 512), (136, 264), (45, 70), (512, 1024)])
@pytest.mark.parametrize("part", [0.0, 0.4, 1.0, 5.0])
def test_device_count(cuda_ops, rows, block, c, f, part):
    x, wg, wu, wd, _ = _inputs(rows, c, f, torch.float16, seed=rows + c)
    blocks = rows // block
    count = int(round(part * blocks))
    live = min(count, blocks)
    x = x.view(blocks, block, c)
    x[live:] = math.nan
    out = torch.full_like(x, -7.0)
    n = torch.tensor([count], dtype=torch.int32, device="cuda")
    res = ops.gated_ffn_dyn(x, n, wg, wu, wd, "gelu", out=out)
    assert res.data_ptr() == out.data_ptr() and (out[live:] == -7).all()
    if live:
        xs = x[:live].reshape(-1, c).contiguous()
        exp = _expected("gelu", xs, wg, wu, wd)
        _check(out[:live].reshape(-1, c), exp, "y", x.dtype)
    n.fill_(-1)
    out.fill_(3)
    ops.gated_ffn_dyn(x, n, wg, wu, wd, "gelu", out=out)
    assert (out == 3).all()


@pytest.mark.parametrize("off", [1, 2, 4])
@pytest.mark.parametrize("rows", [3, 150])
def test_tensors_off_a_16_byte_boundary(cuda_ops, off, rows):
    c, f, dtype = 64, 96, torch.bfloat16
    place = lambda t: torch.full((t.numel() + 16,), math.nan, dtype=t.dtype, device="cuda")[off:off + t.numel()].view(t.shape).copy_(t)
    args = _inputs(rows, c, f, dtype)
    exp = _expected("silu", *args)
    x, wg, wu, wd, dy = (place(t) for t in args)
    buf = torch.full((rows * c + 64,), 7.0, dtype=dtype, device="cuda")
    out = buf[16 + off:16 + off + rows * c].view(rows, c)
    ops.gated_ffn(x, wg, wu, wd, out=out)
    _check(out, exp, "y", dtype)
    assert (buf[:16 + off] == 7).all() and (buf[16 + off + rows * c:] == 7).all()
    got = _run("silu", x, wg, wu, wd, dy)
    for n in NAMES:
        _check(got[n], exp, n, dtype)


def test_rows_that_are_not_finite_stay_alone(cuda_ops):
    for rows in (6, 200):
        x, wg, wu, wd, _ = _inputs(rows, 128, 256, torch.float16)
        want = ops.gated_ffn(x, wg, wu, wd)
        x[1, 5], x[4, 0] = math.inf, math.nan
        y = ops.gated_ffn(x, wg, wu, wd)
        keep = [i for i in range(rows) if i not in (1, 4)]
        assert torch.equal(y[keep], want[keep])
        assert torch.isnan(y[1]).all() and torch.isnan(y[4]).all()


def test_asked_for_gradients_only(cuda_ops):
    x, wg, wu, wd, dy = _inputs(260, 72, 136, torch.bfloat16)
    full = ops.gated_ffn_grad(dy, x, wg, wu, wd)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        part = ops.gated_ffn_grad(dy, x, wg, wu, wd, "silu", *need)
        for got, want, asked in zip(part, full, (need[0], need[1], need[1], need[2])):
            assert (got is None) == (not asked) and (got is None or torch.equal(got, want))


def test_no_rows(cuda_ops):
    x, wg, wu, wd, dy = (t.requires_grad_(True) for t in _inputs(0, 24, 40, torch.float16))
    y = sb.gated_ffn(x, wg, wu, wd)
    gx, g1, g2, g3 = torch.autograd.grad(y, (x, wg, wu, wd), dy.detach())
    assert y.shape == gx.shape == x.shape and not (g1.any() or g2.any() or g3.any())


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_autograd_against_differences(cuda_ops, act):
    """Central differences of the 64-bit definition along a random direction, against the kernel's gradients."""
    args = _inputs(40, 48, 56, torch.float16, seed=9)
    leaves = [t.clone().requires_grad_(True) for t in args[:4]]
    y = sb.gated_ffn(*leaves, activation=act)
    grads = torch.autograd.grad(y, leaves, args[4])
    dy = args[4].double()

    def f(*t):
        g, up = t[0] @ t[1].T, t[0] @ t[2].T
        return float((((_act64(act, g)[0] * up) @ t[3].T) * dy).sum())
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    exp = _expected(act, *args)
    for k, (g, name) in enumerate(zip(grads, NAMES[1:])):
        base = [t.double() for t in args[:4]]
        d = torch.randn(base[k].shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-4
        num = (f(*[t + h * d if i == k else t for i, t in enumerate(base)]) -
               f(*[t - h * d if i == k else t for i, t in enumerate(base)])) / (2 * h)
        ana = float((g.double() * d).sum())
        assert abs(num - ana) <= float((exp[name][1] * d.abs()).sum()) + 1e-4 * abs(num) + 1e-4, (name, num, ana)


def test_another_stream_and_captured_graphs(cuda_ops):
    """Two captured graphs and an eager call share nothing: each has a workspace of its own."""
    args = _inputs(300, 128, 256, torch.float16, seed=2)
    x, wg, wu, wd, dy = args
    want = _run("silu", *args)
    few = ops.gated_ffn(x[:3].contiguous(), wg, wu, wd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run("silu", *args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in NAMES)
    graphs = []
    for _ in range(2):
        g, xs = torch.cuda.CUDAGraph(), torch.zeros_like(x)
        with torch.cuda.graph(g):
            res = _run("silu", xs, wg, wu, wd, dy)
            small = ops.gated_ffn(xs[:3].contiguous(), wg, wu, wd)
        graphs.append((g, xs, res, small))
    for _, xs, _, _ in graphs:
        xs.copy_(x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for (g, _, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, _, res, small in graphs:
            assert all(torch.equal(res[n], want[n]) for n in NAMES) and torch.equal(small, few)


def test_many_rows(cuda_ops):
    """Row offsets past 2^31 elements of the hidden products."""
    rows, c, f = 140_000, 264, 16_384
    x, wg, wu, wd, _ = _inputs(256, c, f, torch.bfloat16, seed=4)
    big = torch.zeros((rows, c), dtype=x.dtype, device="cuda")
    big[-256:] = x
    y = ops.gated_ffn(big, wg, wu, wd)
    _check(y[-256:].contiguous(), _expected("silu", x, wg, wu, wd), "y", x.dtype)
    assert not y[:1000].any()


def test_a_thread_that_has_no_context_yet(cuda_ops):
    """Every call from a fresh thread whose memory all comes from the allocator's cache, so that the library's call is the
    thread's first."""
    import threading
    args = _inputs(700, 64, 136, torch.float16)
    few = [args[0][:3].contiguous(), *args[1:4]]
    many = _inputs(12_000, 64, 136, torch.float16)
    calls = [lambda: ops.gated_ffn(*args[:4]), lambda: ops.gated_ffn_grad(args[4], *args[:4])[1], lambda: ops.gated_ffn(*few),
             lambda: ops.gated_ffn(*many[:4]), lambda: ops.gated_ffn(*args[:4], keep=True)[0], lambda: ops.layer_norm(args[0])]
    for call in calls:
        want, got = call(), []
        torch.cuda.synchronize()
        thread = threading.Thread(target=lambda: got.append(call()))
        thread.start()
        thread.join()
        torch.cuda.synchronize()
        assert got and torch.equal(got[0], want)


def test_two_threads_on_streams_of_their_own(cuda_ops):
    import threading
    jobs = [_inputs(500 + 300 * i, 128, 264, torch.bfloat16, seed=i) for i in range(2)]
    want = [ops.gated_ffn_grad(j[4], *j[:4]) for j in jobs]
    torch.cuda.synchronize()
    results = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                results[i] = ops.gated_ffn_grad(jobs[i][4], *jobs[i][:4])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for got, exp in zip(results, want):
        assert all(torch.equal(g, e) for g, e in zip(got, exp))


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (3,), (0, 3), (1, 2, 3)])
def test_some_leaves_only_and_gradients_that_are_not_contiguous(cuda_ops, which):
    args = _inputs(150, 72, 136, torch.bfloat16, seed=8)
    leaves = [t.clone().requires_grad_(i in which) for i, t in enumerate(args[:4])]
    y = sb.gated_ffn(*leaves, activation="relu")
    # the gradient of a sum over the transposed result: a broadcast scalar, no memory of its own
    (y.t().sum() * 2).backward()
    exp = _expected("relu", *args[:4], torch.full_like(args[0], 2))
    for i, (leaf, name) in enumerate(zip(leaves, NAMES[1:])):
        assert (leaf.grad is not None) == (i in which)
        if i in which:
            _check(leaf.grad, exp, name, leaf.dtype, norm=False)


def test_one_matrix_for_both_projections_and_shapes_of_any_rank(cuda_ops):
    x, wg, _, wd, dy = _inputs(2 * 3 * 35, 48, 80, torch.float16, seed=6)
    shaped, dys = x.view(2, 3, 35, 48), dy.view(2, 3, 35, 48)
    y = ops.gated_ffn(shaped, wg, wg, wd)
    assert y.shape == shaped.shape
    exp = _expected("silu", x, wg, wg, wd, dy)
    _check(y.view(-1, 48), exp, "y", x.dtype)
    got = ops.gated_ffn_grad(dys, shaped, wg, wg, wd)
    for n, v in zip(NAMES[1:], got):
        _check(v.reshape(exp[n][0].shape), exp, n, x.dtype)


def test_second_derivatives_are_refused(cuda_ops):
    leaves = [t.requires_grad_(True) for t in _inputs(20, 16, 24, torch.float16)[:4]]
    y = sb.gated_ffn(*leaves)
    (g,) = torch.autograd.grad(y.float().square().sum(), leaves[:1], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|twice"):
        g.float().sum().backward()


FIRST_CALL = """
import sys
sys.path.insert(0, %r)
import torch
from sbnet_b200 import ops
x = torch.randn(%d, %d, device="cuda").half()
w = [torch.randn(s, device="cuda").half() * 0.05 for s in ((96, %d), (96, %d), (%d, 96))]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = ops.gated_ffn(ops.layer_norm(x), *w)
    d = ops.gated_ffn_grad(x, x, *w)
g.replay()
torch.cuda.synchronize()
first = y.clone(), [t.clone() for t in d]
assert torch.equal(first[0], ops.gated_ffn(ops.layer_norm(x), *w))
assert all(torch.equal(a, b) for a, b in zip(first[1], ops.gated_ffn_grad(x, x, *w)))
"""


@pytest.mark.parametrize("rows,c", [(5, 64), (300, 520), (10_000, 72)])
def test_the_first_call_of_a_process_may_be_captured(cuda_ops, rows, c):
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", FIRST_CALL % (root, rows, c, c, c, c)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
