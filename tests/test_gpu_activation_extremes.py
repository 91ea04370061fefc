"""The gated feed-forward block at pre-activations far from zero, against the 64-bit definition.

The weights pick single channels, so that every product and sum is exact: G[r, f] = x[r, 0] * sign[f], U[r, f] = x[r, 1],
Y[r, f] = H[r, f] for f < F, and dX[r, F + f] = dG[r, f] (the one non-zero weight in that column).  What is left are the
element-wise steps and the rounding of H and dG to the tensors' type (u, half a step; the second rounding of the same
value is exact):

* silu: 2^x with x = -g log2(e), |x| <= 60 where it matters: the constant and the product are off by 2^-24 of x each,
  which is 120 ln 2 * 2^-24 < 2^-17.5 of the result; the instruction adds 2^-22, reciprocal and products a few 2^-23.
  Hence 2^-17 of sig, of a = g sig and of a (1 - sig) each.  Sigmoids below 2^-60 read as 2^-60, at most 42 * 2^-60 in a.
* gelu: Phi is off by 0.75e-7 (the approximation) and some 2^-22 where it is not 0 or 1 to fp32, |g| < 8: 2^-21 of that g.
* relu: exact.
"""
import math

import pytest
import torch

from sbnet_b200 import lib, ops

pytestmark = pytest.mark.gpu

F, C = 16, 32
MAGNITUDES = [0.0, 2.0 ** -10, 0.5, 1.0, 4.0, 10.0, 16.0, 40.0, 41.5, 42.0, 60.0, 88.0, 104.0, 1000.0, 2.0 ** 14, 60000.0]
LARGER = [1e6, 1e8, 1e12, 1e18, 1e20, 1e30]


def _case(dtype, rows, up):
    values = MAGNITUDES + (LARGER if dtype == torch.bfloat16 else [])
    values = torch.tensor(values + [-v for v in values], dtype=torch.float64)
    x = torch.zeros(rows, C, dtype=torch.float64)
    x[:, 0] = values[torch.arange(rows) % len(values)]
    x[:, 1] = up
    wg, wu, wd = torch.zeros(F, C), torch.zeros(F, C), torch.zeros(C, F)
    f = torch.arange(F)
    wg[f, 0] = torch.where(f % 3 == 0, -1.0, 1.0)       # pairs of neighbours of one sign and of both
    for k, small in ((1, 0.0), (2, 2.0 ** -14), (4, 2.0 ** -16), (8, -2.0 ** -15), (10, 2.0 ** -12), (12, 2.0 ** -30), (14, 2.0 ** -18)):
        wg[k, 0] = small                                # beside a neighbour whose gate is large
    wg[f, F + f] = 1.0                                  # x is zero there
    wu[f, 1] = 1.0
    wd[f, f] = 1.0
    dy = torch.zeros(rows, C)
    dy[:, :F] = 1.0
    return [t.to(dtype).cuda() for t in (x, wg, wu, wd, dy)]


def _reference(act, x, wg, up):
    g = x.double()[:, :1] * wg.double()[:, 0]
    if act == "silu":
        s = torch.sigmoid(g)
        a, slope = g * s, s * (1 + g * torch.sigmoid(-g))
        ta, ts = 2.0 ** -17 * a.abs() + 42 * 2.0 ** -60, 2.0 ** -17 * (s + (a * torch.sigmoid(-g)).abs()) + 43 * 2.0 ** -60
    elif act == "gelu":
        cdf, density = torch.special.ndtr(g), torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        a, slope = g * cdf, cdf + g * density
        near = g.abs().clamp(max=8)
        ta, ts = 2.0 ** -21 * near + 2.0 ** -22 * a.abs(), 2.0 ** -20 * (1 + near)
    else:
        a, slope = g.clamp(min=0), (g > 0).double()
        ta = ts = torch.zeros_like(g)
    return a * up, ta * abs(up), slope * up, ts * abs(up)


def _near(got, want, tol, dtype):
    u, info = torch.finfo(dtype).eps / 2, torch.finfo(dtype)
    err = (got.double() - want).abs()
    bar = tol + u * (want.abs() + tol) + info.smallest_normal * info.eps
    bad = ~(err <= bar)
    assert not bad.any(), [(float(want[i, j]), float(got[i, j]), float(bar[i, j])) for i, j in bad.nonzero()[:8].tolist()]


# the forms for a few rows, for some and for many
@pytest.mark.parametrize("rows", [4, 16, 32, 64, 300, 9217])
@pytest.mark.parametrize("up", [1.0, -0.75])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_far_from_zero(cuda_ops, dtype, act, up, rows):
    all_x, wg, wu, wd, all_dy = _case(dtype, max(rows, 64), up)
    for first in range(0, all_x.shape[0] - rows + 1, rows):
        x, dy = all_x[first:first + rows].contiguous(), all_dy[first:first + rows].contiguous()
        h, th, dg, tg = _reference(act, x, wg, up)
        y, kept = ops.gated_ffn(x, wg, wu, wd, act, keep=True)
        for out in (ops.gated_ffn(x, wg, wu, wd, act), y):
            _near(out[:, :F], h, th, dtype)
        for k in (None, kept):
            dx, _, _, dwd = ops.gated_ffn_grad(dy, x, wg, wu, wd, act, kept=k)
            _near(dx[:, F:2 * F], dg, tg, dtype)
    assert lib.wait_timeouts() == 0


@pytest.mark.parametrize("rows", [4, 300, 9217])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_a_gate_that_is_not_a_number_is_not_hidden(cuda_ops, act, rows):
    x, wg, wu, wd, _ = _case(torch.bfloat16, rows, 1.0)
    assert torch.isfinite(ops.gated_ffn(x, wg, wu, wd, act)).all()
    wg[7, 0] = math.nan         # U is finite
    assert torch.isnan(ops.gated_ffn(x, wg, wu, wd, act)).all()


@pytest.mark.parametrize("rows", [16, 300, 9217])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_large_gate_beside_any_neighbour(cuda_ops, dtype, act, rows):
    """Two neighbours share a reciprocal in silu: what it is off by must not be multiplied with a large gate."""
    x, wg, wu, wd, dy = _case(dtype, rows, 1.0)
    top = 15 if dtype == torch.float16 else 40
    x[:, 0] = 2.0 ** torch.linspace(3, top, rows, dtype=torch.float64)[torch.randperm(rows, generator=torch.Generator().manual_seed(rows))]
    x[:, 2] = torch.linspace(-9, 9, rows, dtype=torch.float64)
    wg[:, :3] = 0
    for f in range(F):      # one of each pair is large, either first or second, the other from the sweep
        wg[f, 2 * (f % 4 in (0, 3))] = 1.0
    wu[:, 2] = 0
    g = x.double() @ wg.double().T
    one = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    y, kept = ops.gated_ffn(x, wg, wu, wd, act, keep=True)
    for k in (None, kept):
        dx = ops.gated_ffn_grad(dy, x, wg, wu, wd, act, kept=k)[0]
        for f in range(F):
            h, th, dg, tg = _reference(act, g[:, f:f + 1], one, 1.0)
            _near(dx[:, F + f:F + f + 1], dg, tg, dtype)
            _near(y[:, f:f + 1], h, th, dtype)
