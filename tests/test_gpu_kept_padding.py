"""The padding columns of the kept projections (hidden counts off a multiple of 8) are undefined; whatever they hold, the
backward pass gives the same bits."""
import math

import pytest
import torch

from sbnet_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,c,f", [(130, 40, 33), (3, 16, 1), (300, 72, 257), (777, 333, 1001), (260, 64, 250), (60_001, 16, 17)])
def test_padding_of_the_kept_projections_does_not_matter(cuda_ops, dtype, act, rows, c, f):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows + c + f)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=gen, device="cuda") * scale).to(dtype)
    # gates of some size either side of zero: the rounding of a sigmoid then depends on every step that leads to it
    x, dy = r(rows, c), r(rows, c)
    wg, wu, wd = r(f, c, scale=3 * c ** -0.5), r(f, c, scale=c ** -0.5), r(c, f, scale=f ** -0.5)
    _, kept = ops.gated_ffn(x, wg, wu, wd, act, keep=True)
    kept[..., f:] = 0
    want = ops.gated_ffn_grad(dy, x, wg, wu, wd, act, kept=kept)
    for pad in (50.0, -50.0, -3.0, 1e30, -math.inf, math.nan):
        kept[..., f:] = pad
        for name, g, e in zip(("dx", "dw_gate", "dw_up", "dw_down"), ops.gated_ffn_grad(dy, x, wg, wu, wd, act, kept=kept), want):
            assert torch.equal(g, e), (name, pad)
