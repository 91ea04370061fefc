"""Memory of the differentiable feed-forward block in inference: nothing is kept for a backward pass that cannot come."""
import pytest
import torch

from sbnet_b200 import autograd as sb
from sbnet_b200 import ops
from sbnet_b200.resblock import SparseGatedBlock

pytestmark = pytest.mark.gpu

ROWS, HIDDEN = 4096, 4096
CHANNELS = sb.KEEP_CHANNELS + 8
KEPT = 2 * ROWS * HIDDEN * 4


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode], ids=["no_grad", "inference_mode"])
def test_inference_does_not_hold_the_projections(cuda_ops, mode):
    torch.manual_seed(0)
    block = SparseGatedBlock(CHANNELS, HIDDEN, dtype=torch.bfloat16)
    x = torch.randn(ROWS, CHANNELS, device="cuda", dtype=torch.bfloat16)
    args = (x, block.w_gate, block.w_up, block.w_down)
    want = ops.gated_ffn(*args)
    peak = {}
    for name, cm in (("inference", mode()), ("training", torch.enable_grad())):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        with cm:
            y = sb.gated_ffn(*args)
        peak[name] = torch.cuda.max_memory_allocated() - before
        assert y.requires_grad == (name == "training") and torch.equal(y, want)
        del y
    assert peak["training"] >= KEPT > peak["inference"]


@pytest.mark.parametrize("channels", [64, CHANNELS])
def test_the_block_in_inference_equals_training(cuda_ops, channels):
    torch.manual_seed(1)
    block = SparseGatedBlock(channels, 136, (8, 8))
    x = torch.randn(2, 40, 24, channels, device="cuda").half()
    mask = (torch.rand(2, 40, 24, 1, device="cuda") > 0.9).float()
    trained = block(x, mask)
    with torch.no_grad():
        assert torch.equal(block(x, mask), trained.detach())
