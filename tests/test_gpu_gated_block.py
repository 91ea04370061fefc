"""The gated residual block on active blocks: the block ops, layer norm and the gated feed-forward block together,
against a dense evaluation in 64 bits, forward, backward and without a host round trip."""
import math

import pytest
import torch

from sbnet_b200 import configs as cfg
from sbnet_b200.resblock import SparseGatedBlock

pytestmark = pytest.mark.gpu


def _setup(N, H, W, C, F, act, dtype, bsize, seed=0, density=0.3):
    torch.manual_seed(seed)
    block = SparseGatedBlock(C, F, bsize, act, dtype=dtype)
    with torch.no_grad():
        block.norm_weight.add_(0.2 * torch.randn_like(block.norm_weight))
        block.norm_bias.add_(0.2 * torch.randn_like(block.norm_bias))
    x = (torch.randn((N, H, W, C), device="cuda") * 1.5 + 0.2).to(dtype)
    gh, gw = -(-H // bsize[0]), -(-W // bsize[1])
    live = torch.rand((N, gh, gw), device="cuda") < density
    live[0, 0, 0] = True
    mask = live.repeat_interleave(bsize[0], 1).repeat_interleave(bsize[1], 2)[:, :H, :W, None].float().contiguous()
    return block, x, mask


def _dense(block, x, mask):
    """x + FFN(LN(x)) in 64 bits where the mask is set (it is constant on blocks)."""
    p = [t.double() for t in (x, block.norm_weight, block.norm_bias, block.w_gate, block.w_up, block.w_down)]
    var, mean = torch.var_mean(p[0], dim=-1, unbiased=False, keepdim=True)
    u = (p[0] - mean) / torch.sqrt(var + block.eps) * p[1] + p[2]
    g = u @ p[3].T
    g = {"silu": lambda: g * torch.sigmoid(g), "gelu": lambda: g * torch.special.ndtr(g), "relu": lambda: g.clamp(min=0)}[block.activation]()
    return p[0] + mask.double() * ((g * (u @ p[4].T)) @ p[5].T)


CASES = [(2, 48, 40, 64, 128, "silu", torch.float16, (16, 16)), (1, 31, 45, 24, 56, "gelu", torch.bfloat16, (8, 4)),
         (1, 30, 30, 33, 70, "relu", torch.float16, (7, 9)), (3, 128, 128, 128, 256, "silu", torch.bfloat16, (16, 16))]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[1]}x{c[2]}x{c[3]}")
def test_forward_and_gradients(cuda_ops, case):
    """Rounded to the tensors' type on the way: x, LN(x), H, the branch and the sum (each off by u = eps/2 of itself) --
    five independent roundings, each of which reaches the result with no more than its own size for random
    weights.  The norm of the error stays below 4u of the result's for y, and of the gradients' (dY, dG and dU,
    the norm's input gradient, its sum with dY, LN(x)) below 6u."""
    block, x, mask = _setup(*case)
    u = torch.finfo(x.dtype).eps / 2
    x.requires_grad_(True)
    y = block(x, mask)
    want = _dense(block, x, mask)
    assert float((y.detach().double() - want.detach()).norm() / want.detach().norm()) <= 4 * u
    off = (mask == 0).expand_as(x)
    assert torch.equal(y.detach()[off], x.detach()[off])
    dy = torch.randn_like(y)
    leaves = [x, block.norm_weight, block.norm_bias, block.w_gate, block.w_up, block.w_down]
    got = torch.autograd.grad(y, leaves, dy)
    exp = torch.autograd.grad(want, leaves, dy.double())
    for g, e, leaf in zip(got, exp, leaves):
        # torch casts the 64-bit gradient to the leaf's type: one more rounding
        assert g.dtype == leaf.dtype and float((g.double() - e.double()).norm() / e.double().norm()) <= 6 * u


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[1]}x{c[2]}x{c[3]}")
def test_device_count_form_gives_the_same_bits(cuda_ops, case):
    block, x, mask = _setup(*case, seed=3)
    want = block(x, mask).detach()
    assert torch.equal(block.forward_async(x, mask), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = block.forward_async(x, mask)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(side, want)


def test_captured_in_a_graph_with_changing_counts(cuda_ops):
    block, x, mask = _setup(2, 64, 64, 64, 128, "silu", torch.float16, (16, 16), seed=5)
    xs, ms = torch.zeros_like(x), torch.zeros_like(mask)
    block.forward_async(xs, ms)      # first calls outside of a capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = block.forward_async(xs, ms)
    for seed in range(4):
        _, x, mask = _setup(2, 64, 64, 64, 128, "silu", torch.float16, (16, 16), seed=seed, density=0.25 * seed)
        xs.copy_(x), ms.copy_(mask)
        g.replay()
        assert torch.equal(y, block(x, mask).detach())


def test_training_step_captured_in_a_graph(cuda_ops):
    """Forward and backward in one graph, after eager steps of the same parameters whose results (not whose autograd
    graphs: torch ties a leaf's accumulation to the stream of the first graph that lives) are kept."""
    torch.manual_seed(1)
    from sbnet_b200 import autograd as sb
    x = torch.randn((300, 72), device="cuda").bfloat16()
    ws = [torch.randn(s, device="cuda").mul_(0.1).bfloat16().requires_grad_(True) for s in ((120, 72), (120, 72), (72, 120))]
    w = torch.ones(72, device="cuda", requires_grad=True)
    b = torch.zeros(72, device="cuda", requires_grad=True)
    dy = torch.randn_like(x)

    def step(inp):
        y = sb.gated_ffn(sb.layer_norm(inp, w, b), *ws, activation="gelu")
        return y.detach(), torch.autograd.grad(y, (w, b, *ws), dy)
    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x)
    torch.cuda.current_stream().wait_stream(side)
    xs = torch.zeros_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(xs)
    xs.copy_(x)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and all(torch.equal(p, q) for p, q in zip(got[1], want[1]))


def test_parameters_train(cuda_ops):
    """One optimiser step changes every parameter and nothing is left undefined."""
    block, x, mask = _setup(1, 32, 32, 64, 128, "gelu", torch.bfloat16, (16, 16))
    opt = torch.optim.SGD(block.parameters(), lr=0.1)
    before = [p.detach().clone() for p in block.parameters()]
    block(x, mask).float().square().mean().backward()
    opt.step()
    for p, q in zip(block.parameters(), before):
        assert torch.isfinite(p).all() and not torch.equal(p, q)
