"""What the differentiable per-position operators ask of the kernels in each grad mode: a call that nothing can be
differentiated through keeps nothing for a backward pass.  Kernels are replaced by their definitions on the CPU."""
import contextlib

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from sbnet_b200 import autograd as sb
from sbnet_b200 import ops

CHANNELS = sb.KEEP_CHANNELS + 8


@pytest.fixture
def calls(monkeypatch):
    seen = []

    def gated_ffn(x, w_gate, w_up, w_down, activation="silu", out=None, keep=False):
        seen.append(keep)
        g, u = x @ w_gate.t(), x @ w_up.t()
        y = (F.silu(g) * u) @ w_down.t()
        return (y, torch.stack((g, u))) if keep else y

    def layer_norm(x, weight=None, bias=None, eps=1e-5, out=None, stats=False):
        seen.append(stats)
        y = F.layer_norm(x, x.shape[-1:], weight, bias, eps)
        return (y, torch.zeros(2, x.numel() // x.shape[-1])) if stats else y
    monkeypatch.setattr(ops, "gated_ffn", gated_ffn)
    monkeypatch.setattr(ops, "layer_norm", layer_norm)
    return seen


def _ffn(channels=CHANNELS, hidden=8, grad=True):
    gen = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=gen)
    return r(3, channels), *(nn.Parameter(t, requires_grad=grad) for t in (r(hidden, channels), r(hidden, channels), r(channels, hidden)))


MODES = {"no_grad": torch.no_grad, "inference_mode": torch.inference_mode, "grad": contextlib.nullcontext}


@pytest.mark.parametrize("mode", ["no_grad", "inference_mode"])
def test_projections_are_not_kept_without_a_graph(calls, mode):
    args = _ffn()
    with MODES[mode]():
        y = sb.gated_ffn(*args)
    assert calls == [False] and not y.requires_grad
    kept = sb.gated_ffn(*args)
    assert calls == [False, True] and kept.requires_grad and torch.equal(kept.detach(), y)


def test_projections_are_not_kept_for_constants(calls):
    assert not sb.gated_ffn(*_ffn(grad=False)).requires_grad and calls == [False]


@pytest.mark.parametrize("which", range(4))
def test_projections_are_kept_for_any_leaf(calls, which):
    args = [t.detach().requires_grad_(i == which) for i, t in enumerate(_ffn())]
    y = sb.gated_ffn(*args)
    assert y.requires_grad and calls == [True] and y.grad_fn.saved_tensors[-1] is not None


def test_projections_are_not_kept_up_to_the_limit(calls):
    assert sb.gated_ffn(*_ffn(sb.KEEP_CHANNELS)).requires_grad and calls == [False]


def test_a_graph_inside_and_outside_a_block_without_one(calls):
    args = _ffn()
    with torch.no_grad():
        sb.gated_ffn(*args)
        with torch.enable_grad():
            assert sb.gated_ffn(*args).requires_grad
        sb.gated_ffn(*args)
    assert calls == [False, True, False]


def _norm(weight=True, grad=True):
    x = torch.randn(5, 16, generator=torch.Generator().manual_seed(2))
    return x, *((nn.Parameter(torch.ones(16), requires_grad=grad), nn.Parameter(torch.zeros(16), requires_grad=grad)) if weight else (None, None))


@pytest.mark.parametrize("mode", ["no_grad", "inference_mode"])
def test_statistics_are_not_written_without_a_graph(calls, mode):
    with MODES[mode]():
        y = sb.layer_norm(*_norm())
    trained = sb.layer_norm(*_norm())
    assert calls == [False, True] and not y.requires_grad and trained.requires_grad and torch.equal(trained.detach(), y)


@pytest.mark.parametrize("weight", [True, False])
def test_statistics_are_not_written_for_constants(calls, weight):
    assert not sb.layer_norm(*_norm(weight, grad=False)).requires_grad and calls == [False]


@pytest.mark.parametrize("which", range(3))
def test_statistics_are_written_for_any_leaf(calls, which):
    y = sb.layer_norm(*[t.detach().requires_grad_(i == which) for i, t in enumerate(_norm())])
    assert y.requires_grad and calls == [True] and y.grad_fn.saved_tensors[-1] is not None
