"""Differentiable wrappers of the block ops for torch.autograd.

The reference registers its gradients in Python as compositions of the same ops
(``benchmark/sparse_conv_lib.py:80-147``, ``sbnet_ops/tests/test_sparse_blocks.py:36-98``):

* d(sparse_gather)/dx      = sparse_scatter(grad, ..., zeros_like(x), add=True, atomic=True)
* d(sparse_scatter)/dx     = sparse_gather(grad, ...)
* d(sparse_scatter)/dybase = grad                       (add=True)
                           = grad with the scattered pixels stamped out   (add=False)

Two differences from the reference, both deliberate: the scatter gradient passes ``transpose`` on to
the gather (the reference drops it, so its gradient has the wrong layout for transposed stacks), and
the stamp-out for ``add=False`` overwrites the scattered pixels of a copy of ``grad`` with zeros
directly instead of building a ones/zeros mask and multiplying.
``layer_norm`` and ``gated_ffn`` (the per-position operators of ``ops``) are differentiable once.  Their backward
passes can be captured in a CUDA graph like any other; torch's own rule applies, that no eager autograd graph of
the same leaves is alive then (it ties their gradients to the stream it was built on).

All heavy lifting happens in the CUDA library; nothing here computes on tensors itself except
allocating the zero base.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _SparseGather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bin_counts, indices, bsize, bstride, boffset, transpose):
        ctx.save_for_backward(indices)
        ctx.meta = (int(bin_counts.reshape(-1)[0]), tuple(bsize), tuple(bstride), tuple(boffset),
                    bool(transpose), x.shape, x.dtype)
        return ops.sparse_gather(x, bin_counts, indices, bsize, bstride, boffset, transpose=transpose)

    @staticmethod
    def backward(ctx, grad):
        (indices,) = ctx.saved_tensors
        nb, bsize, bstride, boffset, transpose, shape, dtype = ctx.meta
        base = torch.zeros(shape, dtype=dtype, device=grad.device)
        gx = ops.sparse_scatter_var(grad.contiguous(), [nb], indices, base, bsize, bstride, boffset,
                                    add=True, atomic=True, transpose=transpose)
        return gx, None, None, None, None, None, None


class _SparseScatter(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, bin_counts, indices, ybase, bsize, bstride, boffset, add, atomic, transpose):
        ctx.save_for_backward(indices)
        ctx.meta = (int(bin_counts.reshape(-1)[0]), tuple(bsize), tuple(bstride), tuple(boffset),
                    bool(add), bool(transpose), x.shape)
        return ops.sparse_scatter(x, bin_counts, indices, ybase, bsize, bstride, boffset, add=add,
                                  atomic=atomic, transpose=transpose)

    @staticmethod
    def backward(ctx, grad):
        (indices,) = ctx.saved_tensors
        nb, bsize, bstride, boffset, add, transpose, xshape = ctx.meta
        grad = grad.contiguous()
        gx = ops.sparse_gather(grad, [nb], indices, bsize, bstride, boffset, transpose=transpose)
        if add:
            gbase = grad
        else:   # scattered pixels do not depend on ybase: zero them in a copy of grad
            zeros = torch.zeros(xshape, dtype=grad.dtype, device=grad.device)
            gbase = ops.sparse_scatter(zeros, [nb], indices, grad, bsize, bstride, boffset, add=False,
                                       transpose=transpose)
        return gx, None, None, gbase, None, None, None, None, None, None


def sparse_gather(x, bin_counts, active_block_indices, dynamic_bsize, dynamic_bstride, dynamic_boffset,
                  transpose=False):
    """Differentiable ``SparseGather`` (gradient flows to ``x``)."""
    return _SparseGather.apply(x, bin_counts, active_block_indices, dynamic_bsize, dynamic_bstride,
                               dynamic_boffset, transpose)


def sparse_scatter(x, bin_counts, active_block_indices, ybase, dynamic_bsize, dynamic_bstride,
                   dynamic_boffset, add, atomic=False, transpose=False):
    """Differentiable ``SparseScatter`` (gradients flow to the block stack ``x`` and to ``ybase``)."""
    return _SparseScatter.apply(x, bin_counts, active_block_indices, ybase, dynamic_bsize,
                                dynamic_bstride, dynamic_boffset, add, atomic, transpose)


def _will_differentiate(*inputs):
    """Whether a backward pass can follow a call made now.  Asked before ``apply``: inside ``forward`` the grad mode is
    always off, and ``ctx.needs_input_grad`` speaks of the leaves whatever the mode."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, keep):
        stats = None
        if keep:
            y, stats = ops.layer_norm(x, weight, bias, eps, stats=True)
        else:
            y = ops.layer_norm(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        param = weight if weight is not None else bias
        wdtype = ops._DTYPES[x.dtype if param is None else param.dtype]
        gx, gw, gb = ops._layer_norm_grad_call(grad.contiguous(), x, stats, weight, bias, stats.shape[1], x.shape[-1],
                                               wdtype, need[1] or need[2])
        return gx, gw, gb, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Differentiable :func:`sbnet_b200.ops.layer_norm` (gradients flow to ``x``, ``weight`` and ``bias``)."""
    return _LayerNorm.apply(x, weight, bias, eps, _will_differentiate(x, weight, bias))


# Beyond this many channels the forward pass of the gated feed-forward block keeps its two projections (8 bytes per
# hidden element) for the backward pass, where one can follow; up to it they are multiplied again.  Forward + backward
# in bf16, kept against multiplied again: 32,768 x 512 x 2,048 690 / 670 us, 16,384 x 768 x 2,304 573 / 588,
# 16,384 x 896 x 3,584 994 / 1,109, 16,384 x 1,024 x 4,096 1,171 / 1,306; with 300 rows keeping costs 6 us more at 1,024
# channels (115 / 109).  The limit is on the channels alone: at 768 many rows would be 3 % quicker kept, which does not
# pay for the memory.
KEEP_CHANNELS = 768


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation, keep):
        kept = None
        if keep:
            y, kept = ops.gated_ffn(x, w_gate, w_up, w_down, activation, keep=True)
        else:
            y = ops.gated_ffn(x, w_gate, w_up, w_down, activation)
        ctx.save_for_backward(x, w_gate, w_up, w_down, kept)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, w_gate, w_up, w_down, kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        channels = x.shape[-1]
        return (*ops._gated_ffn_grad_call(grad.contiguous(), x, w_gate, w_up, w_down, x.numel() // channels, channels,
                                          w_gate.shape[0], ops._lib.SBNET_ACT[ctx.activation],
                                          need[0], need[1] or need[2], need[3], kept), None, None)


def gated_ffn(x, w_gate, w_up, w_down, activation="silu"):
    """Differentiable :func:`sbnet_b200.ops.gated_ffn` (gradients flow to ``x`` and the three weights).  Up to
    ``KEEP_CHANNELS`` channels nothing but the inputs is kept for the backward pass."""
    keep = x.dim() > 0 and x.shape[-1] > KEEP_CHANNELS and _will_differentiate(x, w_gate, w_up, w_down)
    return _GatedFfn.apply(x, w_gate, w_up, w_down, activation, keep)
