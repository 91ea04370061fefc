"""Residual blocks on the block ops: y = x + F(x) evaluated only on active blocks.

:class:`SparseBottleneck`: the sparse ResNet bottleneck.  Mirrors the structure of the reference's ``sparse_res_block_bottleneck``
(``benchmark/sparse_conv_lib.py:677-824``): sparse_gather of 18x18 (in general ``bsize``) windows ->
BN-ReLU-1x1, BN-ReLU-3x3 VALID, BN-ReLU-1x1 on the block stack (the host framework's dense ops, here
torch / cuDNN in NCHW, i.e. ``transpose=True``) -> sparse_scatter(add=True) of the ``bsize_out``
interiors onto the residual.  The convolutions are NOT part of this library; the module exists so
the op pipeline can be exercised and timed in its real setting.

:class:`SparseGatedBlock`: a per-position residual branch (layer norm, then the gated feed-forward block) on the
same pipeline; the branch itself is this library's (``ops.layer_norm``, ``ops.gated_ffn``).
"""
from __future__ import annotations

from typing import Sequence

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import autograd as sb
from . import geometry, ops


class SparseBottleneck(nn.Module):
    def __init__(self, channels: int, mid: int, bsize: Sequence[int] = (18, 18), dtype=torch.float16,
                 device="cuda"):
        super().__init__()
        self.channels, self.mid, self.bsize = channels, mid, tuple(bsize)
        kw = dict(device=device, dtype=dtype)
        self.bn = nn.ModuleList([nn.BatchNorm2d(channels, **kw), nn.BatchNorm2d(mid, **kw), nn.BatchNorm2d(mid, **kw)])
        self.conv1 = nn.Conv2d(channels, mid, 1, bias=False, **kw)
        self.conv2 = nn.Conv2d(mid, mid, 3, bias=False, **kw)          # VALID: 18x18 -> 16x16
        self.conv3 = nn.Conv2d(mid, channels, 1, bias=False, **kw)
        for c in (self.conv1, self.conv2, self.conv3):
            nn.init.kaiming_normal_(c.weight, nonlinearity="relu")

    def block_params(self, x_shape) -> geometry.BlockParams:
        N, H, W, C = x_shape
        ks = [[1, 1, C, self.mid], [3, 3, self.mid, self.mid], [1, 1, self.mid, C]]
        return geometry.calc_block_params_res_block([N, H, W, C], [1, *self.bsize, 1], ks, [1, 1, 1, 1], "SAME")

    def residual(self, p: torch.Tensor) -> torch.Tensor:
        q = self.conv1(F.relu(self.bn[0](p)))
        q = self.conv2(F.relu(self.bn[1](q)))
        return self.conv3(F.relu(self.bn[2](q)))

    def forward(self, x: torch.Tensor, mask: torch.Tensor, tol: float = 0.5, avgpool: bool = False):
        """``x`` NHWC, ``mask`` [N,H,W,1] fp32.  Returns NHWC ``x + F(x)`` on active blocks, ``x`` elsewhere."""
        bp = self.block_params(x.shape)
        idx, cnt = ops.reduce_mask(mask, bp.bcount, bp.bsize, bp.bstrides, bp.boffset, tol=tol, avgpool=avgpool)
        p = sb.sparse_gather(x, cnt, idx, bp.bsize, bp.bstrides, bp.boffset, transpose=True)
        q = self.residual(p).contiguous()
        return sb.sparse_scatter(q, cnt, idx, x, bp.bsize_out, bp.bsize_out, [0, 0], add=True, transpose=True)


class SparseGatedBlock(nn.Module):
    """``y = x + FFN(LN(x))`` on the active blocks of an NHWC image, ``x`` elsewhere.

    The branch looks at one position at a time, so blocks need no halo: ``bsize`` blocks on a pitch of ``bsize``,
    gathered in the rows layout (``[nB, bh, bw, C]``), normed over the channels, sent through the gated feed-forward
    block ``(act(u Wg^T) * (u Wu^T)) Wd^T`` and scattered back with ``add=True``.  ``dtype``: float16 or bfloat16 (the
    feed-forward block's types); the norm's parameters are float32."""

    def __init__(self, channels: int, hidden: int, bsize: Sequence[int] = (16, 16), activation: str = "silu",
                 eps: float = 1e-5, dtype=torch.float16, device="cuda"):
        super().__init__()
        self.channels, self.hidden, self.bsize = channels, hidden, tuple(bsize)
        self.activation, self.eps = activation, eps
        self.norm_weight = nn.Parameter(torch.ones(channels, device=device))
        self.norm_bias = nn.Parameter(torch.zeros(channels, device=device))
        kw = dict(device=device, dtype=dtype)
        self.w_gate = nn.Parameter(torch.empty(hidden, channels, **kw).normal_(std=channels ** -0.5))
        self.w_up = nn.Parameter(torch.empty(hidden, channels, **kw).normal_(std=channels ** -0.5))
        self.w_down = nn.Parameter(torch.empty(channels, hidden, **kw).normal_(std=hidden ** -0.5))

    def _geometry(self, x_shape):
        """``(bcount, bsize, bstride, boffset)`` of the blocks that tile an image."""
        bcount = [-(-x_shape[1] // self.bsize[0]), -(-x_shape[2] // self.bsize[1])]
        return bcount, self.bsize, self.bsize, (0, 0)

    def residual(self, p: torch.Tensor) -> torch.Tensor:
        u = sb.layer_norm(p, self.norm_weight, self.norm_bias, self.eps)
        return sb.gated_ffn(u, self.w_gate, self.w_up, self.w_down, self.activation)

    def forward(self, x: torch.Tensor, mask: torch.Tensor, tol: float = 0.5, avgpool: bool = False):
        """``x`` NHWC of the block's dtype, ``mask`` [N,H,W,1] fp32.  Differentiable."""
        geom = self._geometry(x.shape)
        idx, cnt = ops.reduce_mask(mask, *geom, tol=tol, avgpool=avgpool)
        p = sb.sparse_gather(x, cnt, idx, *geom[1:])
        return sb.sparse_scatter(self.residual(p), cnt, idx, x, *geom[1:], add=True)

    @torch.no_grad()
    def forward_async(self, x: torch.Tensor, mask: torch.Tensor, tol: float = 0.5, avgpool: bool = False,
                      max_blocks: int = None) -> torch.Tensor:
        """:meth:`forward` for inference without a host round trip: the block count stays on the device from the mask
        to the scatter, and the call can be captured in a CUDA graph.  ``max_blocks``: room in the block stacks
        (default: every block of the image); blocks past it are left out."""
        geom = self._geometry(x.shape)
        total = x.shape[0] * geom[0][0] * geom[0][1]
        room = total if max_blocks is None else min(int(max_blocks), total)
        idx, count = ops.reduce_mask_async(mask, *geom, tol=tol, avgpool=avgpool)
        p = ops.sparse_gather_dyn(x, count, room, idx, *geom[1:])
        u = ops.layer_norm_dyn(p, count, self.norm_weight, self.norm_bias, self.eps)
        q = ops.gated_ffn_dyn(u, count, self.w_gate, self.w_up, self.w_down, self.activation, out=p)
        y = ops.copy_tensor(torch.empty_like(x), x)
        return ops.sparse_scatter_var_dyn(q, count, room, idx, y, *geom[1:], add=True)
