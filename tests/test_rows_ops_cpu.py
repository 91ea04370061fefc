"""Argument rules of the per-position operators (layer norm, gated feed-forward), checked without a GPU: every
wrapper raises ValueError, and every C entry returns an error status, before anything could be launched."""
import pytest
import torch

from sbnet_b200 import ops

BAD = -1


@pytest.fixture(scope="module")
def handle():
    from sbnet_b200 import build, lib
    build.build_library()
    return lib.load()


def test_row_rules():
    assert ops._check_rows(torch.zeros(2, 3, 5), "x") == (6, 5)
    assert ops._check_rows(torch.zeros(0, 5), "x") == (0, 5)
    assert ops._check_rows(torch.zeros(7), "x") == (1, 7)
    with pytest.raises(ValueError, match="at least one channel"):
        ops._check_rows(torch.zeros(4, 0), "x")
    with pytest.raises(ValueError, match="dtype"):
        ops._check_rows(torch.zeros(4, 4, dtype=torch.float64), "x")
    with pytest.raises(ValueError, match="contiguous"):
        ops._check_rows(torch.zeros(4, 6).t(), "x")
    assert ops._blocks_of(torch.zeros(4, 2, 3, 8)) == (4, 6)
    with pytest.raises(ValueError, match="block stack"):
        ops._blocks_of(torch.zeros(8))
    with pytest.raises(ValueError, match="at least one row"):
        ops._blocks_of(torch.zeros(4, 0, 8))


def test_layer_norm_rules():
    x = torch.zeros(4, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.layer_norm(x)
    for w, why in [(torch.zeros(7), r"\[8\]"), (torch.zeros(8, 1), r"\[8\]"), (torch.zeros(16)[::2], "contiguous"),
                   (torch.zeros(8, dtype=torch.bfloat16), "float32")]:
        with pytest.raises(ValueError, match=why):
            ops.layer_norm(x, w)
        with pytest.raises(ValueError, match=why):
            ops.layer_norm(x, None, w)
    with pytest.raises(ValueError, match="share a dtype"):
        ops.layer_norm(x, torch.zeros(8), torch.zeros(8, dtype=torch.float16))
    for out in (torch.zeros(4, 7, dtype=torch.float16), torch.zeros(4, 8), torch.zeros(8, 4, dtype=torch.float16).t()):
        with pytest.raises(ValueError, match="out"):
            ops.layer_norm(x, out=out)
    with pytest.raises(ValueError, match="count_dev"):
        ops.layer_norm_dyn(x, None)
    with pytest.raises(ValueError, match="int32"):
        ops.layer_norm_dyn(x, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError, match="grad"):
        ops.layer_norm_grad(torch.zeros(4, 8), x, torch.zeros(2, 4))
    for bad in (torch.zeros(2, 3), torch.zeros(8), torch.zeros(2, 4, dtype=torch.float16), torch.zeros(4, 2).t()):
        with pytest.raises(ValueError, match="stats"):
            ops.layer_norm_grad(x, x, bad)


def test_layer_norm_c_entries_refuse(handle):
    norm, dyn, grad = handle.sbnet_layer_norm, handle.sbnet_layer_norm_dyn, handle.sbnet_layer_norm_grad
    a, b, c = 1 << 20, 1 << 24, 1 << 28        # addresses that are never touched
    assert norm(a, 9, 4, 8, None, None, 0, 1e-5, b, None, None, None) == BAD            # dtype
    assert norm(a, 0, -1, 8, None, None, 0, 1e-5, b, None, None, None) == BAD           # rows
    assert norm(a, 0, 4, 0, None, None, 0, 1e-5, b, None, None, None) == BAD            # channels
    assert norm(a, 0, 1 << 40, 8, None, None, 0, 1e-5, b, None, None, None) == -2       # too many elements
    assert norm(a, 1, 4, 8, c, None, 2, 1e-5, b, None, None, None) == BAD               # weight type
    assert norm(a, 0, 4, 8, None, None, 0, -1.0, b, None, None, None) == BAD            # eps
    assert norm(a, 0, 4, 8, None, None, 0, float("nan"), b, None, None, None) == BAD
    assert norm(a, 0, 4, 8, None, None, 0, 1e-5, b, c, None, None) == BAD               # mean without rstd
    assert norm(None, 0, 4, 8, None, None, 0, 1e-5, b, None, None, None) == BAD
    assert norm(a, 0, 4, 8, None, None, 0, 1e-5, a + 64, None, None, None) == BAD       # overlap
    assert norm(a + 1, 1, 4, 8, None, None, 1, 1e-5, b, None, None, None) == BAD        # alignment
    assert norm(a, 0, 0, 8, None, None, 0, 1e-5, b, None, None, None) == 0              # nothing to do
    assert dyn(a, 0, 4, 2, None, 8, None, None, 0, 1e-5, b, None, None, None) == BAD    # no count
    assert dyn(a, 0, 4, 0, c, 8, None, None, 0, 1e-5, b, None, None, None) == BAD       # empty blocks
    assert grad(a, a, 0, 4, 8, None, 0, None, None, b, None, None, None, 0, None) == BAD
    assert grad(a, a, 0, 4, 8, None, 0, c, c, a, None, None, None, 0, None) == BAD      # overlap
    assert grad(a, a, 0, 4, 8, c, 0, c, c, b, c, None, None, 0, None) == BAD            # no workspace
    need = handle.sbnet_layer_norm_grad_workspace(4, 8)
    assert need > 0 and grad(a, a, 0, 4, 8, c, 0, c, c, b, c, None, c, need - 1, None) == BAD
    assert handle.sbnet_last_error()


def _ffn_args(c=8, f=16, dtype=torch.float16, rows=4):
    return (torch.zeros(rows, c, dtype=dtype), torch.zeros(f, c, dtype=dtype), torch.zeros(f, c, dtype=dtype),
            torch.zeros(c, f, dtype=dtype))


def test_gated_ffn_rules():
    x, wg, wu, wd = _ffn_args()
    with pytest.raises(ValueError, match="CUDA"):
        ops.gated_ffn(x, wg, wu, wd)
    with pytest.raises(ValueError, match="float16 and bfloat16"):
        ops.gated_ffn(*_ffn_args(dtype=torch.float32))
    with pytest.raises(ValueError, match="dtype"):
        ops.gated_ffn(*_ffn_args(dtype=torch.float64))
    with pytest.raises(ValueError, match="activation"):
        ops.gated_ffn(x, wg, wu, wd, "tanh")
    for bad, why in [((x, wg[:, :7].contiguous(), wu, wd), "w_gate"), ((x, wg[0], wu, wd), "w_gate"),
                     ((x, wg, wu[:8], wd), "w_up"), ((x, wg, wu, wd.t()), "w_down"),
                     ((x, wg, wu, wd.t().contiguous()), "w_down"), ((x, wg.float(), wu, wd), "w_gate"),
                     ((x, wg, wu.bfloat16(), wd), "w_up"), ((x, wg.t().contiguous().t(), wu, wd), "w_gate"),
                     ((x.t(), wg, wu, wd), "contiguous"), ((x, wg[:0], wu[:0], wd[:, :0].contiguous()), "w_gate")]:
        for call in (ops.gated_ffn, lambda *a: ops.gated_ffn_grad(a[0], *a)):
            with pytest.raises(ValueError, match=why):
                call(*bad)
    with pytest.raises(ValueError, match="out"):
        ops.gated_ffn(x, wg, wu, wd, out=torch.zeros(4, 9, dtype=torch.float16))
    with pytest.raises(ValueError, match="count_dev"):
        ops.gated_ffn_dyn(x, None, wg, wu, wd)
    with pytest.raises(ValueError, match="int32"):
        ops.gated_ffn_dyn(x, torch.zeros(1), wg, wu, wd)
    with pytest.raises(ValueError, match="grad"):
        ops.gated_ffn_grad(x[:3], x, wg, wu, wd)
    with pytest.raises(ValueError, match="CUDA"):
        ops.gated_ffn_grad(x, x, wg, wu, wd)
    kept = torch.zeros(2, 4, 16)
    for bad in (kept[:1], kept[:, :3].contiguous(), kept[..., :15], kept.half()):
        with pytest.raises(ValueError, match="kept"):
            ops.gated_ffn_grad(x, x, wg, wu, wd, kept=bad)


def test_gated_ffn_c_entries_refuse(handle):
    ffn, dyn, grad = handle.sbnet_gated_ffn, handle.sbnet_gated_ffn_dyn, handle.sbnet_gated_ffn_grad
    x, w, y, ws = 1 << 20, 1 << 24, 1 << 28, 1 << 30        # addresses that are never touched
    need = handle.sbnet_gated_ffn_workspace(4, 8, 16, 0, 1)
    assert need > 0 and handle.sbnet_gated_ffn_workspace(4, 7, 16, 0, 1) > need     # rows that have to be copied
    assert handle.sbnet_gated_ffn_workspace(4, 8, 16, 0, 0) > need
    assert handle.sbnet_gated_ffn_workspace(0, 8, 16, 0, 1) == 0

    def call(x=x, dtype=1, rows=4, c=8, f=16, wg=w, wu=w, wd=w, act=0, y=y, kept=None, ws=ws, n=need):
        return ffn(x, dtype, rows, c, f, wg, wu, wd, act, y, kept, ws, n, None)
    for bad in (dict(dtype=0), dict(dtype=7), dict(rows=-1), dict(c=0), dict(f=0), dict(act=3), dict(act=-1), dict(x=None),
                dict(y=None), dict(wd=None), dict(kept=(1 << 29) + 4), dict(x=x + 1), dict(y=y + 1), dict(y=x + 32), dict(y=w), dict(ws=None), dict(ws=ws + 16), dict(n=need - 1)):
        assert call(**bad) == BAD, bad
        assert handle.sbnet_last_error()
    assert call(rows=1 << 31) == -2 and call(c=1 << 25) == -2 and call(f=1 << 25) == -2
    assert call(rows=(1 << 30), f=1 << 20) == -2
    assert call(rows=0) == 0
    assert dyn(x, 1, 4, 2, None, 8, 16, w, w, w, 0, y, ws, 1 << 20, None) == BAD
    assert dyn(x, 1, 4, 0, ws, 8, 16, w, w, w, 0, y, ws, 1 << 20, None) == BAD
    assert dyn(x, 1, -1, 2, ws, 8, 16, w, w, w, 0, y, ws, 1 << 20, None) == BAD

    gneed = handle.sbnet_gated_ffn_workspace(4, 8, 16, 1, 1)

    def back(dy=x, x=x, kept=1 << 29, dtype=1, rows=4, wd=w, act=0, dx=y, dwg=None, dwu=None, dwd=None, ws=ws, n=gneed):
        return grad(dy, x, kept, dtype, rows, 8, 16, w, w, wd, act, dx, dwg, dwu, dwd, ws, n, None)
    for bad in (dict(dtype=0), dict(act=5), dict(dy=None), dict(dwg=y + 4096),
                dict(dwu=y + 4096), dict(dx=y + 1), dict(dx=x), dict(dx=1 << 29), dict(kept=(1 << 29) + 4), dict(dwd=w), dict(ws=None), dict(n=gneed - 1),
                dict(wd=None), dict(x=x + 1)):
        assert back(**bad) == BAD, bad
