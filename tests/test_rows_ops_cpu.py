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
        ops.layer_norm_grad(torch.zeros(4, 8), x, torch.zeros(4), torch.zeros(4))
    with pytest.raises(ValueError, match="mean"):
        ops.layer_norm_grad(x, x, torch.zeros(3), torch.zeros(4))
    with pytest.raises(ValueError, match="rstd"):
        ops.layer_norm_grad(x, x, torch.zeros(4), torch.zeros(4, dtype=torch.float16))


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
