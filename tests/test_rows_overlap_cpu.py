"""Row operators at the C ABI: memory that one kernel would write while another thread reads or writes it is refused
before anything is launched.  Addresses are made up and never touched."""
import pytest

BAD = -1
ROWS, C, F = 64, 32, 48
X, DY, Y, W, B, MEAN, RSTD, DW, DB, WS, K = (1 << 20 | n << 24 for n in range(1, 12))
XB, WB, SB, KB = ROWS * C * 2, C * 2, ROWS * 4, 2 * ROWS * F * 4       # bytes of x, weight, mean; G and U in fp32
FB = F * C * 2


@pytest.fixture(scope="module")
def handle():
    from sbnet_b200 import build, lib
    build.build_library()
    return lib.load()


def _refused(handle, rc):
    return rc == BAD and b"overlap" in handle.sbnet_last_error()


@pytest.mark.parametrize("bad", [dict(y=X), dict(y=X + XB - 2), dict(y=W - XB + 2), dict(y=W + WB - 2), dict(y=B), dict(y=MEAN),
                                 dict(y=RSTD + SB - 4), dict(rstd=MEAN), dict(rstd=MEAN + SB - 4), dict(mean=X), dict(mean=X + XB - 4),
                                 dict(rstd=W), dict(mean=B)], ids=str)
def test_layer_norm(handle, bad):
    def call(y=Y, mean=MEAN, rstd=RSTD):
        return handle.sbnet_layer_norm(X, 1, ROWS, C, W, B, 1, 1e-5, y, mean, rstd, None)
    assert _refused(handle, call(**bad))


@pytest.mark.parametrize("bad", [dict(dx=X), dict(dx=DY + XB - 2), dict(dx=W), dict(dx=MEAN + SB - 4), dict(dx=RSTD), dict(dx=DW),
                                 dict(dx=DB - XB + 2), dict(db=DW), dict(db=DW + WB - 2), dict(dw=DB + WB - 2)], ids=str)
def test_layer_norm_grad(handle, bad):
    need = handle.sbnet_layer_norm_grad_workspace(ROWS, C)

    def call(dx=Y, dw=DW, db=DB):
        return handle.sbnet_layer_norm_grad(DY, X, 1, ROWS, C, W, 1, MEAN, RSTD, dx, dw, db, WS, need, None)
    assert _refused(handle, call(**bad))


@pytest.mark.parametrize("bad", [dict(y=X), dict(y=W + FB - 2), dict(kept=Y), dict(kept=Y - KB + 16), dict(kept=X), dict(kept=X - KB + 16),
                                 dict(kept=W), dict(kept=B), dict(kept=DW + FB - 16)], ids=str)
def test_gated_ffn(handle, bad):
    need = handle.sbnet_gated_ffn_workspace(ROWS, C, F, 2, 1)

    def call(y=Y, kept=K):
        return handle.sbnet_gated_ffn(X, 1, ROWS, C, F, W, B, DW, 0, y, kept, WS, need, None)
    assert _refused(handle, call(**bad))


@pytest.mark.parametrize("bad", [dict(dx=X), dict(dx=K), dict(dwd=W), dict(dwg=RSTD), dict(dwu=MEAN + FB - 2), dict(dwd=MEAN),
                                 dict(dx=MEAN), dict(dx=RSTD - XB + 2), dict(dwd=RSTD + FB - 2)], ids=str)
def test_gated_ffn_grad(handle, bad):
    need = handle.sbnet_gated_ffn_workspace(ROWS, C, F, 1, 1)

    def call(dx=Y, dwg=MEAN, dwu=RSTD, dwd=1 << 29):
        return handle.sbnet_gated_ffn_grad(DY, X, K, 1, ROWS, C, F, W, B, DW, 0, dx, dwg, dwu, dwd, WS, need, None)
    assert _refused(handle, call(**bad))
