"""The norm's argument checks, which come before anything is launched (no GPU; the addresses here belong to nothing)."""

import pytest
import torch


def test_forward_refusals(built_library):
    from sonicmoe._lib import lib

    at = 4096

    def call(x=at, ld=64, res=None, res_ld=0, w=at, wt=1, y=at, h=None, rstd=None, q=None, q_ld=0, scale=None, dtype=1, rows=4, H=64, eps=1e-6):
        return lib.smoe_rms_norm(x, ld, res, res_ld, w, wt, y, h, rstd, q, q_ld, scale, dtype, rows, H, eps, None)

    assert call(dtype=2) == call(wt=3) == call(wt=4) == call(dtype=0, wt=1) == -6  # weights of another 16-bit type, or narrower ones
    assert call(rows=-1) == call(rows=2 ** 31) == call(H=0) == call(H=2 ** 30 + 1) == call(ld=-1) == call(eps=-1.0) == call(eps=float("nan")) == -1
    assert call(x=None) == call(w=None) == call(y=None) == call(h=at) == call(q=at, q_ld=64) == call(scale=at) == -1
    assert call(res=at, res_ld=-64) == call(q=at, scale=at, q_ld=48) == call(q=at, scale=at, q_ld=2 ** 17, H=131072) == -1
    assert call(x=at + 1) == call(y=at + 1) == call(w=at + 2, wt=0) == call(rstd=at + 2) == call(res=at + 1, h=at) == -2
    assert call(q=at + 8, scale=at, q_ld=64) == call(q=at, scale=at, q_ld=72) == call(q=at, scale=at + 2, q_ld=64) == -2
    assert call(rows=0) == 0


def test_backward_refusals(built_library):
    from sonicmoe._lib import lib

    at = 4096

    def call(dy=at, ld=64, dh=None, h=at, w=at, wt=1, rstd=at, dx=at, dw=at, dtype=1, rows=4, H=64, ws=at):
        return lib.smoe_rms_norm_backward(dy, ld, dh, ld, h, ld, w, wt, rstd, dx, dw, dtype, rows, H, ws, None)

    assert call(dtype=3) == call(wt=4) == call(dtype=0) == -6
    assert call(rows=-1) == call(rows=2 ** 31) == call(H=0) == call(ld=-1) == call(dx=None, dw=None) == -1
    assert call(dy=None) == call(h=None) == call(w=None) == call(rstd=None) == -1
    assert call(dy=at + 1) == call(dh=at + 1) == call(dx=at + 1) == call(dw=at + 1) == call(rstd=at + 2) == call(ws=at + 8) == -2
    assert call(ws=None) == -7
    assert call(rows=0, dw=None, dy=None, h=None, rstd=None) == 0
    size = lib.smoe_rms_norm_backward_workspace_bytes
    assert size(0, 64) == 0 and size(-1, 64) == 0 and size(3, 64) >= 3 * 256 and size(10 ** 6, 64) == size(2 * 10 ** 6, 64)


def test_python_refusals(built_library):
    import sonicmoe
    from sonicmoe import SonicMoEError

    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    for call in (sonicmoe.rms_norm, sonicmoe.rms_norm_quantize):
        with pytest.raises(SonicMoEError, match="no CPU path"):
            call(x, w)
        with pytest.raises(TypeError, match="rows"):
            call(x.int(), w)
        with pytest.raises(TypeError, match="rows"):
            call(x[0, 0], w)
        with pytest.raises(ValueError, match="rows of 1"):
            call(x[:, :0], w)
        for eps in (-1e-6, float("nan"), float("inf")):
            with pytest.raises(ValueError, match="eps"):
                call(x, w, eps)
