"""What the 8-bit products refuse, before anything is launched (no GPU; the addresses here belong to nothing)."""

import pytest
import torch


def test_quantize_refusals(built_library):
    from sonicmoe._lib import lib

    at = 4096

    def call(x=at, ld=64, dtype=1, q=at, q_ld=64, scale=at, rows=4, cols=64):
        return lib.smoe_int8_quantize_rows(x, ld, dtype, q, q_ld, scale, rows, cols, None)

    assert call(dtype=2) == call(dtype=5) == -6
    assert call(rows=-1) == call(cols=0) == call(cols=131072, q_ld=131072) == call(q_ld=48) == call(ld=-1) == call(rows=2 ** 31) == -1
    assert call(x=None) == call(q=None) == call(scale=None) == -1
    assert call(x=at + 1) == call(dtype=0, x=at + 2) == call(q=at + 8) == call(q_ld=72) == call(scale=at + 2) == -2
    assert call(rows=0) == 0


def test_linear_refusals(built_library):
    from sonicmoe._lib import lib

    at = 4096

    def call(x=at, ld=64, x_type=1, xs=None, wq=at, w_ld=64, ws=at, bias=None, bias_type=0, out=at, out_type=1, off=at, freq=None,
             gather=None, T=16, rows=16, N=32, cols=64, E=4, act=-1, work=at, status=at):
        return lib.smoe_int8_linear(x, ld, x_type, xs, wq, w_ld, ws, bias, bias_type, out, out_type, off, freq, gather, T, rows, N, cols,
                                    E, act, work, status, None)

    given = dict(x_type=5, xs=at, work=None)  # 8-bit rows
    assert call(x_type=2) == call(out_type=2) == call(out_type=5) == call(bias=at, bias_type=3) == -6
    for bad in (dict(T=-1), dict(rows=-1), dict(T=2 ** 31 - 1, rows=2 ** 31 - 1), dict(E=1024, N=2 ** 21), dict(N=0), dict(cols=0), dict(cols=131072, ld=131072, w_ld=131072), dict(E=0), dict(E=1025),
                dict(w_ld=48), dict(ld=-1), dict(act=-2), dict(act=7), dict(act=0, N=33), dict(off=None), dict(off=None, E=1, freq=at),
                dict(rows=17), dict(rows=9), dict(gather=at, T=0), dict(given, ld=48), dict(x=None), dict(wq=None), dict(ws=None), dict(out=None), dict(xs=at), dict(x_type=5)):
        assert call(**bad) == -1, bad
    assert call(work=None) == -7
    for bad in (dict(x=at + 1), dict(given, x=at + 8), dict(given, ld=72), dict(wq=at + 8), dict(w_ld=72), dict(ws=at + 2),
                dict(given, xs=at + 2), dict(out=at + 1), dict(out_type=0, out=at + 2), dict(bias=at + 1, bias_type=1), dict(off=at + 2),
                dict(freq=at + 2), dict(gather=at + 1), dict(work=at + 16)):
        assert call(**bad) == -2, bad
    assert call(T=0, rows=0) == 0
    size = lib.smoe_int8_linear_workspace_bytes
    assert size(5, 100, 100, 64, 64, 4) == 0 and size(1, 0, 100, 64, 64, 4) == 0
    assert size(1, 100, 9, 64, 65, 4) == size(1, 100, 5, 64, 65, 1) == 100 * 80 + 192 + 512
    # few rows are quantised inside the kernel
    assert size(1, 100, 8, 64, 64, 4) == size(1, 4, 4, 64, 64, 1) == size(1, 1, 1, 14336, 4096, 1) == 0 and size(1, 5, 5, 14336, 4096, 1) > 0


def test_python_refusals(built_library):
    from sonicmoe import SonicMoEError
    from sonicmoe.functional import int8

    x, w = torch.zeros(4, 32), torch.zeros(8, 32, dtype=torch.int8)
    s = torch.ones(8)
    with pytest.raises(SonicMoEError, match="no CPU path"):
        int8.quantize_rows(x)
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        int8.quantize_rows(x.double())
    with pytest.raises(ValueError, match="1 to 131071"):
        int8.quantize_rows(torch.zeros(2, 0))
    with pytest.raises(SonicMoEError, match="no CPU path"):
        int8.int8_linear(x, w, s)
    with pytest.raises(NotImplementedError, match="no gradient"):
        int8.int8_linear(x.clone().requires_grad_(True), w, s)
    with pytest.raises(TypeError, match="has to be int8"):
        int8.int8_linear(x, w.float(), s)
    with pytest.raises(TypeError, match="has to be int8"):
        int8.int8_linear(x, w[None], s)
    with pytest.raises(ValueError, match="inconsistent shapes"):
        int8.int8_linear(x[:, :31], w, s)
    with pytest.raises(ValueError, match="int8_linear is the product"):
        int8.int8_grouped_linear(x, w[None], s[None], None)
    with pytest.raises(ValueError, match="is not a valid"):
        int8.int8_linear(x, w, s, activation_type="tanh")


def test_layer_refusals(built_library):
    from sonicmoe import SonicMoEError
    from sonicmoe.functional import int8

    w1, w2 = torch.zeros(8, 4, 16, dtype=torch.int8), torch.zeros(8, 16, 2, dtype=torch.int8)
    experts = int8.Int8Experts(w1, torch.ones(8, 4), None, w2, torch.ones(8, 16), None)
    x, router = torch.zeros(3, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16)
    with pytest.raises(SonicMoEError, match="no CPU path"):
        int8.moe_int8_softmax_topk_layer(x, router, experts, 2)
    with pytest.raises(NotImplementedError, match="no gradient"):
        int8.moe_int8_softmax_topk_layer(x.requires_grad_(True), router, experts, 2)
    with pytest.raises(AssertionError):
        int8.quantize_experts(torch.zeros(4, 16, 8), None, torch.zeros(16, 2, 8), torch.zeros(8, 16))
    with pytest.raises(ValueError, match="inconsistent shapes"):
        int8.quantize_experts(torch.zeros(4, 16, 8), None, torch.zeros(12, 2, 8), None)


def test_forward_mode_derivatives_are_refused(built_library):
    """A dual tensor does not require a gradient, and torch.no_grad() leaves its tangent alone."""
    from torch.autograd import forward_ad

    from sonicmoe.functional import int8

    x, w = torch.zeros(4, 32), torch.zeros(8, 32, dtype=torch.int8)
    s, xs, bias = torch.ones(8), torch.ones(4), torch.zeros(8)
    experts = int8.Int8Experts(torch.zeros(8, 4, 16, dtype=torch.int8), torch.ones(8, 4), None,
                               torch.zeros(8, 16, 2, dtype=torch.int8), torch.ones(8, 16), None)
    t, router = torch.zeros(3, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16)
    with forward_ad.dual_level(), torch.no_grad():
        dual = lambda v: forward_ad.make_dual(v, torch.ones_like(v))
        off = torch.zeros(2, dtype=torch.int32)
        for call in (lambda: int8.int8_linear(dual(x), w, s), lambda: int8.int8_linear(x, w, dual(s)),
                     lambda: int8.int8_linear(x.to(torch.int8), w, s, x_scale=dual(xs)),
                     lambda: int8.int8_linear(x, w, s, bias=dual(bias)),
                     lambda: int8.int8_grouped_linear(dual(x), w[None], s[None], off),
                     lambda: int8.moe_int8_softmax_topk_layer(dual(t), router, experts, 2),
                     lambda: int8.moe_int8_softmax_topk_layer(t, dual(router), experts, 2)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
