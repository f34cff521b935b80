"""The norm and its gradients against plain implementations in 64 bits, at the widths, layouts and values where it can go wrong.

Tolerances, in units u = 2^-24 of fp32's half step.  The sum of H squares, each thread's by one fused step per value and then over at most
ten levels and sixteen warps: within (EP + 26) u of its value with EP <= 16 values per thread and round; rows above 8192 values
add H / 8192 rounds of 16.  The mean and eps: 2 u more; the root halves all that and adds 1 u; (h w) r adds 2 u.  `chain(H)` is half of the first
plus 5.  An output adds half a step of its own type, at its smallest where the value is subnormal."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -24
EPS = 1e-6


def half_step(dtype, value):
    f = torch.finfo(dtype)
    return f.eps / 2 * value.abs() + f.smallest_normal * f.eps / 2


def chain(H):
    return ((16 * -(-H // 8192) + 28) / 2 + 5) * U


def source(rows, H, dtype, seed, pitch=0, offset=0):
    """(rows, H) on the device, `pitch` values longer per row in memory and `offset` values into its buffer."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.empty(offset + rows * (H + pitch), dtype=dtype, device="cuda")
    view = flat[offset:].view(rows, H + pitch)[:, :H]
    view.copy_(torch.randn(rows, H, generator=g) * (1 + 9 * (torch.rand(H, generator=g) < 0.02)))
    return view


def weights(H, dtype, seed, offset=0):
    g = torch.Generator().manual_seed(seed)
    flat = torch.empty(H + offset, dtype=dtype, device="cuda")
    flat[offset:].copy_(1 + 0.1 * torch.randn(H, generator=g))
    return flat[offset:]


def plain(x, w, eps=EPS, residual=None):
    h = x if residual is None else (x.double() + residual.double()).float().to(x.dtype)
    d = h.double()
    r = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    return d * r * w.double(), h, r


def check_y(y, want, H):
    bound = chain(H) * want.abs()
    bound = bound + half_step(y.dtype, want.abs() + bound)
    assert ((y.double() - want).abs() <= bound).all()


#: (width, values between rows, values before the first)
LAYOUTS = [(64, 0, 0), (128, 0, 0), (512, 8, 0), (24, 0, 8), (1005, 0, 0), (1030, 0, 0), (17, 3, 1), (1, 0, 0), (2, 1, 1), (4096, 0, 0),
           (4104, 0, 4), (8192, 0, 0), (8193, 0, 0), (8200, 0, 0), (16384, 0, 0), (20001, 2, 3)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,pitch,offset", LAYOUTS)
def test_forward(built_library, dtype, H, pitch, offset):
    import sonicmoe

    for T in (1, 37):
        for wt in {dtype, torch.float32}:
            x, res = source(T, H, dtype, 1, pitch, offset), source(T, H, dtype, 2, 0, offset)
            w = weights(H, wt, 3, offset % 2)
            y = sonicmoe.rms_norm(x, w)
            check_y(y, plain(x, w)[0], H)
            y, h = sonicmoe.rms_norm(x, w, EPS, residual=res)
            want, wh, _ = plain(x, w, EPS, res)
            assert torch.equal(h, wh) and y.is_contiguous() and h.is_contiguous()
            check_y(y, want, H)


def test_rows_of_many_dimensions_and_views(built_library):
    import sonicmoe

    w = weights(64, torch.bfloat16, 0)
    qkv = source(33, 6 * 64, torch.bfloat16, 1).view(33, 6, 64)
    for x in (qkv, qkv[:, 1:3], qkv[:, 2], qkv.transpose(0, 1), qkv[0, 0], qkv[5], qkv[:1, 1:2], qkv[:, 0, None, :].expand(33, 5, 64),
              qkv[:, 0].repeat_interleave(2, 1)[:, ::2], qkv[:0], qkv[:, :0]):
        y = sonicmoe.rms_norm(x, w)
        assert y.shape == x.shape
        check_y(y, plain(x, w)[0], 64)
        y, h = sonicmoe.rms_norm(x, w, EPS, residual=x)
        assert torch.equal(h, x + x)
        r = sonicmoe.rms_norm_quantize(x, w, EPS, residual=x, keep_y=True)
        assert torch.equal(r.y, y) and torch.equal(r.h, h) and r.q.shape == x.shape and r.scale.shape == x.shape[:-1]


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_zeros_infinities_and_nans(built_library, dtype):
    import sonicmoe

    x = source(8, 136, dtype, 5).clone()
    x[0] = 0
    x[1, 7] = float("inf")
    x[2, 135] = float("nan")
    x[3, 0] = -float("inf")
    x[4] = torch.finfo(dtype).smallest_normal
    w = weights(136, dtype, 6)
    y = sonicmoe.rms_norm(x, w)
    assert (y[0] == 0).all()
    # an infinity's root is infinite: its own column is NaN, the others are zeros
    assert y[1, 7].isnan() and y[3, 0].isnan() and (y[1, :7] == 0).all() and (y[3, 1:] == 0).all()
    assert y[2].isnan().all()
    check_y(y[4:], plain(x[4:], w)[0], 136)
    r = sonicmoe.rms_norm_quantize(x, w)
    assert (r.q[0] == 0).all() and r.scale[0] == 1
    assert (r.q[1:4] == 0).all() and r.scale[1:4].isnan().all()  # as quantize_rows gives rows that hold a NaN
    assert r.scale[4:].isfinite().all() and (r.q[4:].abs().amax(1) == 127).all()
    assert sonicmoe.rms_norm(x[:1], w, 0.0).isnan().all()  # 0 / 0


def check_quantised(q, scale, want, H):
    """q within half a step of 127 y / amax, and an error of y and of amax, relative to theirs."""
    amax = want.abs().amax(-1)
    live = amax > 0
    assert (scale[~live] == 1).all() and (q[~live] == 0).all()
    assert ((scale.double() - amax / 127).abs() <= (chain(H) + 2 * U) * amax / 127)[live].all()
    exact = 127 * want[live] / amax[live].unsqueeze(1)
    # errors of both, and the quantiser's own of up to 2^-14
    assert ((q[live].double() - exact).abs() <= 0.5 + 127 * 2 * (chain(H) + 2 * U) + 2.0 ** -14).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,pitch,offset", LAYOUTS)
def test_quantised(built_library, dtype, H, pitch, offset):
    import sonicmoe

    T = 37
    x, res = source(T, H, dtype, 1, pitch, offset), source(T, H, dtype, 2, 0, offset)
    for wt in {dtype, torch.float32}:
        w = weights(H, wt, 3, offset % 2)
        for residual in (None, res):
            r = sonicmoe.rms_norm_quantize(x, w, EPS, residual=residual, keep_y=True)
            want, h, _ = plain(x, w, EPS, residual)
            check_quantised(r.q, r.scale, want, H)
            alone = sonicmoe.rms_norm_quantize(x, w, EPS, residual=residual)
            assert torch.equal(alone.q, r.q) and torch.equal(alone.scale, r.scale) and alone.y is None
            y = sonicmoe.rms_norm(x, w, EPS, residual=residual)
            if residual is None:
                assert r.h is None and torch.equal(r.y, y)
            else:
                assert torch.equal(r.h, h) and torch.equal(r.y, y[0]) and torch.equal(r.h, y[1])
            whole = r.q.as_strided((T, -(-H // 16) * 16), (r.q.stride(0), 1))
            assert (whole[:, H:] == 0).all() and r.q.stride(0) % 16 == 0


def test_fp32_rows_are_quantised_as_quantize_rows_does(built_library):
    import sonicmoe
    from sonicmoe.functional import int8

    for H in (64, 1005, 4096, 9000):
        x, w = source(50, H, torch.float32, 7), weights(H, torch.float32, 8)
        r = sonicmoe.rms_norm_quantize(x, w, keep_y=True)
        q, scale = int8.quantize_rows(r.y)
        assert torch.equal(r.q, q) and torch.equal(r.scale, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H", [17, 1005, 16376, 16378, 16381, 16383, 16387, 24570, 24573, 24575, 32761, 131071])
def test_columns_behind_8_bit_rows(built_library, dtype, H):
    """Zeros up to the next multiple of 16, whatever was there, for rows of every shift; nothing behind that is written."""
    import sonicmoe
    from sonicmoe import _lib

    T, width = 17, -(-H // 16) * 16
    x, w = source(T, H, dtype, 1), weights(H, dtype, 2)
    want = sonicmoe.rms_norm_quantize(x, w, EPS)
    q = torch.full((T, width + 16), 85, dtype=torch.int8, device="cuda")
    scale = torch.empty(T, dtype=torch.float32, device="cuda")
    code = {torch.float32: _lib.SMOE_F32, torch.bfloat16: _lib.SMOE_BF16, torch.float16: _lib.SMOE_F16}[dtype]
    _lib.check(_lib.lib.smoe_rms_norm(x.data_ptr(), H, None, 0, w.data_ptr(), code, None, None, None, q.data_ptr(), width + 16, scale.data_ptr(),
                                      code, T, H, EPS, _lib.stream_ptr(x.device)), "rms_norm")
    assert torch.equal(q[:, :H], want.q) and torch.equal(scale, want.scale)
    assert (q[:, H:width] == 0).all() and (q[:, width:] == 85).all()


def plain_gradients(x, w, eps, residual, dy, dh):
    _, h, r = plain(x, w, eps, residual)
    u = h.double() * r
    g = dy.double() * w.double()
    along = (g * u).mean(-1, keepdim=True)
    dx = r * (g - u * along)
    size = r * (g.abs() + u.abs() * (g * u).abs().mean(-1, keepdim=True))  # magnitudes of the terms
    if dh is not None:
        dx, size = dx + dh.double(), size + dh.double().abs()
    return dx, size, (dy.double() * u).sum(0), (dy.double() * u).abs().sum(0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,pitch,offset", LAYOUTS)
def test_gradients(built_library, dtype, H, pitch, offset):
    import sonicmoe

    for T in (1, 50):
        for wt in {dtype, torch.float32}:
            x, res = source(T, H, dtype, 1, pitch, offset).requires_grad_(), source(T, H, dtype, 2, 0, offset).requires_grad_()
            w = weights(H, wt, 3, offset % 2).requires_grad_()
            dy, dh = source(T, H, dtype, 4, pitch), source(T, H, dtype, 5, 0, offset)
            for residual in (None, res):
                if residual is None:
                    y = sonicmoe.rms_norm(x, w)
                    dx, dw = torch.autograd.grad(y, (x, w), dy)
                else:
                    y, h = sonicmoe.rms_norm(x, w, EPS, residual=res)
                    dx, dres, dw = torch.autograd.grad((y, h), (x, res, w), (dy, dh))
                    assert torch.equal(dx, dres)
                want, size, want_dw, size_dw = plain_gradients(x.detach(), w.detach(), EPS, None if residual is None else res.detach(),
                                                               dy, None if residual is None else dh)
                # two sums over a row, the root's errors and some ten steps more
                bound = (3 * chain(H) + 10 * U) * size
                assert ((dx.double() - want).abs() <= bound + half_step(dtype, want.abs() + bound)).all()
                # the sum over the rows: one addition for each, and the terms' own errors
                bound = ((T + 34) * U + chain(H) + 3 * U) * size_dw
                assert ((dw.double() - want_dw).abs() <= bound + half_step(wt, want_dw.abs() + bound)).all()
                assert dw.dtype == wt and dx.dtype == dtype


def test_gradients_over_many_rows(built_library):
    """More rows than blocks take at once: many rows to a block, several rows at a time, one row at a time, rows read twice."""
    import sonicmoe

    for T, H in ((40000, 64), (70001, 10), (3000, 2056), (1300, 4100), (700, 8200)):
        x = source(T, H, torch.float32, 1).requires_grad_()
        w = weights(H, torch.float32, 2).requires_grad_()
        dy = source(T, H, torch.float32, 3)
        dx, dw = torch.autograd.grad(sonicmoe.rms_norm(x, w), (x, w), dy)
        want, size, want_dw, size_dw = plain_gradients(x.detach(), w.detach(), EPS, None, dy, None)
        bound = (3 * chain(H) + 10 * U) * size
        assert ((dx.double() - want).abs() <= bound + U * want.abs()).all()
        # a thread's rows one by one, then the threads of a block, then the blocks
        bound = ((min(T, T / 148 + 400) + 34) * U + chain(H) + 3 * U) * size_dw
        assert ((dw.double() - want_dw).abs() <= bound + U * want_dw.abs()).all()
        again = torch.autograd.grad(sonicmoe.rms_norm(x, w), (x, w), dy)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H", [(3000, 2049), (3000, 1005), (200000, 10), (1500, 7169), (1300, 8197), (1300, 16389), (3000, 2056), (150000, 24), (1300, 16400)])
def test_gradients_of_many_rows_of_every_type(built_library, dtype, T, H):
    """Several rows of a thread, which start anywhere or on 16-byte boundaries, with a residual and an upstream gradient of h."""
    import sonicmoe

    x, res, w = source(T, H, dtype, 1).requires_grad_(), source(T, H, dtype, 2).requires_grad_(), weights(H, dtype, 3).requires_grad_()
    dy, dh = source(T, H, dtype, 4), source(T, H, dtype, 5)
    dx, dres, dw = torch.autograd.grad(sonicmoe.rms_norm(x, w, EPS, residual=res), (x, res, w), (dy, dh))
    want, size, want_dw, size_dw = plain_gradients(x.detach(), w.detach(), EPS, res.detach(), dy, dh)
    bound = (3 * chain(H) + 10 * U) * size
    assert ((dx.double() - want).abs() <= bound + half_step(dtype, want.abs() + bound)).all() and torch.equal(dx, dres)
    # as in test_gradients_over_many_rows, and the weight's own type
    bound = ((min(T, T / 148 + 400) + 34) * U + chain(H) + 3 * U) * size_dw
    assert ((dw.double() - want_dw).abs() <= bound + half_step(dtype, want_dw.abs() + bound)).all()
    again = torch.autograd.grad(sonicmoe.rms_norm(x, w, EPS, residual=res), (x, res, w), (dy, dh))
    assert torch.equal(again[0], dx) and torch.equal(again[2], dw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,pitch,offset", [(64, 0, 0), (64, 3, 1), (4096, 0, 0), (32768, 0, 0), (32768, 3, 1)])
def test_gradients_of_rows_whose_root_squared_leaves_the_range(built_library, dtype, H, pitch, offset):
    """eps 0 and rows of 1 to 3 times 2^-66: r is some 2^65 and r^2 past fp32's range, dx some 2^65.  The squares are whole multiples of 2^-132, their
    mean one of 2^-147, at most 9 H of them, which fp32 holds: sums and mean are exact, and the bounds of other rows hold."""
    import sonicmoe

    T = 5
    g = torch.Generator().manual_seed(1)
    x = source(T, H, dtype, 1, pitch, offset)
    x.copy_(torch.randint(1, 4, (T, H), generator=g) * (2 * torch.randint(0, 2, (T, H), generator=g) - 1) * 2.0 ** -66)
    x.requires_grad_()
    w, dy = weights(H, dtype, 2).requires_grad_(), source(T, H, dtype, 3)
    y = sonicmoe.rms_norm(x, w, 0.0)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    check_y(y.detach(), plain(x.detach(), w.detach(), 0.0)[0], H)
    want, size, want_dw, size_dw = plain_gradients(x.detach(), w.detach(), 0.0, None, dy, None)
    bound = (3 * chain(H) + 10 * U) * size
    assert ((dx.double() - want).abs() <= bound + half_step(dtype, want.abs() + bound)).all()
    bound = ((T + 34) * U + chain(H) + 3 * U) * size_dw
    assert ((dw.double() - want_dw).abs() <= bound + half_step(dtype, want_dw.abs() + bound)).all()


def test_gradients_against_differences(built_library):
    """fp32 differences of the loss <y, a> + <h, b> along random directions, by 64-bit evaluations of the formula."""
    import sonicmoe

    T, H = 9, 40
    x, res, w = (source(T, H, torch.float32, i).requires_grad_() for i in (1, 2)), None, None
    x, res = x
    w = weights(H, torch.float32, 3).requires_grad_()
    a, b = source(T, H, torch.float32, 4), source(T, H, torch.float32, 5)
    y, h = sonicmoe.rms_norm(x, w, 1e-3, residual=res)
    grads = torch.autograd.grad((y, h), (x, res, w), (a, b))

    def loss(xx, rr, ww):
        hh = xx + rr
        yy = hh / torch.sqrt((hh * hh).mean(-1, keepdim=True) + 1e-3) * ww
        return ((yy * a.double()).sum() + (hh * b.double()).sum()).item()

    at = [t.detach().double() for t in (x, res, w)]
    for i in range(3):
        g = torch.Generator().manual_seed(i)
        d = torch.randn(at[i].shape, generator=g).cuda().double()
        step = 1e-5
        up, down = [t + step * d if j == i else t for j, t in enumerate(at)], [t - step * d if j == i else t for j, t in enumerate(at)]
        slope = (loss(*up) - loss(*down)) / (2 * step)
        # third derivatives are of the order of the loss's terms: step^2 of their sum; h's rounding 2^-24 of its terms
        size = (grads[i].double().abs() * d.abs()).sum().item()
        assert abs((grads[i].double() * d).sum().item() - slope) <= 1e-5 * size


def test_gradients_where_only_some_are_asked_for(built_library):
    import sonicmoe

    T, H = 20, 72
    full = [source(T, H, torch.bfloat16, 1), weights(H, torch.bfloat16, 2), source(T, H, torch.bfloat16, 3)]
    dy, dh = source(T, H, torch.bfloat16, 4), source(T, H, torch.bfloat16, 5)

    def grads(needs, gy=True, gh=True):
        x, w, r = (t.detach().clone().requires_grad_(n) for t, n in zip(full, needs))
        y, h = sonicmoe.rms_norm(x, w, EPS, residual=r)
        outs = [(t, g) for t, g, use in ((y, dy, gy), (h, dh, gh)) if use]
        torch.autograd.backward([o for o, _ in outs], [g for _, g in outs])
        return x.grad, w.grad, r.grad

    every = grads((True, True, True))
    for needs in ((True, False, False), (False, True, False), (False, False, True), (True, True, False), (False, True, True)):
        for got, want, need in zip(grads(needs), every, needs):
            assert torch.equal(got, want) if need else got is None
    # h alone: its gradient passes; y alone: no gradient of h
    x, w, r = grads((True, True, True), gy=False)
    assert torch.equal(x, dh) and torch.equal(r, dh) and (w is None or (w == 0).all())
    x, w, r = grads((True, True, True), gh=False)
    want, size, _, _ = plain_gradients(full[0], full[1], EPS, full[2], dy, None)
    bound = (3 * chain(H) + 10 * U) * size
    assert ((x.double() - want).abs() <= bound + half_step(torch.bfloat16, want.abs() + bound)).all() and torch.equal(w, every[1])


def test_broadcast_inputs_and_gradients(built_library):
    import sonicmoe

    one = source(1, 48, torch.float32, 1).requires_grad_()
    w = weights(48, torch.float32, 2).requires_grad_()
    y = sonicmoe.rms_norm(one.expand(30, 48), w)
    y.sum().backward()  # a gradient of one value, broadcast
    ref = one.detach().double().requires_grad_()
    wref = w.detach().double().requires_grad_()
    (30 * ref / torch.sqrt((ref * ref).mean() + EPS) * wref).sum().backward()
    assert torch.allclose(one.grad.double(), ref.grad, rtol=1e-4, atol=1e-4) and torch.allclose(w.grad.double(), wref.grad, rtol=1e-5)


def test_derivatives_that_are_refused(built_library):
    import sonicmoe
    from torch.autograd import forward_ad

    x, w = source(4, 16, torch.float32, 1).requires_grad_(), weights(16, torch.float32, 2).requires_grad_()
    dx, = torch.autograd.grad(sonicmoe.rms_norm(x, w).sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError, match="first derivatives"):
        torch.autograd.grad(dx.sum(), x)
    with forward_ad.dual_level():
        with pytest.raises((NotImplementedError, RuntimeError)):
            sonicmoe.rms_norm(forward_ad.make_dual(x.detach(), torch.ones_like(x)), w.detach())
        with pytest.raises(NotImplementedError, match="forward-mode"):
            sonicmoe.rms_norm_quantize(forward_ad.make_dual(x.detach(), torch.ones_like(x)), w.detach())
    for bad in ((x, w.detach()), (x.detach(), w)):
        with pytest.raises(NotImplementedError, match="no gradient"):
            sonicmoe.rms_norm_quantize(*bad)
    with torch.no_grad():
        sonicmoe.rms_norm_quantize(x, w)


def test_refusals_on_the_device(built_library):
    import sonicmoe

    x, w = source(4, 16, torch.bfloat16, 1), weights(16, torch.bfloat16, 2)
    for call in (sonicmoe.rms_norm, sonicmoe.rms_norm_quantize):
        for bad in (w[:8], w.cpu(), weights(32, torch.bfloat16, 2)[::2], w.view(1, 16)):
            with pytest.raises(ValueError, match="weight has to be"):
                call(x, bad)
        with pytest.raises(TypeError, match="or fp32"):
            call(x, w.half())
        for bad in (x[:2], x.float(), x.cpu()):
            with pytest.raises(ValueError, match="residual has to be"):
                call(x, w, EPS, residual=bad)
    with pytest.raises(ValueError, match="at most"):
        sonicmoe.rms_norm_quantize(source(1, 131072, torch.bfloat16, 1), weights(131072, torch.bfloat16, 1))


def test_on_another_stream_and_in_a_graph(built_library):
    import sonicmoe

    x, res = source(40, 512, torch.bfloat16, 1), source(40, 512, torch.bfloat16, 2)
    w = weights(512, torch.bfloat16, 3)
    want = sonicmoe.rms_norm_quantize(x, w, EPS, residual=res, keep_y=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sonicmoe.rms_norm_quantize(x, w, EPS, residual=res, keep_y=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    xs, ws, rs = (t.detach().clone().requires_grad_() for t in (x, w, res))
    dy, dh = source(40, 512, torch.bfloat16, 4), source(40, 512, torch.bfloat16, 5)
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y, h = sonicmoe.rms_norm(xs, ws, EPS, residual=rs)
        grads = torch.autograd.grad((y, h), (xs, rs, ws), (dy, dh))
    for seed in (7, 8):
        with torch.no_grad():
            xs.copy_(source(40, 512, torch.bfloat16, seed))
        graph.replay()
        xe = xs.detach().clone().requires_grad_()
        ye, he = sonicmoe.rms_norm(xe, ws.detach(), EPS, residual=rs.detach())
        assert torch.equal(y, ye) and torch.equal(h, he)
        assert torch.equal(grads[0], torch.autograd.grad((ye, he), xe, (dy, dh))[0])


@pytest.mark.parametrize("T", [1, 40, 3000])
@pytest.mark.parametrize("residual", [False, True])
def test_the_8_bit_layer_takes_the_rows(built_library, T, residual):
    """The layer on a norm's 8-bit rows against the layer on those of quantize_rows, which differ where a value is next to a border, and the layer's
    own quantising against rows that are given: the same bits."""
    import sonicmoe
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(12)
    H, I, E, K = 256, 64, 8, 2
    x = torch.randn(T, H, generator=g).bfloat16().cuda()
    h0 = torch.randn(T, H, generator=g).bfloat16().cuda() if residual else None
    weight = (1 + 0.1 * torch.randn(H, generator=g)).bfloat16().cuda()
    router = (torch.randn(E, H, generator=g) * 0.1).bfloat16().cuda()
    w1 = (torch.randn(E, 2 * I, H, generator=g) * 2 / H ** 0.5).bfloat16().cuda()
    w2 = (torch.randn(E, H, I, generator=g) / I ** 0.5).bfloat16().cuda()
    experts = int8.quantize_experts(w1.permute(1, 2, 0), None, w2.permute(1, 2, 0), None)
    r = sonicmoe.rms_norm_quantize(x, weight, residual=h0, keep_y=True)
    o, logits, frequency = int8.moe_int8_softmax_topk_layer(r.y, router, experts, K, x_q=r.q, x_scale=r.scale)
    h = (x if h0 is None else r.h).double()
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6) * weight.double()
    q, scale = int8.quantize_rows(y.float())
    # fp32 sums of 256 squares, a root and three products: under 2^-19 of y and of the scale, so that a value within 127 2^-19 of a step of a border may
    # go to the other side: 127 2^-18 of all values, evenly spread, and 8 for the spread of a small number
    assert (r.q != q).sum() <= 8 + T * H * 127 * 2.0 ** -18 and (r.q.int() - q.int()).abs().max() <= 1
    assert ((r.scale - scale).abs() <= 2.0 ** -19 * scale).all()
    same = int8.moe_int8_softmax_topk_layer(r.y, router, experts, K, x_q=q, x_scale=scale)
    assert torch.equal(same[1], logits) and torch.equal(same[2], frequency)
    # a value by a step changes its row by under 1 / 127 (its largest value, 1/16 of the row's norm at least, over 127), and what follows is rounded twice
    # to bf16 (2^-8) and once to 8 bits (1 / 127) where it changes
    assert ((o.double() - same[0].double()).norm() / o.double().norm()).item() < 4 / 127
    own = int8.moe_int8_softmax_topk_layer(r.y, router, experts, K)
    q, scale = int8.quantize_rows(r.y)
    given = int8.moe_int8_softmax_topk_layer(r.y, router, experts, K, x_q=q, x_scale=scale)
    assert all(torch.equal(a, b) for a, b in zip(own, given))


def test_rows_that_the_8_bit_layer_refuses(built_library):
    from sonicmoe.functional import int8

    x = torch.randn(4, 256, device="cuda").bfloat16()
    router = torch.randn(8, 256, device="cuda").bfloat16()
    experts = int8.quantize_experts(torch.randn(128, 256, 8, device="cuda").bfloat16(), None, torch.randn(256, 64, 8, device="cuda").bfloat16(), None)
    q, scale = int8.quantize_rows(x)
    for bad in ({"x_q": q}, {"x_scale": scale}):
        with pytest.raises(ValueError, match="belong together"):
            int8.moe_int8_softmax_topk_layer(x, router, experts, 2, **bad)
    for bad in (q[:3], q[:, :128], q.short(), q.cpu()):
        with pytest.raises(ValueError, match="x_q has to be"):
            int8.moe_int8_softmax_topk_layer(x, router, experts, 2, x_q=bad, x_scale=scale)
    for bad in (scale[:3], scale.double(), scale.cpu()):
        with pytest.raises(ValueError, match="x_scale has to be"):
            int8.moe_int8_softmax_topk_layer(x, router, experts, 2, x_q=q, x_scale=bad)
