"""Low-rank adapters against a plain implementation in 64 bits, at the sizes, ranks, layouts and loads where they can go wrong.

Tolerances.  A step of the tensor core adds 16 products to an fp32 sum; the sum is taken to be off by at most 2^-22 of the magnitudes in it
after each step, and additions of parts (64 at most, in three levels) by 2^-24 each.  So s = a x is within (H / 16 + 20) 2^-22 of
sum |a| |x|.  Its two 16-bit parts leave out 2^-16 of it (bf16: eight bits cut, eight more rounded) or 2^-22 and 2^-38 of the row's largest
(fp16).  The second product has 2 r / 16 steps over |b| |s|; the result is within half a step of its type of all that."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def half_step(dtype, value):
    f = torch.finfo(dtype)
    return f.eps / 2 * value.abs() + f.smallest_normal * f.eps / 2


def rows_of(T, width, dtype, gen, pitch=0, offset=0):
    flat = torch.empty(offset + T * (width + pitch), dtype=dtype, device="cuda")
    view = flat[offset:].view(T, width + pitch)[:, :width]
    view.copy_(torch.randn(T, width, generator=gen))
    return view


def make(T, H, N, n, r, dtype, seed=0, dropped=0.2, runs=3, pitch=0, offset=0):
    g = torch.Generator().manual_seed(seed)
    idx = torch.where(torch.rand(T, generator=g) < dropped, -1, torch.randint(0, n, (T,), generator=g))
    idx = idx[torch.arange(T) // runs * runs]  # runs of tokens of one request
    a = (torch.randn(n, r, H, generator=g) * H ** -0.5).to(dtype).cuda()
    b = (torch.randn(n, N, r, generator=g) * r ** -0.5).to(dtype).cuda()
    scale = (2.0 ** torch.randint(-2, 3, (n,), generator=g)).cuda()
    return (rows_of(T, H, dtype, g, pitch, offset), a, b, idx.to(torch.int32).cuda(), rows_of(T, N, dtype, g, pitch, offset), scale)


def check(out, x, a, b, idx, base, scale):
    """out against base + scale b (a x), and its error against the bound."""
    dtype, H, r = x.dtype, x.shape[1], a.shape[1]
    want = torch.zeros(x.shape[0], b.shape[1], dtype=torch.float64, device="cuda") if base is None else base.double()
    bound = torch.zeros_like(want)
    for e in torch.unique(idx).tolist():
        if not 0 <= e < a.shape[0]:
            continue
        mine = torch.nonzero(idx == e).reshape(-1)
        k = 1.0 if scale is None else scale[e].item()
        xe, ae, be = x[mine].double(), a[e].double(), b[e].double()
        s = xe @ ae.T
        off = (H / 16 + 20) * 2.0 ** -22 * (xe.abs() @ ae.abs().T) + 2.0 ** -16 * s.abs()
        if dtype == torch.float16:
            off = off - 2.0 ** -16 * s.abs() + 2.0 ** -22 * s.abs() + 2.0 ** -38 * s.abs().amax(1, keepdim=True)
        want[mine] += k * (s @ be.T)
        bound[mine] = k * (off @ be.abs().T + (r / 8 + 3) * 2.0 ** -22 * (s.abs() @ be.abs().T))
    bound = bound + half_step(dtype, want.abs() + bound) + 2.0 ** -24 * want.abs()
    wrong = (out.double() - want).abs() > bound
    assert not wrong.any(), (int(wrong.sum()), torch.nonzero(wrong)[:4].tolist())
    none = (idx < 0) | (idx >= a.shape[0])
    assert torch.equal(out[none], torch.zeros_like(out[none]) if base is None else base[none])


def permutation(idx, n, align):
    import sonicmoe

    return sonicmoe.token_permutation(idx.view(-1, 1), n, align=align)


#: tokens, H, N, adapters, rank, align
SIZES = [(1, 64, 64, 1, 16, 16), (1, 4096, 4096, 5, 16, 16), (3, 40, 24, 7, 8, 16), (16, 520, 264, 2, 32, 16), (17, 1000, 72, 60, 24, 48),
         (37, 64, 1032, 3, 64, 128), (64, 2048, 512, 64, 128, 16), (256, 96, 32, 4, 40, 64), (300, 128, 64, 4, 8, 32),
         (300, 136, 40, 1, 16, 32), (600, 1032, 520, 9, 32, 64), (1000, 192, 256, 3, 64, 128), (700, 264, 264, 5, 128, 128),
         (1500, 64, 64, 400, 16, 16), (400, 3000, 96, 2, 104, 64), (5000, 64, 40, 6, 16, 128), (9600, 72, 64, 40, 32, 64),
         (19000, 64, 64, 7, 64, 128), (1030, 520, 72, 33, 48, 32), (4500, 520, 264, 3, 16, 16), (4500, 1000, 520, 500, 32, 16),
         (4400, 264, 776, 5, 64, 32), (5000, 136, 64, 12, 128, 48), (4224, 2048, 256, 1, 8, 128), (1000, 72, 296, 900, 24, 16),
         (10000, 192, 64, 100, 128, 16), (4300, 8, 8, 70, 40, 64),
         (4400, 520, 1032, 5, 128, 16), (4700, 2048, 136, 2, 24, 16), (4096, 64, 2048, 60, 64, 16), (11000, 264, 200, 3, 8, 16),
         (4500, 128, 8, 2, 104, 32)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,N,n,r,align", SIZES)
def test_whole_pieces(built_library, dtype, T, H, N, n, r, align):
    import sonicmoe

    x, a, b, idx, base, scale = make(T, H, N, n, r, dtype)
    p = permutation(idx, n, align)
    check(sonicmoe.adapter_linear(x, a, b, p, base=base, scale=scale), x, a, b, idx, base, scale)
    check(sonicmoe.adapter_linear(x, a, b, p), x, a, b, idx, None, None)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,N,n,r,align", [
    (1, 1, 1, 1, 1, 16), (1, 65, 33, 3, 16, 16), (5, 1030, 1001, 60, 12, 64), (33, 255, 7, 2, 5, 16), (64, 4097, 2049, 9, 100, 16),
    (300, 130, 66, 5, 16, 32), (300, 1031, 515, 1, 3, 128), (1027, 1030, 1001, 60, 12, 64), (900, 517, 30, 4, 127, 64), (5001, 61, 63, 6, 33, 128),
    (4500, 523, 261, 3, 16, 16), (4501, 999, 519, 300, 32, 16), (4400, 260, 770, 5, 63, 32), (5000, 131, 65, 12, 128, 48),
    (10001, 67, 300, 9, 5, 128), (4300, 1, 1, 70, 1, 64),
    (4400, 520, 1031, 5, 128, 16), (4700, 2048, 139, 2, 24, 16), (4096, 64, 2046, 60, 64, 16), (11000, 264, 193, 3, 8, 16), (4500, 128, 7, 2, 40, 32)])
def test_odd_sizes(built_library, dtype, T, H, N, n, r, align):
    import sonicmoe

    for pitch, offset in ((0, 0), (3, 1)):
        x, a, b, idx, base, scale = make(T, H, N, n, r, dtype, pitch=pitch, offset=offset)
        p = permutation(idx, n, align)
        check(sonicmoe.adapter_linear(x, a, b, p, base=base, scale=scale), x, a, b, idx, base, scale)
        check(sonicmoe.adapter_linear(x, a, b, p), x, a, b, idx, None, None)


@pytest.mark.parametrize("T,align", [(40, 16), (4500, 64)])
def test_strides(built_library, T, align):
    import sonicmoe

    x, a, b, idx, base, scale = make(T, 64, 48, 5, 16, torch.bfloat16)
    p = permutation(idx, 5, align)
    # (layouts go by different kernels, whose sums are in different orders: the same bound, not the same bits)
    for pitch, offset in ((8, 0), (0, 8), (2, 0), (3, 5)):
        flat = torch.empty(offset + T * (64 + pitch), dtype=x.dtype, device="cuda")[offset:].view(T, 64 + pitch)[:, :64]
        flat.copy_(x)
        wide = torch.empty(T, 48 + pitch + offset, dtype=x.dtype, device="cuda")[:, offset:offset + 48]
        wide.copy_(base)
        check(sonicmoe.adapter_linear(flat, a, b, p, base=wide, scale=scale), x, a, b, idx, base, scale)
        check(sonicmoe.adapter_linear(x, a, b, p, base=wide, scale=scale), x, a, b, idx, base, scale)
        check(sonicmoe.adapter_linear(flat, a, b, p, base=base, scale=scale), x, a, b, idx, base, scale)
    check(sonicmoe.adapter_linear(x.t().contiguous().t(), a, b, p, base=base.t().contiguous().t(), scale=scale), x, a, b, idx, base, scale)
    one = x[:1].expand(T, 64)
    check(sonicmoe.adapter_linear(one, a, b, p, base=base[:1].expand(T, 48), scale=scale), one, a, b, idx, base[:1].expand(T, 48), scale)


@pytest.mark.parametrize("T,align,N", [(40, 16, 48), (4500, 64, 48), (40, 16, 37), (4500, 16, 37), (4500, 16, 333)])
def test_in_place_into_a_slice(built_library, T, align, N):
    import sonicmoe

    x, a, b, idx, base, scale = make(T, 64, N, 5, 16, torch.bfloat16)
    p = permutation(idx, 5, align)
    qkv = torch.randn(T, 3 * N, device="cuda").bfloat16()
    before = qkv.clone()
    before[:, N:2 * N] = sonicmoe.adapter_linear(x, a, b, p, base=qkv[:, N:2 * N], scale=scale)
    got = sonicmoe.adapter_linear(x, a, b, p, base=qkv[:, N:2 * N], scale=scale, inplace=True)
    assert torch.equal(qkv, before) and got.data_ptr() == qkv[:, N:].data_ptr()


def test_in_place_counts_as_a_change(built_library):
    """What autograd has saved of a base that is added to in place is no longer what a backward pass needs: it refuses, as after base.add_()."""
    import sonicmoe

    x, a, b, idx, base, scale = make(40, 64, 48, 5, 16, torch.bfloat16)
    p = sonicmoe.adapter_permutation(idx, 5)
    y = base.clone().requires_grad_().sigmoid()
    version = y._version
    sonicmoe.adapter_linear(x, a, b, p, base=y.detach(), scale=scale)
    assert y._version == version
    y.sum().backward(retain_graph=True)
    sonicmoe.adapter_linear(x, a, b, p, base=y.detach(), scale=scale, inplace=True)
    assert y._version == version + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    leaf = base.clone().requires_grad_()
    w = torch.ones(48, dtype=base.dtype, device="cuda")
    z, h = sonicmoe.rms_norm(leaf, w, residual=base)
    with torch.no_grad():  # the first half of the columns alone
        sonicmoe.adapter_linear(x, a, b[:, :24].contiguous(), p, base=h[:, :24], scale=scale, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    with torch.inference_mode():  # tensors without a count, and those of outside
        for own in (base.clone(), base):
            want = sonicmoe.adapter_linear(x, a, b, p, base=own, scale=scale)
            assert torch.equal(sonicmoe.adapter_linear(x, a, b, p, base=own, scale=scale, inplace=True), want)


@pytest.mark.parametrize("T,n,r", [(30, 4, 16), (900, 40, 16), (4400, 5, 16), (4400, 5, 64)])
def test_in_place_into_the_rows_that_are_read(built_library, T, n, r):
    import sonicmoe

    for H in (256, 251):
        x, a, b, idx, _, scale = make(T, H, H, n, r, torch.bfloat16)
        p = sonicmoe.adapter_permutation(idx, n)
        want = sonicmoe.adapter_linear(x, a, b, p, base=x, scale=scale)
        check(want, x, a, b, idx, x, scale)
        assert torch.equal(sonicmoe.adapter_linear(x, a, b, p, base=x, scale=scale, inplace=True), want)
    flat = torch.zeros((T + 1) * 256, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="other tokens' rows"):
        sonicmoe.adapter_linear(flat[:-256].view(T, 256), a.new_zeros(n, r, 256), b.new_zeros(n, 256, r), p, base=flat[256:].view(T, 256), inplace=True)


@pytest.mark.parametrize("T,align", [(30, 16), (600, 32), (4400, 16), (4400, 128)])
def test_loads(built_library, T, align):
    """All tokens with one adapter, none with any, every token with its own, the first or the last one alone."""
    import sonicmoe

    n = 700
    x, a, b, _, base, scale = make(T, 64, 40, n, 8, torch.bfloat16)
    only = torch.full((T,), -1)
    for idx in (torch.full((T,), 3), only, torch.arange(T), torch.full((T,), n - 1), only.clone().index_fill_(0, torch.tensor([0]), 5),
                only.clone().index_fill_(0, torch.tensor([T - 1]), 0), torch.full((T,), n), torch.full((T,), -2 ** 31)):
        idx = idx.to(torch.int32).cuda()
        p = permutation(idx, n, align)
        check(sonicmoe.adapter_linear(x, a, b, p, base=base, scale=scale), x, a, b, idx, base, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,N,n,r", [(2048, 136, 264, 512, 64), (8192, 264, 136, 256, 32), (4400, 72, 96, 4096, 16), (4200, 131, 257, 300, 128),
                                       (6000, 264, 201, 700, 128), (3000, 520, 264, 2000, 8)])
def test_few_adapters_of_many_in_use(built_library, dtype, T, H, N, n, r):
    """Long prompts of eight requests, one without an adapter, with hundreds of adapters to choose from."""
    import sonicmoe

    x, a, b, _, base, scale = make(T, H, N, n, r, dtype)
    g = torch.Generator().manual_seed(6)
    request = torch.randint(0, 8, (T,), generator=g).sort().values
    idx = torch.randperm(n, generator=g)[:8].index_fill_(0, torch.tensor([5]), -1)[request].to(torch.int32).cuda()
    p = sonicmoe.adapter_permutation(idx, n)
    check(sonicmoe.adapter_linear(x, a, b, p, base=base, scale=scale), x, a, b, idx, base, scale)
    check(sonicmoe.adapter_linear(x, a, b, p), x, a, b, idx, None, None)


def test_two_threads(built_library):
    """Calls of two host threads, each on a stream of its own."""
    import threading

    import sonicmoe

    inputs = [make(T, 200, 136, 6, r, torch.float16, seed=T) for T, r in ((50, 16), (4400, 64))]
    x = [i[0] for i in inputs]
    w = torch.ones(200, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(k):
        try:
            xk, a, b, idx, base, scale = inputs[k]
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    leaf = xk.detach().clone().requires_grad_()
                    y = sonicmoe.rms_norm(leaf, w)
                    g, = torch.autograd.grad(y, leaf, xk)
                    out = sonicmoe.adapter_linear(xk, a, b, sonicmoe.adapter_permutation(idx, 6), base=base, scale=scale)
            stream.synchronize()
            got[k] = (y.detach(), g, out)
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for k, (xk, a, b, idx, base, scale) in enumerate(inputs):
        leaf = x[k].detach().clone().requires_grad_()
        y = sonicmoe.rms_norm(leaf, w)
        g, = torch.autograd.grad(y, leaf, x[k])
        assert torch.equal(got[k][0], y) and torch.equal(got[k][1], g)
        check(got[k][2], xk, a, b, idx, base, scale)


@pytest.mark.parametrize("T,align", [(30, 16), (4400, 64)])
def test_tokens_dropped_after_the_sort(built_library, T, align):
    import sonicmoe

    x, a, b, idx, base, scale = make(T, 64, 40, 5, 8, torch.bfloat16, dropped=0.0)
    p = permutation(idx, 5, align)
    gone = torch.arange(T, device="cuda") % 3 == 1
    p.s_reverse_scatter_idx[gone] = -1
    check(sonicmoe.adapter_linear(x, a, b, p, base=base, scale=scale), x, a, b, torch.where(gone, -1, idx), base, scale)


@pytest.mark.parametrize("T,align", [(20, 16), (4400, 32)])
def test_numbers_that_are_not_finite_stay_in_their_rows(built_library, T, align):
    import sonicmoe

    for dtype in TYPES:
        x, a, b, idx, base, scale = make(T, 72, 40, 3, 8, dtype, dropped=0.0, runs=1)
        p = permutation(idx, 3, align)
        want = sonicmoe.adapter_linear(x, a, b, p, base=base, scale=scale)
        x[3, 5], x[7, 0], base[9, 2] = float("nan"), float("inf"), -float("inf")
        got = sonicmoe.adapter_linear(x, a, b, p, base=base, scale=scale)
        rest = torch.ones(T, dtype=torch.bool)
        rest[[3, 7, 9]] = False
        assert torch.equal(got[rest], want[rest]) and got[3].isnan().all() and not got[7].isfinite().any()
        assert got[9, 2] == -float("inf") and torch.equal(got[9, 3:], want[9, 3:])


@pytest.mark.parametrize("T,align", [(20, 16), (4400, 32)])
def test_fp16_products_past_its_range(built_library, T, align):
    """a x beyond fp16's largest value, and below its smallest, on the way to results within its range."""
    import sonicmoe

    x, a, b, idx, base, scale = make(T, 512, 40, 3, 16, torch.float16, dropped=0.0)
    p = permutation(idx, 3, align)
    for up, down in ((2.0 ** 10, 2.0 ** -12), (2.0 ** -12, 2.0 ** 6)):
        big, small = (x * up, b * down) if up > 1 else (x * up, b * down)
        strong = a * (2.0 ** 8 if up > 1 else 2.0 ** -8)
        check(sonicmoe.adapter_linear(big, strong, small, p, base=base, scale=scale), big, strong, small, idx, base, scale)


def test_the_same_bits_every_time_and_in_a_graph(built_library):
    import sonicmoe

    for T in (30, 700, 4400):
        x, a, b, idx, base, scale = make(T, 520, 264, 6, 16, torch.bfloat16)
        p = sonicmoe.adapter_permutation(idx, 6)
        want = sonicmoe.adapter_linear(x, a, b, p, base=base, scale=scale)
        check(want, x, a, b, idx, base, scale)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(sonicmoe.adapter_linear(x, a, b, p, base=base, scale=scale), want)
        graph = torch.cuda.CUDAGraph()
        live = idx.clone()
        with torch.cuda.graph(graph, stream=side):
            got = sonicmoe.adapter_linear(x, a, b, sonicmoe.adapter_permutation(live, 6), base=base, scale=scale)
        graph.replay()
        assert torch.equal(got, want)
        live.copy_(idx.roll(1))
        graph.replay()
        check(got, x, a, b, live, base, scale)
        torch.cuda.synchronize()


def test_between_other_kernels_with_tensor_memory(built_library):
    """Tiles by tensor memory with products that want all of it right behind them, on two streams."""
    import sonicmoe
    from sonicmoe.functional import int8

    x, a, b, idx, base, scale = make(9000, 512, 512, 3, 64, torch.bfloat16)
    p = sonicmoe.adapter_permutation(idx, 3)
    g = torch.Generator().manual_seed(4)
    wq, w_scale = int8.quantize_rows((torch.randn(512, 512, generator=g) * 0.05).cuda())

    def chain():
        out = x
        for _ in range(6):
            out = sonicmoe.adapter_linear(out, a, b, p, base=int8.int8_linear(out, wq, w_scale, out_dtype=torch.bfloat16), scale=scale)
            out = out / 4
        return out

    want = chain()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(chain())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got)
    sonicmoe.check_status()


def test_adapter_permutation(built_library):
    import sonicmoe

    for T, n in ((0, 4), (1, 1), (1000, 1000), (1000, 8)):
        idx = torch.randint(-1, n, (T,), dtype=torch.int64, device="cuda")
        p = sonicmoe.adapter_permutation(idx, n)
        want = sonicmoe.token_permutation(idx.view(T, 1), n, align=16)
        assert p.align == 16 and p.s_reverse_scatter_idx.shape == (T, 1)
        assert torch.equal(p.s_reverse_scatter_idx, want.s_reverse_scatter_idx) and torch.equal(p.x_gather_idx, want.x_gather_idx)


def test_no_tokens(built_library):
    import sonicmoe

    x, a, b, idx, base, scale = make(0, 64, 40, 3, 8, torch.bfloat16)
    assert sonicmoe.adapter_linear(x, a, b, sonicmoe.adapter_permutation(idx, 3), base=base, scale=scale).shape == (0, 40)


def test_refusals_on_the_device(built_library):
    import sonicmoe
    from torch.autograd import forward_ad

    x, a, b, idx, base, scale = make(40, 64, 48, 5, 16, torch.bfloat16)
    p = sonicmoe.adapter_permutation(idx, 5)
    f = sonicmoe.adapter_linear
    for bad in (a.transpose(0, 1).contiguous().transpose(0, 1), a.cpu()):
        with pytest.raises(ValueError, match="a has to be a contiguous"):
            f(x, bad, b, p)
    with pytest.raises(ValueError, match="b has to be a contiguous"):
        f(x, a, b.transpose(1, 2).contiguous().transpose(1, 2), p)
    with pytest.raises(ValueError, match="of \\(40, 1\\) pairs"):
        f(x, a, b, sonicmoe.token_permutation(idx.view(20, 2), 5, align=16))
    with pytest.raises(ValueError, match="by 5 adapters"):
        f(x, a, b, sonicmoe.adapter_permutation(idx, 6))
    for align in (1, 8, 40):
        with pytest.raises(ValueError, match="multiple of 16"):
            f(x, a, b, sonicmoe.token_permutation(idx.view(-1, 1), 5, align=align))
    for bad in (scale.bfloat16(), scale[:4], scale.cpu()):
        with pytest.raises(ValueError, match="scale has to be"):
            f(x, a, b, p, scale=bad)
    for bad in (base.float(), base[:, :40], base[:30], base.cpu()):
        with pytest.raises(ValueError, match="base has to be"):
            f(x, a, b, p, base=bad)
    with pytest.raises(ValueError, match="no base"):
        f(x, a, b, p, inplace=True)
    for bad in (base.t().contiguous().t(), base[:1].expand(40, 48)):
        with pytest.raises(ValueError, match="contiguous and apart"):
            f(x, a, b, p, base=bad, inplace=True)
    for k in range(3):
        args = [t.detach().clone() for t in (x, a, b)]
        args[k].requires_grad_()
        with pytest.raises(NotImplementedError, match="no gradient"):
            f(*args, p)
        with torch.no_grad():
            f(*args, p)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(forward_ad.make_dual(x, torch.ones_like(x)), a, b, p)


def test_norm_8_bit_projection_and_adapters_together(built_library):
    """A serving block's order: norm to 8-bit rows, shared projection, adapters beside it, the residual of the next norm."""
    import sonicmoe
    from sonicmoe.functional import int8

    for T in (1, 50, 4400):
        x, a, b, idx, _, scale = make(T, 256, 256, 6, 16, torch.bfloat16)
        g = torch.Generator().manual_seed(9)
        h0 = rows_of(T, 256, torch.bfloat16, g)
        weight = (1 + 0.1 * torch.randn(256, generator=g)).bfloat16().cuda()
        w = (torch.randn(256, 256, generator=g) * 0.05).cuda()
        wq, w_scale = int8.quantize_rows(w)
        p = sonicmoe.adapter_permutation(idx, 6)
        r = sonicmoe.rms_norm_quantize(x, weight, residual=h0, keep_y=True)
        z = int8.int8_linear(r.q, wq, w_scale, x_scale=r.scale)
        out = sonicmoe.adapter_linear(r.y, a, b, p, base=z, scale=scale)
        check(out, r.y, a, b, idx, z, scale)
        again = sonicmoe.adapter_linear(r.y, a, b, p, base=z.clone(), scale=scale, inplace=True)
        assert torch.equal(again, out)
        # the whole against 64 bits: values of 8-bit rows and weights are off evenly over a step, rms 1 / sqrt(12) of it, the step 1/127 of the largest of
        # 256 normal numbers, under 4.5 of their rms: 1.02 % each, 1.45 % together, which the adapters' part does not have; and three roundings to bf16,
        # under 0.25 % each.  Twice that.
        h = (x.double() + h0.double()).bfloat16().double()
        y = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * weight.double()
        want = y @ w.double().T
        for t in range(T):
            if idx[t] >= 0:
                want[t] += scale[idx[t]].double() * (b[idx[t]].double() @ (a[idx[t]].double() @ y[t]))
        assert (out.double() - want).norm() <= 0.03 * want.norm()
        y2, h2 = sonicmoe.rms_norm(out, weight, residual=r.h)
        assert torch.equal(h2, (out.double() + r.h.double()).float().bfloat16()) and y2.isfinite().all()
