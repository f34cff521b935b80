"""8-bit integer products: quantisation bit for bit, products against 64-bit sums of the same integers.

Tolerances.  The sum of a product is exact, so z = sum * x_scale * w_scale + bias is off by at most dz = 4 * 2^-24 (|z - bias| +
|bias|): the sum's rounding, two products and an addition.  An activation adds its slope times that and 2^-15 of its value (the
fast exponential: 2 + 1.16 |z| units in the last place, |z| < 60 here; erfc's 4 units).  The result is rounded to its type: half
a step, eps / 2 of the value, or of the smallest normal value below it."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTIVATIONS = [None, "swiglu", "geglu", "reglu", "relu_sq", "relu", "gelu", "silu"]
GATED = ("swiglu", "geglu", "reglu")


def exact_quantize(x):
    """(127 x / amax rounded half to even, by its remainder; amax / 127 in fp32)."""
    amax32 = x.float().abs().amax(-1, keepdim=True)
    amax = torch.where(amax32 > 0, amax32, torch.ones_like(amax32)).double()
    twice = 254 * x.double() + amax
    q = torch.floor(twice / (2 * amax))
    tie = (twice == 2 * q * amax) & (torch.remainder(q, 2) == 1)
    return torch.where(tie, q - 1, q), torch.where(amax32 > 0, amax32 / 127, torch.ones_like(amax32)).squeeze(-1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pitch,offset", [
    (1, 1, 0, 0), (3, 15, 0, 0), (5, 16, 0, 0), (70, 17, 0, 0), (9, 64, 0, 0), (130, 1005, 0, 0), (33, 1030, 0, 0), (40, 1024, 8, 8),
    (7, 4096, 0, 0), (5, 4098, 0, 1), (2, 40000, 0, 0), (1, 131071, 0, 0)])
def test_quantize_rows(built_library, dtype, rows, cols, pitch, offset):
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(cols)
    flat = torch.zeros(offset + rows * (cols + pitch), dtype=dtype, device="cuda")
    x = flat[offset:].view(rows, cols + pitch)[:, :cols]
    x.copy_(torch.randn(rows, cols, generator=g) * torch.rand(rows, 1, generator=g) * 5)
    q, scale = int8.quantize_rows(x)
    want, want_scale = exact_quantize(x.cpu())
    assert q.dtype == torch.int8 and torch.equal(q.cpu().double(), want) and torch.equal(scale.cpu(), want_scale)
    assert q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
    padded = torch.as_strided(q, (rows, q.stride(0)), (q.stride(0), 1))
    assert not padded[:, cols:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_special_rows(built_library, dtype):
    """Rows of zeros, of halves (127 x / amax is k + 1/2), of the type's smallest and largest values, with infinities and NaN."""
    from sonicmoe.functional import int8

    f = torch.finfo(dtype)
    cols = 508
    x = torch.zeros(12, cols, dtype=torch.float64)
    x[1] = torch.arange(cols) - 254                    # amax 254: every odd value is a tie
    x[2] = x[1] * 2.0 ** -12
    x[3, ::3] = f.smallest_normal * f.eps              # the smallest subnormal value alone
    x[4] = (torch.arange(cols) - 254) * f.smallest_normal * f.eps
    x[5] = torch.linspace(-1, 1, cols, dtype=torch.float64) * f.max
    x[6] = (torch.arange(cols) % 255 - 127) * 2.0 ** -8
    x[7, 0], x[7, 1:] = -1, torch.linspace(0, 1, cols - 1, dtype=torch.float64)
    x = x.to(dtype)
    x[8, 3], x[9, 4], x[10, 5], x[10, 6] = float("inf"), float("-inf"), float("nan"), float("inf")
    x[8:11, 100:] = 1
    q, scale = int8.quantize_rows(x.cuda())
    want, want_scale = exact_quantize(x)
    fine = [i for i in range(12) if i not in (8, 9, 10)]
    assert torch.equal(q.cpu().double()[fine], want[fine]) and torch.equal(scale.cpu()[fine], want_scale[fine])
    assert not q[8:11].any() and scale[8].item() == scale[9].item() == float("inf") and scale[10].isnan()
    w = torch.ones(3, cols, dtype=dtype, device="cuda")
    y = int8.int8_linear(x.cuda(), *int8.quantize_rows(w))
    assert bool(y[8:11].isnan().all()) and not y[fine].isnan().any()


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_next_to_borders(built_library, dtype):
    """The values nearest to every border k + 1/2 of rows with random largest values: a few steps of the type to either side."""
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(1)
    amax = (torch.rand(400, 1, generator=g, dtype=torch.float64) + 0.5).to(dtype)
    amax[:17, 0] = torch.arange(8, 25) * 127.0 / 2048  # of 16-bit types: those that have more borders than one
    border = ((torch.arange(254) - 126.5) * amax.double() / 127).to(dtype)
    bits = border.view(torch.int32 if dtype == torch.float32 else torch.int16)
    near = torch.cat([(bits + d).view(dtype) for d in (-2, -1, 0, 1, 2)], dim=1)
    x = torch.cat([amax, near.clamp(-amax, amax)], dim=1)
    for scale in (1.0, 2.0 ** -130 if dtype == torch.float32 else 1.0, 2.0 ** 125 if dtype != torch.float16 else 1.0):
        scaled = (x.double() * scale).to(dtype)
        q, s = int8.quantize_rows(scaled.cuda())
        want, want_scale = exact_quantize(scaled)
        assert torch.equal(q.cpu().double(), want) and torch.equal(s.cpu(), want_scale)


def test_quantize_leading_dimensions_and_empty(built_library):
    from sonicmoe.functional import int8

    w = torch.randn(3, 5, 40, device="cuda")
    q, s = int8.quantize_rows(w)
    q2, s2 = int8.quantize_rows(w.transpose(0, 1))
    assert q.shape == (3, 5, 40) and torch.equal(q2.transpose(0, 1), q) and torch.equal(s2.t(), s)
    assert q.stride(1) == 48 and q.stride(0) == 5 * 48
    q, s = int8.quantize_rows(w[:0])
    assert q.shape == (0, 5, 40) and s.shape == (0, 5)
    q, s = int8.quantize_rows(w[0, 0])
    assert q.shape == (40,) and s.dim() == 0
    assert int8.int8_linear(w[0, :0], *int8.quantize_rows(w[1])).shape == (0, 5)


def act_value(name, z):
    """(value, largest slope near z)"""
    one = torch.ones_like(z)
    if name in ("swiglu", "silu"):
        return z * torch.sigmoid(z), 1.2 * one
    if name in ("geglu", "gelu"):
        return 0.5 * z * torch.special.erfc(-z / 2 ** 0.5), 1.2 * one
    if name == "relu_sq":
        return z.clamp_min(0) ** 2, 2 * z.abs() + 1
    if name in ("relu", "reglu"):
        return z.clamp_min(0), one
    return z, one


def check(y, acc, xs, ws, bias, activation):
    """y against the exact sums acc (rows, N), scales (rows, 1) and (rows or 1, N), bias like ws."""
    plain = acc * xs.double() * ws.double()
    b = torch.zeros_like(plain) if bias is None else bias.double().expand_as(plain)
    z, dz = plain + b, 4 * 2.0 ** -24 * (plain.abs() + b.abs())
    if activation in GATED:
        a, slope = act_value(activation, z[:, 0::2])
        want = a * z[:, 1::2]
        off = a.abs() * dz[:, 1::2] + slope * (z[:, 1::2].abs() + dz[:, 1::2]) * dz[:, 0::2] + 2.0 ** -15 * want.abs()
    else:
        want, slope = act_value(activation, z)
        off = slope * dz + (2.0 ** -15 if activation else 0) * want.abs()
    f = torch.finfo(y.dtype)
    bound = off + f.eps / 2 * (want.abs() + off) + f.smallest_normal * f.eps / 2
    bad = (y.double() - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), torch.nonzero(bad)[:4].tolist())


def product(q, wq):
    """Exact sums of 8-bit products in 64 bits."""
    return q.double() @ wq.double().transpose(-1, -2)


SIZES = [(1, 1, 1), (1, 128, 4096), (3, 7, 17), (4, 34, 130), (5, 34, 130), (9, 64, 16), (128, 700, 264), (256, 520, 400), (16, 96, 128), (33, 100, 520), (64, 2048, 256), (100, 4096, 1000),
         (129, 258, 384), (300, 130, 1000), (257, 512, 131), (1000, 300, 640), (2049, 514, 136), (700, 4096, 2048)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_linear(built_library, M, N, K, dtype, with_bias):
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(M + N + K)
    x = torch.randn(M, K, generator=g).to(dtype).cuda()
    wq, ws = int8.quantize_rows((torch.randn(N, K, generator=g) * 0.05).cuda())
    bias = torch.randn(N, generator=g).to(dtype).cuda() if with_bias else None
    q, xs = int8.quantize_rows(x)
    acc = product(q, wq)
    check(int8.int8_linear(x, wq, ws, bias=bias), acc, xs[:, None], ws, bias, None)
    y = int8.int8_linear(q, wq, ws, x_scale=xs, bias=bias, out_dtype=dtype)
    assert torch.equal(y, int8.int8_linear(x, wq, ws, bias=bias))


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("M,N,K", [(2, 128, 64), (40, 200, 520), (300, 260, 264), (1500, 640, 1024)])
@pytest.mark.parametrize("out_dtype", TYPES)
def test_activations(built_library, activation, M, N, K, out_dtype):
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(N)
    x = (torch.randn(M, K, generator=g) * 3).bfloat16().cuda()
    wq, ws = int8.quantize_rows((torch.randn(N, K, generator=g) * 2 / K ** 0.5).cuda())
    bias = torch.randn(N, generator=g).cuda()
    q, xs = int8.quantize_rows(x)
    for b in (None, bias):
        y = int8.int8_linear(x, wq, ws, bias=b, activation_type=activation, out_dtype=out_dtype)
        assert y.dtype == out_dtype
        check(y, product(q, wq), xs[:, None], ws, b, activation)


@pytest.mark.parametrize("M,N", [(1, 9), (20, 200), (300, 300)])
def test_largest_sums(built_library, M, N):
    """131071 products of -128 and -128 is the largest sum that 32 bits hold."""
    from sonicmoe.functional import int8

    K = 131071
    q = torch.zeros(M, K + 1, dtype=torch.int8, device="cuda")[:, :K]
    wq = torch.zeros(N, K + 1, dtype=torch.int8, device="cuda")[:, :K]
    q.fill_(-128)
    wq.fill_(-128)
    wq[1::3] = 127
    one = torch.ones(max(M, N), device="cuda")
    y = int8.int8_linear(q, wq, one[:N], x_scale=one[:M], out_dtype=torch.float32)
    sums = torch.full((N,), 2 ** 14 * K, dtype=torch.int64)
    sums[1::3] = -128 * 127 * K
    assert torch.equal(y.cpu(), sums.float().expand(M, N))


def test_columns_behind_the_last_do_not_count(built_library):
    """8-bit rows whose buffer goes on behind the last column with values of another use."""
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(0)
    for M, N, K in ((2, 16, 37), (50, 140, 200), (600, 300, 333)):
        q = torch.randint(-128, 128, (M, 1024), generator=g, dtype=torch.int8).cuda()
        wq = torch.randint(-128, 128, (N, 1024), generator=g, dtype=torch.int8).cuda()
        one = torch.ones(max(M, N), device="cuda")
        y = int8.int8_linear(q[:, :K], wq[:, :K], one[:N], x_scale=one[:M], out_dtype=torch.float32)
        assert torch.equal(y.double(), product(q[:, :K], wq[:, :K]))  # at most 333 * 2^14 < 2^24: exact in fp32


@pytest.fixture(autouse=True)
def no_wait_was_abandoned():
    yield
    from sonicmoe import _lib

    _lib.check_status()


def grouped_case(T, K, E, align, dropped, seed=0):
    import sonicmoe

    g = torch.Generator().manual_seed(seed + T + E)
    bias = torch.randn(E, generator=g)
    idx = (torch.randn(T, E, generator=g) + bias).topk(K, dim=1).indices
    idx = torch.where(torch.rand(T, K, generator=g) < dropped, -1, idx)
    return sonicmoe.token_permutation(idx.cuda(), E, align)


def grouped_reference(p, q, xs, wq, ws, bias, E, gather, frequency):
    """(rows of experts, exact sums, row scales, channel scales, bias) of the rows that an expert has."""
    first = p.expert_frequency_offset.tolist()
    count = p.expert_frequency.tolist() if frequency else [b - a for a, b in zip(first, first[1:])]
    rows = torch.cat([torch.arange(first[e], first[e] + count[e]) for e in range(E)]).cuda()
    expert = torch.cat([torch.full((count[e],), e) for e in range(E)]).cuda()
    at = p.x_gather_idx.long()[rows] if gather else rows
    qr = torch.where((at >= 0)[:, None], q[at.clamp_min(0)].double(), 0.0)
    sr = torch.where(at >= 0, xs[at.clamp_min(0)], 0.0)
    acc = torch.zeros(rows.numel(), wq.shape[1], dtype=torch.float64, device="cuda")
    for e in range(E):
        of = expert == e
        acc[of] = qr[of] @ wq[e].double().t()
    return rows, acc, sr[:, None], ws[expert], None if bias is None else bias[expert]


@pytest.mark.parametrize("T,K,E,align,dropped,N,cols", [
    (1, 1, 1, 1, 0.0, 64, 64), (1, 8, 64, 1, 0.0, 256, 512), (5, 2, 4, 16, 0.5, 130, 200), (64, 4, 32, 1, 0.0, 512, 256),
    (200, 2, 3, 128, 0.1, 96, 1030), (1000, 3, 5, 1, 0.0, 300, 144), (1027, 4, 60, 64, 0.1, 200, 130), (600, 2, 300, 1, 0.0, 64, 80),
    (3000, 2, 4, 1, 0.0, 512, 256), (40, 2, 1000, 8, 0.0, 34, 48), (30, 2, 6, 4, 1.0, 64, 64), (2000, 8, 16, 1, 0.3, 256, 384),
    (512, 8, 64, 1, 0.0, 1536, 256), (700, 8, 64, 1, 0.0, 312, 272), (130, 2, 2, 1, 0.0, 384, 1024)])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("activation,with_bias,dtype", [(None, True, torch.float32), ("swiglu", False, torch.bfloat16),
                                                        ("gelu", True, torch.float16)])
def test_grouped(built_library, T, K, E, align, dropped, N, cols, gather, activation, with_bias, dtype):
    from sonicmoe.functional import int8

    p = grouped_case(T, K, E, align, dropped)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(T if gather else p.num_rows, cols, generator=g).to(dtype).cuda()
    wq, ws = int8.quantize_rows((torch.randn(E, N, cols, generator=g) * 2 / cols ** 0.5).cuda())
    bias = torch.randn(E, N, generator=g).to(dtype).cuda() if with_bias else None
    q, xs = int8.quantize_rows(x)
    for frequency in (False, True):
        y = int8.int8_grouped_linear(x, wq, ws, p.expert_frequency_offset, p.x_gather_idx if gather else None,
                                     p.expert_frequency if frequency else None, bias=bias, activation_type=activation)
        rows, *parts = grouped_reference(p, q, xs, wq, ws, bias, E, gather, frequency)
        check(y[rows], *parts, activation)
        rest = torch.ones(p.num_rows, dtype=torch.bool, device="cuda")
        rest[rows] = False
        assert not y[rest].any() and not y[rest].isnan().any()
        again = int8.int8_grouped_linear(q, wq, ws, p.expert_frequency_offset, p.x_gather_idx if gather else None,
                                         p.expert_frequency if frequency else None, x_scale=xs, bias=bias,
                                         activation_type=activation, out_dtype=dtype)
        assert torch.equal(again, y)


def test_grouped_load_in_one_expert(built_library):
    from sonicmoe.functional import int8

    E, N, cols = 9, 128, 192
    g = torch.Generator().manual_seed(2)
    wq, ws = int8.quantize_rows(torch.randn(E, N, cols, generator=g).cuda())
    for R in (3, 100, 700, 5000):
        x = torch.randn(R, cols, generator=g).cuda()
        off = torch.tensor([0] * 5 + [R] * 5, dtype=torch.int32, device="cuda")
        y = int8.int8_grouped_linear(x, wq, ws, off)
        q, xs = int8.quantize_rows(x)
        check(y, product(q, wq[4]), xs[:, None], ws[4], None, None)


@pytest.mark.parametrize("N,K", [(1, 16), (64, 128), (65, 400), (200, 520), (1030, 2064), (2048, 1152), (4800, 144), (9473, 256)])
def test_every_number_of_rows(built_library, N, K):
    """Where the kernel and its tiles change with the rows: scales of one and fp32 results, so that an exact sum has one answer."""
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(N + K)
    wq = torch.empty(N, (K + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :K]
    wq.copy_(torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8))
    q = torch.empty(300, wq.stride(0), dtype=torch.int8, device="cuda")[:, :K]
    q.copy_(torch.randint(-128, 128, (300, K), generator=g, dtype=torch.int8))
    want, one = product(q, wq).float(), torch.ones(max(N, 300), device="cuda")
    for M in (1, 2, 3, 4, 5, 6, 7, 8, 9, 31, 32, 33, 63, 64, 65, 96, 97, 127, 128, 129, 191, 192, 193, 256, 257, 300):
        first = (300 - M) // 2
        y = int8.int8_linear(q[first : first + M], wq, one[:N], x_scale=one[:M], out_dtype=torch.float32)
        assert torch.equal(y, want[first : first + M]), M
        if N % 2 == 0:
            z = int8.int8_linear(q[first : first + M], wq, one[:N], x_scale=one[:M], activation_type="reglu", out_dtype=torch.float32)
            assert torch.equal(z, want[first : first + M, 0::2].clamp_min(0) * want[first : first + M, 1::2]), M


@pytest.mark.parametrize("counts", [[9, 0, 3], [1, 60, 3], [0, 0, 64], [40, 50, 30], [128, 0, 0], [1, 1, 90]])
def test_few_sorted_rows_of_few_experts(built_library, counts):
    """Small tiles with expert offsets: an expert's last rows next to the following one's first."""
    from sonicmoe.functional import int8

    R, E, N, K = sum(counts), len(counts), 328, 700
    g = torch.Generator().manual_seed(R)
    wq, ws = int8.quantize_rows(torch.randn(E, N, K, generator=g).cuda())
    x = torch.randn(R + 7, K, generator=g).bfloat16().cuda()
    off = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    q, xs = int8.quantize_rows(x)
    y = int8.int8_grouped_linear(x, wq, ws, off, out_dtype=torch.float32)
    for e, n in enumerate(counts):
        rows = slice(int(off[e]), int(off[e]) + n)
        check(y[rows], product(q[rows], wq[e]), xs[rows, None], ws[e], None, None)
    assert not y[R:].any()
    assert torch.equal(y, int8.int8_grouped_linear(q, wq, ws, off, x_scale=xs, out_dtype=torch.float32))


@pytest.mark.parametrize("rows,E,N", [(32, 16, 200), (32, 128, 72), (31, 300, 64), (9, 5, 640), (8, 64, 1536), (17, 16, 30)])
@pytest.mark.parametrize("spread", [1, 3, 100])
def test_few_rows_of_many_experts(built_library, rows, E, N, spread):
    """Rows shared out in small units: every row in one expert, in three, in as many as there are, and rows that none has between."""
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(rows + E + spread)
    K = 320
    wq, ws = int8.quantize_rows(torch.randn(E, N, K, generator=g).cuda())
    chosen = torch.randperm(E, generator=g)[:spread]
    owner = chosen[torch.randint(0, len(chosen), (rows,), generator=g)].sort().values
    count = torch.bincount(owner, minlength=E)
    gap = (torch.rand(E, generator=g) < 0.02).int()  # a row that no expert has behind some of them
    off = torch.cat([torch.zeros(1, dtype=torch.long), (count + gap).cumsum(0)])
    R = int(off[-1])
    x = torch.randn(5, K, generator=g).bfloat16().cuda()
    take = torch.randint(-1, 5, (R,), generator=g, dtype=torch.int32).cuda()
    bias = torch.randn(E, N, generator=g).cuda()
    out = int8.int8_grouped_linear(x, wq, ws, off.int().cuda(), take, count.int().cuda(), bias=bias, out_dtype=torch.float32)
    q, xs = int8.quantize_rows(x)
    for e in range(E):
        r = torch.arange(int(off[e]), int(off[e] + count[e]), device="cuda")
        if len(r):
            src, none = take[r].long().clamp_min(0), take[r] < 0
            acc = product(q[src], wq[e])
            acc[none] = 0
            check(out[r], acc, xs[src, None], ws[e], bias[e], None)
        assert not out[int(off[e] + count[e]) : int(off[e + 1])].any()


def test_many_tiles_of_every_kind(built_library):
    """Loads whose last tiles have 1 to 256 rows, many tiles to a CTA pair, long reductions, again and again: the roles of the
    tile kernel must not lose one another where a tile's rows are few."""
    from sonicmoe.functional import int8

    E, N, cols, T, K = 64, 1024, 2048, 2500, 4
    g = torch.Generator().manual_seed(7)
    wq = torch.randint(-127, 128, (E, N, cols), generator=g, dtype=torch.int8).cuda()
    ws = torch.rand(E, N, generator=g).cuda() * 1e-4
    q = torch.randint(-127, 128, (T, cols), generator=g, dtype=torch.int8).cuda()
    xs = torch.rand(T, generator=g).cuda()
    for seed in range(4):
        p = grouped_case(T, K, E, 1, 0.0, seed)
        rows, *parts = grouped_reference(p, q, xs, wq, ws, None, E, True, False)
        for _ in range(5):
            y = int8.int8_grouped_linear(q, wq, ws, p.expert_frequency_offset, p.x_gather_idx, x_scale=xs, out_dtype=torch.float32)
        check(y[rows], *parts, None)
        sorted_x = q[p.x_gather_idx.long()].contiguous()
        again = int8.int8_grouped_linear(sorted_x, wq, ws, p.expert_frequency_offset, x_scale=xs[p.x_gather_idx.long()].contiguous(),
                                         out_dtype=torch.float32)
        assert torch.equal(again, y)


def test_offsets_and_gather_indices_out_of_range(built_library):
    """They are cut to the rows that exist; a gathered row that does not counts as zeros."""
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(3)
    for R in (12, 400):
        wq, ws = int8.quantize_rows(torch.randn(2, 64, 96, generator=g).cuda())
        x = torch.randn(R, 96, generator=g).cuda()
        off = torch.tensor([0, R // 2, 2 ** 30], dtype=torch.int32, device="cuda")
        gather = torch.arange(R, dtype=torch.int32, device="cuda")
        gather[1], gather[R // 2 + 1], gather[R - 1] = -7, R, 2 ** 31 - 1
        bias = torch.randn(2, 64, generator=g).cuda()
        y = int8.int8_grouped_linear(x, wq, ws, off, gather, bias=bias)
        q, xs = int8.quantize_rows(x)
        xs[[1, R // 2 + 1, R - 1]] = 0
        for e, rows in ((0, slice(0, R // 2)), (1, slice(R // 2, R))):
            check(y[rows], product(q[rows], wq[e]), xs[rows, None], ws[e], bias[e], None)


def test_streams_graphs_and_repeats(built_library):
    """On a stream of its own, captured and replayed on new values and another load: the same bits as outside."""
    from sonicmoe import _lib
    from sonicmoe.functional import int8

    T, K, E, N, cols = 700, 2, 8, 256, 320
    g = torch.Generator().manual_seed(4)
    wq, ws = int8.quantize_rows(torch.randn(E, N, cols, generator=g).cuda())
    plans = [grouped_case(T, K, E, 1, 0.2, seed) for seed in (0, 5)]
    xs = [torch.randn(T, cols, generator=g).bfloat16().cuda() for _ in range(2)]

    def run(x, off, gather):
        return (int8.int8_grouped_linear(x, wq, ws, off, gather, activation_type="swiglu"),
                int8.int8_linear(x[:9], wq[0], ws[0]), int8.int8_linear(x[:100], wq[1], ws[1]))

    want = [run(x, p.expert_frequency_offset, p.x_gather_idx) for x, p in zip(xs, plans)]
    assert all(torch.equal(a, b) for a, b in zip(want[0], run(xs[0], plans[0].expert_frequency_offset, plans[0].x_gather_idx)))
    static = [xs[0].clone(), plans[0].expert_frequency_offset.clone(), plans[0].x_gather_idx.clone()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = run(*static)
    for i in (1, 0):
        for t, v in zip(static, (xs[i], plans[i].expert_frequency_offset, plans[i].x_gather_idx)):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))
    _lib.check_status()


def test_sort_quantise_multiply_combine(built_library):
    """The operators together, as an MoE layer of 8-bit experts: against the dequantised values in 64 bits."""
    import sonicmoe
    from sonicmoe.functional import int8

    T, K, E, H, I = 300, 2, 8, 128, 64
    g = torch.Generator().manual_seed(6)
    x = torch.randn(T, H, generator=g).cuda()
    idx = torch.randn(T, E, generator=g).topk(K, dim=1).indices.cuda()
    idx[5] = -1
    s = torch.rand(T, K, generator=g).cuda()
    w1, w2 = torch.randn(E, 2 * I, H, generator=g).cuda() / H ** 0.5, torch.randn(E, H, I, generator=g).cuda() / I ** 0.5
    (w1q, w1s), (w2q, w2s) = int8.quantize_rows(w1), int8.quantize_rows(w2)
    p = sonicmoe.token_permutation(idx, E, 16)
    y1 = int8.int8_grouped_linear(x, w1q, w1s, p.expert_frequency_offset, p.x_gather_idx, p.expert_frequency, activation_type="swiglu")
    y2 = int8.int8_grouped_linear(y1, w2q, w2s, p.expert_frequency_offset, expert_frequency=p.expert_frequency)
    o = sonicmoe.unpermute_tokens(y2, p, s)
    assert not o[5].any()
    d1, d2 = w1q.double() * w1s.double().unsqueeze(-1), w2q.double() * w2s.double().unsqueeze(-1)
    safe = idx.clamp_min(0)
    h = torch.einsum("th,tknh->tkn", x.double(), d1[safe])
    a = h[..., 0::2] * torch.sigmoid(h[..., 0::2]) * h[..., 1::2]
    want = (torch.einsum("tki,tkni->tkn", a, d2[safe]) * (s.double() * (idx >= 0)).unsqueeze(-1)).sum(1)
    # one quantised value is off by half a scale, 1 / 254 of its row's largest (about 3.5 of its rms, independent of one
    # another): 0.8 % of the sum of such products per quantised operand, rms; two of them, and the first's goes through SwiGLU
    assert ((o.double() - want).norm() / want.norm()).item() < 3 * 0.008


@pytest.mark.parametrize("T,H,I,E,K,activation,biased", [
    (0, 128, 64, 8, 2, "swiglu", False), (1, 256, 128, 32, 4, "swiglu", False), (77, 192, 64, 8, 1, "gelu", True),
    (1000, 512, 256, 64, 8, "swiglu", False), (513, 136, 72, 6, 3, "relu_sq", True), (3000, 256, 128, 4, 2, "silu", False)])
def test_layer(built_library, T, H, I, E, K, activation, biased):
    """The layer against its steps in 64 bits, with the routing of the logits that it returns."""
    from sonicmoe.enums import ActivationType
    from sonicmoe.functional import int8, moe_TC_softmax_topk_layer

    g = torch.Generator().manual_seed(8)
    n1 = 2 * I if activation in GATED else I
    x = torch.randn(T, H, generator=g).bfloat16().cuda()
    router = (torch.randn(E, H, generator=g) * 0.1).bfloat16().cuda()
    w1 = (torch.randn(E, n1, H, generator=g) * 2 / H ** 0.5).bfloat16().cuda()
    w2 = (torch.randn(E, H, I, generator=g) / I ** 0.5).bfloat16().cuda()
    b1, b2 = (torch.randn(E, n, generator=g).bfloat16().cuda() if biased else None for n in (n1, H))
    experts = int8.quantize_experts(w1.permute(1, 2, 0), b1, w2.permute(1, 2, 0), b2)
    o, logits, frequency = int8.moe_int8_softmax_topk_layer(x, router, experts, K, ActivationType(activation))
    assert o.shape == x.shape and o.dtype == torch.bfloat16 and logits.shape == (T, E) and int(frequency.sum()) == T * K
    if T == 0:
        return
    top, idx = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    scores, idx = torch.softmax(top[:, :K].double(), dim=1), idx[:, :K]
    assert torch.equal(frequency.long().cpu(), torch.bincount(idx.reshape(-1).cpu(), minlength=E))
    d1 = experts.w1q.double() * experts.w1_scale.double().unsqueeze(-1)
    d2 = experts.w2q.double() * experts.w2_scale.double().unsqueeze(-1)
    q, s = exact_quantize(x)
    xd = q * s.double().unsqueeze(-1)
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for e in range(E):
        t, k = torch.nonzero(idx == e, as_tuple=True)
        z = xd[t] @ d1[e].t() + (0 if b1 is None else b1[e].double())
        y = act_value(activation, z[:, 0::2])[0] * z[:, 1::2] if activation in GATED else act_value(activation, z)[0]
        q, s = exact_quantize(y.bfloat16())
        y = (q * s.double().unsqueeze(-1)) @ d2[e].t() + (0 if b2 is None else b2[e].double())
        want.index_add_(0, t, y * scores[t, k].unsqueeze(1))
    # bf16 roundings of the two projections' results and of the sum, at most 2^-8 each, rms a third of that; a value of y1 that
    # is rounded to the neighbouring bf16 may be quantised to the neighbouring step: 2^-8 of it again
    assert ((o.double() - want).norm() / want.norm()).item() < 4 * 2.0 ** -8 / 3 ** 0.5
    bf16 = moe_TC_softmax_topk_layer(x, router, w1.permute(1, 2, 0), b1, w2.permute(1, 2, 0), b2, K, 0, ActivationType(activation),
                                     True)[0] if H % 64 == 0 and I % 64 == 0 and n1 % 128 == 0 else None
    if bf16 is not None:  # 8-bit operands: 0.8 % rms each, three of them and the activation's slope
        assert ((o.double() - bf16.double()).norm() / bf16.double().norm()).item() < 0.06


def test_quantising_a_dual_tensor_is_refused(built_library):
    from torch.autograd import forward_ad

    from sonicmoe.functional import int8

    w = torch.randn(2, 6, 16, device="cuda")
    with forward_ad.dual_level():
        for call in (int8.quantize_rows, lambda v: int8.quantize_experts(v.permute(1, 2, 0), None, v.permute(2, 1, 0), None)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(forward_ad.make_dual(w, torch.ones_like(w)))
        assert int8.quantize_rows(w)[0].shape == w.shape


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("N,K", [(200, 520), (1030, 144), (9602, 256)])
def test_the_same_bits_from_every_kernel(built_library, activation, N, K):
    """A row's result does not depend on the rows beside it, on x being quantised before, on the way there or inside, or on an expert's
    other rows: dot products of eight and of two rows, tiles of every kind, with scales and biases of any value."""
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(N + K)
    R = 600
    x = torch.randn(R, K, generator=g).bfloat16().cuda()
    wq, ws = int8.quantize_rows((torch.randn(N, K, generator=g) * torch.rand(N, 1, generator=g)).cuda())
    bias = torch.randn(N, generator=g).cuda()
    q, xs = int8.quantize_rows(x)
    for b in (bias, None):
        call = dict(bias=b, activation_type=activation, out_dtype=torch.float32)
        want = int8.int8_linear(q, wq, ws, x_scale=xs, **call)
        for M in (1, 2, 3, 4, 8, 9, 31, 33, 64, 65, 100, 128, 129, 200, 224, 225, 300, 512):
            for first in (0, R - M):
                rows = slice(first, first + M)
                assert torch.equal(int8.int8_linear(q[rows], wq, ws, x_scale=xs[rows], **call), want[rows]), M
                assert torch.equal(int8.int8_linear(x[rows], wq, ws, **call), want[rows]), M
        many = wq.unsqueeze(0).expand(6, N, K).contiguous() if K % 16 == 0 else int8_copies(wq, 6)
        scales, biases = ws.expand(6, N).contiguous(), None if b is None else b.expand(6, N).contiguous()
        for off in ([0, 0, 3, 5, 9, 20, 31], [0, 5, 45, 190, 420, 599, 600], [0, 0, 0, 600, 600, 600, 600]):
            take = torch.arange(R, dtype=torch.int32, device="cuda")[: off[-1]]
            y = int8.int8_grouped_linear(q, many, scales, torch.tensor(off, dtype=torch.int32, device="cuda"), take, x_scale=xs,
                                         bias=biases, activation_type=activation, out_dtype=torch.float32)
            assert torch.equal(y, want[: off[-1]]), off


def int8_copies(wq, n):
    """n experts with the same 8-bit rows, laid out as quantize_rows does."""
    N, K = wq.shape
    out = torch.zeros(n, N, (K + 15) // 16 * 16, dtype=torch.int8, device=wq.device)[..., :K]
    return out.copy_(wq)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 40, 8192), (1, 33, 18001), (1, 24, 18432), (2, 72, 4097), (2, 40, 7168), (3, 40, 3400), (1, 200, 4112)])
def test_few_long_rows_quantised_on_the_way(built_library, dtype, M, N, K):
    """More columns than the kernel has in shared memory at a time: the same bits as from rows quantised before."""
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(K)
    x = (torch.randn(M, K, generator=g) * torch.rand(M, 1, generator=g)).to(dtype).cuda()
    x[0, -1] = 9  # the largest value is one of the last
    wq, ws = int8.quantize_rows(torch.randn(N, K, generator=g).cuda())
    bias = torch.randn(N, generator=g).cuda()
    q, xs = int8.quantize_rows(x)
    y = int8.int8_linear(x, wq, ws, bias=bias, out_dtype=torch.float32)
    assert torch.equal(y, int8.int8_linear(q, wq, ws, x_scale=xs, bias=bias, out_dtype=torch.float32))
    check(y, product(q, wq), xs[:, None], ws, bias, None)
    shifted = torch.zeros(M, K + 3, dtype=dtype, device="cuda")[:, 1 : K + 1].copy_(x)  # rows that start anywhere
    assert torch.equal(int8.int8_linear(shifted, wq, ws, bias=bias, out_dtype=torch.float32), y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,E,N,K", [(8, 5, 64, 9001), (24, 13, 40, 9001), (16, 40, 32, 18432), (5, 3, 32, 18433)])
def test_few_long_rows_of_experts(built_library, dtype, rows, E, N, K):
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(rows)
    wq, ws = int8.quantize_rows(torch.randn(E, N, K, generator=g).cuda())
    x = torch.randn(7, K, generator=g).to(dtype).cuda()
    take = torch.randint(-1, 7, (rows,), generator=g, dtype=torch.int32).cuda()
    first = torch.randint(0, rows + 1, (E - 1,), generator=g).sort().values.tolist()
    off = torch.tensor([0, *first, rows], dtype=torch.int32, device="cuda")
    q, xs = int8.quantize_rows(x)
    y = int8.int8_grouped_linear(x, wq, ws, off, take, out_dtype=torch.float32)
    assert torch.equal(y, int8.int8_grouped_linear(q, wq, ws, off, take, x_scale=xs, out_dtype=torch.float32))
    for e in range(E):
        r = torch.arange(int(off[e]), int(off[e + 1]), device="cuda")
        if len(r):
            src, none = take[r].long().clamp_min(0), take[r] < 0
            acc = product(q[src], wq[e])
            acc[none] = 0
            check(y[r], acc, xs[src, None], ws[e], None, None)


@pytest.mark.parametrize("N,K", [(8448, 4096), (4096, 8200)])
def test_few_rows_of_large_weights(built_library, N, K):
    """Above 32 MB of weights the kernels change at other numbers of rows."""
    from sonicmoe.functional import int8

    g = torch.Generator().manual_seed(N)
    wq, ws = int8.quantize_rows(torch.randn(N, K, generator=g).cuda())
    x = torch.randn(9, K, generator=g).bfloat16().cuda()
    q, xs = int8.quantize_rows(x)
    want = int8.int8_linear(q, wq, ws, x_scale=xs, out_dtype=torch.float32)
    check(want, product(q, wq), xs[:, None], ws, None, None)
    for M in range(1, 9):
        assert torch.equal(int8.int8_linear(x[:M], wq, ws, out_dtype=torch.float32), want[:M]), M
        assert torch.equal(int8.int8_linear(q[:M], wq, ws, x_scale=xs[:M], out_dtype=torch.float32), want[:M]), M


def test_captured_by_a_thread_of_its_own(built_library):
    """The first call of a thread is part of a capture there; so is the first one of the bf16 layer."""
    import threading

    import sonicmoe
    from sonicmoe.functional import int8

    x = torch.randn(100, 256, device="cuda")
    wq, ws = int8.quantize_rows(torch.randn(64, 256, device="cuda"))
    m = sonicmoe.MoE(32, 2, 128, 64, sonicmoe.ActivationType.SWIGLU, False, 0.05).cuda().bfloat16()
    t = torch.randn(3000, 128, device="cuda").bfloat16()

    def calls():
        with torch.no_grad():
            return int8.int8_linear(x, wq, ws), m(t, is_inference_mode=True)[0]

    want, got = calls(), []  # (kernels are loaded and workspaces of the library exist)
    torch.cuda.synchronize()

    def run():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            out = calls()
        graph.replay()
        torch.cuda.synchronize()
        got.extend(v.clone() for v in out)

    thread = threading.Thread(target=run)
    thread.start()
    thread.join()
    assert len(got) == 2 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows(built_library):
    """No tokens, and tokens none of which is gathered."""
    from sonicmoe.functional import int8

    E, N, K = 3, 40, 64
    wq, ws = int8.quantize_rows(torch.randn(E, N, K, device="cuda"))
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    for dtype in TYPES:
        x = torch.randn(30, K, device="cuda").to(dtype)
        q, xs = int8.quantize_rows(x)
        for activation, width in ((None, N), ("swiglu", N // 2)):
            call = dict(activation_type=activation)
            for y in (int8.int8_grouped_linear(x, wq, ws, off, none, **call), int8.int8_grouped_linear(x[:0], wq, ws, off, none, **call),
                      int8.int8_grouped_linear(x[:0], wq, ws, off, **call), int8.int8_linear(x[:0], wq[0], ws[0], **call),
                      int8.int8_grouped_linear(q, wq, ws, off, none, x_scale=xs, out_dtype=dtype, **call),
                      int8.int8_linear(q[:0], wq[0], ws[0], x_scale=xs[:0], out_dtype=dtype, **call)):
                assert y.shape == (0, width) and y.dtype == dtype and y.is_cuda
    with pytest.raises(ValueError, match="no rows to gather"):
        int8.int8_grouped_linear(x[:0], wq, ws, off, torch.zeros(2, dtype=torch.int32, device="cuda"))
