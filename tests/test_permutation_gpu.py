"""Tokens sorted by expert and back against plain implementations in 64 bits, at the sizes, masks, strides and alignments where
the index arithmetic can go wrong.

Tolerances: an output is within half a step of its type (eps / 2 of its value) of the fp32 sum, and that within `terms` * 2^-24
of the sum of the terms' magnitudes, one rounding per product and addition.  Below its smallest normal value a type's steps no
longer shrink with the value: half a step is smallest_normal * eps / 2 there (fp16: 2^-14 * 2^-10 / 2 = 2^-25), the last term of
`half_step`."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype, value):
    f = torch.finfo(dtype)
    return f.eps / 2 * value.abs() + f.smallest_normal * f.eps / 2


def indices(T, K, E, dropped=0.0, dtype=torch.int32, seed=0):
    g = torch.Generator().manual_seed(seed + T + 7 * E)
    idx = torch.randint(0, E, (T, K), generator=g)  # repeated experts in a row are allowed
    out = torch.randint(0, 3, (T, K), generator=g)
    lost = torch.tensor([-1, E, -2 ** 31])[out]
    return torch.where(torch.rand(T, K, generator=g) < dropped, lost, idx).to(dtype)


def plain_permutation(idx, E, align):
    """One pair at a time."""
    T, K = idx.shape
    n = T * K
    rows = (n + min(E, n) * (align - 1)) // align * align
    flat = idx.reshape(-1).tolist()
    count, offset = [0] * E, [0]
    for e in flat:
        if 0 <= e < E:
            count[e] += 1
    for c in count:
        offset.append(offset[-1] + -(-c // align) * align)
    at, slot, row = offset[:-1], [-1] * rows, [-1] * n
    at = list(at)
    for p, e in enumerate(flat):
        if 0 <= e < E:
            slot[at[e]], row[p] = p, at[e]
            at[e] += 1
    token = [s // K if s >= 0 else -1 for s in slot]
    return dict(expert_frequency=count, expert_frequency_offset=offset, x_gather_idx=token, s_scatter_idx=slot,
                s_reverse_scatter_idx=row)


def check_permutation(p, idx, E, align):
    for name, want in plain_permutation(idx, E, align).items():
        got = getattr(p, name)
        assert got.dtype == torch.int32 and got.reshape(-1).tolist() == want, name


@pytest.mark.parametrize("T,K,E,align,dropped", [
    (0, 2, 4, 1, 0.0), (0, 2, 4, 16, 0.0), (1, 1, 1, 1, 0.0), (1, 8, 128, 1, 0.0), (1, 1, 5, 128, 0.0), (1, 3, 2, 4, 1.0),
    (33, 3, 7, 1, 0.2), (100, 2, 3, 64, 0.3), (1024, 8, 128, 1, 0.0), (1025, 8, 60, 16, 0.1), (8192, 1, 1024, 1, 0.0),
    (8192, 1, 1025, 3, 0.0), (8193, 1, 33, 1, 0.0), (5000, 4, 1, 8, 0.5), (30000, 3, 4096, 1, 0.1), (40000, 8, 256, 128, 0.05),
    (300, 7, 2000, 2, 1.0),
    (2049, 1, 7, 1, 0.0), (4097, 2, 128, 4, 0.2), (16385, 1, 1000, 1, 0.0), (10000, 5, 64, 16, 0.1), (65536, 1, 256, 1, 0.0),
    (65537, 1, 256, 8, 0.0)])
def test_permutation(built_library, T, K, E, align, dropped):
    import sonicmoe

    for dtype in (torch.int32, torch.int64):
        idx = indices(T, K, E, dropped, dtype)
        check_permutation(sonicmoe.token_permutation(idx.cuda(), E, align), idx, E, align)
    assert sonicmoe.token_permutation(idx.cuda(), E, align).num_rows % align == 0


def test_permutation_of_a_load_in_one_expert(built_library):
    import sonicmoe

    for T, K in ((4000, 2), (70000, 8)):  # one block, many
        idx = torch.full((T, K), 5)
        check_permutation(sonicmoe.token_permutation(idx.cuda(), 9, 32), idx, 9, 32)


def test_permutation_takes_strided_indices_and_ids_past_32_bits(built_library):
    import sonicmoe

    wide = indices(50, 6, 9, dtype=torch.int64)
    check_permutation(sonicmoe.token_permutation(wide.cuda()[:, 1:4], 9), wide[:, 1:4], 9, 1)
    wide[3, 1] = 2 ** 32 + 2  # not expert 2
    check_permutation(sonicmoe.token_permutation(wide.cuda(), 9), wide, 9, 1)


def source(rows, H, dtype, seed, pitch=0, offset=0):
    """(rows, H) on the device, `pitch` values longer per row in memory and `offset` values into its buffer."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.empty(offset + rows * (H + pitch), dtype=dtype, device="cuda")
    view = flat[offset:].view(rows, H + pitch)[:, :H]
    view.copy_(torch.randn(rows, H, generator=g))
    return view


#: widths and layouts: 32-byte, 16-byte, 4-byte and 2-byte pieces, one value, more than one round of a block
LAYOUTS = [(64, 0, 0), (512, 8, 0), (24, 0, 8), (1005, 0, 0), (1030, 0, 0), (17, 3, 1), (1, 0, 0), (4104, 0, 0), (9000, 2, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,pitch,offset", LAYOUTS)
def test_permute(built_library, dtype, H, pitch, offset):
    import sonicmoe

    T, K, E, align = 37, 3, 6, 8
    idx = indices(T, K, E, 0.2)
    p = sonicmoe.token_permutation(idx.cuda(), E, align)
    x = source(T, H, dtype, 1, pitch, offset)
    x[0, 0], x[1, -1] = float("nan"), float("inf")
    leaf = x.detach().requires_grad_(True)
    rows = sonicmoe.permute_tokens(leaf, p)
    token = p.x_gather_idx.long()
    want = torch.where((token >= 0).unsqueeze(1), x[token.clamp_min(0)], torch.zeros_like(x[:1]))
    assert torch.equal(rows.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0)) and torch.equal(rows.isnan(), want.isnan())

    drows = source(p.num_rows, H, dtype, 2, pitch, offset)
    drows[token < 0] = float("nan")  # gradients of rows without a pair go nowhere
    dx, = torch.autograd.grad(rows, leaf, drows)
    live = token >= 0
    exact = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, token[live], drows.double()[live])
    size = torch.zeros_like(exact).index_add_(0, token[live], drows.double().abs()[live])
    bound = half_step(dtype, exact) + 2 * (K + 1) * 2.0 ** -24 * size
    assert dx.dtype == dtype and bool(((dx.double() - exact).abs() <= bound).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,pitch,offset", LAYOUTS)
@pytest.mark.parametrize("K,score_type", [(1, torch.float32), (5, torch.bfloat16), (40, torch.float16), (8, None)])
def test_unpermute(built_library, dtype, H, pitch, offset, K, score_type):
    """More than 32 pairs of a token are the backward pass's second chunk; a token without any pair gets zeros."""
    import sonicmoe

    T, E, align = 21, 6, 4
    idx = indices(T, K, E, 0.25)
    idx[4] = -1
    p = sonicmoe.token_permutation(idx.cuda(), E, align)
    slot, token = p.s_scatter_idx.long(), p.x_gather_idx.long()
    live = slot >= 0
    y = source(p.num_rows, H, dtype, 3, pitch, offset)
    y[~live] = float("nan")
    y.requires_grad_(True)
    g = torch.Generator().manual_seed(4)
    scores = None
    weight = torch.ones(p.num_rows, dtype=torch.float64, device="cuda")
    if score_type is not None:
        scores = torch.rand(T, K, generator=g).to(score_type).cuda()
        scores[p.s_reverse_scatter_idx < 0] = float("nan")
        scores.requires_grad_(True)
        weight = scores.detach().double().reshape(-1)[slot.clamp_min(0)]
    out = sonicmoe.unpermute_tokens(y, p, scores)
    unit = 2.0 ** -24
    terms = (y.detach().double() * weight.unsqueeze(1))[live]
    exact = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, token[live], terms)
    size = torch.zeros_like(exact).index_add_(0, token[live], terms.abs())
    assert out.dtype == dtype
    assert bool(((out.double() - exact).abs() <= half_step(dtype, exact) + 2 * (K + 1) * unit * size).all())
    assert bool((out[4] == 0).all())

    dout = source(T, H, dtype, 5, pitch, offset)
    leaves = (y,) if scores is None else (y, scores)
    grads = torch.autograd.grad(out, leaves, dout)
    dy = torch.zeros(p.num_rows, H, dtype=torch.float64, device="cuda")
    dy[live] = (dout.double()[token.clamp_min(0)] * weight.unsqueeze(1))[live]
    assert bool(((grads[0].double() - dy).abs() <= half_step(dtype, dy) + 2 * unit * dy.abs()).all())
    if scores is not None:
        products = dout.double()[token.clamp_min(0)] * y.detach().double()
        want = torch.zeros(T * K, dtype=torch.float64, device="cuda")
        size = torch.zeros_like(want)
        want[slot[live]], size[slot[live]] = products[live].sum(1), products[live].abs().sum(1)
        deep = H / 32 + 48  # a thread's values, five steps over the lanes, the warps
        bound = half_step(score_type, want) + 2 * deep * unit * size
        assert grads[1].dtype == score_type and bool(((grads[1].double().reshape(-1) - want).abs() <= bound).all())


def test_gradients_against_differences(built_library):
    """Both operators are linear in each argument: a difference is exact but for its roundings."""
    import sonicmoe

    T, K, E, H = 50, 4, 5, 96
    p = sonicmoe.token_permutation(indices(T, K, E, 0.1).cuda(), E, 4)
    x, v = source(T, H, torch.float32, 1).requires_grad_(True), source(T, H, torch.float32, 2)
    c = source(p.num_rows, H, torch.float32, 3)
    dx, = torch.autograd.grad(sonicmoe.permute_tokens(x, p), x, c)
    moved = ((sonicmoe.permute_tokens(x + v, p) - sonicmoe.permute_tokens(x, p)).double() * c).sum()
    # every product is off by at most three roundings of values up to 8
    assert abs(moved - (dx.double() * v).sum()) <= p.num_rows * H * 8 * 2.0 ** -22
    y, s = source(p.num_rows, H, torch.float32, 4).requires_grad_(True), torch.rand(T, K, device="cuda", requires_grad=True)
    d, vs = source(T, H, torch.float32, 5), torch.rand(T, K, device="cuda")
    out = sonicmoe.unpermute_tokens(y, p, s)
    dy, ds = torch.autograd.grad(out, (y, s), d)
    by_rows = ((sonicmoe.unpermute_tokens(y + c, p, s) - out).double() * d).sum()
    by_scores = ((sonicmoe.unpermute_tokens(y, p, s + vs) - out).double() * d).sum()
    assert abs(by_rows - (dy.double() * c).sum()) <= p.num_rows * H * 8 * 2.0 ** -21
    assert abs(by_scores - (ds.double() * vs).sum()) <= p.num_rows * H * 8 * 2.0 ** -21


def test_sort_an_own_expert_and_combine(built_library):
    """The operators as they are used: sorted rows through one matrix per expert and back, against the sum written out."""
    import sonicmoe

    T, K, E, H, N = 200, 2, 4, 64, 32
    g = torch.Generator().manual_seed(0)
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)])
    x = torch.randn(T, H, generator=g).cuda().requires_grad_(True)
    w = torch.randn(E, N, H, generator=g).cuda().requires_grad_(True)
    s = torch.rand(T, K, generator=g).cuda().requires_grad_(True)
    p = sonicmoe.token_permutation(idx.cuda(), E)
    rows = sonicmoe.permute_tokens(x, p).split(p.expert_frequency.tolist())
    out = sonicmoe.unpermute_tokens(torch.cat([r @ w[e].t() for e, r in enumerate(rows)]), p, s)
    want = torch.einsum("tk,tknh,th->tn", s.double(), w.double()[idx.cuda()], x.double())
    # fp32 products of 64 terms of a few units each, and their gradients of up to 200 x 32
    assert (out.double() - want).abs().max() < 64 * 30 * 2.0 ** -22
    c = torch.randn(T, N, generator=g).cuda()
    for got, ref in zip(torch.autograd.grad(out, (x, w, s), c), torch.autograd.grad(want, (x, w, s), c.double())):
        assert (got.double() - ref).abs().max() < 200 * 64 * 10 * 2.0 ** -22


def test_broadcast_gradients(built_library):
    """A summed output's gradient is one value for all rows (strides of zero)."""
    import sonicmoe

    T, K, E, H = 30, 3, 4, 40
    p = sonicmoe.token_permutation(indices(T, K, E).cuda(), E)
    x = source(T, H, torch.bfloat16, 1).requires_grad_(True)
    rows = sonicmoe.permute_tokens(x, p)
    assert bool((torch.autograd.grad(rows.sum(), x)[0] == K).all())
    y = rows.detach().requires_grad_(True)
    s = torch.rand(T, K, device="cuda", requires_grad=True)
    row = torch.ones(1, H, dtype=torch.bfloat16, device="cuda").expand(T, H)
    dy, ds = torch.autograd.grad(sonicmoe.unpermute_tokens(y, p, s), (y, s), row)
    want = s.detach().reshape(-1)[p.s_scatter_idx.long()].bfloat16()
    assert torch.equal(dy, want.unsqueeze(1).expand(-1, H))


def test_fields_replaced_before_the_backward_pass(built_library):
    """Gradients belong to the permutation of the forward pass, whatever its object holds by then (here: fewer, other rows)."""
    import sonicmoe

    T, K, E, H = 50, 2, 4, 24
    p, q = (sonicmoe.token_permutation(indices(t, K, E, 0.2, seed=t).cuda(), E) for t in (T, 20))
    x = source(T, H, torch.float32, 1).requires_grad_(True)
    y = source(T * K, H, torch.float32, 2).requires_grad_(True)
    s = torch.rand(T, K, device="cuda", requires_grad=True)
    drows, dout = source(T * K, H, torch.float32, 3), source(T, H, torch.float32, 4)

    def outputs():
        return sonicmoe.permute_tokens(x, p), sonicmoe.unpermute_tokens(y, p), sonicmoe.unpermute_tokens(y, p, s)

    want = torch.autograd.grad(outputs(), (x, y, s), (drows, dout, dout))
    held = outputs()
    p.s_reverse_scatter_idx, p.s_scatter_idx = q.s_reverse_scatter_idx, q.s_scatter_idx
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(held, (x, y, s), (drows, dout, dout))))


def test_streams_graphs_and_repeats(built_library):
    """On a stream of its own, captured with its backward pass and replayed on new values: the same bits as outside."""
    import sonicmoe

    T, K, E, H = 3000, 4, 16, 264
    idx = [indices(T, K, E, 0.1, seed=s).cuda() for s in (1, 2)]
    xs = [source(T, H, torch.bfloat16, s) for s in (1, 2)]
    scores = torch.rand(T, K, device="cuda")
    dout = source(T, H, torch.bfloat16, 3)

    def step(idx, x):
        x, s = x.detach().requires_grad_(True), scores.detach().requires_grad_(True)
        p = sonicmoe.token_permutation(idx, E, 16)
        rows = sonicmoe.permute_tokens(x, p)
        out = sonicmoe.unpermute_tokens(rows * 2, p, s)
        return (out.detach(), p.s_scatter_idx, *torch.autograd.grad(out, (x, s), dout))

    want = [step(i, x) for i, x in zip(idx, xs)]
    again = step(idx[0], xs[0])
    assert all(torch.equal(a, b) for a, b in zip(want[0], again))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    static_idx, static_x = idx[0].clone(), xs[0].clone()
    with torch.cuda.stream(side):
        step(static_idx, static_x)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(static_idx, static_x)
    for i in (1, 0):
        static_idx.copy_(idx[i])
        static_x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))


def test_rows_past_32_bit_offsets(built_library):
    """More than 2^31 values: the last rows are where they belong."""
    import sonicmoe

    T, K, E, H = 131072 + 5, 4, 8, 4104
    idx = torch.arange(T * K, device="cuda").view(T, K) % E
    p = sonicmoe.token_permutation(idx, E)
    x = torch.arange(T, device="cuda", dtype=torch.float32).fmod(251).to(torch.bfloat16).unsqueeze(1).expand(T, H)
    rows = sonicmoe.permute_tokens(x, p)
    assert rows.numel() > 2 ** 31
    assert torch.equal(rows[:, 0], x[:, 0][p.x_gather_idx.long()]) and torch.equal(rows[:, -1], rows[:, 0])
    assert torch.equal(sonicmoe.unpermute_tokens(rows, p)[:, ::513], (x[:, ::513].float() * K).bfloat16())


def test_row_numbers_out_of_range_count_as_none(built_library):
    import sonicmoe

    T, K, E, H = 6, 2, 3, 32
    p = sonicmoe.token_permutation(indices(T, K, E).cuda(), E)
    broken = p.s_reverse_scatter_idx.clone()
    broken[0, 0], broken[1, 1], broken[2, 0] = p.num_rows, -5, 2 ** 31 - 1
    q = sonicmoe.TokenPermutation(p.expert_frequency, p.expert_frequency_offset, p.x_gather_idx, p.s_scatter_idx, broken)
    y = source(p.num_rows, H, torch.float32, 1)
    ok = (broken >= 0) & (broken < p.num_rows)
    want = torch.where(ok.unsqueeze(2), y[torch.where(ok, broken, 0).long()], torch.zeros(1, 1, 1, device="cuda")).sum(1)
    assert torch.allclose(sonicmoe.unpermute_tokens(y, q), want, rtol=0, atol=2.0 ** -20)


def test_forward_mode_derivatives_are_refused(built_library):
    """A dual tensor does not require a gradient: its tangent must not be lost without a word, under torch.no_grad() either."""
    from torch.autograd import forward_ad

    import sonicmoe

    T, K, E, H = 20, 2, 3, 16
    p = sonicmoe.token_permutation(indices(T, K, E).cuda(), E)
    x, y, s = source(T, H, torch.float32, 1), source(T * K, H, torch.float32, 2), torch.rand(T, K, device="cuda")
    plain = sonicmoe.permute_tokens(x, p), sonicmoe.unpermute_tokens(y, p, s)
    for enabled in (True, False):
        with forward_ad.dual_level(), torch.set_grad_enabled(enabled):
            dual = lambda v: forward_ad.make_dual(v, torch.ones_like(v))
            for call in (lambda: sonicmoe.permute_tokens(dual(x), p), lambda: sonicmoe.unpermute_tokens(dual(y), p),
                         lambda: sonicmoe.unpermute_tokens(dual(y), p, s), lambda: sonicmoe.unpermute_tokens(y, p, dual(s))):
                with pytest.raises(NotImplementedError, match="jvp"):
                    call()
            again = sonicmoe.permute_tokens(x, p), sonicmoe.unpermute_tokens(y, p, s)
            assert all(torch.equal(a, b) and not b.requires_grad for a, b in zip(plain, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,pitch,offset", LAYOUTS)
def test_pairs_dropped_after_the_sort(built_library, dtype, H, pitch, offset):
    """A pair taken out of s_reverse_scatter_idx alone (a capacity applied later): its row is zeros, in the gradients too, whatever
    the memory held before.  Every number here is a value of the inputs or a product of two: one rounding each."""
    import sonicmoe

    T, K, E, align = 37, 3, 6, 8
    p = sonicmoe.token_permutation(indices(T, K, E, 0.1).cuda(), E, align)
    kept = p.s_reverse_scatter_idx.clone()
    g = torch.Generator().manual_seed(9)
    lost = (torch.rand(T, K, generator=g) < 0.4).cuda()
    kept[lost] = torch.where(torch.rand(T, K, generator=g) < 0.5, -1, p.num_rows).int().cuda()[lost]
    q = sonicmoe.TokenPermutation(p.expert_frequency, p.expert_frequency_offset, p.x_gather_idx, p.s_scatter_idx, kept, align)
    has_row = (kept >= 0) & (kept < p.num_rows)
    rows = kept[has_row].long()
    token = torch.arange(T, device="cuda").unsqueeze(1).expand(T, K)[has_row]
    x, y, dout = source(T, H, dtype, 1, pitch, offset), source(p.num_rows, H, dtype, 2, pitch, offset), source(T, H, dtype, 3, pitch, offset)
    s = torch.rand(T, K, generator=g).cuda()

    def poisoned(call):
        junk = torch.full((p.num_rows, H), float("nan"), dtype=dtype, device="cuda")  # the block that the rows get
        del junk
        return call()

    def expected(values, weights=None):
        want = torch.zeros(p.num_rows, H, dtype=torch.float64, device="cuda")
        want[rows] = values.double()[token] * (1 if weights is None else weights.double()[has_row].unsqueeze(1))
        return want

    assert torch.equal(poisoned(lambda: sonicmoe.permute_tokens(x, q)).double(), expected(x))
    for scores, leaves in ((None, 1), (s, 1), (s, 2)):  # by the rows, by the rows with constant scores, by both
        rows_in = y.detach().requires_grad_(True)
        weights = None if scores is None else scores.clone().requires_grad_(leaves == 2)
        out = sonicmoe.unpermute_tokens(rows_in, q, weights)
        grads = poisoned(lambda: torch.autograd.grad(out, (rows_in, weights)[:leaves], dout))
        want = expected(dout, scores)
        assert bool(((grads[0].double() - want).abs() <= half_step(dtype, want) + 2.0 ** -24 * want.abs()).all())
        if leaves == 2:
            assert not grads[1][~has_row].any()


def test_the_largest_permutation(built_library):
    """As many pairs as there may be, and row numbers within a block's step of 2^31: rows behind the last pair are marked, and
    nothing else is written."""
    import sonicmoe

    n, E, align = 2 ** 31 - 2 ** 16 - 1, 512, 64
    if torch.cuda.mem_get_info()[0] < 6 * 4 * n:
        pytest.skip("needs 52 GB")
    for expert in (3, -1):
        p = sonicmoe.token_permutation(torch.full((n, 1), expert, dtype=torch.int32, device="cuda"), E, align)
        kept = n if expert >= 0 else 0
        assert p.num_rows > 2 ** 31 - 2 ** 15 - 1024 and int(p.expert_frequency.sum()) == kept
        assert p.expert_frequency_offset.tolist() == [0] * 4 + [-(-kept // align) * align] * (E - 3)
        for got in (p.s_scatter_idx, p.x_gather_idx):
            assert bool((got[kept:] == -1).all())
        count = torch.arange(n, dtype=torch.int32, device="cuda")
        for got in (p.s_scatter_idx[:kept], p.x_gather_idx[:kept], p.s_reverse_scatter_idx[:kept, 0]):
            assert torch.equal(got, count[:kept])
        assert bool((p.s_reverse_scatter_idx[kept:] == -1).all())
        del p, got, count


def test_fields_changed_in_place_before_the_backward_pass(built_library):
    """The counts and the other index vectors are the caller's to change; a change of those that the gradient takes is noticed."""
    import sonicmoe

    T, K, E, H = 30, 2, 4, 16
    x, drows = source(T, H, torch.float32, 1).requires_grad_(True), source(T * K, H, torch.float32, 2)
    s = torch.rand(T, K, device="cuda", requires_grad=True)
    dout = source(T, H, torch.float32, 3)
    for inference in (False, True):
        with torch.inference_mode(inference):
            p = sonicmoe.token_permutation(indices(T, K, E).cuda(), E)
        if inference:  # still what it was
            assert all(t.is_inference() for t in (p.expert_frequency, p.s_reverse_scatter_idx))
            continue
        want = torch.autograd.grad(sonicmoe.permute_tokens(x, p), x, drows)[0]
        rows = sonicmoe.permute_tokens(x, p)
        out = sonicmoe.unpermute_tokens(rows.detach(), p, s)
        first = p.expert_frequency_offset.clone()
        p.expert_frequency.add_(7)
        p.expert_frequency_offset.zero_()
        p.x_gather_idx.fill_(-1)
        assert torch.equal(torch.autograd.grad(rows, x, drows)[0], want) and bool(first.any())
        torch.autograd.grad(out, s, dout)
        rows = sonicmoe.permute_tokens(x, p)
        p.s_reverse_scatter_idx.copy_(p.s_reverse_scatter_idx.flip(0))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(rows, x, drows)


def test_gradients_of_gradients(built_library):
    """create_graph alone asks for nothing; without scores every order follows, with scores the second one is refused."""
    import sonicmoe

    T, K, E, H = 30, 3, 4, 16
    p = sonicmoe.token_permutation(indices(T, K, E, 0.2).cuda(), E, 4)
    token = p.x_gather_idx.long()
    live = token >= 0
    x, y = source(T, H, torch.float32, 1).requires_grad_(True), source(p.num_rows, H, torch.float32, 2).requires_grad_(True)
    s = torch.rand(T, K, device="cuda", requires_grad=True)

    def penalty(leaf, call):  # |d sum(out^3) / d leaf|^2 and its gradient
        first, = torch.autograd.grad(call(leaf).pow(3).sum(), leaf, create_graph=True)
        return torch.autograd.grad(first.pow(2).sum(), leaf)[0]

    def plain_permute(v):
        return torch.where(live.unsqueeze(1), v[token.clamp_min(0)], 0.0)

    def plain_unpermute(v):
        return torch.zeros(T, H, dtype=v.dtype, device="cuda").index_add(0, token[live], v[live])

    for leaf, own, plain in ((x, sonicmoe.permute_tokens, plain_permute), (y, sonicmoe.unpermute_tokens, plain_unpermute)):
        got, want = penalty(leaf, lambda v: own(v, p)), penalty(leaf.detach().double().requires_grad_(True), plain)
        # powers and sums of K values of up to 5: a few roundings of each, relative to the largest
        assert bool(((got.double() - want).abs() <= 64 * 2.0 ** -24 * want.abs().max()).all())

    dout = source(T, H, torch.float32, 3)
    for leaves in ((y, s), (y,)):
        out = sonicmoe.unpermute_tokens(y, p, s if len(leaves) == 2 else s.detach())
        want = torch.autograd.grad(out, leaves, dout, retain_graph=True)
        first = torch.autograd.grad(out, leaves, dout, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(first, want))
    out = sonicmoe.unpermute_tokens(y, p, s)
    d = dout.clone().requires_grad_(True)
    for i, by in ((0, s), (1, y), (0, d), (1, d)):  # the score is in the rows' gradient, the rows in the score's
        first = torch.autograd.grad(out, (y, s), d, create_graph=True)
        with pytest.raises(NotImplementedError, match="first derivatives only"):
            torch.autograd.grad(first[i].sum(), by)


def test_forward_mode_tangents_of_upstream_gradients_are_refused(built_library):
    from torch.autograd import forward_ad

    import sonicmoe

    T, K, E, H = 20, 2, 3, 16
    p = sonicmoe.token_permutation(indices(T, K, E).cuda(), E)
    x, y = source(T, H, torch.float32, 1).requires_grad_(True), source(T * K, H, torch.float32, 2).requires_grad_(True)
    s = torch.rand(T, K, device="cuda", requires_grad=True)
    for call, leaves in ((lambda: sonicmoe.permute_tokens(x, p), x), (lambda: sonicmoe.unpermute_tokens(y, p), y),
                         (lambda: sonicmoe.unpermute_tokens(y, p, s), (y, s)), (lambda: sonicmoe.unpermute_tokens(y, p, s.detach()), y)):
        out = call()
        g = torch.ones_like(out)
        want = torch.autograd.grad(out, leaves, g, retain_graph=True)
        with forward_ad.dual_level():
            assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, g, retain_graph=True), want))
            with pytest.raises(NotImplementedError, match="jvp"):
                torch.autograd.grad(out, leaves, forward_ad.make_dual(g, torch.ones_like(g)))


@pytest.mark.parametrize("T,K,E,align,dropped", [
    (2048, 1, 1024, 1, 0.0), (2047, 1, 1023, 3, 0.0), (1025, 1, 7, 1, 0.0), (256, 8, 128, 1, 0.2), (1024, 2, 8, 128, 0.0),
    (2048, 1, 1025, 1, 0.0), (2049, 1, 1024, 1, 0.1), (683, 3, 1000, 2, 1.0)])
def test_permutation_by_one_block_and_next_to_it(built_library, T, K, E, align, dropped):
    """Up to 2048 pairs of 1024 experts one block sorts, 32 pairs of a warp or up to 64 in turn; one pair or expert more is another form."""
    import sonicmoe

    for dtype in (torch.int32, torch.int64):
        idx = indices(T, K, E, dropped, dtype)
        check_permutation(sonicmoe.token_permutation(idx.cuda(), E, align), idx, E, align)
    idx = torch.full((T, K), E - 1, dtype=torch.int32)
    check_permutation(sonicmoe.token_permutation(idx.cuda(), E, align), idx, E, align)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,pitch,offset", LAYOUTS)
@pytest.mark.parametrize("score_type", TYPES)
def test_gradients_of_one_argument(built_library, dtype, H, pitch, offset, score_type):
    """By the rows where the scores are constant, a product with one rounding, and by the scores where the rows are."""
    import sonicmoe

    T, K, E, align = 21, 3, 6, 4
    p = sonicmoe.token_permutation(indices(T, K, E, 0.25).cuda(), E, align)
    slot, token = p.s_scatter_idx.long(), p.x_gather_idx.long()
    live = slot >= 0
    g = torch.Generator().manual_seed(11)
    y, dout = source(p.num_rows, H, dtype, 3, pitch, offset), source(T, H, dtype, 5, pitch, offset)
    scores = torch.rand(T, K, generator=g).to(score_type).cuda()
    rows = y.detach().requires_grad_(True)
    got, = torch.autograd.grad(sonicmoe.unpermute_tokens(rows, p, scores), rows, dout)
    want = torch.where(live.unsqueeze(1), dout.double()[token.clamp_min(0)] * scores.double().reshape(-1)[slot.clamp_min(0)].unsqueeze(1), 0.0)
    assert got.dtype == dtype and bool(((got.double() - want).abs() <= half_step(dtype, want) + 2.0 ** -24 * want.abs()).all())
    leaf = scores.detach().requires_grad_(True)
    got, = torch.autograd.grad(sonicmoe.unpermute_tokens(y, p, leaf), leaf, dout)
    both, = torch.autograd.grad(sonicmoe.unpermute_tokens(rows, p, leaf), leaf, dout)
    assert torch.equal(got, both) and got.dtype == score_type
