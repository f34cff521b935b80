"""The adapters' argument checks, which come before anything is launched (no GPU; the addresses here belong to nothing)."""

import pytest
import torch


def test_refusals(built_library):
    from sonicmoe._lib import lib

    at = 4096

    def call(x=at, ld=64, a=at, b=at, scale=None, base=None, base_ld=0, out=at, out_ld=32, dtype=1, off=at, count=at, gather=at, reverse=at, T=5000,
             rows=5120, H=64, N=32, n=4, r=8, align=32, status=None):
        return lib.smoe_adapter_linear(x, ld, a, b, scale, base, base_ld, out, out_ld, dtype, off, count, gather, reverse, T, rows, H, N, n, r, align, status, None)

    assert call(dtype=0) == call(dtype=2) == -6
    assert call(T=-1) == call(rows=-1) == call(H=0) == call(N=0) == call(n=0) == call(n=4097) == call(r=0) == call(r=129) == -1
    assert call(align=0) == call(align=8) == call(align=-16) == call(align=40) == call(ld=-1) == call(out_ld=31) == call(base=at, base_ld=-1) == -1
    assert call(H=2 ** 28 + 1) == call(N=2 ** 28 + 1, out_ld=2 ** 30) == call(rows=2 ** 31 - 2 ** 15) == call(T=2 ** 31 - 2 ** 15) == -1
    assert call(x=None) == call(a=None) == call(b=None) == call(out=None) == call(off=None) == call(count=None) == call(gather=None) == call(reverse=None) == -1
    assert call(x=at + 1) == call(a=at + 1) == call(b=at + 1) == call(out=at + 1) == call(base=at + 1) == -2
    assert call(scale=at + 2) == call(off=at + 2) == call(count=at + 2) == call(gather=at + 2) == call(reverse=at + 2) == call(status=at + 2) == -2
    assert call(T=0) == 0


def test_python_refusals(built_library):
    import sonicmoe
    from sonicmoe import SonicMoEError

    x, a, b = (torch.zeros(s, dtype=torch.bfloat16) for s in ((4, 64), (3, 8, 64), (3, 32, 8)))
    p = sonicmoe.TokenPermutation(*[torch.zeros(n, dtype=torch.int32) for n in (3, 4, 64, 64)], torch.zeros(4, 1, dtype=torch.int32), 16)
    with pytest.raises(SonicMoEError, match="no CPU path"):
        sonicmoe.adapter_linear(x, a, b, p)
    for bad in ((x[0], a, b), (x, a[0], b), (x, a, b[0])):
        with pytest.raises(ValueError, match="has to be"):
            sonicmoe.adapter_linear(*bad, p)
    for bad in ((x[:, :32], a, b), (x, a[:2], b), (x, a[:, :4], b)):
        with pytest.raises(ValueError, match="inconsistent"):
            sonicmoe.adapter_linear(*bad, p)
    for bad in ((x.float(), a.float(), b.float()), (x.half(), a, b), (x, a, b.half())):
        with pytest.raises(TypeError, match="bf16 or fp16"):
            sonicmoe.adapter_linear(*bad, p)
    wide = torch.zeros(3, 129, 64, dtype=torch.bfloat16), torch.zeros(3, 32, 129, dtype=torch.bfloat16)
    for bad in (wide, (a[:, :0], b[:, :, :0]), (a[:0], b[:0]), (a, b[:, :0])):
        with pytest.raises(ValueError, match="are needed"):
            sonicmoe.adapter_linear(x, *bad, p)
    idx = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="has to be"):
        sonicmoe.adapter_permutation(idx[None], 3)
    for n in (0, 4097):
        with pytest.raises(ValueError, match="are needed"):
            sonicmoe.adapter_permutation(idx, n)
    with pytest.raises(TypeError, match="int32 or int64"):
        sonicmoe.adapter_permutation(idx.float(), 3)
    with pytest.raises(SonicMoEError, match="no CPU path"):
        sonicmoe.adapter_permutation(idx, 3)


def test_rows_that_share_memory(built_library):
    from sonicmoe.functional.adapters import _meets_other_rows

    flat = torch.zeros(4000, dtype=torch.bfloat16)
    wide = flat.view(40, 100)

    def brute(x, out):
        at = lambda t: (t.data_ptr() - flat.data_ptr()) // 2
        rows = lambda t: [set(range(at(t[i]), at(t[i]) + t.shape[1])) for i in range(t.shape[0])]
        xs, outs = rows(x), rows(out)
        return any(xs[i] & outs[j] for i in range(len(xs)) for j in range(len(outs)) if i != j)

    for x, out in ((wide[:10, :60], wide[:10, 60:]), (wide[:10, 60:], wide[:10, :60]), (wide[:10, :60], wide[:10, 20:90]), (wide[:10], wide[:10]),
                   (wide[:10], wide[10:20]), (wide[:10], wide[9:19]), (wide[1:11, :30], wide[:10, 40:]), (wide[:1], wide[:1, :7]),
                   (wide[0].expand(10, 100), wide[:10]), (wide[0].expand(10, 100), wide[1:11]), (flat[5:1005].view(10, 100), wide[:10]),
                   (wide[5:15], wide[:5]), (flat[:500].view(5, 100), flat[500:1500].view(5, 200)), (flat[:500].view(5, 100), flat[400:1400].view(5, 200))):
        # (rows at different distances that only share their range are taken to meet)
        assert _meets_other_rows(x[:out.shape[0]], out) >= brute(x[:out.shape[0]], out)
        if x.stride(0) == out.stride(0):
            assert _meets_other_rows(x[:out.shape[0]], out) == brute(x[:out.shape[0]], out)
    assert not _meets_other_rows(wide[:10, :60], wide[:10, 60:]) and not _meets_other_rows(wide[1:11, :30], wide[:10, 40:])
