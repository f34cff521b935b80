"""What the sorted-token operators refuse, before anything is launched (no GPU; the addresses here belong to nothing)."""

import pytest
import torch


def test_sizes_of_the_sorted_layout(built_library):
    from sonicmoe._lib import lib

    rows = lib.smoe_token_permutation_rows
    assert rows(100, 8, 1) == 100 and rows(0, 8, 128) == 0 and rows(1, 8, 128) == 128
    assert rows(100, 8, 16) == (100 + 8 * 15) // 16 * 16 and rows(3, 8, 16) == 48
    assert rows(-1, 8, 1) == -1 and rows(1, 0, 1) == -1 and rows(1, 8, 0) == -1
    ws = lib.smoe_token_permutation_workspace_bytes
    assert ws(2048, 1024) == 0 and ws(2049, 8) > 0 and ws(8, 1025) >= 4 * 1025


def test_permutation_refusals(built_library):
    from sonicmoe._lib import lib

    at = 4096

    def call(dtype=2, T=5000, K=2, E=8, align=1, idx=at, ws=at, **bad):
        names = ("freq", "off", "gather", "scatter", "reverse")
        return lib.smoe_token_permutation(idx, dtype, T, K, E, align, *[bad.get(n, at) for n in names], ws, None)

    assert call(T=-1) == call(K=0) == call(E=0) == call(E=4097) == call(align=0) == call(align=-4) == -1
    assert call(T=2 ** 30, K=2) == -1 and call(T=2 ** 31 - 2 ** 16, K=1) == -1 and call(align=2 ** 29) == -1
    assert call(dtype=0) == call(dtype=4) == -6
    assert call(ws=None) == -7
    assert call(idx=None) == -1 and call(idx=at + 2) == -2 and call(dtype=3, idx=at + 4) == -2 and call(ws=at + 8) == -2
    for name in ("freq", "off", "gather", "scatter", "reverse"):
        assert call(**{name: None}) == -1 and call(**{name: at + 2}) == -2, name


def test_row_mover_refusals(built_library):
    from sonicmoe._lib import lib

    at = 4096

    def permute(dtype=1, x=at, rows=at, w=None, wt=0, rev=at, scat=at, T=4, K=2, H=8, R=8):
        return lib.smoe_permute_rows(x, H, rows, dtype, w, wt, rev, scat, T, K, H, R, None)

    def unpermute(dtype=1, rows=at, out=at, w=None, wt=0, rev=at, T=4, K=2, H=8, R=8):
        return lib.smoe_unpermute_rows(rows, H, out, dtype, w, wt, rev, T, K, H, R, None)

    def backward(dtype=1, dout=at, rows=at, drows=at, w=at, dw=at, wt=0, rev=at, scat=at, T=4, K=2, H=8, R=8):
        return lib.smoe_unpermute_rows_backward(dout, H, rows, H, drows, dtype, w, dw, wt, rev, scat, T, K, H, R, None)

    for call in (permute, unpermute, backward):
        assert call(dtype=2) == call(dtype=7) == call(w=at, wt=3) == -6
        assert call(T=-1) == call(K=0) == call(H=0) == call(R=-1) == call(R=2 ** 31) == call(T=2 ** 30, K=2) == call(H=2 ** 30) == -1
        assert call(rows=None) == call(rev=None) == -1
        assert call(rows=at + 1) == call(rev=at + 2) == call(w=at + 2, wt=0) == call(w=at + 1, wt=1) == call(dtype=0, rows=at + 2) == -2
    assert permute(x=None) == permute(scat=None) == unpermute(out=None) == backward(dout=None) == backward(dw=None) == backward(w=None) == -1
    assert backward(drows=None) == backward(scat=None) == -1 and backward(dw=at + 2) == backward(scat=at + 2) == -2
    assert permute(T=0, R=0) == 0 and unpermute(T=0) == 0 and backward(T=0, R=0) == 0


def test_python_refusals(built_library):
    import sonicmoe
    from sonicmoe import SonicMoEError

    idx = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(SonicMoEError, match="no CPU path"):
        sonicmoe.token_permutation(idx, 8)
    for bad in (idx[0], idx[None]):
        with pytest.raises(ValueError, match="has to be"):
            sonicmoe.token_permutation(bad, 8)
    with pytest.raises(TypeError, match="int32 or int64"):
        sonicmoe.token_permutation(idx.float(), 8)
    for E, align in ((0, 1), (4097, 1), (8, 0)):
        with pytest.raises(ValueError, match="are needed"):
            sonicmoe.token_permutation(idx, E, align)
    with pytest.raises(ValueError, match="32-bit"):
        sonicmoe.token_permutation(idx, 8, 2 ** 29)
    p = sonicmoe.TokenPermutation(*[torch.zeros(n, dtype=torch.int32) for n in (8, 9, 8, 8)], idx)
    assert p.num_rows == 8 and p.align == 1
    with pytest.raises(SonicMoEError, match="no CPU path"):
        sonicmoe.permute_tokens(torch.zeros(4, 16), p)
    with pytest.raises(SonicMoEError, match="no CPU path"):
        sonicmoe.unpermute_tokens(torch.zeros(8, 16), p)


def test_grids_past_the_limit_are_refused(built_library):
    """Broadcast rows (ld 0) and rows of one value allow for more blocks than a grid has, although all of it fits into memory."""
    from sonicmoe._lib import lib

    at, T, H = 4096, 2 ** 31 - 1, 2 ** 20
    # 2^31 rows of 2^18 pieces of 16 bytes are 2^41 blocks: zero in 32 bits
    assert lib.smoe_permute_rows(at, 0, at, 0, None, 0, at, at, T, 1, H, 64, None) == -1
    assert lib.smoe_permute_rows(at + 4, 0, at, 0, None, 0, at, at, T, 1, H + 1, 64, None) == -1
    assert lib.smoe_unpermute_rows(at, 0, at, 0, None, 0, at, T, 1, H, 64, None) == -1
    assert lib.smoe_unpermute_rows(at + 2, 0, at, 1, None, 0, at, T, 1, H + 1, 64, None) == -1
    # a block per token and one per 64 rows
    n = 2 ** 31 - 2 ** 16 - 1
    assert lib.smoe_unpermute_rows_backward(at, 1, at, 1, at, 1, at, at, 0, at, at, n, 1, 1, n, None) == -1
