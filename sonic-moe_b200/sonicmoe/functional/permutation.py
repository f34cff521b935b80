"""Tokens sorted by expert and back: for experts that are not this library's own GEMMs (other layers, adapters, 8-bit
products), which take their rows expert by expert.

    p = token_permutation(topk_indices, E)           # stable sort of the (token, slot) pairs by expert
    rows = permute_tokens(x, p)                      # rows[r] = x[token of row r]
    y = experts(rows, p.expert_frequency_offset)     # expert e has rows [offset[e], offset[e] + expert_frequency[e])
    o = unpermute_tokens(y, p, scores)               # o[t] = sum over k of scores[t, k] y[row of pair (t, k)]

Both directions have gradients (the sums over a token's rows, the rows' dot products for the scores).  A pair whose expert is
outside [0, E) (-1, say: a token beyond an expert's capacity, a padding token) is dropped: it has no row, adds nothing, and its
score is not read.  A pair may also be dropped after the sort, by -1 in ``s_reverse_scatter_idx``.  ``align`` starts every
expert's rows at a multiple of it; rows without a pair are zeros in `permute_tokens`, ignored by `unpermute_tokens` whatever they
hold, and get zero gradients.

The gradients have gradients of their own, any number of times, where there are no scores; with scores that is refused.

fp32, bf16 and fp16 rows of any width; sums in fp32 in the order of k, rounded once: the same bits every time.  The number of
rows follows from the shapes alone, so nothing here waits for the device and all of it can be captured in a graph.  (For a captured
backward pass autograd itself asks that no graph recorded outside the capture still holds the same leaves.)
The reference has no such operators: its GEMMs gather and scatter (sonicmoe/functional/__init__.py:19-82 makes the indices).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._lib import check, lib, ptr, stream_ptr

_ROW_TYPES = {torch.float32: _lib.SMOE_F32, torch.bfloat16: _lib.SMOE_BF16, torch.float16: _lib.SMOE_F16}
_MAX_EXPERTS = 4096


@dataclass
class TokenPermutation:
    """Index vectors of one routing decision (int32, contiguous, on the tokens' device; the names are those of `Route`)."""

    expert_frequency: torch.Tensor         # (E,)   pairs of each expert
    expert_frequency_offset: torch.Tensor  # (E+1,) first row of each expert, multiples of `align`; [E]: end of the last
    x_gather_idx: torch.Tensor             # (rows,) token of each row, -1: none
    s_scatter_idx: torch.Tensor            # (rows,) flat (token, slot) pair of each row, -1: none
    s_reverse_scatter_idx: torch.Tensor    # (T, K) row of each pair, -1: dropped
    align: int = 1

    @property
    def num_rows(self) -> int:
        return self.s_scatter_idx.numel()


def token_permutation(topk_indices: torch.Tensor, E: int, align: int = 1) -> TokenPermutation:
    """The stable sort by expert of the pairs of ``topk_indices`` (T, K), int32 or int64: pairs of one expert stay in the order
    of (token, slot).  The number of rows is T K, or with ``align`` > 1 what every load fits into."""
    if topk_indices.dim() != 2:
        raise ValueError(f"topk_indices has to be (T, K), got {tuple(topk_indices.shape)}")
    if topk_indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"topk_indices has to be int32 or int64, got {topk_indices.dtype}")
    T, K = topk_indices.shape
    n = T * K
    if not 0 < E <= _MAX_EXPERTS or align <= 0 or K == 0:
        raise ValueError(f"1 <= E <= {_MAX_EXPERTS}, 1 <= K and 1 <= align are needed, got E {E}, K {K}, align {align}")
    rows = lib.smoe_token_permutation_rows(n, E, align)
    if rows + E * align >= 2 ** 31 or n >= 2 ** 31 - 2 ** 16:
        raise ValueError(f"{n} pairs of {E} experts aligned to {align} do not fit into 32-bit row numbers")
    _lib.require_cuda(topk_indices, "topk_indices")
    idx = topk_indices.detach().contiguous()
    dev = idx.device
    with _lib.on_device(dev):
        # tensors in their own right: views of one buffer would share the count of in-place changes that autograd looks at
        freq, off, gather, scatter, reverse = torch.empty(
            2 * E + 1 + 2 * rows + n, dtype=torch.int32, device=dev).unsafe_split_with_sizes((E, E + 1, rows, rows, n))
        ws = lib.smoe_token_permutation_workspace_bytes(n, E)
        ws = _lib.workspace(ws, dev) if ws else None
        check(lib.smoe_token_permutation(
            idx.data_ptr(), _lib.dtype_code(idx.dtype), T, K, E, align, freq.data_ptr(), off.data_ptr(), gather.data_ptr(),
            scatter.data_ptr(), reverse.data_ptr(), ptr(ws), stream_ptr(dev)), "token_permutation")
    return TokenPermutation(freq, off, gather, scatter, reverse.view(T, K), align)


def _check_permutation(pair: torch.Tensor, row: torch.Tensor, dev: torch.device) -> None:
    if pair.dim() != 2 or row.dim() != 1 or pair.shape[1] == 0:
        raise ValueError("a permutation's s_reverse_scatter_idx is (T, K) and its s_scatter_idx (rows,)")
    if not (pair.dtype == row.dtype == torch.int32 and pair.device == row.device == dev and pair.is_contiguous() and row.is_contiguous()):
        raise ValueError(f"a permutation's index vectors are contiguous int32 tensors on {dev}")


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """A 2D tensor of a known type whose rows are contiguous (their distance may be anything)."""
    if t.dim() != 2:
        raise ValueError(f"{name} has to be 2-dimensional, got {tuple(t.shape)}")
    if t.dtype not in _ROW_TYPES:
        raise TypeError(f"{name} has to be fp32, bf16 or fp16, got {t.dtype}")
    if t.shape[1] == 0:
        raise ValueError(f"{name} has rows of no values")
    return t if t.stride(1) == 1 else t.contiguous()


def _spread(x, pair, row, scores):
    x = _rows(x, "x")
    (T, K), R, H, dev = pair.shape, row.numel(), x.shape[1], x.device
    with _lib.on_device(dev):
        rows = x.new_empty((R, H))
        check(lib.smoe_permute_rows(
            x.data_ptr(), x.stride(0), rows.data_ptr(), _ROW_TYPES[x.dtype], ptr(scores),
            0 if scores is None else _ROW_TYPES[scores.dtype], pair.data_ptr(), row.data_ptr(), T, K, H, R, stream_ptr(dev)),
            "permute_rows")
    return rows


def _collect(rows, pair, scores):
    rows = _rows(rows, "rows")
    (T, K), (R, H), dev = pair.shape, rows.shape, rows.device
    with _lib.on_device(dev):
        out = rows.new_empty((T, H))
        check(lib.smoe_unpermute_rows(
            rows.data_ptr(), rows.stride(0), out.data_ptr(), _ROW_TYPES[rows.dtype], ptr(scores),
            0 if scores is None else _ROW_TYPES[scores.dtype], pair.data_ptr(), T, K, H, R, stream_ptr(dev)), "unpermute_rows")
    return out


class _FirstDerivative(torch.autograd.Function):
    """A gradient as it is; its own derivative, by what it was computed from, is refused where one is asked for."""

    @staticmethod
    def forward(ctx, grad, *of):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise NotImplementedError("unpermute_tokens has first derivatives only where there are scores")


# Both keep the index vectors themselves: the fields of a permutation may be replaced before the backward pass.  Gradients are recorded
# there where the caller wants to differentiate them again: without scores each function's gradient is the other one.  What may have
# a forward-mode tangent goes by the functions too, here and below, which refuse it; the kernels alone would lose it.
class _Permute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pair, row):
        ctx.save_for_backward(pair, row)
        return _spread(x, pair, row, None)

    @staticmethod
    def backward(ctx, drows):
        pair, row = ctx.saved_tensors
        again = torch.is_grad_enabled() or forward_ad._current_level >= 0
        return _Unpermute.apply(drows, pair, row, None) if again else _collect(drows, pair, None), None, None


class _Unpermute(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, pair, row, scores):
        ctx.save_for_backward(pair, row, scores, rows if scores is not None and ctx.needs_input_grad[3] else None)
        return _collect(rows, pair, scores)

    @staticmethod
    def backward(ctx, dout):
        pair, row, scores, rows = ctx.saved_tensors
        again = torch.is_grad_enabled() or forward_ad._current_level >= 0
        if scores is None:
            return _Permute.apply(dout, pair, row) if again else _spread(dout, pair, row, None), None, None, None
        if rows is None:
            drows = _spread(dout, pair, row, scores)
            return _FirstDerivative.apply(drows, dout, scores) if again else drows, None, None, None
        g, y = _rows(dout, "dout"), _rows(rows, "rows")
        (T, K), (R, H), dev = pair.shape, y.shape, y.device
        with _lib.on_device(dev):
            drows = y.new_empty((R, H))
            dscores = torch.empty_like(scores)
            check(lib.smoe_unpermute_rows_backward(
                g.data_ptr(), g.stride(0), y.data_ptr(), y.stride(0), drows.data_ptr(), _ROW_TYPES[y.dtype],
                scores.data_ptr(), dscores.data_ptr(), _ROW_TYPES[scores.dtype], pair.data_ptr(), row.data_ptr(), T, K, H, R,
                stream_ptr(dev)), "unpermute_rows_backward")
        if again:
            drows, dscores = _FirstDerivative.apply(drows, dout, scores), _FirstDerivative.apply(dscores, dout, rows)
        return drows, None, None, dscores


def permute_tokens(x: torch.Tensor, permutation: TokenPermutation) -> torch.Tensor:
    """rows (permutation.num_rows, H): x[token] of every row's pair, zeros in rows without one.  x (T, H); the gradient of x is
    the sum of its tokens' rows."""
    _lib.require_cuda(x, "x")
    pair, row = permutation.s_reverse_scatter_idx, permutation.s_scatter_idx
    _check_permutation(pair, row, x.device)
    if x.dim() != 2 or x.shape[0] != pair.shape[0]:
        raise ValueError(f"x has to be ({pair.shape[0]}, H), got {tuple(x.shape)}")
    if torch.is_grad_enabled() and x.requires_grad or forward_ad._current_level >= 0:
        return _Permute.apply(x, pair, row)
    return _spread(x, pair, row, None)


def unpermute_tokens(rows: torch.Tensor, permutation: TokenPermutation, scores: torch.Tensor | None = None) -> torch.Tensor:
    """out (T, H): the sum over each token's pairs of score * row (``scores`` (T, K) fp32, bf16 or fp16; None: 1).  Gradients flow
    to rows and scores."""
    _lib.require_cuda(rows, "rows")
    pair, row = permutation.s_reverse_scatter_idx, permutation.s_scatter_idx
    _check_permutation(pair, row, rows.device)
    if rows.dim() != 2 or rows.shape[0] != row.shape[0]:
        raise ValueError(f"rows has to be ({row.shape[0]}, H), got {tuple(rows.shape)}")
    if scores is not None:
        if scores.shape != pair.shape or scores.device != rows.device:
            raise ValueError(f"scores has to be {tuple(pair.shape)} on {rows.device}, got "
                             f"{tuple(scores.shape)} on {scores.device}")
        if scores.dtype not in _ROW_TYPES:
            raise TypeError(f"scores has to be fp32, bf16 or fp16, got {scores.dtype}")
        scores = scores.contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or scores is not None and scores.requires_grad) or forward_ad._current_level >= 0:
        return _Unpermute.apply(rows, pair, row, scores)
    return _collect(rows, pair, scores)
