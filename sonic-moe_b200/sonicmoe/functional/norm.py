"""Root-mean-square norm of the rows in front of the layer, with the residual's addition, and as 8-bit rows for the 8-bit products.

    y, h = rms_norm(x, weight, residual=h)               # h = x + residual, the new residual stream; y = its norm
    o, aux = moe(y)

    r = rms_norm_quantize(x, weight, residual=h, keep_y=True)   # serving: r.q, r.scale, r.h and r.y
    z = int8.int8_linear(r.q, wq, w_scale, x_scale=r.scale)

y = h / sqrt(mean(h^2) + eps) * weight over the last dimension.  h is rounded to the type of x once, and y is the norm of that h; the
sum of squares and everything up to y's one rounding is fp32.  So are products of two of h, weight and the gradients: h weight is formed before
it is multiplied by the root.  Squares past fp32's range, of values above 1.8e19, make a row zeros; where eps is 0, or below 1e-38 (it is taken as
fp32 too), squares of values below 1e-19 lose bits, and rows of values below 1e-23 have none left: their root is infinite, and so are they.  The 8-bit
rows are those of the unrounded y: scale = amax / 127, values rounded half to even, as `int8.quantize_rows` makes them of fp32 rows (of bf16
and fp16 x by one multiply-add: a value within 1.6e-5 of a step of a border may go to the other side).  They are what `int8.int8_linear` and
`int8.moe_int8_softmax_topk_layer` take as x and x_q.

fp32, bf16 and fp16 rows of any width; weights of the same type or fp32.  `rms_norm` has gradients for x, the residual and the
weight (its sum over the rows is fp32, in the same order every time; the residual's gradient is that of x); second derivatives and forward-mode
ones are refused.  `rms_norm_quantize` has none.  For a captured backward pass autograd itself asks that no graph recorded outside
the capture still holds the same leaves.
The reference has no norm.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._lib import check, lib, ptr, stream_ptr
from .int8 import MAX_COLS
from .permutation import _ROW_TYPES

_MAX_WIDTH = 2 ** 28


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """(rows, H): a view where the rows lie at one distance from one another, a copy otherwise."""
    if t.dim() != 2:
        try:
            t = t.view(-1, t.shape[-1])
        except RuntimeError:
            t = t.reshape(-1, t.shape[-1])
    # (the distance of a single row means nothing, and that of broadcast rows is 0)
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _check(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None) -> None:
    if x.dim() < 1 or x.dtype not in _ROW_TYPES:
        raise TypeError(f"x has to be fp32, bf16 or fp16 rows, got {x.dtype} {tuple(x.shape)}")
    H = x.shape[-1]
    if not 0 < H <= _MAX_WIDTH:
        raise ValueError(f"rows of 1 to {_MAX_WIDTH} values are needed, got {H}")
    if not 0 <= eps < float("inf"):
        raise ValueError(f"eps has to be a finite number that is not negative, got {eps}")
    _lib.require_cuda(x, "x")
    if weight.shape != (H,) or weight.device != x.device or weight.stride(0) != 1 and H > 1:
        raise ValueError(f"weight has to be a contiguous ({H},) tensor on {x.device}, got {tuple(weight.shape)} on {weight.device}")
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise TypeError(f"weight has to be {x.dtype} or fp32, got {weight.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual has to be {x.dtype} {tuple(x.shape)} on {x.device}, got {residual.dtype} "
                         f"{tuple(residual.shape)} on {residual.device}")
    if x.numel() // H >= 2 ** 31:
        raise ValueError(f"{x.numel() // H} rows do not fit into 32-bit numbers")


def _like(x: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of the shape and type of x (a copy of its layout is the cheapest way to one)."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _norm(x, weight, eps, residual, keep_rstd=False, keep_y=True, quantise=False):
    """(y, h, rstd, q, scale), each None where it is not asked for; h is None without a residual."""
    shape, dev, code = x.shape, x.device, _ROW_TYPES[x.dtype]
    H = shape[-1]
    rows = x.numel() // H
    with _lib.on_device(dev):
        x2 = _as_rows(x)
        y = _like(x) if keep_y else None
        h = q = scale = rstd = res = None
        res_ld = q_ld = 0
        if residual is not None:
            r2 = _as_rows(residual)
            res, res_ld, h = r2.data_ptr(), r2.stride(0), _like(x)
        if keep_rstd:
            rstd = x.new_empty(rows, dtype=torch.float32)
        if quantise:
            q_ld = -(-H // 16) * 16
            q = x.new_empty((*shape[:-1], q_ld), dtype=torch.int8)
            scale = x.new_empty(shape[:-1], dtype=torch.float32)
        check(lib.smoe_rms_norm(x2.data_ptr(), x2.stride(0), res, res_ld, weight.data_ptr(), _ROW_TYPES[weight.dtype], ptr(y), ptr(h),
                                ptr(rstd), ptr(q), q_ld, ptr(scale), code, rows, H, eps, stream_ptr(dev)), "rms_norm")
    return y, h, rstd, q if q_ld in (0, H) else q[..., :H], scale


class _FirstDerivative(torch.autograd.Function):
    """Gradients as they are; their own derivatives, by what they were computed from, are refused where they are asked for."""

    @staticmethod
    def forward(ctx, grad, *of):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise NotImplementedError("rms_norm has first derivatives only")


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        y, h, rstd, _, _ = _norm(x, weight, eps, residual, keep_rstd=True)
        ctx.save_for_backward(x if residual is None else h, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        if dy is None:  # h alone was used
            return dh, None, None, dh
        h, weight, rstd = ctx.saved_tensors
        need_dx, need_dw = ctx.needs_input_grad[0] or ctx.needs_input_grad[3], ctx.needs_input_grad[1]
        rows, H, dev = rstd.numel(), weight.numel(), h.device
        with _lib.on_device(dev):
            dy2, h2 = _as_rows(dy), _as_rows(h)
            dh2 = None if dh is None or not need_dx else _as_rows(dh)
            dx = _like(h) if need_dx else None
            dw = torch.empty_like(weight) if need_dw else None
            ws = lib.smoe_rms_norm_backward_workspace_bytes(rows, H) if need_dw else 0
            ws = weight.new_empty(ws, dtype=torch.uint8) if ws else None
            check(lib.smoe_rms_norm_backward(
                dy2.data_ptr(), dy2.stride(0), ptr(dh2), 0 if dh2 is None else dh2.stride(0), h2.data_ptr(), h2.stride(0),
                weight.data_ptr(), _ROW_TYPES[weight.dtype], rstd.data_ptr(), ptr(dx), ptr(dw), _ROW_TYPES[h.dtype], rows, H,
                ptr(ws), stream_ptr(dev)), "rms_norm_backward")
        if torch.is_grad_enabled() or forward_ad._current_level >= 0:
            of = [t for t in (dy, dh, h, weight) if t is not None]
            dx = None if dx is None else _FirstDerivative.apply(dx, *of)
            dw = None if dw is None else _FirstDerivative.apply(dw, *of)
        return dx, dw, None, dx if ctx.needs_input_grad[3] else None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             residual: torch.Tensor | None = None) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """y, or with a ``residual`` (y, h) with h = x + residual.  x, residual (..., H), weight (H,)."""
    _check(x, weight, eps, residual)
    if (torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or residual is not None and residual.requires_grad)
            or forward_ad._current_level >= 0):
        return _RmsNorm.apply(x, weight, eps, residual)
    y, h, _, _, _ = _norm(x, weight, eps, residual)
    return y if residual is None else (y, h)


class NormedRows(NamedTuple):
    """8-bit rows of a norm as `int8.int8_linear` and `int8.int8_grouped_linear` take them (x, x_scale), and what else was asked for."""

    q: torch.Tensor             # (..., H) int8, rows on 16-byte boundaries
    scale: torch.Tensor         # (...) fp32
    y: torch.Tensor | None      # (..., H) in the type of x, with keep_y
    h: torch.Tensor | None      # (..., H) x + residual, with a residual


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                      keep_y: bool = False) -> NormedRows:
    """The rows of `rms_norm` quantised to 8 bits, one scale each; ``keep_y`` returns them in the type of x as well (for a router, for
    adapters)."""
    _check(x, weight, eps, residual)
    if x.shape[-1] > MAX_COLS:
        raise ValueError(f"8-bit rows have at most {MAX_COLS} values, got {x.shape[-1]}")
    for t in (x, weight, residual):
        if t is not None and torch.is_grad_enabled() and t.requires_grad:
            raise NotImplementedError("8-bit rows have no gradient: call rms_norm_quantize under torch.no_grad()")
        if t is not None and forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("8-bit rows have no forward-mode derivative")
    y, h, _, q, scale = _norm(x, weight, eps, residual, keep_y=keep_y, quantise=True)
    return NormedRows(q, scale, y, h)
