"""8-bit integer products for serving: activations quantised per token, weights per output channel, dense or grouped by expert.

    wq, w_scale = quantize_rows(w)                       # once: w (E, N, cols), one scale per expert and channel
    y = int8_grouped_linear(x, wq, w_scale, p.expert_frequency_offset, x_gather_idx=p.x_gather_idx)

or the whole layer, with the router's logits, top-K choice and combine of the bf16 one (under torch.no_grad()):

    experts = quantize_experts(moe.c_fc.weight.permute(1, 2, 0), moe.c_fc.bias, moe.c_proj.weight.permute(1, 2, 0), moe.c_proj.bias)
    o, router_logits, expert_frequency = moe_int8_softmax_topk_layer(x, moe.router.weight, experts, K)

scale = amax / 127 of the row (1 for a row of zeros), values = 127 x / amax rounded half to even; the sum of a product is exact
in 32-bit integers and rounded once, so results do not depend on how the work is shared out.  It is multiplied by the row's scale
and then by the channel's in fp32: rows whose largest value is 0 or from 2^-119 to 2^103 leave its range only where the result does.
Rows that hold an infinity or a NaN give NaN.  8-bit rows start on 16-byte boundaries: `quantize_rows` lays them out so, whatever their width.

There is no gradient: arguments that require one are refused where gradients are recorded, and those with a forward-mode
tangent everywhere.  The FP8 experts (`functional.fp8`) are the path for training.  The reference has no 8-bit path.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from .. import _lib
from .._lib import check, lib, ptr, stream_ptr
from ..enums import ActivationType, is_glu
from .permutation import _ROW_TYPES as _FLOAT_TYPES

MAX_COLS = 131071  # sums of that many products of 8-bit integers fit into 32 bits
MAX_EXPERTS = 1024

_ACTIVATIONS = {ActivationType.SWIGLU: 0, ActivationType.GEGLU: 1, ActivationType.REGLU: 2, ActivationType.RELU_SQ: 3,
                ActivationType.RELU: 4, ActivationType.GELU: 5, ActivationType.SILU: 6}


def _refuse_gradients(*tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise NotImplementedError("the 8-bit products have no gradient: call them under torch.no_grad()")
    if forward_ad._current_level >= 0:  # (torch.no_grad() does not stop these)
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("the 8-bit products have no forward-mode derivative")


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x (..., cols) fp32, bf16 or fp16 -> (q (..., cols) int8, scale (...) fp32), one scale per row."""
    if x.dim() < 1 or x.dtype not in _FLOAT_TYPES:
        raise TypeError(f"x has to be fp32, bf16 or fp16 rows, got {x.dtype} {tuple(x.shape)}")
    cols = x.shape[-1]
    if not 0 < cols <= MAX_COLS:
        raise ValueError(f"rows of 1 to {MAX_COLS} values are needed, got {cols}")
    _lib.require_cuda(x, "x")
    _refuse_gradients(x)
    dev = x.device
    rows = x.numel() // cols
    if x.dim() != 2 or (cols > 1 and x.stride(1) != 1):
        x2 = x.contiguous().view(rows, cols)
    else:
        x2 = x
    with _lib.on_device(dev):
        q = torch.empty(*x.shape[:-1], -(-cols // 16) * 16, dtype=torch.int8, device=dev)
        scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
        check(lib.smoe_int8_quantize_rows(x2.data_ptr(), x2.stride(0), _FLOAT_TYPES[x.dtype], q.data_ptr(), q.shape[-1],
                                          scale.data_ptr(), rows, cols, stream_ptr(dev)), "int8_quantize_rows")
    return q if q.shape[-1] == cols else q[..., :cols], scale


def _activation_code(activation_type) -> int:
    if activation_type is None:
        return -1
    if isinstance(activation_type, str):
        activation_type = ActivationType(activation_type)
    return _ACTIVATIONS[activation_type]


def _rows_16(t: torch.Tensor, name: str) -> int:
    """Distance of the rows of an 8-bit tensor in bytes."""
    if t.stride(-1) != 1 and t.shape[-1] > 1 or t.stride(-2) % 16 != 0 or t.stride(-2) < t.shape[-1] or t.data_ptr() % 16 != 0:
        raise ValueError(f"the rows of {name} have to start on 16-byte boundaries, as quantize_rows lays them out "
                         f"(strides {t.stride()})")
    return t.stride(-2)


def _check_vector(t: torch.Tensor, name: str, dtype: torch.dtype, shape, dev: torch.device) -> None:
    if t.dtype != dtype or t.shape != shape or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} has to be a contiguous {dtype} tensor {tuple(shape)} on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")


def _linear(x, wq, w_scale, x_scale, bias, out_dtype, activation, offset, frequency, gather):
    grouped = offset is not None
    _refuse_gradients(x, w_scale, x_scale, bias)
    if wq.dtype != torch.int8 or wq.dim() != (3 if grouped else 2):
        raise TypeError(f"wq has to be int8 {'(E, N, cols)' if grouped else '(N, cols)'}, got {wq.dtype} {tuple(wq.shape)}")
    if x.dim() != 2 or x.shape[1] != wq.shape[-1]:
        raise ValueError(f"inconsistent shapes: x {tuple(x.shape)}, wq {tuple(wq.shape)}")
    N, cols = wq.shape[-2:]
    E = wq.shape[0] if grouped else 1
    if not 0 < cols <= MAX_COLS or N == 0 or not 0 < E <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_COLS} columns, 1 to {MAX_EXPERTS} experts and a channel are needed, got wq {tuple(wq.shape)}")
    dev = x.device
    _lib.require_cuda(x, "x")
    _check_vector(w_scale, "w_scale", torch.float32, wq.shape[:-1], dev)
    if x_scale is not None:
        _check_vector(x_scale, "x_scale", torch.float32, x.shape[:1], dev)
    if grouped:
        _check_vector(offset, "expert_frequency_offset", torch.int32, (E + 1,), dev)
        if frequency is not None:
            _check_vector(frequency, "expert_frequency", torch.int32, (E,), dev)
        if gather is not None:
            _check_vector(gather, "x_gather_idx", torch.int32, (gather.numel(),), dev)
    if wq.device != dev:
        raise ValueError(f"wq is on {wq.device}, x on {dev}")
    w_ld = _rows_16(wq, "wq")
    if grouped and E > 1 and wq.stride(0) != N * w_ld:
        raise ValueError(f"the experts of wq have to follow one another (strides {wq.stride()})")
    if x.dtype == torch.int8:
        if x_scale is None:
            raise ValueError("8-bit x needs x_scale")
        x_type, ld = _lib.SMOE_I8, _rows_16(x, "x") if x.shape[0] else 0
        out_dtype = out_dtype or torch.bfloat16
    elif x.dtype in _FLOAT_TYPES:
        if x_scale is not None:
            raise ValueError("x_scale belongs to 8-bit x")
        if x.stride(1) != 1 and cols > 1:
            x = x.contiguous()
        x_type, ld = _FLOAT_TYPES[x.dtype], x.stride(0)
        out_dtype = out_dtype or x.dtype
    else:
        raise TypeError(f"x has to be int8, fp32, bf16 or fp16, got {x.dtype}")
    if out_dtype not in _FLOAT_TYPES:
        raise TypeError(f"out_dtype has to be fp32, bf16 or fp16, got {out_dtype}")
    if activation >= 0 and activation <= 2 and N % 2:
        raise ValueError(f"a gated activation needs an even number of channels, got {N}")
    if bias is not None:
        if bias.dtype not in _FLOAT_TYPES or bias.shape != wq.shape[:-1] or bias.device != dev:
            raise ValueError(f"bias has to be {tuple(wq.shape[:-1])} on {dev}, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
        bias = bias.contiguous()
    T = x.shape[0]
    rows = gather.numel() if gather is not None else T
    if T == 0 and rows > 0:
        raise ValueError("x has no rows to gather")
    if max(T, rows) > 2 ** 31 - 2 ** 16 or E * N >= 2 ** 31 - 256:
        raise ValueError(f"{max(T, rows)} rows or {E * N} channels do not fit into 32-bit numbers")
    with _lib.on_device(dev):
        out = torch.empty(rows, N // 2 if 0 <= activation <= 2 else N, dtype=out_dtype, device=dev)
        if rows == 0:  # (an empty gather index has no address, which would stand for no gathering)
            return out
        ws = lib.smoe_int8_linear_workspace_bytes(x_type, T, rows, N, cols, E)
        ws = _lib.workspace(ws, dev) if ws else None
        check(lib.smoe_int8_linear(
            x.data_ptr(), ld, x_type, ptr(x_scale), wq.data_ptr(), w_ld, w_scale.data_ptr(), ptr(bias),
            0 if bias is None else _FLOAT_TYPES[bias.dtype], out.data_ptr(), _FLOAT_TYPES[out_dtype], ptr(offset),
            ptr(frequency), ptr(gather), T, rows, N, cols, E, activation, ptr(ws), _lib.device_state(dev).status.data_ptr(),
            stream_ptr(dev)), "int8_linear")
    return out


def int8_linear(x: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, x_scale: torch.Tensor | None = None,
                bias: torch.Tensor | None = None, activation_type: ActivationType | str | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """act(x w^T + bias) (M, N) with w = wq * w_scale: wq (N, cols) int8, w_scale (N,).  x (M, cols): fp32, bf16 or fp16, quantised
    row by row on the way, or int8 with ``x_scale`` (M,).  The result has x's type (8-bit x: bf16) unless ``out_dtype`` says
    otherwise; a gated activation takes the channels 2j and 2j + 1 as gate and up and gives N / 2."""
    return _linear(x, wq, w_scale, x_scale, bias, out_dtype, _activation_code(activation_type), None, None, None)


def int8_grouped_linear(x: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, expert_frequency_offset: torch.Tensor,
                        x_gather_idx: torch.Tensor | None = None, expert_frequency: torch.Tensor | None = None,
                        x_scale: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                        activation_type: ActivationType | str | None = None,
                        out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """`int8_linear` with the weights of each row's expert: wq (E, N, cols), w_scale and bias (E, N).

    Expert e has the rows from ``expert_frequency_offset[e]`` on, as many as ``expert_frequency[e]`` (None: up to the next
    expert's first); rows that no expert has are zeros.  ``x_gather_idx`` (rows,): the row of x that each takes (-1: a row of
    zeros); None: x is sorted already.  These are the fields of `TokenPermutation`."""
    if expert_frequency_offset is None:
        raise ValueError("expert_frequency_offset is needed: int8_linear is the product without experts")
    return _linear(x, wq, w_scale, x_scale, bias, out_dtype, _activation_code(activation_type), expert_frequency_offset,
                   expert_frequency, x_gather_idx)


@dataclass
class Int8Experts:
    """The experts of a layer as `quantize_rows` lays them out: w1q (E, N1, H), w2q (E, H, I), scales and biases like their rows."""

    w1q: torch.Tensor
    w1_scale: torch.Tensor
    b1: torch.Tensor | None
    w2q: torch.Tensor
    w2_scale: torch.Tensor
    b2: torch.Tensor | None


@torch.no_grad()
def quantize_experts(w1: torch.Tensor, b1: torch.Tensor | None, w2: torch.Tensor, b2: torch.Tensor | None) -> Int8Experts:
    """w1 (N1, H, E) and w2 (H, I, E), the ``permute(1, 2, 0)`` views that the other layer functions take; biases (E, N1), (E, H)."""
    if (b1 is None) != (b2 is None):
        raise AssertionError("b1 and b2 has to be None or not None at the same time!")
    if w1.dim() != 3 or w2.dim() != 3 or w1.shape[2] != w2.shape[2] or w1.shape[1] != w2.shape[0]:
        raise ValueError(f"inconsistent shapes: w1 {tuple(w1.shape)}, w2 {tuple(w2.shape)}")
    return Int8Experts(*quantize_rows(w1.permute(2, 0, 1)), b1, *quantize_rows(w2.permute(2, 0, 1)), b2)


def moe_int8_softmax_topk_layer(
    x: torch.Tensor,
    router_w: torch.Tensor,
    experts: Int8Experts,
    K: int,
    activation_type: ActivationType | str = ActivationType.SWIGLU,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Inference forward of the token-choice top-K layer with 8-bit experts: (o (T, H), router_logits (T, E), expert_frequency
    (E,) int32), as `moe_TC_softmax_topk_layer`.  x (T, H) bf16, quantised per token; the activations between the projections are
    rounded to bf16 and quantised per row."""
    from . import _FusedRouter, _route_metadata, fused_router_applies, topk_softmax

    if isinstance(activation_type, str):
        activation_type = ActivationType(activation_type)
    _refuse_gradients(x, router_w, experts.w1_scale, experts.b1, experts.w2_scale, experts.b2)
    _lib.require_cuda(x, "x")
    if x.dtype != torch.bfloat16 or x.dim() != 2:
        raise TypeError(f"x has to be (T, H) bf16, got {x.dtype} {tuple(x.shape)}")
    T, H = x.shape
    E, n1 = experts.w1q.shape[:2]
    if router_w.shape != (E, H) or experts.w1q.shape[2] != H or experts.w2q.shape[:2] != (E, H):
        raise ValueError(f"inconsistent shapes: x {tuple(x.shape)}, router {tuple(router_w.shape)}, w1q {tuple(experts.w1q.shape)}, "
                         f"w2q {tuple(experts.w2q.shape)}")
    if experts.w2q.shape[2] * (2 if is_glu(activation_type) else 1) != n1:
        raise ValueError(f"{n1} rows of the up projection do not fit {experts.w2q.shape[2]} columns of the down projection")
    if not 1 <= K <= E:
        raise ValueError(f"1 <= K <= {E} is needed, got {K}")
    if H % 8:
        raise ValueError("the hidden size has to be a multiple of 8")  # the combine's accesses
    with torch.no_grad():
        if T > 0 and fused_router_applies(x, router_w, K):
            router_logits, scores, indices = _FusedRouter.apply(x, router_w, K)[:3]
        else:
            router_logits = F.linear(x if x.dtype == router_w.dtype else x.to(router_w.dtype), router_w)
            scores, indices = topk_softmax(router_logits, K)
        route = _route_metadata(indices.reshape(-1), None, E, K)
        code = _ACTIVATIONS[activation_type]
        y1 = _linear(x, experts.w1q, experts.w1_scale, None, experts.b1, None, code, route.expert_frequency_offset, None,
                     route.x_gather_idx)
        y2 = _linear(y1, experts.w2q, experts.w2_scale, None, experts.b2, None, -1, route.expert_frequency_offset, None, None)
        with _lib.on_device(x.device):
            o = torch.empty_like(x, memory_format=torch.contiguous_format)
            check(lib.smoe_gather_sum(y2.data_ptr(), o.data_ptr(), scores.data_ptr(), _lib.SMOE_F32,
                                      route.s_reverse_scatter_idx.data_ptr(), None, T, H, K, stream_ptr(x.device)), "gather_sum")
    return o, router_logits, route.expert_frequency
