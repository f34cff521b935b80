"""Low-rank adapters of many requests beside a shared projection, for serving.

    p = adapter_permutation(adapter_idx, n)              # once for a batch: adapter_idx (T,), -1 for tokens without an adapter
    y = int8.int8_linear(x, wq, w_scale)                 # or any other projection of all tokens
    y = adapter_linear(x, a, b, p, base=y, scale=scale)  # y[t] + scale[e] b[e] (a[e] x[t]) with e the adapter of token t

The tokens are sorted by adapter as they are by expert (`token_permutation`), once for all projections and layers of a batch.  bf16 and fp16,
adapters of ranks up to 128 (smaller ones padded with zeros to the largest); sums in fp32, the product of the first projection goes on
without being rounded to 16 bits, and the result is rounded once.

There is no gradient: arguments that require one are refused where gradients are recorded, and those with a forward-mode tangent
everywhere.  The reference has no adapters.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from .. import _lib
from .._lib import check, lib, ptr, stream_ptr
from .permutation import TokenPermutation, _check_permutation, token_permutation

MAX_ADAPTERS = 4096
MAX_RANK = 128
_MAX_WIDTH = 2 ** 28
_TYPES = {torch.bfloat16: _lib.SMOE_BF16, torch.float16: _lib.SMOE_F16}


def adapter_permutation(adapter_idx: torch.Tensor, num_adapters: int) -> TokenPermutation:
    """The tokens sorted by adapter.  adapter_idx (T,) int32 or int64; a token whose index is outside [0, num_adapters) (-1, say) has
    no adapter."""
    if adapter_idx.dim() != 1:
        raise ValueError(f"adapter_idx has to be (T,), got {tuple(adapter_idx.shape)}")
    if not 0 < num_adapters <= MAX_ADAPTERS:
        raise ValueError(f"1 to {MAX_ADAPTERS} adapters are needed, got {num_adapters}")
    return token_permutation(adapter_idx.unsqueeze(1), num_adapters, align=16)


def _refuse_gradients(*tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise NotImplementedError("the adapters have no gradient: call them under torch.no_grad()")
    if forward_ad._current_level >= 0:  # (torch.no_grad() does not stop these)
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError("the adapters have no forward-mode derivative")


def _meets_other_rows(x: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether rows of out, at the distance of out.stride(0), share memory with rows of x of other tokens."""
    (T, H), N = x.shape, out.shape[1]
    if T <= 1:
        return False
    ahead, ld = (out.data_ptr() - x.data_ptr()) // x.element_size(), x.stride(0)
    if ahead >= (T - 1) * ld + H or -ahead >= (T - 1) * out.stride(0) + N:
        return False
    return ld != out.stride(0) or ahead + N > ld or H - ahead > ld


def adapter_linear(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, permutation: TokenPermutation,
                   base: torch.Tensor | None = None, scale: torch.Tensor | None = None, inplace: bool = False) -> torch.Tensor:
    """out (T, N) = base + scale[e] b[e] (a[e] x), and base where a token has no adapter (None: zeros).

    x (T, H), base (T, N), a (n, r, H) and b (n, N, r), all bf16 or all fp16; scale (n,) fp32, None: 1.  ``permutation``: of the T tokens by
    n adapters, K = 1, an ``align`` that is a multiple of 16 (`adapter_permutation`).  ``inplace`` adds to base, which is returned, and
    leaves the rows of tokens without an adapter as they are; base may be a slice of columns, and share memory with the same tokens' rows of x
    (not with those of others).  Autograd counts it as a change of base, as it does base.add_()."""
    if x.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        raise ValueError(f"x has to be (T, H), a (n, r, H) and b (n, N, r), got {tuple(x.shape)}, {tuple(a.shape)} and {tuple(b.shape)}")
    (T, H), (n, r), N = x.shape, a.shape[:2], b.shape[1]
    if a.shape != (n, r, H) or b.shape != (n, N, r):
        raise ValueError(f"inconsistent shapes: x {tuple(x.shape)}, a {tuple(a.shape)}, b {tuple(b.shape)}")
    if x.dtype not in _TYPES or a.dtype != x.dtype or b.dtype != x.dtype:
        raise TypeError(f"x, a and b have to be bf16 or fp16, all of one type, got {x.dtype}, {a.dtype} and {b.dtype}")
    if not (0 < n <= MAX_ADAPTERS and 0 < r <= MAX_RANK and 0 < H <= _MAX_WIDTH and 0 < N <= _MAX_WIDTH):
        raise ValueError(f"1 to {MAX_ADAPTERS} adapters of ranks 1 to {MAX_RANK} and widths of 1 to {_MAX_WIDTH} are needed, got "
                         f"a {tuple(a.shape)}, b {tuple(b.shape)}")
    dev = x.device
    _lib.require_cuda(x, "x")
    _refuse_gradients(x, a, b, base, scale)
    for t, name in ((a, "a"), (b, "b")):
        if t.device != dev or not t.is_contiguous():
            raise ValueError(f"{name} has to be a contiguous tensor on {dev}, got strides {t.stride()} on {t.device}")
    pair, row = permutation.s_reverse_scatter_idx, permutation.x_gather_idx
    offset, count = permutation.expert_frequency_offset, permutation.expert_frequency
    _check_permutation(pair, row, dev)
    if pair.shape != (T, 1):
        raise ValueError(f"the permutation has to be of ({T}, 1) pairs, got {tuple(pair.shape)}")
    for t, size in ((offset, n + 1), (count, n)):
        if t.dtype != torch.int32 or t.shape != (size,) or t.device != dev or not t.is_contiguous():
            raise ValueError(f"the permutation has to be by {n} adapters, contiguous int32 tensors on {dev}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
    align = permutation.align
    if align <= 0 or align % 16:
        raise ValueError(f"the permutation's align has to be a multiple of 16, got {align} (adapter_permutation chooses one)")
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != (n,) or scale.device != dev or not scale.is_contiguous()):
        raise ValueError(f"scale has to be a contiguous fp32 tensor ({n},) on {dev}, got {scale.dtype} {tuple(scale.shape)} on {scale.device}")
    if base is not None and (base.dtype != x.dtype or base.shape != (T, N) or base.device != dev):
        raise ValueError(f"base has to be {x.dtype} ({T}, {N}) on {dev}, got {base.dtype} {tuple(base.shape)} on {base.device}")
    if inplace:
        if base is None:
            raise ValueError("there is no base to add to in place")
        if N > 1 and base.stride(1) != 1 or T > 1 and base.stride(0) < N:
            raise ValueError(f"the rows of a base that is added to in place have to be contiguous and apart, got strides {base.stride()}")
    rows = row.numel()
    if max(T, rows) > 2 ** 31 - 2 ** 16:
        raise ValueError(f"{max(T, rows)} rows do not fit into 32-bit numbers")
    with _lib.on_device(dev):
        x = x if x.stride(1) == 1 or H == 1 else x.contiguous()
        if inplace and _meets_other_rows(x, base):
            raise ValueError("a base that is added to in place shares memory with other tokens' rows of x")
        if base is not None and base.stride(1) != 1 and N > 1:
            base = base.contiguous()
        # (the distance of a single row means nothing)
        base_ld = 0 if base is None else base.stride(0) if T > 1 else max(N, base.stride(0))
        out = base if inplace else torch.empty_like(base) if base is not None and base.is_contiguous() else x.new_empty((T, N))
        check(lib.smoe_adapter_linear(
            x.data_ptr(), x.stride(0), a.data_ptr(), b.data_ptr(), ptr(scale), ptr(base), base_ld, out.data_ptr(),
            base_ld if inplace else N, _TYPES[x.dtype], offset.data_ptr(), count.data_ptr(), row.data_ptr(), pair.data_ptr(), T, rows, H, N, n, r, align,
            _lib.device_state(dev).status.data_ptr(), stream_ptr(dev)), "adapter_linear")
    if inplace:  # (the library writes through an address, which autograd does not see; tensors of inference mode have no count, and that is no error)
        increment_version(base)
    return out
