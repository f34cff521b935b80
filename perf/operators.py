"""Operators around the experts of an MoE layer, as timed cases: tokens sorted by expert and back, and products of 8-bit
integers with one scale per token and output channel, dense and grouped by expert.

Kinds of cases
  sort     the expert of every (token, slot) pair in, the permutation and the rows sorted by expert out; training adds the
           gradient of x, the sum over each token's rows
  combine  sorted rows and the router's scores in, the weighted sum of each token's rows out; training adds the gradients
           of the rows and of the scores
  linear   rows quantised to 8 bits, one scale each, times 8-bit weights with one scale per output channel, plus a bias
  grouped  the same with the weights of the row's expert; rows gathered by token, SwiGLU of the interleaved gate and up
           channels where the case says so

Sizes are the layer shapes of this repository's benchmark and tests, and generic ones of the same kind.  Activations and
upstream gradients are N(0, 1), weights N(0, 0.02); a token's experts are the largest of N(0, 1) logits plus a bias per expert.
"""

import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _sort(name, T, H, E, K, dtype, train, align=1, dropped=0.0):
    return dict(name=name, kind="sort", T=T, H=H, E=E, K=K, dtype=dtype, train=train, align=align, dropped=dropped)


def _combine(name, T, H, E, K, dtype, train, align=1, dropped=0.0):
    return dict(name=name, kind="combine", T=T, H=H, E=E, K=K, dtype=dtype, train=train, align=align, dropped=dropped)


def _linear(name, T, N, H, dtype, bias):
    return dict(name=name, kind="linear", T=T, N=N, H=H, dtype=dtype, bias=bias)


def _grouped(name, T, N, H, E, K, dtype, gather, swiglu, bias, align=1, dropped=0.0):
    return dict(name=name, kind="grouped", T=T, N=N, H=H, E=E, K=K, dtype=dtype, gather=gather, swiglu=swiglu, bias=bias,
                align=align, dropped=dropped)


def listed():
    return [
        # one token of a decode step: nothing but latency
        _sort("sort_decode_1", 1, 4096, 128, 8, "bf16", False),
        # the benchmark layer's training step
        _sort("sort_train_32768", 32768, 4096, 128, 8, "bf16", True),
        # fp32 rows of an odd width, experts padded to tiles of 128 rows, a tenth of the pairs dropped (capacity, padding)
        _sort("sort_padded_4099", 4099, 1005, 60, 6, "fp32", True, 128, 0.1),
        # the combine of a decode step with a batch of 64
        _combine("combine_decode_64", 64, 4096, 128, 8, "bf16", False),
        # a training step of the mid-size layer with fine-grained experts
        _combine("combine_train_24576", 24576, 1536, 128, 8, "bf16", True),
        # fp16, a width that is no multiple of 8, padded experts, dropped pairs
        _combine("combine_ragged_5003", 5003, 1030, 40, 3, "fp16", True, 16, 0.2),
        # one token through a dense projection
        _linear("linear_decode_1", 1, 4096, 4096, "bf16", False),
        # a small decode batch through a wide projection
        _linear("linear_decode_33", 33, 7168, 2048, "bf16", True),
        # a long prefill
        _linear("linear_prefill_8192", 8192, 7168, 4096, "bf16", False),
        # the up projection of the benchmark layer for a decode batch of 64: about four rows per expert
        _grouped("grouped_decode_64", 64, 2048, 4096, 128, 8, "bf16", True, True, False),
        # the same for a prefill of 8192 tokens
        _grouped("grouped_prefill_8192", 8192, 2048, 4096, 128, 8, "bf16", True, True, False),
        # rows sorted by the caller, padded experts, odd sizes, fp32 result with bias
        _grouped("grouped_padded_1027", 1027, 1000, 1030, 60, 4, "fp32", False, False, True, 64, 0.1),
    ]


def _log(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def _odd(rng, n, step):
    """n as it is, or the multiple of `step` below it: half of the sizes are round ones."""
    return n if rng.random() < 0.5 else max(step, n // step * step)


def draw(rng):
    kind = rng.choice(["sort", "combine", "linear", "grouped"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    T = _odd(rng, _log(rng, 1, 32768), 64)
    E = _log(rng, 8, 256)
    K = rng.randint(1, min(8, E))
    align = rng.choice([1, 1, 16, 128])
    dropped = rng.choice([0.0, 0.0, 0.1, 0.5])
    if kind in ("sort", "combine"):
        H = _odd(rng, _log(rng, 64, 7168), 64)
        while T * K * H * _BYTES[dtype] > 2 ** 30:
            T = max(1, T // 2)
        make = _sort if kind == "sort" else _combine
        case = make("", T, H, E, K, dtype, rng.random() < 0.5, align, dropped)
    elif kind == "linear":
        N, H = _odd(rng, _log(rng, 64, 8192), 64), _odd(rng, _log(rng, 64, 8192), 64)
        while T * N * H > 2 ** 37:
            T = max(1, T // 2)
        case = _linear("", T, N, H, dtype, rng.random() < 0.5)
    else:
        N, H = 2 * _odd(rng, _log(rng, 64, 1024), 64), _odd(rng, _log(rng, 64, 4096), 64)
        while T * K * N * H > 2 ** 38:
            T = max(1, T // 2)
        case = _grouped("", T, N, H, E, K, dtype, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5, align, dropped)
    del case["name"]
    return case


def _num_rows(case):
    """Rows that hold every load: each expert that has any is padded by less than `align`."""
    pairs, align = case["T"] * case["K"], case["align"]
    return (pairs + min(case["E"], pairs) * (align - 1)) // align * align


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _pitched(q):
    """8-bit rows that start on 16-byte boundaries: how the products take their weights."""
    cols = q.shape[-1]
    buffer = torch.zeros(*q.shape[:-1], (cols + 15) // 16 * 16, dtype=torch.int8, device=q.device)
    buffer[..., :cols] = q
    return buffer[..., :cols]


def _weights(gen, shape, out):
    """(values int8, one scale per channel) of N(0, 0.02) weights."""
    w = torch.randn(shape, generator=gen, device="cuda") * 0.02
    scale = w.abs().amax(-1) / 127
    out["wq"] = _pitched(torch.round(w / scale.unsqueeze(-1)).to(torch.int8))
    out["w_scale"] = scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(_TYPES[case["dtype"]])

    s = {"case": case}
    T, kind = case["T"], case["kind"]
    if kind != "linear":
        E, K = case["E"], case["K"]
        logits = torch.randn(T, E, generator=gen, device="cuda") + 0.5 * torch.randn(E, generator=gen, device="cuda")
        top = logits.topk(K, dim=1)
        drop = torch.rand(T, K, generator=gen, device="cuda") < case["dropped"]
        s["idx"] = torch.where(drop, -1, top.indices).to(torch.int32)
        s["rows"] = _num_rows(case)
    if kind == "sort":
        s["x"] = normal(T, case["H"]).requires_grad_(case["train"])
        s["drows"] = normal(s["rows"], case["H"]) if case["train"] else None
    elif kind == "combine":
        s["perm"] = _permutation(s["idx"], E, case["align"], s["rows"])
        s["y"] = normal(s["rows"], case["H"]).requires_grad_(case["train"])
        s["scores"] = torch.softmax(top.values, dim=1).requires_grad_(case["train"])
        s["dout"] = normal(T, case["H"]) if case["train"] else None
    else:
        N, H = case["N"], case["H"]
        s["bias"] = normal(N) if kind == "linear" and case["bias"] else None
        if kind == "linear":
            s["x"] = normal(T, H)
            _weights(gen, (N, H), s)
        else:
            _weights(gen, (E, N, H), s)
            s["bias"] = normal(E, N) if case["bias"] else None
            s["perm"] = _permutation(s["idx"], E, case["align"], s["rows"])
            s["x"] = normal(T, H)
            s["most"] = max(1, int(s["perm"]["expert_frequency"].max()))  # rows of the fullest expert
            if not case["gather"]:
                token = s["perm"]["x_gather_idx"].long()
                s["x"] = torch.where((token >= 0).unsqueeze(1), s["x"][token.clamp_min(0)], torch.zeros_like(s["x"][:1]))
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _permutation(idx, E, align, rows):
    """The stable sort of the (token, slot) pairs by expert; an expert's rows start at a multiple of `align`.  Pairs whose
    expert is not in [0, E) are dropped; -1 stands for a pair without a row and for a row without a pair."""
    T, K = idx.shape
    dev = idx.device
    flat = idx.reshape(-1).long()
    kept = (flat >= 0) & (flat < E)
    key = torch.where(kept, flat, E)
    order = torch.argsort(key, stable=True)
    count = torch.zeros(E + 1, dtype=torch.int64, device=dev).scatter_add_(0, key, torch.ones_like(key))
    padded = torch.cat([(count[:E] + align - 1) // align * align, count[E:]])
    first, start = padded.cumsum(0) - padded, count.cumsum(0) - count
    expert = key[order]
    row = first[expert] + torch.arange(T * K, device=dev) - start[expert]
    row = torch.where(expert < E, row, rows)  # dropped pairs meet in a row of their own behind the last
    slot_row = torch.full((T * K,), -1, dtype=torch.int64, device=dev).scatter(0, order, torch.where(expert < E, row, -1))
    row_slot = torch.full((rows + 1,), -1, dtype=torch.int64, device=dev).scatter(0, row, order)[:rows]
    token = torch.div(row_slot, K, rounding_mode="floor")  # -1 stays -1
    offset = torch.cat([first[:E], (first[E - 1] + padded[E - 1]).reshape(1)])
    i32 = torch.int32
    return {"expert_frequency": count[:E].to(i32), "expert_frequency_offset": offset.to(i32), "x_gather_idx": token.to(i32),
            "s_scatter_idx": row_slot.to(i32), "s_reverse_scatter_idx": slot_row.to(i32).view(T, K)}


def _rows_of(x, index):
    """x[index] in 32 bits, zeros where the index is -1."""
    index = index.long()
    return torch.where((index >= 0).unsqueeze(-1), x[index.clamp_min(0)].float(), 0.0)


def _plain_sort(s):
    case, x = s["case"], s["x"].detach()
    p = _permutation(s["idx"], case["E"], case["align"], s["rows"])
    out = {"rows": _rows_of(x, p["x_gather_idx"]).to(x.dtype), **p}
    if case["train"]:
        out["dx"] = _rows_of(s["drows"], p["s_reverse_scatter_idx"].reshape(-1)).view(case["T"], case["K"], -1).sum(1).to(x.dtype)
    return out


def _plain_combine(s):
    case, p, y, w = s["case"], s["perm"], s["y"].detach(), s["scores"].detach()
    T, K = case["T"], case["K"]
    mine = _rows_of(y, p["s_reverse_scatter_idx"].reshape(-1)).view(T, K, -1)
    out = {"out": (mine * w.unsqueeze(-1)).sum(1).to(y.dtype)}
    if case["train"]:
        out["dscores"] = (mine * s["dout"].float().unsqueeze(1)).sum(-1)
        slot = p["s_scatter_idx"].long()
        weight = torch.where(slot >= 0, w.reshape(-1)[slot.clamp_min(0)], 0.0)
        out["drows"] = (_rows_of(s["dout"], p["x_gather_idx"]) * weight.unsqueeze(-1)).to(y.dtype)
    return out


def _plain_quantize(x):
    """(whole numbers of at most 127, scale) of each row; quotients next to a border in 64 bits."""
    amax = x.float().abs().amax(-1, keepdim=True)
    some = torch.where(amax > 0, amax, 1.0)
    return torch.round(x.double() * 127 / some.double()).float(), torch.where(amax > 0, amax / 127, 1.0)


def _plain_linear(s):
    q, scale = _plain_quantize(s["x"])
    y = (q @ s["wq"].float().t()) * scale * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_grouped(s):
    case, p, x = s["case"], s["perm"], s["x"]
    q, scale = _plain_quantize(x)
    if case["gather"]:
        token = p["x_gather_idx"]
        q, scale = _rows_of(q, token), _rows_of(scale, token)
    first, count = p["expert_frequency_offset"].long(), p["expert_frequency"].long()
    place = torch.arange(s["most"], device=x.device)
    at = torch.where(place < count.unsqueeze(1), first[:-1].unsqueeze(1) + place, -1)  # (E, rows of the fullest expert)
    y = torch.bmm(_rows_of(q, at), s["wq"].float().transpose(1, 2)) * _rows_of(scale, at) * s["w_scale"].unsqueeze(1)
    if s["bias"] is not None:
        y = y + s["bias"].float().unsqueeze(1)
    if case["swiglu"]:
        gate, up = y[..., 0::2], y[..., 1::2]
        y = gate / (1 + torch.exp(-gate)) * up
    # rows without a pair are zeros, whatever the bias
    row = torch.where(at >= 0, at, s["rows"]).reshape(-1)
    out = torch.zeros(s["rows"] + 1, y.shape[-1], device=x.device).index_copy_(0, row, y.reshape(row.numel(), -1))
    return out[:-1].to(x.dtype)


# ------------------------------------------------------------------------------------------------
# the framework's operators
# ------------------------------------------------------------------------------------------------
def _package():
    package = os.path.join(os.getcwd(), "sonic-moe_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import sonicmoe

    return sonicmoe


def _own(s):
    sonicmoe = _package()
    case = s["case"]
    kind = case["kind"]
    if kind == "sort":
        p = sonicmoe.token_permutation(s["idx"], case["E"], align=case["align"])
        rows = sonicmoe.permute_tokens(s["x"], p)
        out = {"rows": rows.detach(), "expert_frequency": p.expert_frequency,
               "expert_frequency_offset": p.expert_frequency_offset, "x_gather_idx": p.x_gather_idx,
               "s_scatter_idx": p.s_scatter_idx, "s_reverse_scatter_idx": p.s_reverse_scatter_idx}
        if case["train"]:
            out["dx"], = torch.autograd.grad(rows, s["x"], s["drows"])
        return out
    if kind == "combine":
        p = sonicmoe.TokenPermutation(**s["perm"], align=case["align"])
        o = sonicmoe.unpermute_tokens(s["y"], p, s["scores"])
        out = {"out": o.detach()}
        if case["train"]:
            out["drows"], out["dscores"] = torch.autograd.grad(o, (s["y"], s["scores"]), s["dout"])
        return out
    from sonicmoe.functional import int8

    if kind == "linear":
        return int8.int8_linear(s["x"], s["wq"], s["w_scale"], bias=s["bias"])
    p = s["perm"]
    return int8.int8_grouped_linear(
        s["x"], s["wq"], s["w_scale"], p["expert_frequency_offset"], x_gather_idx=p["x_gather_idx"] if case["gather"] else None,
        expert_frequency=p["expert_frequency"], bias=s["bias"], activation_type="swiglu" if case["swiglu"] else None)


def run(state):
    if own:
        return _own(state)
    plain = {"sort": _plain_sort, "combine": _plain_combine, "linear": _plain_linear, "grouped": _plain_grouped}
    with torch.no_grad():
        return plain[state["case"]["kind"]](state)


def work(case):
    T, H, kind = case["T"], case["H"], case["kind"]
    size = _BYTES[case["dtype"]]
    if kind in ("sort", "combine"):
        K, rows = case["K"], _num_rows(case)
        pairs = T * K
        kept = pairs * (1 - case["dropped"])
        index = 4 * (2 * pairs + 2 * rows + 2 * case["E"])
        if kind == "sort":  # x in, rows out; the rows' gradient in, that of x out
            passes = T * H * size + rows * H * size
            both = passes + (kept + T) * H * size
            return {"bytes": index + (both if case["train"] else passes), "flops": kept * H if case["train"] else 0}
        passes = (kept + T) * H * size + 8 * pairs
        # the rows again for the scores' gradient, the result's gradient in, the rows' out
        both = passes + (kept + T + rows) * H * size + 4 * pairs + 8 * rows
        return {"bytes": both if case["train"] else passes, "flops": kept * H * (5 if case["train"] else 2)}
    N = case["N"]
    if kind == "linear":
        return {"bytes": T * H * size + N * H + 4 * N + T * N * size + (N * size if case["bias"] else 0), "flops": 2 * T * N * H}
    E, pairs = case["E"], case["T"] * case["K"] * (1 - case["dropped"])
    used = E * (1 - (1 - 1 / E) ** pairs)  # experts that have rows, for even loads
    rows, cols = _num_rows(case), N // 2 if case["swiglu"] else N
    x_bytes = (T if case["gather"] else pairs) * H * size
    return {"bytes": x_bytes + used * (N * H + 4 * N + (N * size if case["bias"] else 0)) + rows * cols * size + 4 * (rows + 2 * E),
            "flops": 2 * pairs * N * H}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_quantize(x):
    """round(127 x / amax), ties to even, as a whole number found by its remainder."""
    x = x.detach().double()
    amax = x.abs().amax(-1, keepdim=True)
    amax = torch.where(amax == 0, torch.full_like(amax, 127.0), amax)
    twice = 254 * x + amax
    q = torch.floor(twice / (2 * amax))
    tie = (twice - q * 2 * amax == 0) & (torch.remainder(q, 2) == 1)
    return torch.where(tie, q - 1, q), amax / 127


def _exact_rows(s):
    """For every row its slot (-1: none), found expert by expert."""
    case, flat = s["case"], s["idx"].reshape(-1)
    slots = torch.full((s["rows"],), -1, dtype=torch.int64, device=flat.device)
    at = 0
    for e in range(case["E"]):
        mine = torch.nonzero(flat == e).reshape(-1)
        slots[at:at + mine.numel()] = mine
        at += -(-mine.numel() // case["align"]) * case["align"]
    return slots


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind == "linear":
            q, scale = _exact_quantize(s["x"])
            y = scale * (q @ s["wq"].double().T) * s["w_scale"].double()
            return y if s["bias"] is None else y + s["bias"].double()
        slots = _exact_rows(s)
        live = torch.nonzero(slots >= 0).reshape(-1)
        slot = slots[live]
        token = slot // case["K"]
        if kind == "sort":
            rows = torch.zeros(s["rows"], case["H"], dtype=torch.float64, device="cuda")
            rows[live] = s["x"].detach().double()[token]
            out = {"rows": rows, **dict.fromkeys(("expert_frequency", "expert_frequency_offset", "x_gather_idx",
                                                  "s_scatter_idx", "s_reverse_scatter_idx"))}
            if case["train"]:
                out["dx"] = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda").index_add_(
                    0, token, s["drows"].double()[live])
            return out
        if kind == "combine":
            y, w = s["y"].detach().double()[live], s["scores"].detach().double().reshape(-1)[slot].unsqueeze(1)
            o = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
            out = {"out": o.index_add_(0, token, y * w)}
            if case["train"]:
                g = s["dout"].double()[token]
                out["dscores"] = torch.zeros(case["T"] * case["K"], dtype=torch.float64, device="cuda").index_copy_(
                    0, slot, (g * y).sum(1)).view(case["T"], case["K"])
                out["drows"] = torch.zeros(s["rows"], case["H"], dtype=torch.float64, device="cuda").index_copy_(0, live, g * w)
            return out
        q, scale = _exact_quantize(s["x"])
        expert = s["idx"].reshape(-1)[slot].long()
        source = token if case["gather"] else live
        y = torch.zeros(s["rows"], case["N"], dtype=torch.float64, device="cuda")
        for e in range(case["E"]):
            of = expert == e
            at = source[of]
            z = scale[at] * (q[at] @ s["wq"][e].double().T) * s["w_scale"][e].double()
            y[live[of]] = z if s["bias"] is None else z + s["bias"][e].double()
        if case["swiglu"]:
            gate, up = y[:, 0::2], y[:, 1::2]
            y = gate * torch.sigmoid(gate) * up
        return y
