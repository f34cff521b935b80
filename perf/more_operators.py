"""Operators in front of and beside the projections of an MoE layer, as timed cases: root-mean-square norm with the residual's
addition, in the activations' type or as 8-bit rows, and the low-rank adapters of many requests beside a shared projection.

Kinds of cases
  norm      h = x + residual (or x) and y = h / sqrt(mean(h^2) + eps) * weight out; training adds the gradients of x, of the
            residual and of the weight
  norm8     the same rows y as 8-bit values with one scale each, as the 8-bit products take them; h, and y where the case says so
  adapters  out[t] = base[t] + scale[e] b[e] (a[e] x[t]) with e the adapter of token t, which may be none

Sizes are the layer shapes of this repository's benchmark and tests, and generic ones of the same kind.  Activations and
upstream gradients are N(0, 1), a hundredth of the channels of x ten times as large; a norm's weights are 1 + N(0, 0.1).  The
rows of an adapter's a are N(0, 1 / H), of its b N(0, 0.3^2 / r).  The tokens of a request follow one another and share an adapter.
"""

import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def _norm(name, T, H, dtype, weights, residual, train, eps=1e-6):
    return dict(name=name, kind="norm", T=T, H=H, dtype=dtype, weights=weights, residual=residual, train=train, eps=eps)


def _norm8(name, T, H, dtype, weights, residual, keep, eps=1e-6):
    return dict(name=name, kind="norm8", T=T, H=H, dtype=dtype, weights=weights, residual=residual, keep=keep, eps=eps)


def _adapters(name, T, requests, H, N, n, r, dtype, base, dropped=0.0, align=16):
    return dict(name=name, kind="adapters", T=T, requests=requests, H=H, N=N, n=n, r=r, dtype=dtype, base=base, dropped=dropped,
                align=align)


def listed():
    return [
        # one token of a decode step: nothing but latency
        _norm("norm_decode_1", 1, 4096, "bf16", "bf16", True, False),
        # the benchmark layer's training step
        _norm("norm_train_32768", 32768, 4096, "bf16", "bf16", True, True),
        # fp32 rows of an odd width, no residual
        _norm("norm_train_4099", 4099, 1005, "fp32", "fp32", False, True, 1e-5),
        # the norm of attention heads: many short rows, fp32 weights
        _norm("norm_heads_262144", 262144, 128, "bf16", "fp32", False, True),
        # in front of the 8-bit projections, a decode batch of 64; the router reads y
        _norm8("norm8_decode_64", 64, 4096, "bf16", "bf16", True, True),
        # the same for a prefill of 8192 tokens, 8-bit rows alone
        _norm8("norm8_prefill_8192", 8192, 4096, "bf16", "bf16", True, False),
        # fp16, a width that is no multiple of 8
        _norm8("norm8_ragged_5003", 5003, 1030, "fp16", "fp32", False, False, 1e-5),
        # one token, one adapter
        _adapters("adapters_decode_1", 1, 1, 4096, 4096, 64, 16, "bf16", True),
        # a decode batch of 64 requests with 64 adapters to choose from, some with none
        _adapters("adapters_decode_64", 64, 64, 4096, 2048, 64, 16, "bf16", True, 0.1),
        # a prefill of twelve requests
        _adapters("adapters_prefill_8192", 8192, 12, 4096, 4096, 8, 64, "bf16", True, 0.0, 128),
        # many short prompts
        _adapters("adapters_mixed_2048", 2048, 100, 4096, 1024, 100, 32, "bf16", True, 0.05, 32),
        # fp16, odd sizes, half of the requests without an adapter, the adapters' part alone
        _adapters("adapters_ragged_1027", 1027, 40, 1030, 1001, 60, 12, "fp16", False, 0.5, 64),
    ]


def _log(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def _odd(rng, n, step):
    """n as it is, or the multiple of `step` below it: half of the sizes are round ones."""
    return n if rng.random() < 0.5 else max(step, n // step * step)


def draw(rng):
    kind = rng.choice(["norm", "norm8", "adapters"])
    if kind == "adapters":
        T = _odd(rng, _log(rng, 1, 16384), 64)
        H, N = _odd(rng, _log(rng, 64, 8192), 64), _odd(rng, _log(rng, 64, 8192), 64)
        n, r = _log(rng, 1, 512), rng.choice([8, 16, 32, 64, 128, _log(rng, 1, 128)])
        while n * r * (H + N) > 2 ** 28:
            n = max(1, n // 2)
        while T * r * (H + N) > 2 ** 33:
            T = max(1, T // 2)
        requests = T if rng.random() < 0.3 else rng.randint(1, min(T, 64))
        case = _adapters("", T, requests, H, N, n, r, rng.choice(["bf16", "bf16", "fp16"]), rng.random() < 0.8,
                         rng.choice([0.0, 0.1, 0.5]), rng.choice([16, 32, 64, 128]))
    else:
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        weights = rng.choice([dtype, "fp32"])
        T, H = _odd(rng, _log(rng, 1, 262144), 64), _odd(rng, _log(rng, 64, 16384), 64)
        while T * H * _BYTES[dtype] > 2 ** 28:
            T = max(1, T // 2)
        make = _norm if kind == "norm" else _norm8
        case = make("", T, H, dtype, weights, rng.random() < 0.5, rng.random() < 0.5, rng.choice([1e-6, 1e-5]))
    del case["name"]
    return case


def _num_rows(case):
    """Rows that hold every load: each adapter that has any is padded by less than `align`."""
    T, align = case["T"], case["align"]
    return (T + min(case["n"], T) * (align - 1)) // align * align


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=case["dtype"]):
        return torch.randn(shape, generator=gen, device="cuda").to(_TYPES[dtype])

    T, H = case["T"], case["H"]
    loud = 1 + 9 * (torch.rand(H, generator=gen, device="cuda") < 0.01).float()
    s = {"case": case, "x": (torch.randn(T, H, generator=gen, device="cuda") * loud).to(_TYPES[case["dtype"]])}
    if case["kind"] == "adapters":
        n, r, N = case["n"], case["r"], case["N"]
        s["a"] = (torch.randn(n, r, H, generator=gen, device="cuda") * H ** -0.5).to(s["x"].dtype)
        s["b"] = (torch.randn(n, N, r, generator=gen, device="cuda") * 0.3 * r ** -0.5).to(s["x"].dtype)
        s["scale"] = 2.0 ** torch.randint(-1, 3, (n,), generator=gen, device="cuda").float()
        s["base"] = normal(T, N) if case["base"] else None
        # every request has a token; the other boundaries between requests are drawn
        cuts = torch.zeros(T, dtype=torch.int64, device="cuda")
        cuts[1:][torch.randperm(T - 1, generator=gen, device="cuda")[:case["requests"] - 1]] = 1
        adapter = torch.randint(0, n, (T,), generator=gen, device="cuda")
        none = torch.rand(T, generator=gen, device="cuda") < case["dropped"]
        s["idx"] = torch.where(none, -1, adapter)[cuts.cumsum(0)].to(torch.int32)
        s["perm"] = _permutation(s["idx"], n, case["align"], _num_rows(case))
        return s
    train = case.get("train", False)
    s["x"].requires_grad_(train)
    s["residual"] = normal(T, H).requires_grad_(train) if case["residual"] else None
    s["weight"] = (1 + 0.1 * torch.randn(H, generator=gen, device="cuda")).to(_TYPES[case["weights"]]).requires_grad_(train)
    s["dy"] = normal(T, H) if train else None
    s["dh"] = normal(T, H) if train and case["residual"] else None
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _permutation(idx, n, align, rows):
    """The tokens sorted by adapter, in the order of the tokens; an adapter's rows start at a multiple of `align`.  -1 stands for a
    token without an adapter and for a row without a token."""
    T, dev = idx.numel(), idx.device
    key = torch.where(idx >= 0, idx.long(), n)
    order = torch.argsort(key, stable=True)
    count = torch.zeros(n + 1, dtype=torch.int64, device=dev).scatter_add_(0, key, torch.ones_like(key))
    padded = (count + align - 1) // align * align
    first, start = padded.cumsum(0) - padded, count.cumsum(0) - count
    adapter = key[order]
    row = torch.where(adapter < n, first[adapter] + torch.arange(T, device=dev) - start[adapter], rows)
    token_row = torch.full((T,), -1, dtype=torch.int64, device=dev).scatter(0, order, torch.where(adapter < n, row, -1))
    row_token = torch.full((rows + 1,), -1, dtype=torch.int64, device=dev).scatter(0, row, order)[:rows]
    i32 = torch.int32
    return {"expert_frequency": count[:n].to(i32), "expert_frequency_offset": first.to(i32), "x_gather_idx": row_token.to(i32),
            "s_scatter_idx": row_token.to(i32), "s_reverse_scatter_idx": token_row.to(i32).view(T, 1)}


def _normed(s):
    """(h in the type of x, its fp32 values, 1 / sqrt(mean(h^2) + eps) in fp32)"""
    x = s["x"].detach()
    h = x if s["residual"] is None else (x.float() + s["residual"].detach().float()).to(x.dtype)
    f = h.float()
    return h, f, torch.rsqrt((f * f).mean(-1, keepdim=True) + s["case"]["eps"])


def _plain_norm(s):
    h, f, r = _normed(s)
    w = s["weight"].detach().float()
    out = {"y": (f * r * w).to(h.dtype)}
    if s["residual"] is not None:
        out["h"] = h
    if s["case"]["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = r * (g - f * r * (g * f * r).mean(-1, keepdim=True))
        if s["residual"] is not None:
            dx = dx + s["dh"].float()
            out["dresidual"] = dx.to(h.dtype)
        out["dx"] = dx.to(h.dtype)
        out["dweight"] = (dy * f * r).sum(0).to(s["weight"].dtype)
    return out


def _values(q, scale):
    """What 8-bit rows stand for; 8 bits fit into a bf16 value."""
    return torch.mul(q, scale.unsqueeze(1), out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))


def _plain_norm8(s):
    h, f, r = _normed(s)
    y = f * r * s["weight"].float()
    amax = y.abs().amax(-1, keepdim=True)
    some = torch.where(amax > 0, amax, 1.0)
    q = torch.round(y.double() * 127 / some.double()).to(torch.int8)  # quotients next to a border in 64 bits
    scale = torch.where(amax > 0, amax / 127, 1.0).squeeze(1)
    out = {"values": _values(q, scale), "scale": scale}
    if s["residual"] is not None:
        out["h"] = h
    if s["case"]["keep"]:
        out["y"] = y.to(h.dtype)
    return out


def _plain_adapters(s):
    case, p, x = s["case"], s["perm"], s["x"]
    align, n = case["align"], case["n"]
    token = p["x_gather_idx"].long()
    rows = torch.where((token >= 0).unsqueeze(1), x[token.clamp_min(0)].float(), 0.0).view(-1, align, case["H"])
    # the adapter of every `align` rows: the last that begins there or before; what lies behind the last row is zeros
    start = torch.arange(rows.shape[0], device=x.device) * align
    e = (torch.searchsorted(p["expert_frequency_offset"].long(), start, right=True) - 1).clamp(0, n - 1)
    t = torch.bmm(rows, s["a"][e].float().transpose(1, 2))
    delta = torch.bmm(t, s["b"][e].float().transpose(1, 2)) * s["scale"][e].view(-1, 1, 1)
    row = p["s_reverse_scatter_idx"].view(-1).long()
    mine = torch.where((row >= 0).unsqueeze(1), delta.view(-1, case["N"])[row.clamp_min(0)], 0.0)
    return (mine if s["base"] is None else s["base"].float() + mine).to(x.dtype)


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
    if case["kind"] == "norm":
        if s["residual"] is None:
            y, h = sonicmoe.rms_norm(s["x"], s["weight"], case["eps"]), None
            out = {"y": y.detach()}
        else:
            y, h = sonicmoe.rms_norm(s["x"], s["weight"], case["eps"], residual=s["residual"])
            out = {"y": y.detach(), "h": h.detach()}
        if case["train"] and h is None:
            out["dx"], out["dweight"] = torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"])
        elif case["train"]:
            out["dx"], out["dresidual"], out["dweight"] = torch.autograd.grad(
                (y, h), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dh"]))
        return out
    if case["kind"] == "norm8":
        r = sonicmoe.rms_norm_quantize(s["x"], s["weight"], case["eps"], residual=s["residual"], keep_y=case["keep"])
        out = {"values": _values(r.q, r.scale), "scale": r.scale}
        if r.h is not None:
            out["h"] = r.h
        if r.y is not None:
            out["y"] = r.y
        return out
    p = sonicmoe.TokenPermutation(**s["perm"], align=case["align"])
    return sonicmoe.adapter_linear(s["x"], s["a"], s["b"], p, base=s["base"], scale=s["scale"])


def run(state):
    if own:
        return _own(state)
    plain = {"norm": _plain_norm, "norm8": _plain_norm8, "adapters": _plain_adapters}
    with torch.no_grad():
        return plain[state["case"]["kind"]](state)


def work(case):
    T, H = case["T"], case["H"]
    size = _BYTES[case["dtype"]]
    if case["kind"] == "adapters":
        n, r, N = case["n"], case["r"], case["N"]
        kept = T * (1 - case["dropped"])
        used = n * (1 - (1 - 1 / n) ** (case["requests"] * (1 - case["dropped"])))  # adapters that a request has
        return {"bytes": size * (kept * H + T * N * (2 if case["base"] else 1) + used * r * (H + N)) + 8 * T,
                "flops": 2 * kept * r * (H + N)}
    row, weight = T * H * size, H * _BYTES[case["weights"]]
    both = 2 if case["residual"] else 1  # x and the residual in; h out beside y
    if case["kind"] == "norm8":
        return {"bytes": row * (both + (1 if case["residual"] else 0) + (1 if case["keep"] else 0)) + T * H + 4 * T + weight,
                "flops": 6 * T * H}
    if not case["train"]:
        return {"bytes": row * 2 * both + weight, "flops": 5 * T * H}
    # the upstream gradients and h in once more, the gradient of x (which is the residual's) and of the weight out
    return {"bytes": row * (2 * both + both + 2) + 3 * weight, "flops": 16 * T * H}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_adapters(s):
    out = torch.zeros(s["case"]["T"], s["case"]["N"], dtype=torch.float64, device="cuda") if s["base"] is None else s["base"].double()
    for e in torch.unique(s["idx"]).tolist():
        if e >= 0:
            mine = torch.nonzero(s["idx"] == e).reshape(-1)
            low = torch.einsum("th,rh->tr", s["x"][mine].double(), s["a"][e].double())
            out.index_add_(0, mine, s["scale"][e].double() * torch.einsum("tr,nr->tn", low, s["b"][e].double()))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "adapters":
            return _exact_adapters(s)
        h = s["x"].detach().double()
        if s["residual"] is not None:  # the rows that are kept, and normalised, have the type of x
            h = (h + s["residual"].detach().double()).to(s["x"].dtype).double()
        w = s["weight"].detach().double()
        root = torch.sqrt(torch.linalg.vector_norm(h, dim=1).square() / case["H"] + case["eps"]).unsqueeze(1)
        unit = h / root
        y = unit * w
        out = {"h": h} if s["residual"] is not None else {}
        if case["kind"] == "norm8":
            scale = torch.linalg.vector_norm(y, ord=float("inf"), dim=1) / 127
            scale = torch.where(scale == 0, torch.ones_like(scale), scale)
            out.update(values=torch.round(y / scale.unsqueeze(1)) * scale.unsqueeze(1), scale=scale)
            if case["keep"]:
                out["y"] = y
            return out
        out["y"] = y
        if case["train"]:
            g = s["dy"].double()
            out["dweight"] = torch.einsum("th,th->h", g, unit)
            g = g * w
            along = torch.einsum("th,th->t", g, unit).unsqueeze(1) / case["H"]
            out["dx"] = (g - unit * along) / root
            if s["residual"] is not None:
                out["dx"] = out["dx"] + s["dh"].double()
                out["dresidual"] = out["dx"]
        return out
