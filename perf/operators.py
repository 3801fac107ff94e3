"""What the operators around the quantised matmuls cost: cases over their real range, their inputs, one pass through
each, and what a pass cannot do without.

Four kinds of case:

* ``norm``      residual addition, root-mean-square norm and quantisation of the result: to int8 with one scale per token
                (the A operand of the W8A8 matmuls) or to fp8 with one E8M0 scale per 32 elements (the A operand of the
                MX matmuls);
* ``dispatch``  tokens sorted by expert, and their rows and scales copied into expert order (the A operand of the grouped
                matmuls);
* ``combine``   the experts' rows brought back to their tokens and added up with the router's weights, and ``grad``, the
                gradient of that step;
* ``adapter``   low-rank adapters of many requests at once, added to the result of a shared projection.

``own`` False computes them in elementary torch operations in 32 bits, ``own`` True through ``asc_devkit_b200.ops``."""
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_FP8 = {"e4m3": (torch.float8_e4m3fn, 8, 448.0, 3, -6), "e5m2": (torch.float8_e5m2, 15, 57344.0, 2, -14)}
_EPS = 1e-6


def listed():
    return [
        # one decode step of one request: the call's own latency
        {"name": "norm_i8_one_token", "kind": "norm", "M": 1, "N": 4096, "dtype": "bf16", "out": "i8", "residual": True},
        # a batch of requests of uneven lengths in front of a W8A8 matmul; first layer: nothing to add yet
        {"name": "norm_i8_ragged_batch", "kind": "norm", "M": 1031, "N": 5120, "dtype": "f16", "out": "i8", "residual": False},
        # a long prompt in front of an MX matmul
        {"name": "norm_mx_prompt", "kind": "norm", "M": 16384, "N": 7168, "dtype": "bf16", "out": "e4m3", "residual": True},
        # a decode step of sixteen requests over many experts: most experts get no token or one
        {"name": "dispatch_few_tokens", "kind": "dispatch", "T": 16, "k": 8, "E": 256, "held": 256, "H": 7168, "rows": "i8"},
        # a prompt on the way to the grouped W8A8 matmul
        {"name": "dispatch_prompt", "kind": "dispatch", "T": 8192, "k": 8, "E": 128, "held": 128, "H": 7168, "rows": "i8"},
        # the way back of a decode step on a rank that holds an eighth of the experts
        {"name": "combine_few_tokens", "kind": "combine", "T": 16, "k": 8, "E": 256, "held": 32, "H": 7168, "dtype": "bf16"},
        # the way back of a prompt
        {"name": "combine_prompt", "kind": "combine", "T": 8192, "k": 8, "E": 128, "held": 128, "H": 7168, "dtype": "bf16"},
        # a training step on sequences of odd lengths, a rank with half of the experts
        {"name": "grad_ragged_share", "kind": "grad", "T": 1021, "k": 4, "E": 64, "held": 32, "H": 2056, "dtype": "f16"},
        # a training step on a full batch
        {"name": "grad_batch", "kind": "grad", "T": 8192, "k": 8, "E": 64, "held": 64, "H": 4096, "dtype": "bf16"},
        # a decode step: thirty-two requests, most with adapters of their own
        {"name": "adapter_decode", "kind": "adapter", "M": 32, "K": 4096, "N": 4096, "r": 16, "L": 16, "span": 1, "dtype": "bf16"},
        # prompts of uneven lengths beside a down projection
        {"name": "adapter_ragged", "kind": "adapter", "M": 1337, "K": 11008, "N": 4096, "r": 32, "L": 8, "span": 97, "dtype": "f16"},
        # long prompts beside a square projection
        {"name": "adapter_prompts", "kind": "adapter", "M": 8192, "K": 4096, "N": 4096, "r": 64, "L": 16, "span": 700, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is uniform."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(["norm", "norm", "dispatch", "dispatch", "combine", "grad", "adapter", "adapter"])
    dtype = rng.choice(["bf16", "f16"])
    if kind == "norm":
        out = rng.choice(["i8", "e4m3", "e5m2"])
        n = _spread(rng, 2, 256) * 32 if out != "i8" else _spread(rng, 64, 8192)
        m = _spread(rng, 1, min(16384, 16384 * 7168 // n))
        return {"kind": kind, "M": m, "N": n, "dtype": dtype, "out": out, "residual": rng.random() < 0.75}
    if kind == "adapter":
        r = rng.choice([8, 16, 24, 32, 64, 128])
        lo, k, n = _spread(rng, 1, 64), _spread(rng, 64, 1376) * 8, _spread(rng, 64, 1376) * 8
        most = 8192 * 16 * 64 * 8192 // (lo * r * (k + n))
        m = _spread(rng, 1, max(1, min(8192, most)))
        return {"kind": kind, "M": m, "K": k, "N": n, "r": r, "L": lo, "span": rng.choice([1, _spread(rng, 1, 1024)]), "dtype": dtype}
    e = rng.choice([8, 16, 60, 64, 128, 256])
    k = rng.randint(1, 8)
    h = _spread(rng, 32, 1024) * 8 if rng.random() < 0.8 else _spread(rng, 256, 8192)
    t = _spread(rng, 1, max(1, min(8192, 8192 * 8 * (4096 if kind == "grad" else 7168) // (k * h))))
    case = {"kind": kind, "T": t, "k": k, "E": e, "held": rng.choice([e, e, max(1, e // rng.choice([2, 4, 8]))]), "H": h}
    return case | ({"rows": rng.choice(["i8", "bf16"])} if kind == "dispatch" else {"dtype": dtype})


# ---- inputs ------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _route(g, case):
    """The router's choice: k different experts a token, some experts more popular than others; -1 = held elsewhere."""
    logits = _randn(g, case["T"], case["E"]) + 0.5 * _randn(g, 1, case["E"])
    best, ids = torch.topk(logits, min(case["k"], case["E"]), dim=-1)
    return torch.where(ids < case["held"], ids, -1), torch.softmax(best, dim=-1)


def _sorted(ids, experts):
    """The slots (token * k + choice) in order of expert, equal ones in their own order; kept = the slots with an expert here."""
    flat = ids.reshape(-1)
    valid = (flat >= 0) & (flat < experts)
    order = torch.sort(torch.where(valid, flat, experts), stable=True).indices
    kept = valid.sum()
    at = torch.arange(flat.numel(), device=flat.device)
    row_of_slot = torch.empty_like(at).scatter_(0, order, at)
    row_of_slot = torch.where(valid, row_of_slot, -1).to(torch.int32).reshape(ids.shape)
    slot_of_row = torch.where(at < kept, order, -1).to(torch.int32)
    counts = (flat[:, None] == torch.arange(experts, device=flat.device)).sum(0)
    return counts, slot_of_row, row_of_slot


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["kind"] == "norm":
        dt, m, n = _TYPES[case["dtype"]], case["M"], case["N"]
        s["x"] = _randn(g, m, n, dtype=dt, scale=0.7)
        # a residual stream has channels that stand out
        s["res"] = (_randn(g, m, n, scale=1.5) * torch.exp(0.7 * _randn(g, 1, n))).to(dt) if case["residual"] else None
        s["gamma"] = (1.0 + _randn(g, n, scale=0.2)).to(dt)
        s["sum"] = torch.empty_like(s["x"]) if case["residual"] else None
        s["q"] = torch.empty(m, n, dtype=torch.int8 if case["out"] == "i8" else torch.uint8, device="cuda")
        s["scale"] = torch.empty(m, dtype=torch.float32, device="cuda") if case["out"] == "i8" else torch.empty(m, n // 32, dtype=torch.uint8, device="cuda")
        s["values"] = torch.empty(m, n, dtype=dt, device="cuda") if case["out"] == "i8" else None
        return s
    if case["kind"] == "adapter":
        dt, m, n, k, r, lo = _TYPES[case["dtype"]], case["M"], case["N"], case["K"], case["r"], case["L"]
        s["x"] = _randn(g, m, k, dtype=dt)
        s["base"] = _randn(g, m, n, dtype=dt)
        s["a"] = _randn(g, lo, r, k, dtype=dt, scale=k ** -0.5)
        s["b"] = _randn(g, lo, n, r, dtype=dt, scale=r ** -0.5)
        s["scale"] = 0.5 + torch.rand(lo, generator=g, device="cuda")
        requests = -(-m // case["span"])
        ids = torch.randint(-1 if lo > 1 else 0, lo, (requests,), generator=g, device="cuda", dtype=torch.int32)
        s["ids"] = ids.repeat_interleave(case["span"])[:m].contiguous()
        s["y"] = torch.empty(m, n, dtype=dt, device="cuda")
        return s
    ids, weights = _route(g, case)
    t, k, h = ids.shape[0], ids.shape[1], case["H"]
    if case["kind"] == "dispatch":
        s["ids"] = ids
        if case["rows"] == "i8":
            s["x"] = torch.randint(-127, 128, (t, h), generator=g, device="cuda", dtype=torch.int8)
            s["x_scale"] = 0.005 + 0.015 * torch.rand(t, generator=g, device="cuda")
            s["row_scale"] = torch.zeros(t * k, device="cuda")
        else:
            s["x"], s["x_scale"], s["row_scale"] = _randn(g, t, h, dtype=torch.bfloat16), None, None
        s["rows"] = torch.zeros(t * k, h, dtype=s["x"].dtype, device="cuda")
        s["counts"] = torch.empty(case["held"], dtype=torch.int64, device="cuda")
        s["slot_of_row"] = torch.empty(t * k, dtype=torch.int32, device="cuda")
        s["row_of_slot"] = torch.empty(t, k, dtype=torch.int32, device="cuda")
        return s
    dt = _TYPES[case["dtype"]]
    _, s["slot_of_row"], s["row_of_slot"] = _sorted(ids, case["held"])
    s["weights"] = weights
    s["y"] = _randn(g, t * k, h, dtype=dt)
    if case["kind"] == "combine":
        s["out"] = torch.empty(t, h, dtype=dt, device="cuda")
    else:
        s["d_out"] = _randn(g, t, h, dtype=dt, scale=0.1)
        s["d_y"] = torch.zeros(t * k, h, dtype=dt, device="cuda")
        s["d_weights"] = torch.empty(t, k, dtype=torch.float32, device="cuda")
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------
def _norm_plain(s):
    h = s["x"].float() + s["res"].float() if s["residual"] else s["x"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + _EPS) * s["gamma"].float()
    total = h.to(s["x"].dtype) if s["residual"] else None
    if s["out"] == "i8":
        amax = y.abs().amax(-1, keepdim=True)
        scale = torch.where(amax > 0, amax / 127.0, 1.0)
        q = torch.round(y * torch.where(amax > 0, 127.0 / amax, 1.0)).clamp(-128, 127)
        return [(q * scale).to(s["x"].dtype), scale[:, 0], total]
    kind, top, largest, _, _ = _FP8[s["out"]]
    blocks = y.reshape(s["M"], s["N"] // 32, 32)
    amax = blocks.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 1 - top, 0).clamp(-127, 127)
    q = torch.ldexp(blocks, -e).clamp(-largest, largest).to(kind)
    return [q.reshape(s["M"], s["N"]), (e[..., 0] + 127).to(torch.uint8).view(torch.float8_e8m0fnu), total]


def _norm_own(ops, L, s):
    code = {"i8": L.DT_I8, "e4m3": L.DT_FP8_E4M3, "e5m2": L.DT_FP8_E5M2}[s["out"]]
    ops.ResidualRmsNormQuant(s["q"], s["scale"], s["x"], s["gamma"], _EPS, residual=s["res"], residualOut=s["sum"], dst_dtype=code)
    if s["out"] == "i8":
        return [torch.mul(s["q"], s["scale"][:, None], out=s["values"]), s["scale"], s["sum"]]
    return [s["q"].view(_FP8[s["out"]][0]), s["scale"].view(torch.float8_e8m0fnu), s["sum"]]


def _dispatch_plain(s):
    counts, slot_of_row, row_of_slot = _sorted(s["ids"], s["held"])
    kept = slot_of_row >= 0
    token = slot_of_row.clamp(min=0) // s["ids"].shape[1]
    rows = torch.where(kept[:, None], s["x"][token], s["rows"])
    scale = torch.where(kept, s["x_scale"][token], s["row_scale"]) if s["x_scale"] is not None else None
    return [counts, slot_of_row, row_of_slot, rows, scale]


def _dispatch_own(ops, s):
    ops.ExpertSort(s["counts"], s["row_of_slot"], s["ids"], slotOfRow=s["slot_of_row"])
    ops.ExpertDispatch(s["rows"], s["x"], s["row_of_slot"], dstScale=s["row_scale"], srcScale=s["x_scale"])
    return [s["counts"], s["slot_of_row"], s["row_of_slot"], s["rows"], s["row_scale"]]


def _combine_plain(s):
    here = s["row_of_slot"] >= 0
    rows = s["y"].float()[s["row_of_slot"].clamp(min=0).long()]
    return (rows * torch.where(here, s["weights"], 0.0)[..., None]).sum(1).to(s["y"].dtype)


def _grad_plain(s):
    here = s["row_of_slot"] >= 0
    d_out = s["d_out"].float()
    rows = s["y"].float()[s["row_of_slot"].clamp(min=0).long()]
    d_weights = torch.where(here, (rows * d_out[:, None]).sum(-1), 0.0)
    kept, slot = s["slot_of_row"] >= 0, s["slot_of_row"].clamp(min=0).long()
    d_y = s["weights"].reshape(-1)[slot][:, None] * d_out[slot // s["row_of_slot"].shape[1]]
    return [torch.where(kept[:, None], d_y.to(s["y"].dtype), s["d_y"]), d_weights]


def _adapter_plain(s):
    m, lo, r = s["M"], s["L"], s["r"]
    inner = (s["x"].float() @ s["a"].float().reshape(lo * r, -1).T).reshape(m, lo, r)
    mine = s["ids"][:, None] == torch.arange(lo, device="cuda")
    inner = torch.where(mine[..., None], inner * s["scale"][:, None], 0.0).reshape(m, lo * r)
    return (s["base"].float() + inner @ s["b"].float().permute(0, 2, 1).reshape(lo * r, -1)).to(s["base"].dtype)


def run(state):
    s = state
    if own:
        from asc_devkit_b200 import _lib, ops
        if s["kind"] == "norm":
            return _norm_own(ops, _lib, s)
        if s["kind"] == "dispatch":
            return _dispatch_own(ops, s)
        if s["kind"] == "combine":
            return ops.ExpertCombine(s["out"], s["y"], s["row_of_slot"], s["weights"])
        if s["kind"] == "grad":
            ops.ExpertCombineGrad(s["d_y"], s["d_weights"], s["d_out"], s["y"], s["row_of_slot"], s["weights"])
            return [s["d_y"], s["d_weights"]]
        return ops.LowRankAdd(s["y"], s["base"], s["x"], s["a"], s["b"], s["ids"], scale=s["scale"])
    return {"norm": _norm_plain, "dispatch": _dispatch_plain, "combine": _combine_plain, "grad": _grad_plain, "adapter": _adapter_plain}[s["kind"]](s)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "norm":
        e = c["M"] * c["N"]
        scales = c["M"] * 4 if c["out"] == "i8" else e // 32
        return {"bytes": e * (7 if c["residual"] else 3) + scales + 2 * c["N"], "flops": e * (8 if c["residual"] else 7)}
    if c["kind"] == "adapter":
        m, k, n, r = c["M"], c["K"], c["N"], c["r"]
        return {"bytes": 2 * m * (k + 2 * n) + 2 * min(c["L"], -(-m // c["span"])) * r * (k + n) + 4 * m, "flops": 2 * m * r * (k + n)}
    t, k, h = c["T"], min(c["k"], c["E"]), c["H"]
    rows = t * k * c["held"] / c["E"]  # slots whose expert is held here
    if c["kind"] == "dispatch":
        size = 1 if c["rows"] == "i8" else 2
        tokens = t * (1 - (1 - c["held"] / c["E"]) ** k)
        return {"bytes": (tokens + rows) * (h * size + (4 if size == 1 else 0)) + t * k * 16 + c["held"] * 8, "flops": 0}
    if c["kind"] == "combine":
        return {"bytes": (rows + t) * h * 2 + t * k * 8, "flops": 2 * rows * h}
    return {"bytes": (2 * rows + t) * h * 2 + t * k * 12, "flops": 3 * rows * h}


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        h = s["x"].double()
        if case["residual"]:
            h += s["res"].double()
        y = (h / (h.square().sum(1, keepdim=True) / case["N"] + _EPS).sqrt()).mul_(s["gamma"].double())
        total = h if case["residual"] else None
        if case["out"] == "i8":
            step = y.abs().max(1, keepdim=True).values / 127
            step[step == 0] = 1
            return [(y / step).round_().clamp_(-128, 127).mul_(step), step[:, 0], total]
        _, top, largest, digits, lowest = _FP8[case["out"]]
        y = y.reshape(case["M"], -1, 32)
        amax = y.abs().max(2, keepdim=True).values
        unit = torch.where(amax > 0, torch.exp2(torch.floor(torch.log2(amax)) - top), 1).clamp_(2.0 ** -127, 2.0 ** 127)
        v = (y / unit).clamp_(-largest, largest)
        grain = torch.exp2(torch.floor(torch.log2(v.abs().clamp_(min=2.0 ** lowest))) - digits)
        return [(v / grain).round_().mul_(grain).reshape(case["M"], -1), unit[..., 0], total]
    if case["kind"] == "dispatch":
        return None  # nothing is computed: rows, scales and whole numbers
    if case["kind"] == "adapter":
        y = s["base"].double()
        for a in range(case["L"]):
            at = (s["ids"] == a).nonzero()[:, 0]
            inner = torch.einsum("mk,rk->mr", s["x"][at].double(), s["a"][a].double())
            y[at] += s["scale"][a].double() * torch.einsum("mr,nr->mn", inner, s["b"][a].double())
        return y
    w = s["weights"].double()
    if case["kind"] == "combine":
        out = torch.zeros(w.shape[0], case["H"], dtype=torch.float64, device="cuda")
        for j in range(w.shape[1]):
            at = (s["row_of_slot"][:, j] >= 0).nonzero()[:, 0]
            out[at] += w[at, j, None] * s["y"][s["row_of_slot"][at, j].long()].double()
        return out
    d_y, d_w, d_out = s["d_y"].double(), torch.zeros_like(w), s["d_out"].double()
    for j in range(w.shape[1]):
        at = (s["row_of_slot"][:, j] >= 0).nonzero()[:, 0]
        row = s["row_of_slot"][at, j].long()
        d_y[row] = w[at, j, None] * d_out[at]
        d_w[at, j] = torch.einsum("th,th->t", s["y"][row].double(), d_out[at])
    return [d_y, d_w]
