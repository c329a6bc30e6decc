"""The feed-forward products of a transformer layer, dense and by expert, forward and backward: what is measured.

Four operators, each in its plain form (elementary torch operations in 32 bits, one rounding at the end) and as the
library offers it (``own``):

* ``linear``            C = act(A B^T + bias) + residual, optionally with Z = A B^T + bias beside it
* ``linear_backward``   dZ = dC * act'(Z);  dA = dZ B,  dB = dZ^T A,  dbias = column sums of dZ
* ``grouped``           rows [offsets[g], offsets[g+1]) of C = act(those rows of A times B_g^T + bias_g)
* ``grouped_backward``  the same gradients, group by group; a group without rows has a gradient of zero

A is [M, K], B is [N, K] (a stack [G, N, K] for the grouped forms), C is [M, N], all row-major. Rows of A behind
the last group belong to nobody: the rows of C and dA at those places keep what they held.
"""
from __future__ import annotations

import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")

# The most work a drawn case may have, that of the largest listed case, and the most weights it may hold.
MOST_FLOPS = 3.84e12
MOST_BYTES = 3.0e9
MOST_WEIGHTS = 1.0e9


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token through a small projection: nothing but latency
        {"name": "linear_1x1024x1024", "op": "linear", "m": 1, "n": 1024, "k": 1024, "type": "f16", "out": "f16",
         "act": "gelu", "bias": True, "residual": True, "pre": False},
        # a decode batch through the up projection: the weights stream from HBM once
        {"name": "linear_decode_16x14336x4096", "op": "linear", "m": 16, "n": 14336, "k": 4096, "type": "bf16",
         "out": "bf16", "act": "silu", "bias": True, "residual": False, "pre": False},
        # a ragged chunk of a prompt, odd in every size, kept in 32 bits for what adds to it
        {"name": "linear_odd_777x4099x2056", "op": "linear", "m": 777, "n": 4099, "k": 2056, "type": "f16", "out": "f32",
         "act": "none", "bias": True, "residual": True, "pre": False},
        # a training step's up projection, which keeps its pre-activation for the way back
        {"name": "linear_train_8192x14336x4096", "op": "linear", "m": 8192, "n": 14336, "k": 4096, "type": "bf16",
         "out": "bf16", "act": "gelu_tanh", "bias": True, "residual": False, "pre": True},
        # the gradients of a small layer, a short sequence
        {"name": "linear_backward_512x1024x1024", "op": "linear_backward", "m": 512, "n": 1024, "k": 1024, "type": "f16",
         "dweight": "f16", "act": "relu"},
        # no activation, sizes that fill no tile, the weight's gradient in 32 bits
        {"name": "linear_backward_odd_1333x4104x2040", "op": "linear_backward", "m": 1333, "n": 4104, "k": 2040,
         "type": "bf16", "dweight": "f32", "act": "none"},
        # the gradients of the training step above
        {"name": "linear_backward_8192x14336x4096", "op": "linear_backward", "m": 8192, "n": 14336, "k": 4096,
         "type": "bf16", "dweight": "bf16", "act": "gelu_tanh"},
        # decode with eight large experts: eight tokens, two experts each; the weights of the experts that were chosen
        {"name": "grouped_decode_16_of_8x14336x4096", "op": "grouped", "rows": 16, "groups": 8, "n": 14336, "k": 4096,
         "type": "bf16", "act": "silu", "bias": False, "pre": False, "skew": 0.5, "empty": 1, "behind": 0},
        # decode with many small experts, a few rows each, several without any
        {"name": "grouped_decode_48_of_64x1024x2048", "op": "grouped", "rows": 48, "groups": 64, "n": 1024, "k": 2048,
         "type": "f16", "act": "none", "bias": False, "pre": False, "skew": 0.3, "empty": 20, "behind": 3},
        # a training step's tokens over eight experts, unevenly, with padding rows behind
        {"name": "grouped_train_16384_of_8x14336x4096", "op": "grouped", "rows": 16384, "groups": 8, "n": 14336, "k": 4096,
         "type": "bf16", "act": "gelu_tanh", "bias": True, "pre": True, "skew": 0.4, "empty": 0, "behind": 37},
        # the gradients of many small experts, one of which saw nothing; the weights' gradient in 32 bits
        {"name": "grouped_backward_4096_of_32x1024x2048", "op": "grouped_backward", "rows": 4096, "groups": 32, "n": 1024,
         "k": 2048, "type": "f16", "dweight": "f32", "act": "none", "skew": 0.6, "empty": 1, "behind": 5},
        # the gradients of the training step over eight experts
        {"name": "grouped_backward_16384_of_8x14336x4096", "op": "grouped_backward", "rows": 16384, "groups": 8,
         "n": 14336, "k": 4096, "type": "bf16", "dweight": "bf16", "act": "silu", "skew": 0.4, "empty": 0, "behind": 37},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _eights(rng, lo, hi):
    """A multiple of eight, as the row pitch of an operand that is read in 16-byte pieces has to be."""
    return max(lo, 8 * int(round(_log_int(rng, lo, hi) / 8)))


def draw(rng):
    while True:
        op = rng.choice(("linear", "linear_backward", "grouped", "grouped_backward"))
        dtype = rng.choice(("f16", "bf16"))
        act = rng.choice(ACTS)
        k = _eights(rng, 64, 14336)
        if op.startswith("linear"):
            case = {"op": op, "m": _log_int(rng, 1, 8192), "n": _eights(rng, 64, 14336), "k": k, "type": dtype, "act": act}
        else:
            groups = _log_int(rng, 1, 128)
            case = {"op": op, "rows": _log_int(rng, 1, 16384), "groups": groups, "n": _eights(rng, 64, 14336), "k": k,
                    "type": dtype, "act": act, "skew": round(rng.uniform(0.0, 1.2), 2),
                    "empty": rng.randrange(0, max(1, groups // 2) + 1) if groups > 1 else 0, "behind": rng.choice((0, 0, 1, 19, 200))}
        if op in ("linear", "grouped"):
            if rng.random() < 0.4:
                case["n"] += rng.randrange(1, 8)  # the output's width is free
            case["bias"] = rng.random() < 0.6
            case["pre"] = rng.random() < 0.4
            if op == "linear":
                case["out"] = rng.choice((dtype, dtype, "f32"))
                case["residual"] = rng.random() < 0.5
        else:
            # 32-bit gradients are asked for where no 16-bit dZ lies before the product
            case["dweight"] = rng.choice((dtype, "f32")) if act == "none" else dtype
        w = work(case)
        weights = case.get("groups", 1) * case["n"] * case["k"]
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and weights <= MOST_WEIGHTS:
            return case


def _group_sizes(case):
    """Rows of each group, largest first: shares that fall off as a power of the rank, as a router's load does; the
    last ``empty`` groups get none. Which group gets which share is the inputs' business (``prepare``)."""
    live = max(1, case["groups"] - case["empty"])
    weights = [(i + 1.0) ** -case["skew"] for i in range(live)]
    total = sum(weights)
    sizes = [int(case["rows"] * w / total) for w in weights]
    for i in range(case["rows"] - sum(sizes)):
        sizes[i % live] += 1
    return sizes + [0] * (case["groups"] - live)


def work(case):
    b = 2
    n, k = case["n"], case["k"]
    if case["op"] == "linear":
        m, out = case["m"], TYPES[case["out"]].itemsize
        read = b * (m * k + n * k) + (b * n if case["bias"] else 0) + (out * m * n if case["residual"] else 0)
        return {"bytes": read + out * m * n * (2 if case["pre"] else 1), "flops": 2 * m * n * k}
    if case["op"] == "linear_backward":
        m = case["m"]
        read = b * (m * n + m * k + n * k) + (b * m * n if case["act"] != "none" else 0)
        return {"bytes": read + b * m * k + TYPES[case["dweight"]].itemsize * n * k + 4 * n, "flops": 4 * m * n * k}
    rows, groups = case["rows"], case["groups"]
    hit = sum(1 for s in _group_sizes(case) if s > 0)
    if case["op"] == "grouped":
        read = b * (rows * k + hit * n * k) + (b * hit * n if case["bias"] else 0) + 4 * (groups + 1)
        return {"bytes": read + b * rows * n * (2 if case["pre"] else 1), "flops": 2 * rows * n * k}
    read = b * (rows * n + rows * k + hit * n * k) + (b * rows * n if case["act"] != "none" else 0) + 4 * (groups + 1)
    write = b * rows * k + TYPES[case["dweight"]].itemsize * groups * n * k + 4 * groups * n
    return {"bytes": read + write, "flops": 4 * rows * n * k}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _normal(gen, shape, dtype, scale=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 27
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.numel(), generator=gen, device="cuda", dtype=torch.float32).mul_(scale))
    return out


def _inputs(case, seed):
    """Activations ~ N(0, 1), weights ~ N(0, 1/K), gradients of about a hundredth, pre-activations ~ N(0, 1)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op, n, k = TYPES[case["type"]], case["op"], case["n"], case["k"]
    s = {"case": case}
    if op.startswith("linear"):
        rows, stack = case["m"], ()
    else:
        rows, stack = case["rows"] + case["behind"], (case["groups"],)
        order = torch.randperm(case["groups"], generator=gen, device="cuda").tolist()
        sizes = _group_sizes(case)
        bounds = [0]
        for g in order:
            bounds.append(bounds[-1] + sizes[g])
        s["bounds"] = bounds  # the plain form's loop; the library reads the offsets on the device
        s["offsets"] = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    s["A"] = _normal(gen, (rows, k), dtype)
    s["B"] = _normal(gen, stack + (n, k), dtype, 1.0 / math.sqrt(k))
    if op in ("linear", "grouped"):
        out = TYPES[case.get("out", case["type"])]
        s["bias"] = _normal(gen, stack + (n,), dtype, 0.5) if case["bias"] else None
        s["residual"] = _normal(gen, (rows, n), out) if case.get("residual") else None
        s["C"] = torch.zeros((rows, n), dtype=out, device="cuda")
        s["pre"] = torch.zeros((rows, n), dtype=out, device="cuda") if case["pre"] else None
    else:
        s["dC"] = _normal(gen, (rows, n), dtype, 0.01)
        s["pre"] = _normal(gen, (rows, n), dtype) if case["act"] != "none" else None
        s["dA"] = torch.zeros((rows, k), dtype=dtype, device="cuda")
        s["dB"] = torch.zeros(stack + (n, k), dtype=TYPES[case["dweight"]], device="cuda")
        s["dbias"] = torch.zeros(stack + (n,), dtype=torch.float32, device="cuda")
    return s


def prepare(case, seed):
    return _inputs(case, seed)


# ---------------------------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------------------------
def _act(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return 1.0 - (z <= 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * 0.044715 * z * z)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _forward_rows(a, b, bias, residual, act):
    z = a.float() @ b.float().T
    if bias is not None:
        z = z + bias.float()
    c = _act(z, act)
    if residual is not None:
        c = c + residual.float()
    return z, c


def _backward_rows(dc, pre, a, b, act):
    dz = dc.float()
    if act != "none":
        dz = dz * _act_slope(pre.float(), act)
    return dz @ b.float(), dz.T @ a.float(), dz.sum(0)


def _plain(s):
    case = s["case"]
    act = case["act"]
    if case["op"] == "linear":
        z, c = _forward_rows(s["A"], s["B"], s["bias"], s["residual"], act)
        out = TYPES[case["out"]]
        return {"C": c.to(out), "pre": z.to(out)} if case["pre"] else {"C": c.to(out)}
    if case["op"] == "linear_backward":
        da, db, dbias = _backward_rows(s["dC"], s["pre"], s["A"], s["B"], act)
        return {"dA": da.to(s["dA"].dtype), "dB": db.to(s["dB"].dtype), "dbias": dbias}
    bounds = s["bounds"]
    for g in range(case["groups"]):
        lo, hi = bounds[g], bounds[g + 1]
        if case["op"] == "grouped":
            if lo == hi:
                continue
            z, c = _forward_rows(s["A"][lo:hi], s["B"][g], None if s["bias"] is None else s["bias"][g], None, act)
            s["C"][lo:hi] = c.to(s["C"].dtype)
            if case["pre"]:
                s["pre"][lo:hi] = z.to(s["pre"].dtype)
        else:
            pre = None if s["pre"] is None else s["pre"][lo:hi]
            da, db, dbias = _backward_rows(s["dC"][lo:hi], pre, s["A"][lo:hi], s["B"][g], act)
            s["dA"][lo:hi] = da.to(s["dA"].dtype)
            s["dB"][g] = db.to(s["dB"].dtype)
            s["dbias"][g] = dbias
    return _outputs(s)


def _outputs(s):
    if s["case"]["op"] in ("linear", "grouped"):
        return {"C": s["C"], "pre": s["pre"]} if s["case"]["pre"] else {"C": s["C"]}
    return {"dA": s["dA"], "dB": s["dB"], "dbias": s["dbias"]}


# ---------------------------------------------------------------------------------------------------------------
# the library's form
# ---------------------------------------------------------------------------------------------------------------
def _own(s):
    from cuda_hgemm_b200 import api

    case = s["case"]
    if case["op"] == "linear":
        api.hgemm_linear(s["A"], s["B"], s["C"], bias=s["bias"], act=case["act"], residual=s["residual"], pre=s["pre"])
    elif case["op"] == "linear_backward":
        api.hgemm_linear_backward(s["dC"], s["A"], s["B"], act=case["act"], pre=s["pre"], dA=s["dA"], dB=s["dB"],
                                  dbias=s["dbias"])
    elif case["op"] == "grouped":
        api.hgemm_grouped(s["A"], s["B"], s["C"], s["offsets"], bias=s["bias"], act=case["act"], pre=s["pre"])
    else:
        api.hgemm_grouped_backward(s["dC"], s["A"], s["B"], s["offsets"], act=case["act"], pre=s["pre"], dA=s["dA"],
                                   dB=s["dB"], dbias=s["dbias"])
    return _outputs(s)


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _gelu_tanh_parts(z):
    # 0.5 (1 + tanh u) is the logistic function of 2u; both it and its slope follow from there
    c = 2.0 * math.sqrt(2.0 / math.pi)
    gate = torch.sigmoid(c * (z + 0.044715 * z ** 3))
    return gate, gate * (1 - gate) * c * (1 + 0.134145 * z ** 2)


def _exact_act(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0),
            "gelu": lambda: z * torch.special.ndtr(z),
            "gelu_tanh": lambda: z * _gelu_tanh_parts(z)[0],
            "silu": lambda: z * torch.sigmoid(z)}[act]()


def _exact_slope(z, act):
    if act == "relu":
        return torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        gate, slope = _gelu_tanh_parts(z)
        return gate + z * slope
    gate = torch.sigmoid(z)  # silu
    return gate + z * gate * (1 - gate)


def _exact_group(s, rows, a, b, bias, out):
    """One group's results in 64 bits into ``out``: forward a slab of rows at a time, backward in one piece."""
    case, act = s["case"], s["case"]["act"]
    b = b.double()
    if case["op"] in ("linear", "grouped"):
        for lo in range(rows.start, rows.stop, 4096):
            part = slice(lo, min(lo + 4096, rows.stop))
            z = torch.einsum("mk,nk->mn", a[part].double(), b)
            if bias is not None:
                z += bias.double()
            if "pre" in out:
                out["pre"][part] = z
            c = _exact_act(z, act)
            if s["residual"] is not None:
                c = c + s["residual"][part].double()
            out["C"][part] = c
        return None
    dz = s["dC"][rows].double()
    if act != "none":
        dz *= _exact_slope(s["pre"][rows].double(), act)
    out["dA"][rows] = torch.einsum("mn,nk->mk", dz, b)
    return torch.einsum("mn,mk->nk", dz, a[rows].double()), dz.sum(0)


def exact(case, seed):
    s = _inputs(case, seed)
    grouped = not case["op"].startswith("linear")
    out = {name: t.double() for name, t in _outputs(s).items()}  # what lies behind the last group stays
    for g in range(case["groups"] if grouped else 1):
        rows = slice(s["bounds"][g], s["bounds"][g + 1]) if grouped else slice(0, case["m"])
        b = s["B"][g] if grouped else s["B"]
        bias = s.get("bias")
        grads = _exact_group(s, rows, s["A"], b, bias[g] if grouped and bias is not None else bias, out)
        if grads is not None:
            if grouped:
                out["dB"][g], out["dbias"][g] = grads
            else:
                out["dB"], out["dbias"] = grads
    return out
