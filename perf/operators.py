"""The fused linear layer and the grouped (expert) products of arc, as measured cases.

Four operators, each in a plain form (torch, 32 bits) and through the framework:

* linear            y = act(x w^T + bias) + residual, and its gradients
* grouped           rows sorted by expert times that expert's weights, and its gradients
* a8w4_grouped      the same with int8 activations and int4 weights (group-128 scales)
* group_rows        expert ids -> offsets, the row of each place and the place of each choice
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_ACTS = (None, "relu", "gelu", "gelu_tanh", "silu")
_arc_module = None


def _arc():
    """The framework's package, which lies beside this folder in arc-gemm_b200/."""
    global _arc_module
    if _arc_module is None:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "arc-gemm_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        import arc

        _arc_module = arc
    return _arc_module


# ----------------------------------------------------------------------------------
# Cases
# ----------------------------------------------------------------------------------
def _linear(name, m, n, k, act, bias=True, residual=False, train=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "act": act, "bias": bias,
            "residual": residual, "train": train}


def _grouped(name, rows, experts, n, k, behind=0, train=False):
    return {"name": name, "op": "grouped", "rows": rows, "experts": experts, "n": n, "k": k,
            "behind": behind, "train": train}


def _a8w4(name, rows, experts, n, k, behind=0):
    return {"name": name, "op": "a8w4_grouped", "rows": rows, "experts": experts, "n": n, "k": k,
            "behind": behind}


def _route(name, tokens, top, experts, absent=0):
    return {"name": name, "op": "group_rows", "tokens": tokens, "top": top, "experts": experts,
            "absent": absent}


def listed():
    return [
        # one token through a square projection: latency and the weight stream
        _linear("linear 1 token", 1, 4096, 4096, "silu"),
        # a decode batch through a wide projection
        _linear("linear decode batch", 16, 14336, 4096, "gelu_tanh", residual=True),
        # odd sizes: a short prompt, a column count that is no multiple of anything
        _linear("linear odd", 333, 1003, 2056, "relu", residual=True),
        # a prefill chunk through an MLP projection, epilogue in full
        _linear("linear prefill", 4096, 14336, 4096, "gelu", residual=True),
        # a training step of the same layer: output and the gradients of x, w and bias
        _linear("linear training step", 4096, 8192, 4096, "gelu", train=True),
        # a decode batch of 16 tokens that chose 4 of 64 experts each
        _grouped("grouped decode", 64, 64, 2048, 4096),
        # a prefill chunk over 16 experts, rows behind the last group as padding leaves them
        _grouped("grouped prefill", 8190, 16, 4096, 4096, behind=2),
        # a training step of an expert layer: output and the gradients of x and w
        _grouped("grouped training step", 8192, 8, 2048, 4096, train=True),
        # the int8 x int4 recipe at decode: the experts' packed weights stream once
        _a8w4("a8w4 grouped decode", 64, 32, 4096, 4096),
        # and at prefill
        _a8w4("a8w4 grouped prefill", 4093, 8, 14336, 4096, behind=3),
        # the choices of one decode batch
        _route("group rows decode", 16, 8, 64),
        # the choices of a long prefill, some tokens of it padding
        _route("group rows prefill", 65536, 8, 256, absent=100),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "grouped", "grouped", "a8w4_grouped", "group_rows"])
    if op == "linear":
        train = rng.random() < 0.4
        c = {"op": op, "m": _log(rng, 1, 4096), "n": _log(rng, 64, 8192), "k": 8 * _log(rng, 8, 512),
             "act": rng.choice(_ACTS), "bias": rng.random() < 0.7, "residual": rng.random() < 0.5,
             "train": train}
        return c
    if op == "group_rows":
        experts = _log(rng, 4, 256)
        return {"op": op, "tokens": _log(rng, 1, 65536), "top": rng.randint(1, min(8, experts)),
                "experts": experts, "absent": rng.choice([0, 0, 1, 7])}
    experts = _log(rng, 2, 64)
    rows = _log(rng, 1, 8192)
    if op == "grouped":
        train = rng.random() < 0.4
        return {"op": op, "rows": rows, "experts": experts, "n": _log(rng, 128, 2048),
                "k": 8 * _log(rng, 16, 512), "behind": rng.choice([0, 0, 1, 30]), "train": train}
    return {"op": op, "rows": rows, "experts": min(experts, 32), "n": 8 * _log(rng, 16, 512),
            "k": 128 * rng.randint(1, 32), "behind": rng.choice([0, 0, 1, 30])}


# ----------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------
def _normal(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def _group_sizes(case, seed):
    """Rows of each expert: drawn with a popularity that differs from expert to expert."""
    g = torch.Generator().manual_seed(seed)
    popularity = torch.softmax(0.7 * torch.randn(case["experts"], generator=g), 0)
    picks = torch.multinomial(popularity, case["rows"], replacement=True, generator=g)
    sizes = torch.bincount(picks, minlength=case["experts"])
    offsets = torch.zeros(case["experts"] + 1, dtype=torch.int64)
    offsets[1:] = sizes.cumsum(0)
    return offsets.to(torch.int32).cuda(), max(1, int(sizes.max()))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _normal(g, m, k)
        s["w"] = _normal(g, n, k, scale=k ** -0.5)
        s["bias"] = _normal(g, n, scale=0.2) if case["bias"] else None
        s["residual"] = _normal(g, m, n) if case["residual"] else None
        if case["train"]:
            s["dy"] = _normal(g, m, n)
            for name in ("x", "w", "bias", "residual"):
                if s[name] is not None:
                    s[name].requires_grad_()
    elif op == "grouped":
        t, n, k = case["rows"] + case["behind"], case["n"], case["k"]
        s["offsets"], s["most"] = _group_sizes(case, seed)
        s["x"] = _normal(g, t, k)
        s["w"] = _normal(g, case["experts"], n, k, scale=k ** -0.5)
        if case["train"]:
            s["dy"] = _normal(g, t, n)
            s["x"].requires_grad_()
            s["w"].requires_grad_()
    elif op == "a8w4_grouped":
        t, n, k, e = case["rows"] + case["behind"], case["n"], case["k"], case["experts"]
        s["offsets"], s["most"] = _group_sizes(case, seed)
        # what the per-token and per-group quantizers give for normal values
        s["x"] = torch.clamp(torch.round(torch.randn(t, k, generator=g, device="cuda") * 32), -127, 127).to(torch.int8)
        s["sa"] = 0.03 + 0.01 * torch.rand(t, generator=g, device="cuda")
        s["wp"] = torch.randint(0, 256, (e, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        s["sb"] = ((0.5 + torch.rand(e, n, k // 128, generator=g, device="cuda")) * (0.2 * k ** -0.5)).to(torch.bfloat16)
    else:
        t, e = case["tokens"], case["experts"]
        scores = torch.randn(t, e, generator=g, device="cuda") + 0.7 * torch.randn(e, generator=g, device="cuda")
        ids = scores.topk(case["top"], dim=1).indices
        if case["absent"]:
            ids[max(0, t - case["absent"]):] = -1  # padding tokens choose nobody
        s["ids"] = ids.contiguous()
    return s


# ----------------------------------------------------------------------------------
# The plain forms
# ----------------------------------------------------------------------------------
def _act(z, act):
    if act is None:
        return z
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))


def _act_slope(z, act):
    if act is None:
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    h = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1 + h) + 0.5 * z * (1 - h * h) * c * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    case = s["case"]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    z = x @ w.T
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    y = y.to(torch.bfloat16)
    if not case["train"]:
        return y
    dy = s["dy"].float()
    dz = dy * _act_slope(z, case["act"])
    got = {"y": y, "dx": (dz @ w).to(torch.bfloat16), "dw": (dz.T @ x).to(torch.bfloat16)}
    if s["bias"] is not None:
        got["dbias"] = dz.sum(0).to(torch.bfloat16)
    if s["residual"] is not None:
        got["dresidual"] = dy.to(torch.bfloat16)
    return got


def _places(offsets, rows):
    """For each of `rows` rows: whether it is in a group, its group and its place there."""
    at = torch.arange(rows, device=offsets.device, dtype=offsets.dtype)
    group = torch.searchsorted(offsets, at, right=True) - 1
    inside = (at >= offsets[0]) & (at < offsets[-1])
    group = torch.where(inside, group, torch.zeros_like(group))
    place = torch.where(inside, at - offsets[group], torch.zeros_like(at)).long()
    return inside, group, place


def _pad(v, inside, group, place, experts, most):
    """Rows [T, C] -> [experts, most, C], zeros where a group has no row."""
    out = torch.zeros(experts * most + 1, v.shape[1], device=v.device)
    out[torch.where(inside, group * most + place, torch.full_like(place, experts * most))] = v
    return out[:-1].view(experts, most, -1)


def _unpad(v, inside, group, place):
    got = v[group, torch.clamp(place, max=v.shape[1] - 1)]
    return torch.where(inside[:, None], got, torch.zeros_like(got))


def _plain_grouped(s):
    case = s["case"]
    x, w = s["x"].detach().float(), s["w"].detach().float()
    inside, group, place = _places(s["offsets"], x.shape[0])
    xp = _pad(x, inside, group, place, case["experts"], s["most"])
    y = _unpad(torch.bmm(xp, w.transpose(1, 2)), inside, group, place).to(torch.bfloat16)
    if not case["train"]:
        return y
    dyp = _pad(s["dy"].float(), inside, group, place, case["experts"], s["most"])
    dx = _unpad(torch.bmm(dyp, w), inside, group, place).to(torch.bfloat16)
    dw = torch.bmm(dyp.transpose(1, 2), xp).to(torch.bfloat16)
    return {"y": y, "dx": dx, "dw": dw}


def _plain_a8w4(s):
    case = s["case"]
    e, n, k = case["experts"], case["n"], case["k"]
    codes = torch.stack((s["wp"] & 15, s["wp"] >> 4), dim=-1).view(e, n, k // 128, 128).float()
    codes = torch.where(codes >= 8, codes - 16, codes)
    w = (codes * s["sb"].float()[..., None]).view(e, n, k)
    x = s["x"].float() * s["sa"][:, None]
    inside, group, place = _places(s["offsets"], x.shape[0])
    xp = _pad(x, inside, group, place, e, s["most"])
    return _unpad(torch.bmm(xp, w.transpose(1, 2)), inside, group, place).to(torch.bfloat16)


def _plain_group_rows(s):
    case = s["case"]
    e = case["experts"]
    flat = s["ids"].reshape(-1)
    key = torch.where((flat < 0) | (flat >= e), torch.full_like(flat, e), flat)
    ordered, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(ordered, torch.arange(e + 1, device=flat.device))
    positions = torch.empty_like(order)
    positions[order] = torch.arange(order.numel(), device=flat.device)
    return {"offsets": offsets.to(torch.int32), "rows": (order // case["top"]).to(torch.int32),
            "positions": positions.view(s["ids"].shape).to(torch.int32)}


# ----------------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------------
def _own(s):
    arc, case = _arc(), s["case"]
    op = case["op"]
    if op == "linear":
        y = arc.linear(s["x"], s["w"], s["bias"], s["residual"], activation=case["act"])
        if not case["train"]:
            return y
        names = [v for v in ("x", "w", "bias", "residual") if s[v] is not None]
        grads = torch.autograd.grad(y, [s[v] for v in names], s["dy"])
        return {"y": y.detach(), **{"d" + v: d for v, d in zip(names, grads)}}
    if op == "grouped":
        y = arc.grouped_matmul(s["x"], s["w"], s["offsets"])
        if not case["train"]:
            return y
        dx, dw = torch.autograd.grad(y, [s["x"], s["w"]], s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if op == "a8w4_grouped":
        return arc.a8w4_grouped_matmul((s["x"], s["sa"]), (s["wp"], s["sb"]), s["offsets"])
    offsets, rows, positions = arc.group_rows(s["ids"], case["experts"])
    return {"offsets": offsets, "rows": rows, "positions": positions}


def run(state):
    if own:
        return _own(state)
    return {"linear": _plain_linear, "grouped": _plain_grouped, "a8w4_grouped": _plain_a8w4,
            "group_rows": _plain_group_rows}[state["case"]["op"]](state)


# ----------------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------------
def _chosen(rows, experts):
    """Experts that an even draw of `rows` rows reaches, on average."""
    return experts * (1 - (1 - 1 / experts) ** rows)


def work(case):
    op = case["op"]
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        vectors = (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        if case["train"]:  # x, w, dy in; y, dx, dw and the small gradients out
            return {"bytes": 2 * (2 * m * k + 2 * n * k + 2 * m * n + 2 * vectors), "flops": 6 * m * n * k}
        return {"bytes": 2 * (m * k + n * k + m * n + vectors), "flops": 2 * m * n * k}
    if op == "grouped":
        t, n, k, e = case["rows"], case["n"], case["k"], case["experts"]
        weights = _chosen(t, e) * n * k
        if case["train"]:
            return {"bytes": 2 * (2 * t * k + weights + e * n * k + 2 * t * n), "flops": 6 * t * n * k}
        return {"bytes": 2 * (t * k + weights + t * n), "flops": 2 * t * n * k}
    if op == "a8w4_grouped":
        t, n, k, e = case["rows"], case["n"], case["k"], case["experts"]
        weights = _chosen(t, e) * n * (k / 2 + 2 * k / 128)
        return {"bytes": t * (k + 4) + weights + 2 * t * n, "flops": 2 * t * n * k}
    slots = case["tokens"] * case["top"]
    return {"bytes": (8 + 4 + 4) * slots + 4 * (case["experts"] + 1), "flops": 0}


# ----------------------------------------------------------------------------------
# The definition in 64 bits
# ----------------------------------------------------------------------------------
def _exact_linear(s, case):
    f = torch.nn.functional
    leaf = {v: None if s[v] is None else s[v].detach().double().requires_grad_(case["train"])
            for v in ("x", "w", "bias", "residual")}
    acts = {None: lambda z: z, "relu": f.relu, "silu": f.silu, "gelu": f.gelu,
            "gelu_tanh": lambda z: f.gelu(z, approximate="tanh")}
    y = acts[case["act"]](f.linear(leaf["x"], leaf["w"], leaf["bias"]))
    if leaf["residual"] is not None:
        y = y + leaf["residual"]
    if not case["train"]:
        return y
    names = [v for v in leaf if leaf[v] is not None]
    grads = torch.autograd.grad(y, [leaf[v] for v in names], s["dy"].double())
    return {"y": y.detach(), **{"d" + v: d for v, d in zip(names, grads)}}


def _exact_grouped(s, case, x, weight):
    ends = s["offsets"].tolist()
    y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device=x.device)
    train = case.get("train", False)
    dx = torch.zeros_like(x) if train else None
    dw = torch.zeros(s["w"].shape, dtype=torch.float64, device=x.device) if train else None
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        if a == b:
            continue
        w = weight(e)
        y[a:b] = x[a:b] @ w.T
        if train:
            d = s["dy"][a:b].double()
            dx[a:b] = d @ w
            dw[e] = d.T @ x[a:b]
    return {"y": y, "dx": dx, "dw": dw} if train else y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        return _exact_linear(s, case)
    if case["op"] == "grouped":
        return _exact_grouped(s, case, s["x"].detach().double(), lambda e: s["w"][e].detach().double())
    if case["op"] == "a8w4_grouped":
        def weight(e):
            p = s["wp"][e].to(torch.int64)
            w = torch.empty(case["n"], case["k"], dtype=torch.float64, device=p.device)
            w[:, 0::2] = ((p & 15) ^ 8) - 8
            w[:, 1::2] = ((p >> 4) ^ 8) - 8
            return w * s["sb"][e].double().repeat_interleave(128, dim=1)

        return _exact_grouped(s, case, s["x"].double() * s["sa"].double()[:, None], weight)
    return None  # whole numbers: the plain form gives them exactly
