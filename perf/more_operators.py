"""The expert layer of a few tokens and the linear layer with adapters of arc, as measured cases.

Two operators, each in a plain form (torch, 32 bits) and through the framework:

* moe          y[t] = sum_j weights[t, j] (act(x[t] gate_e^T) * (x[t] up_e^T)) w_out_e^T, e = ids[t, j], with
               bf16 or int4 (group-128 scales) weights
* lora_linear  y = act(x w^T + bias + scale_i (x a_i^T) b_i^T) + residual, i = ids[row]
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
def _moe(name, tokens, top, experts, hidden, inner, kind="bf16", gated=True, act="silu", absent=0):
    return {"name": name, "op": "moe", "tokens": tokens, "top": top, "experts": experts, "hidden": hidden,
            "inner": inner, "kind": kind, "gated": gated, "act": act, "absent": absent}


def _lora(name, m, n, k, rank, adapters, act=None, bias=False, residual=False, prompts=0, without=0.0):
    return {"name": name, "op": "lora_linear", "m": m, "n": n, "k": k, "rank": rank, "adapters": adapters, "act": act,
            "bias": bias, "residual": residual, "prompts": prompts, "without": without}


def listed():
    return [
        # one token of one request: latency and the weights of eight experts
        _moe("moe 1 token", 1, 8, 64, 4096, 2048),
        # a decode batch; most experts are chosen, by two tokens on average
        _moe("moe decode batch", 16, 8, 64, 4096, 2048),
        # odd sizes, experts without a gate, padding tokens that choose nobody
        _moe("moe odd", 7, 3, 10, 1032, 520, gated=False, act="gelu", absent=2),
        # few wide experts
        _moe("moe wide experts", 4, 2, 8, 4096, 14336),
        # a large decode batch: 16 tokens an expert
        _moe("moe large batch", 128, 8, 64, 4096, 2048),
        # the same layer on int4 weights
        _moe("moe int4 1 token", 1, 8, 64, 4096, 2048, kind="int4"),
        _moe("moe int4 decode batch", 32, 8, 64, 4096, 2048, kind="int4"),
        # one token with its adapter through a square projection
        _lora("lora 1 token", 1, 4096, 4096, 16, 8),
        # a decode batch of requests with adapters of their own through a wide projection
        _lora("lora decode batch", 32, 14336, 4096, 16, 64, without=0.2),
        # odd sizes, the whole epilogue, rows of every adapter mixed
        _lora("lora odd", 77, 1003, 2056, 24, 5, act="gelu", bias=True, residual=True, without=0.3),
        # a few short prompts
        _lora("lora short prompts", 512, 4096, 4096, 32, 16, act="silu", bias=True, prompts=5),
        # a prefill chunk of several prompts
        _lora("lora prefill", 4096, 14336, 4096, 64, 16, residual=True, prompts=9),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.55:
        kind = rng.choice(["bf16", "bf16", "int4"])
        experts = _log(rng, 4, 64)
        if kind == "int4":
            hidden, inner = 128 * rng.randint(2, 32), 128 * rng.randint(1, 16)
        else:
            hidden, inner = 8 * _log(rng, 16, 512), 8 * _log(rng, 16, 256)
        tokens = _log(rng, 1, 128)
        return {"op": "moe", "tokens": tokens, "top": rng.randint(1, min(8, experts)), "experts": experts,
                "hidden": hidden, "inner": inner, "kind": kind, "gated": rng.random() < 0.75, "act": rng.choice(_ACTS),
                "absent": rng.choice([0, 0, min(1, tokens - 1), tokens // 3])}
    m = _log(rng, 1, 4096)
    return {"op": "lora_linear", "m": m, "n": _log(rng, 64, 8192), "k": 8 * _log(rng, 8, 512),
            "rank": rng.choice([8, 16, 16, 24, 32, 64, 128]), "adapters": _log(rng, 1, 128), "act": rng.choice(_ACTS),
            "bias": rng.random() < 0.5, "residual": rng.random() < 0.5,
            "prompts": 0 if m <= 64 else rng.randint(1, 12), "without": rng.choice([0.0, 0.0, 0.3])}


# ----------------------------------------------------------------------------------
# Inputs
# ----------------------------------------------------------------------------------
def _normal(g, *shape, scale=1.0):
    out = torch.empty(*shape, dtype=torch.bfloat16, device="cuda")
    for part in (out if len(shape) == 3 else [out]):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda") * scale)
    return out


def _int4(g, experts, n, k):
    """Packed codes and their scales, as the group quantizer leaves them for normal values."""
    codes = torch.randint(0, 256, (experts, n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (0.5 + torch.rand(experts, n, k // 128, generator=g, device="cuda")) * (0.2 * k ** -0.5)
    return codes, scales.to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "moe":
        t, e, k, i = case["tokens"], case["experts"], case["hidden"], case["inner"]
        rows = 2 * i if case["gated"] else i
        s["x"] = _normal(g, t, k)
        if case["kind"] == "bf16":
            s["w_in"] = _normal(g, e, rows, k, scale=k ** -0.5)
            s["w_out"] = _normal(g, e, k, i, scale=i ** -0.5)
        else:
            s["w_in"], s["w_out"] = _int4(g, e, rows, k), _int4(g, e, k, i)
        # a router's choices: scores whose experts differ in popularity, softmax over the chosen ones
        scores = torch.randn(t, e, generator=g, device="cuda") + 0.7 * torch.randn(e, generator=g, device="cuda")
        best = scores.topk(case["top"], dim=1)
        s["ids"], s["weights"] = best.indices.contiguous(), torch.softmax(best.values, dim=1)
        if case["absent"]:
            s["ids"][t - case["absent"]:] = -1  # padding tokens choose nobody
    else:
        m, n, k, r, count = case["m"], case["n"], case["k"], case["rank"], case["adapters"]
        s["x"] = _normal(g, m, k)
        s["w"] = _normal(g, n, k, scale=k ** -0.5)
        s["a"] = _normal(g, count, r, k, scale=k ** -0.5)
        s["b"] = _normal(g, count, n, r, scale=r ** -0.5)
        s["scales"] = 0.25 + 0.75 * torch.rand(count, generator=g, device="cuda")
        s["bias"] = _normal(g, n, scale=0.2) if case["bias"] else None
        s["residual"] = _normal(g, m, n) if case["residual"] else None
        if case["prompts"]:  # rows of one request lie together
            host = torch.Generator().manual_seed(seed)
            cuts = torch.randint(0, m + 1, (case["prompts"] - 1,), generator=host).sort().values.tolist()
            owner = torch.randint(0, count, (case["prompts"],), generator=host)
            owner[torch.rand(case["prompts"], generator=host) < case["without"]] = -1
            lengths = torch.tensor([b - a for a, b in zip([0] + cuts, cuts + [m])])
            s["ids"] = torch.repeat_interleave(owner, lengths).to(torch.int32).cuda()
        else:
            ids = torch.randint(0, count, (m,), generator=g, device="cuda", dtype=torch.int32)
            none = torch.rand(m, generator=g, device="cuda") < case["without"]
            s["ids"] = torch.where(none, torch.full_like(ids, -1), ids)
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


def _weights_of(w, e, dtype=torch.float32):
    """Expert e's matrix."""
    if isinstance(w, torch.Tensor):
        return w[e].to(dtype)
    packed, scales = w[0][e], w[1][e].to(dtype)
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).view(packed.shape[0], -1, 128).to(dtype)
    codes = torch.where(codes >= 8, codes - 16, codes)
    return (codes * scales[..., None]).flatten(1)


def _plain_moe(s):
    case = s["case"]
    x, inner = s["x"].float(), case["inner"]
    y = torch.zeros_like(x)
    for e in range(case["experts"]):
        share = (s["weights"].float() * (s["ids"] == e)).sum(1)  # of the tokens that chose e; else 0
        z = x @ _weights_of(s["w_in"], e).T
        h = _act(z[:, :inner], case["act"]) * z[:, inner:] if case["gated"] else _act(z, case["act"])
        y = y + share[:, None] * (h @ _weights_of(s["w_out"], e).T)
    return y.to(torch.bfloat16)


def _plain_lora(s):
    case = s["case"]
    x = s["x"].float()
    z = x @ s["w"].float().T
    # all adapters side by side, the sums of the others' set to zero
    u = x @ s["a"].float().flatten(0, 1).T
    owner = torch.arange(case["adapters"], device=x.device).repeat_interleave(case["rank"])
    scale = s["scales"].repeat_interleave(case["rank"])
    u = torch.where(s["ids"][:, None] == owner, u * scale, torch.zeros_like(u))
    z = z + u @ s["b"].float().transpose(1, 2).flatten(0, 1)
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(torch.bfloat16)


# ----------------------------------------------------------------------------------
# One pass
# ----------------------------------------------------------------------------------
def _own(s):
    arc, case = _arc(), s["case"]
    if case["op"] == "moe":
        return arc.moe(s["x"], s["w_in"], s["w_out"], s["ids"], s["weights"], activation=case["act"])
    return arc.lora_linear(s["x"], s["w"], s["a"], s["b"], s["ids"], s["bias"], s["residual"], scales=s["scales"],
                           activation=case["act"])


def run(state):
    if own:
        return _own(state)
    return _plain_moe(state) if state["case"]["op"] == "moe" else _plain_lora(state)


# ----------------------------------------------------------------------------------
# What a pass cannot do without
# ----------------------------------------------------------------------------------
def _chosen(picks, choices):
    """Of `choices` things, those that an even draw of `picks` reaches, on average."""
    return choices * (1 - (1 - 1 / choices) ** picks)


def work(case):
    if case["op"] == "moe":
        k, i = case["hidden"], case["inner"]
        tokens = case["tokens"] - case["absent"]
        # a token's choices differ
        experts = case["experts"] * (1 - (1 - case["top"] / case["experts"]) ** tokens)
        size = (3 if case["gated"] else 2) * k * i
        each = 2 * size if case["kind"] == "bf16" else size // 2 + 2 * size // 128
        slots = case["tokens"] * case["top"]
        return {"bytes": experts * each + 4 * case["tokens"] * k + 12 * slots, "flops": 2 * tokens * case["top"] * size}
    m, n, k, r = case["m"], case["n"], case["k"], case["rank"]
    with_one = m * (1 - case["without"])
    adapters = _chosen(case["prompts"] or with_one, case["adapters"])
    vectors = (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
    return {"bytes": 2 * (m * k + n * k + m * n + vectors + adapters * r * (n + k)) + 4 * m,
            "flops": 2 * m * n * k + 2 * with_one * r * (n + k)}


# ----------------------------------------------------------------------------------
# The definition in 64 bits
# ----------------------------------------------------------------------------------
def _exact_act(z, act):
    f = torch.nn.functional
    if act == "gelu_tanh":
        return f.gelu(z, approximate="tanh")
    return z if act is None else {"relu": f.relu, "silu": f.silu, "gelu": f.gelu}[act](z)


def _exact_matrix(w, e):
    if isinstance(w, torch.Tensor):
        return w[e].double()
    p = w[0][e].to(torch.int64)
    out = torch.empty(p.shape[0], 2 * p.shape[1], dtype=torch.float64, device=p.device)
    out[:, 0::2] = ((p & 15) ^ 8) - 8
    out[:, 1::2] = ((p >> 4) ^ 8) - 8
    return out * w[1][e].double().repeat_interleave(128, dim=1)


def _exact_moe(s, case):
    x = s["x"].double()
    y = torch.zeros_like(x)
    for e in range(case["experts"]):
        token, choice = torch.nonzero(s["ids"] == e, as_tuple=True)
        if token.numel() == 0:
            continue
        z = x[token] @ _exact_matrix(s["w_in"], e).T
        if case["gated"]:
            gate, up = z.chunk(2, dim=1)
            h = _exact_act(gate, case["act"]) * up
        else:
            h = _exact_act(z, case["act"])
        out = h @ _exact_matrix(s["w_out"], e).T
        y.index_add_(0, token, out * s["weights"][token, choice].double()[:, None])
    return y


def _exact_lora(s, case):
    x = s["x"].double()
    z = x @ s["w"].double().T
    for i in range(case["adapters"]):
        rows = torch.nonzero(s["ids"] == i)[:, 0]
        if rows.numel():
            low = x[rows] @ s["a"][i].double().T
            z[rows] += s["scales"][i].double() * (low @ s["b"][i].double().T)
    if s["bias"] is not None:
        z = z + s["bias"].double()
    y = _exact_act(z, case["act"])
    return y if s["residual"] is None else y + s["residual"].double()


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_moe(s, case) if case["op"] == "moe" else _exact_lora(s, case)
