"""The expert layer in 64 bits, with the bound of the kernel's error by arithmetic.

The rules of linear_bounds: a sum of k fp32 products is off by at most k 2^-23 of the magnitudes' sum (group scales
of int4 weights add one product per 128 terms, within that), a rounding to bf16 by 2^-8 relative. What the
kernel rounds: h (the second product's operand) and y.
"""
from __future__ import annotations

import torch

from linear_bounds import F, H, SUM, act64


def dequantized(pair):
    """(packed [E, n, k/2], scales [E, n, k/128]) -> float64 [E, n, k]."""
    packed, scales = pair
    p = packed.to(torch.int64)
    codes = torch.stack((((p & 15) ^ 8) - 8, ((p >> 4) ^ 8) - 8), dim=-1).flatten(2).double()
    return codes * scales.double().repeat_interleave(128, dim=2)


def moe_reference(x, w_in, w_out, ids, weights, act):
    """(y, bound) in float64. Tokens one by one, experts as each asks for them."""
    w_in = dequantized(w_in) if isinstance(w_in, tuple) else w_in.double()
    w_out = dequantized(w_out) if isinstance(w_out, tuple) else w_out.double()
    experts, n, inner = w_out.shape
    gated = w_in.shape[1] == 2 * inner
    y = torch.zeros(x.shape[0], n, dtype=torch.float64, device=x.device)
    err, mag = torch.zeros_like(y), torch.zeros_like(y)
    k = x.shape[1]
    for e in range(experts):
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        if token.numel() == 0:
            continue
        xe, share = x[token].double(), weights[token, choice].double()[:, None]
        z = xe @ w_in[e].T
        zerr = k * SUM * (xe.abs() @ w_in[e].abs().T)
        a = act64(z[:, :inner], act)
        aerr = 1.2 * zerr[:, :inner] + F * a.abs() + 2.0 ** -22 * z[:, :inner].abs()
        h, herr = a, aerr
        if gated:
            u, uerr = z[:, inner:], zerr[:, inner:]
            h = a * u
            herr = aerr * (u.abs() + uerr) + a.abs() * uerr + F * h.abs()
        herr = herr + H * (h.abs() + herr) + 1e-38
        o, m = h @ w_out[e].T, (h.abs() + herr) @ w_out[e].abs().T
        oerr = herr @ w_out[e].abs().T + inner * SUM * m
        y.index_add_(0, token, share * o)
        err.index_add_(0, token, share.abs() * oerr)
        mag.index_add_(0, token, share.abs() * m)
    err = err + (ids.shape[1] + 2) * SUM * mag
    return y, err + H * (y.abs() + err) + 1e-30
