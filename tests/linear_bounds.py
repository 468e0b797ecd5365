"""Error bounds of the linear and grouped products, by arithmetic, and their 64-bit forms.

A bf16 rounding is off by at most half a step, 2^-8 relative (H). A sum of k fp32 products is off
by at most k * 2^-24 times the sum of their magnitudes; twice that is taken, since the tensor
core aligns addends by truncation. The epilogue's fp32 steps and the approximations of exp and
division add a few units of 2^-22 relative (F) and, where 1 + erf cancels, 2^-22 |z| absolute.
Every activation here has a slope of at most 1.2 and a curvature of at most 1 in magnitude.
"""
from __future__ import annotations

import math

import torch

H = torch.finfo(torch.bfloat16).eps / 2
F = 2.0 ** -18
SUM = 2.0 ** -23


def act64(z, act):
    f = torch.nn.functional
    return {None: lambda v: v, "relu": f.relu, "gelu": f.gelu, "silu": f.silu,
            "gelu_tanh": lambda v: f.gelu(v, approximate="tanh")}[act](z)


def slope64(z, act):
    z = z.detach().clone().requires_grad_()
    return torch.autograd.grad(act64(z, act).sum(), z)[0]


def linear_forward(x, w, bias, residual, act):
    """(y, bound of |kernel - y|, z, bound of the fp32 z) in float64."""
    x, w = x.double(), w.double()
    z = x @ w.T
    zerr = x.shape[1] * SUM * (x.abs() @ w.abs().T)
    if bias is not None:
        z = z + bias.double()
        zerr = zerr + 2.0 ** -23 * (z.abs() + bias.double().abs())
    y = act64(z, act)
    yerr = 1.2 * zerr + F * y.abs() + 2.0 ** -22 * z.abs()
    if residual is not None:
        y = y + residual.double()
    return y, yerr + H * (y.abs() + yerr) + F * y.abs() + 1e-30, z, zerr


def linear_gradients(x, w, z, zerr, dy, act):
    """{name: (value, bound)} of dz, dx, dw and dbias in float64."""
    x, w, dy = x.double(), w.double(), dy.double()
    slope = slope64(z, act)
    if act is None:
        serr = torch.zeros_like(z)
    else:
        zr = zerr + H * (z.abs() + zerr)  # z is kept in bf16
        serr = F + (torch.where(z.abs() <= zerr, 1.0, 0.0).double() if act == "relu" else zr)
    dz = dy * slope
    raw = dy.abs() * serr + F * dz.abs()
    err = raw if act is None else raw + H * (dz.abs() + raw)
    m, n = dz.shape
    dx, dw, db = dz @ w, dz.T @ x, dz.sum(0)
    ex = (err + n * SUM * (dz.abs() + err)) @ w.abs()
    ew = (err + m * SUM * (dz.abs() + err)).T @ x.abs()
    eb = raw.sum(0) + m * SUM * (dz.abs() + raw).sum(0)
    out = {"dz": (dz, err), "dx": (dx, ex), "dw": (dw, ew), "dbias": (db, eb)}
    return {k: (v, e + H * (v.abs() + e) + 1e-30) for k, (v, e) in out.items()}


def assert_within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    if got.numel() == 0:
        return
    over = (got - want).abs() - bound
    worst = over.argmax()
    assert over.flatten()[worst] <= 0, (
        f"{what}: off by {(got - want).abs().flatten()[worst]:.3e}, bound {bound.flatten()[worst]:.3e}, "
        f"at {math.floor(worst / got.shape[-1])},{worst % got.shape[-1]}; {(over > 0).sum()} outside")


def normal(g, *shape, scale=1.0, device="cuda"):
    return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16).to(device)
