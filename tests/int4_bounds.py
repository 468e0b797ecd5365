"""The expert layer on int4 weights without a gate or an activation, in 64 bits, with the bound of its error by arithmetic.

A group of 128 enters the sum as -8 x and (code + 8) x, 256 products, whose magnitudes are (16 + code) |x|: their fp32
sum is off by at most 256 * 2^-23 of those (linear_bounds' SUM), not of |code x|. Sums are held in units of 2^-69, of
which fp32 resolves 2^-149: a product, or a group added to the others, loses up to 2^-80. Then the rules of moe_reference.
"""
from __future__ import annotations

import torch

from linear_bounds import H, SUM
from moe_reference import dequantized

LOST = 2.0 ** -80


def product(v, verr, packed, scales):
    """(v w^T, bound) for v [T, k] with an error of verr, w [n, k] packed with scales [n, k/128]."""
    k = v.shape[1]
    w = dequantized((packed[None], scales[None]))[0]
    wide = scales.double().repeat_interleave(128, dim=1)
    mag = (v.abs() + verr) @ (16 * wide.abs() + w.abs()).T  # (16 + code) is at most 16 + |code|
    lost = LOST * (256 * scales.double().abs().sum(1) + k // 128)
    return v @ w.T, verr @ w.abs().T + (256 + k // 128) * SUM * mag + lost


def moe_int4_linear(x, w_in, w_out, ids, weights):
    """(y, bound) of arc.moe(..., activation=None) for w_in [E, I, K/2]; every token's experts differ."""
    t, n = x.shape[0], w_out[0].shape[1]
    y = torch.zeros(t, n, dtype=torch.float64, device=x.device)
    err, mag = torch.zeros_like(y), torch.zeros_like(y)
    for e in range(w_in[0].shape[0]):
        token, choice = torch.nonzero(ids == e, as_tuple=True)
        if token.numel() == 0:
            continue
        xe, share = x[token].double(), weights[token, choice].double()[:, None]
        h, herr = product(xe, torch.zeros_like(xe), w_in[0][e], w_in[1][e])
        herr = herr + H * (h.abs() + herr) + 2.0 ** -134  # half a step of bf16's smallest numbers
        o, oerr = product(h, herr, w_out[0][e], w_out[1][e])
        y.index_add_(0, token, share * o)
        err.index_add_(0, token, share.abs() * oerr)
        mag.index_add_(0, token, share.abs() * (o.abs() + oerr))
    err = err + (ids.shape[1] + 2) * SUM * mag
    return y, err + H * (y.abs() + err) + 2.0 ** -134
