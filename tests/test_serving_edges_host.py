"""CPU: the 64-bit form and the bound that the int4 tests of the expert layer use."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from int4_bounds import moe_int4_linear, product
from moe_reference import dequantized, moe_reference


def _pair(g, n, k, e=None):
    lead = () if e is None else (e,)
    return (torch.randint(0, 256, (*lead, n, k // 2), generator=g, dtype=torch.uint8),
            (0.01 + 0.02 * torch.rand(*lead, n, k // 128, generator=g)).to(torch.bfloat16))


def test_the_form_is_the_layers():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 256, generator=g).to(torch.bfloat16)
    w_in, w_out = _pair(g, 128, 256, 4), _pair(g, 40, 128, 4)
    ids, weights = torch.tensor([[0, 3], [1, 2], [3, 1], [2, 0], [-1, 1]]), torch.rand(5, 2, generator=g)
    y, bound = moe_int4_linear(x, w_in, w_out, ids, weights)
    want, loose = moe_reference(x, w_in, w_out, ids, weights, None)
    assert torch.equal(y, want) and (bound > 0).all() and (bound <= 4 * loose).all()


@pytest.mark.parametrize("power", [0, -57, -70, -82])
@pytest.mark.parametrize("outlier", [0, 14, 30])
def test_the_bound_holds_for_sums_in_32_bits(power, outlier):
    """The kernel's sums step by step in numpy's fp32: x in units of 2^-69 times code + 8, from -8 x on, a rounding for every
    product; groups by a multiplication and an addition."""
    g = torch.Generator().manual_seed(power + outlier + 100)
    k, n = 256, 24
    packed, scales = _pair(g, n, k)
    packed[:, 2] &= 0x0F
    x = torch.randn(2, k, generator=g)
    x[:, 5] = 1.4 * 2.0 ** outlier
    x = (x * 2.0 ** power).to(torch.bfloat16)
    codes = np.rint((dequantized((packed[None], torch.ones_like(scales)[None]))[0]).numpy()).astype(np.float32)
    xs, s = (x.double().numpy() * 2.0 ** -69).astype(np.float64), scales.float().numpy()
    got = np.zeros((2, n), np.float32)
    for r in range(2):
        for j in range(n):
            for q in range(k // 128):
                part = np.float32(0)
                for i in range(q * 128, q * 128 + 128):
                    part = np.float32(np.float64(part) - 8 * xs[r, i])
                for i in range(q * 128, q * 128 + 128):
                    part = np.float32(np.float64(part) + (np.float64(codes[j, i]) + 8) * xs[r, i])
                got[r, j] = np.float32(np.float64(got[r, j]) + np.float64(s[j, q]) * np.float64(part))
    got = torch.from_numpy(got.astype(np.float64) * 2.0 ** 69)
    want, bound = product(x.double(), torch.zeros_like(x.double()), packed, scales)
    assert ((got - want).abs() <= bound).all()
