"""Linear layer with its epilogue in the GEMM, and its gradients.

    out = act(x . w^T + bias) + residual          x [M, K], w [N, K], bf16

`linear` is one launch of `arc_linear_bf16` (include/arc_b200.h) on the caller's stream: the product accumulates in
fp32, bias, activation and residual are applied to the fp32 value and the result is rounded
to bf16 once. It is differentiable in x, w, bias and residual
(once, in reverse mode; a second derivative or a forward-mode tangent is refused):

    dz = dout * act'(z)   z = x . w^T + bias
    dx = dz . w           dw = dz^T . x         dbias = sum_m dz         dresidual = dout

For the backward pass z is kept in bf16 (only with an activation), and dz is rounded to bf16,
the tensor cores' operand type; the sums run in fp32. No transposed copies are made. The graph
keeps x only for dw and w only for dx. The activations are relatively accurate in their lower
tails too (off by less than 2^-14 of themselves before the rounding to bf16, down to 2^-118).

Shapes and strides: any M (0 included), N and K >= 1. The products read x and w where they lie
if their rows are contiguous and 16-byte aligned (leading dimensions multiples of 8 elements, as
`arc.matmul` asks for); other layouts are copied into such rows first, on every call. A weight
whose K is no multiple of 8 is worth padding once: w = torch.nn.functional.pad(w, (0, -K % 8))[:, :K].
"""
from __future__ import annotations

import torch

from ._lib import ACTIVATIONS, torch_ops


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, *, activation: str | None = None,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """act(x . w^T + bias) + residual. See the module docstring.

    x [M, K], w [N, K], bias [N], residual [M, N], all bf16 on one CUDA device.
    activation: None, "relu", "gelu" (erf), "gelu_tanh" or "silu".
    `out` receives the result. It may be `residual` itself and must not overlap x, w or bias; it
    cannot be combined with inputs that require gradients.
    """
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    return torch_ops().linear(x, w, bias, residual, code, out)
