"""Linear layer with its epilogue in the GEMM, and its gradients.

    out = act(x . w^T + bias) + residual          x [M, K], w [N, K], bf16

`linear` is one launch of `arc_linear_bf16` (include/arc_b200.h): the product accumulates in
fp32, bias, activation and residual are applied to the fp32 value and the result is rounded
to bf16 once. It is differentiable in x, w, bias and residual:

    dz = dout * act'(z)   z = x . w^T + bias
    dx = dz . w           dw = dz^T . x         dbias = sum_m dz         dresidual = dout

For the backward pass z is kept in bf16 (only with an activation), and dz is rounded to bf16,
the tensor cores' operand type; the sums run in fp32. No transposed copies are made.

Shapes and strides: any M (0 included), N and K >= 1. The products read x and w where they lie
if their rows are contiguous and 16-byte aligned (leading dimensions multiples of 8 elements, as
`arc.matmul` asks for); other layouts are copied into such rows first, on every call.
"""
from __future__ import annotations

import torch

from ._lib import ACTIVATIONS, call_on, lib, workspace_bytes
from .mm import _require_cuda_bf16, _row_major


def _same_device(t: torch.Tensor, name: str, dev: torch.device) -> None:
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, expected {dev}")


def _padded(*shape, device) -> torch.Tensor:
    """An empty bf16 tensor whose rows are 16-byte aligned (a view of padded storage)."""
    return torch.empty((*shape[:-1], (shape[-1] + 7) // 8 * 8), dtype=torch.bfloat16, device=device)[..., :shape[-1]]


def product_rows(t: torch.Tensor) -> torch.Tensor:
    """`t` [R, C] itself if TMA can read its rows, else a copy whose rows are 16-byte aligned."""
    r, c = t.shape
    if t.stride(1) == 1 and t.stride(0) >= c and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t
    return _padded(r, c, device=t.device).copy_(t)


def _forward(x, w, bias, residual, activation, out, z):
    call_on(x.device, lib().arc_linear_bf16, "arc.linear", x.data_ptr(), w.data_ptr(),
            bias.data_ptr() if bias is not None else None, residual.data_ptr() if residual is not None else None,
            out.data_ptr(), z.data_ptr() if z is not None else None, x.shape[0], w.shape[0], x.shape[1],
            x.stride(0), w.stride(0), residual.stride(0) if residual is not None else 0, out.stride(0),
            z.stride(0) if z is not None else 0, activation)
    return out


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, activation):
        m, n = x.shape[0], w.shape[0]
        x, w = product_rows(x), product_rows(w)
        out = x.new_empty((m, n))
        z = None
        if m > 0:
            if activation != 0 and any(ctx.needs_input_grad[:3]):
                z = _padded(m, n, device=x.device)
            _forward(x, w, bias, residual, activation, out, z)
        ctx.save_for_backward(x, w, z)
        ctx.activation = activation
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, z = ctx.saved_tensors
        need_x, need_w, need_bias, need_residual, _ = ctx.needs_input_grad
        m, k = x.shape
        n = w.shape[0]
        dx = x.new_empty((m, k)) if need_x else None
        dw = w.new_empty((n, k)) if need_w else None
        dbias = w.new_empty((n,)) if need_bias else None
        dresidual = dy if need_residual else None
        if not (need_x or need_w or need_bias):
            return None, None, None, dresidual, None
        if m == 0:
            return (dx, dw.zero_() if need_w else None, dbias.zero_() if need_bias else None, dresidual, None)
        if dy.stride(1) != 1 or dy.stride(0) < n:
            dy = dy.contiguous()  # an expanded or transposed gradient
        need_dz = (need_x or need_w) and (z is not None or dy.stride(0) % 8 != 0 or dy.data_ptr() % 16 != 0)
        size = workspace_bytes("arc_linear_backward_workspace_bytes", m, n, need_dz, need_bias)
        workspace = x.new_empty(((size + 1) // 2,)) if size else None
        call_on(x.device, lib().arc_linear_backward, "arc.linear backward", dy.data_ptr(), x.data_ptr(), w.data_ptr(),
                z.data_ptr() if z is not None else None, dx.data_ptr() if need_x else None,
                dw.data_ptr() if need_w else None, dbias.data_ptr() if need_bias else None,
                workspace.data_ptr() if size else None, size, m, n, k, dy.stride(0), x.stride(0), w.stride(0),
                z.stride(0) if z is not None else 0, k, k, ctx.activation)
        return dx, dw, dbias, dresidual, None


def linear(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None,
           residual: torch.Tensor | None = None, *, activation: str | None = None,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """act(x . w^T + bias) + residual. See the module docstring.

    x [M, K], w [N, K], bias [N], residual [M, N], all bf16 on one CUDA device.
    activation: None, "relu", "gelu" (erf), "gelu_tanh" or "silu".
    `out` receives the result (it may be `residual`); it cannot be combined with inputs that
    require gradients.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    for t, name in ((x, "x"), (w, "w")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        _require_cuda_bf16(t, name)
    m, k = x.shape
    n, _k = w.shape
    if k != _k:
        raise ValueError(f"Inner dimensions must match: {k} vs {_k}")
    if n == 0 or k == 0:
        raise ValueError(f"w must not be empty, got shape {tuple(w.shape)}")
    dev = x.device
    _same_device(w, "w", dev)
    if bias is not None:
        if bias.dtype != torch.bfloat16 or tuple(bias.shape) != (n,):
            raise ValueError(f"bias must be bfloat16 of shape ({n},), got {bias.dtype} {tuple(bias.shape)}")
        _same_device(bias, "bias", dev)
    if residual is not None:
        _require_cuda_bf16(residual, "residual")
        if tuple(residual.shape) != (m, n):
            raise ValueError(f"residual must have shape {(m, n)}, got {tuple(residual.shape)}")
        _same_device(residual, "residual", dev)
    bias = bias.contiguous() if bias is not None else None
    residual = _row_major(residual) if residual is not None else None
    code = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or
                                    (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        if out is not None:
            raise ValueError("out cannot be given when an input requires a gradient")
        return _Linear.apply(x, w, bias, residual, code)
    if out is None:
        out = x.new_empty((m, n))
    else:
        _require_cuda_bf16(out, "out")
        if tuple(out.shape) != (m, n) or out.device != dev or out.stride(1) != 1 or out.stride(0) < n:
            raise ValueError(f"out must be a row-major bf16 [{m}, {n}] tensor on {dev}")
    if m == 0:
        return out
    return _forward(product_rows(x), product_rows(w), bias, residual, code, out, None)
