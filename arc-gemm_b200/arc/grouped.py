"""Products grouped by expert, with ragged row groups, and the grouping itself.

    offsets, rows, positions = arc.group_rows(ids, E)       ids [T, top]: a router's choices
    xs = x[rows.long()]                                      rows sorted by expert
    ys = arc.grouped_matmul(xs, w, offsets)                  w [E, N, K], one matrix per expert
    y  = (ys[positions.long()] * weights[..., None]).sum(1)  back to tokens

Group e owns the rows [offsets[e], offsets[e+1]); offsets is int32 [E+1] on the GPU and is read
there, so no call waits for the host. Rows of no group (behind the last one, where `group_rows`
places the choices of ids outside [0, E)) never reach a result, whatever they hold; their
output rows are left as they are when `out` is given and are zero otherwise.

`grouped_matmul` is differentiable in x and w; `a8w4_grouped_matmul` is the serving form on
int8 activations and int4 weights, with the operands of `arc.a8w4_matmul`. Offsets that
decrease or leave the rows give unspecified values and set bit 7 of `arc.device_status`.
"""
from __future__ import annotations

import torch

from ._lib import A8W4_PREPACKED, GROUPED_ZERO_OTHERS, call_on, lib, workspace_bytes
from .a8w4 import GROUP_K, _expect
from .linear import _padded, _same_device, product_rows
from .mm import _require_cuda_bf16
from .quant import TensorPair

MAX_GROUPS = 1024


def _check_offsets(offsets: torch.Tensor, groups: int, dev: torch.device) -> None:
    if not 1 <= groups <= MAX_GROUPS:
        raise ValueError(f"between 1 and {MAX_GROUPS} groups are supported, got {groups}")
    _expect(offsets, "offsets", torch.int32, (groups + 1,), dev)


def _product_groups(w: torch.Tensor) -> torch.Tensor:
    """`w` [E, N, K] itself if TMA can read its rows, else a copy whose rows are 16-byte aligned."""
    e, n, k = w.shape
    if (w.stride(2) == 1 and w.stride(1) >= k and w.stride(0) >= (n - 1) * w.stride(1) + k and
            w.stride(1) % 8 == 0 and w.stride(0) % 8 == 0 and w.data_ptr() % 16 == 0):
        return w
    return _padded(e, n, k, device=w.device).copy_(w)


def _forward(x, w, offsets, out, zero_others):
    t, k = x.shape
    e, n, _ = w.shape
    call_on(x.device, lib().arc_grouped_matmul, "arc.grouped_matmul", x.data_ptr(), w.data_ptr(), offsets.data_ptr(),
            out.data_ptr(), t, e, n, k, x.stride(0), w.stride(1), w.stride(0), out.stride(0),
            GROUPED_ZERO_OTHERS if zero_others else 0)
    return out


class _Grouped(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets):
        x, w = product_rows(x), _product_groups(w)
        out = x.new_empty((x.shape[0], w.shape[1]))
        if x.shape[0] > 0:
            _forward(x, w, offsets, out, True)
        ctx.save_for_backward(x, w, offsets)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        need_x, need_w, _ = ctx.needs_input_grad
        if x.shape[0] == 0:
            return x.new_empty(x.shape) if need_x else None, w.new_zeros(w.shape) if need_w else None, None
        dy = product_rows(dy)
        (t, k), (e, n, _) = x.shape, w.shape
        dx = dw = None
        if need_x:
            dx = x.new_empty((t, k))
            call_on(x.device, lib().arc_grouped_matmul_dx, "arc.grouped_matmul backward", dy.data_ptr(), w.data_ptr(),
                    offsets.data_ptr(), dx.data_ptr(), t, e, n, k, dy.stride(0), w.stride(1), w.stride(0), k,
                    GROUPED_ZERO_OTHERS)
        if need_w:
            dw = w.new_empty((e, n, k))
            call_on(x.device, lib().arc_grouped_matmul_dw, "arc.grouped_matmul backward", dy.data_ptr(), x.data_ptr(),
                    offsets.data_ptr(), dw.data_ptr(), t, e, n, k, dy.stride(0), x.stride(0), k, n * k)
        return dx, dw, None


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = x[t] . w[e]^T for the rows t of each group e. See the module docstring.

    x [T, K] and w [E, N, K] bf16, offsets int32 [E+1] on the same device, E <= 1024. Rows that
    are not contiguous and 16-byte aligned (strides multiples of 8) are copied first.
    """
    for t, name in ((x, "x"), (w, "w")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    _require_cuda_bf16(x, "x")
    if w.dim() != 3:
        raise ValueError(f"w must be 3-D [E, N, K], got shape {tuple(w.shape)}")
    dev = x.device
    _same_device(w, "w", dev)
    if w.dtype != torch.bfloat16:
        raise TypeError(f"w must be bfloat16, got {w.dtype}")
    t, k = x.shape
    e, n, _k = w.shape
    if k != _k:
        raise ValueError(f"Inner dimensions must match: {k} vs {_k}")
    if n == 0 or k == 0:
        raise ValueError(f"w must not be empty, got shape {tuple(w.shape)}")
    _check_offsets(offsets, e, dev)
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad):
        if out is not None:
            raise ValueError("out cannot be given when an input requires a gradient")
        return _Grouped.apply(x, w, offsets)
    fresh = out is None
    if fresh:
        out = x.new_empty((t, n))
    else:
        _require_cuda_bf16(out, "out")
        if tuple(out.shape) != (t, n) or out.device != dev or out.stride(1) != 1 or out.stride(0) < n:
            raise ValueError(f"out must be a row-major bf16 [{t}, {n}] tensor on {dev}")
    return _forward(product_rows(x), _product_groups(w), offsets, out, fresh) if t > 0 else out


def a8w4_grouped_matmul(a: TensorPair, b: TensorPair, offsets: torch.Tensor, out: torch.Tensor | None = None, *,
                        prepacked: bool = False) -> torch.Tensor:
    """A8W4 GEMM of each row group with its own weights. See the module docstring.

    a = (x int8 [T, K], sa float32 [T]); b = (wp uint8 [E, N, K/2], sb bfloat16 [E, N, K/128]),
    the operands of `arc.a8w4_matmul` with a leading group dimension. `prepacked=True` says that
    wp is in the layout of `arc.prepack_weights` (of wp viewed as [E*N, K/2]).
    """
    x, sa = a
    wp, sb = b
    for v, name, dims in ((x, "a[0]", 2), (wp, "b[0]", 3)):
        if not isinstance(v, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if v.dim() != dims:
            raise ValueError(f"{name} must be {dims}-D, got shape {tuple(v.shape)}")
    t, k = x.shape
    e, n, k2 = wp.shape
    if k != 2 * k2:
        raise ValueError(f"Inner dimensions must match: {k} vs 2*{k2}")
    if k == 0 or k % GROUP_K != 0 or n == 0:
        raise ValueError(f"K ({k}) must be a positive multiple of {GROUP_K} and N ({n}) positive")
    dev = x.device
    if sa.dim() == 2 and sa.shape[1] == 1:
        sa = sa.reshape(-1)
    _expect(x, "a[0]", torch.int8, (t, k), None)
    _expect(sa, "a[1]", torch.float32, (t,), dev)
    _expect(wp, "b[0]", torch.uint8, (e, n, k // 2), dev)
    _expect(sb, "b[1]", torch.bfloat16, (e, n, k // GROUP_K), dev)
    _check_offsets(offsets, e, dev)
    fresh = out is None
    if fresh:
        out = torch.empty((t, n), dtype=torch.bfloat16, device=dev)
    else:
        _expect(out, "out", torch.bfloat16, (t, n), dev)
    if t == 0:
        return out
    flags = (A8W4_PREPACKED if prepacked else 0) | (GROUPED_ZERO_OTHERS if fresh else 0)
    size = workspace_bytes("arc_a8w4_grouped_workspace_bytes", t, e, k)
    workspace = x.new_empty(size) if size else None
    call_on(dev, lib().arc_a8w4_grouped_gemm, "arc.a8w4_grouped_matmul", x.data_ptr(), sa.data_ptr(), wp.data_ptr(),
            sb.data_ptr(), offsets.data_ptr(), out.data_ptr(), workspace.data_ptr() if size else None, size, t, e, n, k,
            GROUP_K, flags)
    return out


def group_rows(ids: torch.Tensor, num_groups: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A router's choices sorted by group: (offsets [E+1], rows [T*top], positions like ids), int32.

    ids [T, top] or [T], int32 or int64. rows[p] is the token at place p of the sorted order and
    positions[t, j] the place of choice ids[t, j]; inside a group, choices keep their order. An id
    outside [0, num_groups) chooses no group: its place is behind the last group, offsets[E] on.
    """
    if not isinstance(ids, torch.Tensor):
        raise TypeError("ids must be a torch.Tensor")
    if ids.device.type != "cuda":
        raise ValueError(f"ids must be a CUDA tensor (there is no CPU path), got {ids.device}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if ids.dim() not in (1, 2):
        raise ValueError(f"ids must be [T] or [T, top], got shape {tuple(ids.shape)}")
    if not 1 <= num_groups <= MAX_GROUPS:
        raise ValueError(f"between 1 and {MAX_GROUPS} groups are supported, got {num_groups}")
    ids = ids.contiguous()
    dev, slots = ids.device, ids.numel()
    if slots == 0:
        return (torch.zeros(num_groups + 1, dtype=torch.int32, device=dev),
                torch.empty(0, dtype=torch.int32, device=dev), torch.empty(ids.shape, dtype=torch.int32, device=dev))
    offsets = ids.new_empty(num_groups + 1, dtype=torch.int32)
    rows = ids.new_empty(slots, dtype=torch.int32)
    positions = ids.new_empty(ids.shape, dtype=torch.int32)
    size = workspace_bytes("arc_group_rows_workspace_bytes", slots, num_groups)
    workspace = ids.new_empty(size, dtype=torch.uint8) if size else None
    call_on(dev, lib().arc_group_rows, "arc.group_rows", ids.data_ptr(), ids.element_size(), offsets.data_ptr(),
            rows.data_ptr(), positions.data_ptr(), workspace.data_ptr() if size else None, size, slots,
            ids.shape[1] if ids.dim() == 2 else 1, num_groups)
    return offsets, rows, positions
