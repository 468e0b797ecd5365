"""Products grouped by expert, with ragged row groups, and the grouping itself.

    offsets, rows, positions = arc.group_rows(ids, E)       ids [T, top]: a router's choices
    xs = x[rows.long()]                                      rows sorted by expert
    ys = arc.grouped_matmul(xs, w, offsets)                  w [E, N, K], one matrix per expert
    y  = (ys[positions.long()] * weights[..., None]).sum(1)  back to tokens

Group e owns the rows [offsets[e], offsets[e+1]); offsets is int32 [E+1] on the GPU and is read
there, so no call waits for the host. Rows of no group (behind the last one, where `group_rows`
places the choices of ids outside [0, E)) never reach a result, whatever they hold; their
output rows are left as they are when `out` is given and are zero otherwise. The kernel and its row
tile are chosen by the rows per group on average, since the sizes are on the GPU: a batch of which
one expert has most rows is as right, but slower than an even one.

`grouped_matmul` is differentiable in x and w (once, in reverse mode; a second derivative or a
forward-mode tangent is refused); `a8w4_grouped_matmul` is the serving form on
int8 activations and int4 weights, with the operands of `arc.a8w4_matmul`. Offsets that
decrease or leave the rows give unspecified values and set bit 7 of `arc.device_status`.
"""
from __future__ import annotations

import torch

from ._lib import torch_ops
from .quant import TensorPair


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = x[t] . w[e]^T for the rows t of each group e. See the module docstring.

    x [T, K] and w [E, N, K] bf16, offsets int32 [E+1] on the same device, E <= 1024. Rows that
    are not contiguous and 16-byte aligned (strides multiples of 8) are copied first. `out`
    must not overlap x, w or offsets and cannot be combined with inputs that require gradients.
    """
    return torch_ops().grouped_matmul(x, w, offsets, out)


def a8w4_grouped_matmul(a: TensorPair, b: TensorPair, offsets: torch.Tensor, out: torch.Tensor | None = None, *,
                        prepacked: bool = False) -> torch.Tensor:
    """A8W4 GEMM of each row group with its own weights. See the module docstring.

    a = (x int8 [T, K], sa float32 [T]); b = (wp uint8 [E, N, K/2], sb bfloat16 [E, N, K/128]),
    the operands of `arc.a8w4_matmul` with a leading group dimension, contiguous and 16-byte aligned. `prepacked=True` says that
    wp is in the layout of `arc.prepack_weights` (of wp viewed as [E*N, K/2]).

    Up to 128 rows per group on average the int32 group partials are exact, as in
    `arc.a8w4_matmul`; above, code times scale is an exact fp16 operand and the sum over K runs
    in fp32 (scales below 2^-24 of their weight row's largest may round). So the last bits of a
    token's result depend on how many rows and groups share the call.
    """
    x, sa = a
    wp, sb = b
    return torch_ops().a8w4_grouped_matmul(x, sa, wp, sb, offsets, out, prepacked)


def group_rows(ids: torch.Tensor, num_groups: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A router's choices sorted by group: (offsets [E+1], rows [T*top], positions like ids), int32.

    ids [T, top] or [T], int32 or int64. rows[p] is the token at place p of the sorted order and
    positions[t, j] the place of choice ids[t, j]; inside a group, choices keep their order. An id
    outside [0, num_groups) chooses no group: its place is behind the last group, offsets[E] on.
    """
    return torch_ops().group_rows(ids, num_groups)
