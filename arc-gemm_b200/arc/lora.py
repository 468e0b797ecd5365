"""Low-rank adapters of many requests at once beside a shared linear layer.

    y[m] = act(x[m] . w^T + bias + scales[i] (x[m] . a[i]^T) . b[i]^T) + residual[m]      i = ids[m]

Two launches: u = scales[i] (x . a[i]^T) for every row, in bf16, then `arc.linear`'s product with u and b as the end
of its contraction, so that bias, activation and residual stay in its epilogue. The shared product starts while u is
computed. Rows of any order and any mix of adapters are right; rows of one request side by side are fastest, since a
tile of rows pays for every adapter in it. What the adapters add to `arc.linear`'s time is least for decode batches of mixed
adapters and for long prompts. Some 64 to 256 rows that share one adapter pay the most (128 x 4096 x 4096, rank 64: 60 us,
`arc.linear` 14), and hundreds of rows with an adapter each (512 x 4096 x 4096, rank 16, 64 adapters: 75, `arc.linear` 19).

Sums are fp32, u is rounded to bf16 as operand, the result once. It is the serving form: there is no gradient, and
inputs that require one are refused (outside torch.no_grad()).
"""
from __future__ import annotations

import torch

from ._lib import ACTIVATIONS, torch_ops


def lora_linear(x: torch.Tensor, w: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor,
                bias: torch.Tensor | None = None, residual: torch.Tensor | None = None, *,
                scales: torch.Tensor | None = None, activation: str | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """The linear layer of `arc.linear` with the adapter ids[m] in row m. See the module docstring.

    x [M, K], w [N, K], a [L, R, K], b [L, N, R], bias [N], residual [M, N], all bf16; ids [M] int32 or int64, an id
    outside [0, L) chooses no adapter; scales [L] float32 (None: all one). L <= 1024, R <= 256. activation and
    `out` as for `arc.linear`. Operands whose rows are not contiguous and 16-byte aligned are copied first, on every
    call: a rank that is no multiple of 8 is worth padding once, in b.
    """
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    return torch_ops().lora_linear(x, w, a, b, ids, bias, residual, scales, code, out)
