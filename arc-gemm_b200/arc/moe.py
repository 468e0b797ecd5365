"""The expert layer of a few tokens: a decode batch through the experts it has chosen, in two launches.

    h[t, j] = act(x[t] . g_e^T) * (x[t] . u_e^T)      e = ids[t, j]; w_in[e] holds g_e, then u_e
    y[t]    = sum_j weights[t, j] (h[t, j] . w_out[e]^T)

`moe` does what `group_rows`, two `grouped_matmul` and the steps between them do, for batches whose cost
is reading the chosen experts' weights: nothing is sorted in memory, rows are gathered there only where
an expert has many, and the second product's weights are on their way before the first has ended. It is the faster way up to about 8 rows an
expert on average (4096 x 2048, 64 experts, 8 a token, bf16: one token 66 us against 103, 16 tokens 309 and 344, 64 tokens 477 and
490). From about 12 on `grouped_matmul`'s tensor-core tiles win (128 tokens 670 and 575, 256 tokens 1010 and 600; 8 experts of
4096 x 7168, two a token: 32 tokens 236 and 220, 256 tokens 713 and 315). Above 256 tokens `moe` refuses.

Sums are fp32; h is rounded to bf16 as operand of the second product, the result is rounded once. The same call gives the
same bits; beside other tokens a token's sums may be added in another order, so its last bits may differ. It is the serving
form: there is no gradient, and inputs that require one are refused (outside torch.no_grad()).
"""
from __future__ import annotations

import torch

from ._lib import ACTIVATIONS, torch_ops
from .quant import TensorPair


def moe(x: torch.Tensor, w_in: torch.Tensor | TensorPair, w_out: torch.Tensor | TensorPair, ids: torch.Tensor,
        weights: torch.Tensor, *, activation: str | None = "silu", out: torch.Tensor | None = None) -> torch.Tensor:
    """y[t] = sum_j weights[t, j] expert_{ids[t, j]}(x[t]). See the module docstring.

    x [T, K] bf16. w_in [E, 2I, K] bf16 with gate and up rows, or [E, I, K] for experts without a gate
    (h = act(x . w_in^T)); w_out [E, N, I] bf16. Or both int4, as pairs (packed uint8 [E, rows, K/2], scales
    bfloat16 [E, rows, K/128]) in the packing of `arc.a8w4_matmul` (not pre-packed), with K and I multiples
    of 128; the activations stay bf16, and those of 2^63 and more in magnitude (infinities among them) give
    infinities or NaN in their token's result. Codes enter the fp32 sum of a group as code + 8, and 8 x is taken off: the
    sum is rounded relative to 8 |x| beside |code x|, which shows where a large activation meets small codes. A product of a
    code and an activation is held to 2^-80: below 2^-57 it loses bits. The same goes for h, the second product's operand.
    ids [T, top], int32 or int64, and weights [T, top], float32 or bfloat16: a router's choices. An id outside
    [0, E) chooses nobody; an expert chosen twice counts with the sum of its weights. T <= 256, T * top <= 4096,
    E <= 1024; K, I and N at most 2^20. activation: as for `arc.linear`. bf16 operands whose rows are not contiguous and
    16-byte aligned are copied first, on every call. `out` [T, N] receives the result and must not overlap an operand.
    """
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    w_in, s_in = w_in if isinstance(w_in, (tuple, list)) else (w_in, None)
    w_out, s_out = w_out if isinstance(w_out, (tuple, list)) else (w_out, None)
    return torch_ops().moe(x, w_in, s_in, w_out, s_out, ids, weights, code, out)
