"""arc.matmul into a slice of a wider buffer: the columns beside it keep what they hold."""
from __future__ import annotations

import pytest
import torch

import arc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ctas", ["1", "2"])
@pytest.mark.parametrize("m", [37, 300])
def test_nothing_beside_out_is_written(cuda_device, monkeypatch, ctas, m):
    monkeypatch.setenv("ARC_BF16_CTAS", ctas)
    g = torch.Generator().manual_seed(0)
    for n in (*range(1, 42), 255, 257, 515, 600):
        a, b = (torch.randn(r, 72, generator=g).to(torch.bfloat16).cuda() for r in (m, n))
        want = arc.matmul(a, b, torch.empty(m, (n + 7) // 8 * 8, dtype=torch.bfloat16, device="cuda")[:, :n])
        exact = a.double() @ b.double().T
        # one rounding to bf16 (2^-8) and an fp32 sum of 72 terms
        bound = 2.0 ** -8 * exact.abs() + 2 * 72 * 2.0 ** -23 * (a.double().abs() @ b.double().abs().T)
        assert ((want.double() - exact).abs() <= bound).all(), n
        for lead in (0, 8):
            buf = torch.full((m + 3, (n + lead + 15) // 8 * 8), 7.0, dtype=torch.bfloat16, device="cuda")
            out = buf[1:m + 1, lead:lead + n]
            arc.matmul(a, b, out)
            assert torch.equal(out, want), (n, lead)
            out.fill_(7.0)
            assert (buf == 7).all(), (n, lead)
    assert arc.device_status(0) == 0
