"""Edges of the linear layer on the B200: far tails of the activations, what a graph keeps, derivatives that
are not offered."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import arc
from linear_bounds import H, act64, normal, slope64

pytestmark = pytest.mark.gpu


def _on_a_grid(values, act):
    """arc.linear with z = the given bf16 values exactly: x is zero and the bias holds them."""
    b = torch.tensor(values, dtype=torch.float64).to(torch.bfloat16).cuda()
    x = torch.zeros(3, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(b.numel(), 8, dtype=torch.bfloat16, device="cuda")
    return b, arc.linear(x, w, b, activation=act)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_lower_tails_are_relatively_accurate(cuda_device, act):
    """Where an activation is small it is still right relative to itself, as long as it is a normal number.

    The exponential's argument is at most 128 in powers of two and has up to six roundings of 2^-24
    behind it: 6 * 128 * ln 2 * 2^-24 = 2^-15 of the result. The approximations are within 2^-19, the
    products behind them 2^-22. 2^-14 is allowed for all, beside the rounding to bf16.
    """
    z = torch.linspace(-13, 4, 1400).tolist()
    b, got = _on_a_grid(z, act)
    if act == "gelu":  # erfc, not 1 + erf, which cancels in 64 bits too
        want = 0.5 * b.double() * torch.special.erfc(-b.double() * 0.5 ** 0.5)
    elif act == "gelu_tanh":
        u = (2 / torch.pi) ** 0.5 * (b.double() + 0.044715 * b.double() ** 3)
        want = b.double() / (1 + torch.exp(-2 * u))
    else:
        want = act64(b.double(), act)
    normal_range = want.abs() > 2.0 ** -120
    assert normal_range.sum() > 1000
    off = (got.double() - want).abs() / want.abs().clamp_min(2.0 ** -120)
    assert off[:, normal_range].max() <= (H + 2.0 ** -14) * 1.001, off[:, normal_range].max()
    assert (got.double().abs()[:, ~normal_range] <= 2.0 ** -119).all()


@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu"])
def test_slopes_of_far_values(cuda_device, act):
    """d act / dz of the largest finite values is 0 or 1, not NaN."""
    b = torch.tensor([3e38, 1e30, 1e20, 1e19, 1e6, -1e6, -1e19, -1e20, -1e30, -3e38]).to(torch.bfloat16).cuda()
    x = torch.zeros(1, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(10, 8, dtype=torch.bfloat16, device="cuda")
    lb = b.clone().requires_grad_()
    (db,) = torch.autograd.grad(arc.linear(x, w, lb, activation=act), [lb], torch.ones_like(b)[None])
    assert torch.equal(db.double(), (b > 0).double() if act else torch.ones(10, dtype=torch.float64, device="cuda"))


def test_forward_gradients_are_refused(cuda_device):
    """A forward-mode derivative is not offered; it must not be dropped unnoticed."""
    g = torch.Generator().manual_seed(0)
    x, w, b, r = normal(g, 4, 16), normal(g, 24, 16), normal(g, 24), normal(g, 4, 24)
    with forward_ad.dual_level():
        for i in range(4):
            args = [x, w, b, r]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            for no_grad in (False, True):
                with torch.set_grad_enabled(not no_grad), pytest.raises(RuntimeError, match="forward"):
                    arc.linear(*args)
        out = forward_ad.make_dual(r.clone(), torch.ones_like(r))
        with pytest.raises(RuntimeError, match="forward"):
            arc.linear(x, w, b, out=out)
    assert arc.linear(x, w, b, r).shape == (4, 24)


def test_operands_that_no_gradient_needs_may_change(cuda_device):
    """The graph keeps what its gradients need: x for dw, w for dx. The other one may be written."""
    g = torch.Generator().manual_seed(0)
    x, w, dy = normal(g, 4, 16), normal(g, 24, 16), normal(g, 4, 24)
    for act in (None, "silu"):
        slope = slope64(x.double() @ w.double().T, act)
        lx = x.clone().requires_grad_()
        frozen = w.clone()
        y = arc.linear(lx, frozen, activation=act)
        h = lx.detach()
        with torch.no_grad():
            h.mul_(2)  # dx does not need x
        (dx,) = torch.autograd.grad(y, [lx], dy)
        want = (dy.double() * slope) @ w.double()
        assert (dx.double() - want).norm() <= 4 * H * want.norm()
        lw, data = w.clone().requires_grad_(), x.clone()
        y = arc.linear(data, lw, activation=act)
        with torch.no_grad():
            lw.mul_(2)  # dw does not need w
        (dw,) = torch.autograd.grad(y, [lw], dy)
        want = (dy.double() * slope).T @ x.double()
        assert (dw.double() - want).norm() <= 4 * H * want.norm()
        # What a gradient does need is still watched.
        y = arc.linear(data, lw, activation=act)
        data.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, [lw], dy)


def test_frozen_operands_are_not_kept_alive(cuda_device):
    """Activations in front of a frozen layer are freed as soon as their own graph lets them go."""
    w = torch.zeros(64, 4096, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    lx = torch.zeros(4096, 4096, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    h = lx * 1.0
    before = torch.cuda.memory_allocated()
    y = arc.linear(h, w)
    del h
    assert torch.cuda.memory_allocated() <= before - 4096 * 4096 * 2 + 2 * y.numel() * 2
    y.sum().backward()


def test_residual_gradient_can_be_differentiated(cuda_device):
    """dresidual is dy itself, with other gradients asked for or without."""
    g = torch.Generator().manual_seed(0)
    x, w, r = normal(g, 4, 16), normal(g, 24, 16), normal(g, 4, 24)
    for frozen in (True, False):
        lr, lx = r.clone().requires_grad_(), x.clone().requires_grad_(not frozen)
        dy = normal(g, 4, 24).requires_grad_()
        (dr,) = torch.autograd.grad(arc.linear(lx, w, None, lr), [lr], dy, create_graph=True)
        (ddy,) = torch.autograd.grad(dr.sum(), [dy])
        assert (ddy == 1).all()


def _views(buf, *where):
    """Row-major views of one buffer: (rows, columns) slices."""
    return [buf[r, c] for r, c in where]


def test_out_that_overlaps_inside_wider_rows_is_refused(cuda_device):
    """Column slices of one buffer: refused where they share an element, taken where they lie side by side."""
    s = slice
    g = torch.Generator().manual_seed(0)
    buf = normal(g, 40, 96)
    w, b, r = normal(g, 32, 32, scale=0.2), normal(g, 32), normal(g, 32, 32)
    for at_x, at_out in (((s(0, 32), s(0, 32)), (s(0, 32), s(16, 48))),    # columns meet
                         ((s(0, 32), s(0, 32)), (s(0, 32), s(0, 32))),     # two views of one slice
                         ((s(0, 32), s(32, 64)), (s(8, 40), s(56, 88))),   # a corner
                         ((s(0, 32), s(0, 32)), (s(0, 32), s(31, 63))),    # one column
                         ((s(31, 40), s(64, 96)), (s(23, 32), s(64, 96)))):  # one row
        x, out = _views(buf, at_x, at_out)
        with pytest.raises(ValueError, match="overlap"):
            arc.linear(x, w, b, out=out)
        wx, = _views(buf, (s(0, 32), s(0, 32)))
        with pytest.raises(ValueError, match="overlap"):
            arc.linear(normal(g, 32, 32), wx, out=_views(buf, (s(0, 32), s(24, 56)))[0])
    # residual: itself or nothing of it
    for at_r, at_out in (((s(0, 32), s(0, 32)), (s(0, 32), s(8, 40))), ((s(0, 32), s(0, 32)), (s(1, 33), s(0, 32))),
                         ((s(0, 32), s(64, 96)), (s(0, 32), s(63, 95)))):
        res, out = _views(buf, at_r, at_out)
        with pytest.raises(ValueError, match="residual"):
            arc.linear(normal(g, 32, 32), w, b, res, out=out)
    # other pitches, one row, a bias inside out, transposed operands
    flat = torch.zeros(40 * 96, dtype=torch.bfloat16, device="cuda")
    out = flat.view(40, 96)[:32, 8:40]
    for bad in (flat[1000:1000 + 1024].view(32, 32), flat.as_strided((32, 32), (64, 1), 100),
                flat.as_strided((32, 32), (1, 96), 8)):
        with pytest.raises(ValueError, match="overlap"):
            arc.linear(bad, w, b, out=out)
    for bad in (flat[96 * 3 + 8:96 * 3 + 40], flat[96 * 3 + 39:96 * 3 + 71]):
        with pytest.raises(ValueError, match="overlap"):
            arc.linear(r, w, bad, out=out)
    # What shares nothing is taken, and right.
    base = buf.clone()
    for at_x, at_out in (((s(0, 32), s(0, 32)), (s(0, 32), s(32, 64))), ((s(0, 32), s(64, 96)), (s(8, 40), s(32, 64))),
                         ((s(0, 20), s(0, 32)), (s(20, 40), s(0, 32))), ((s(0, 1), s(0, 32)), (s(1, 2), s(0, 32)))):
        buf.copy_(base)
        x, out = _views(buf, at_x, at_out)
        want = arc.linear(x.clone(), w, b)
        assert torch.equal(arc.linear(x, w, b, out=out), want)
    gap = flat[96 * 3 + 40:96 * 3 + 72].copy_(b)  # a bias in the columns beside out
    out = flat.view(40, 96)[:32, 8:40]
    assert torch.equal(arc.linear(r, w, gap, out=out), arc.linear(r, w, b))
    res, = _views(buf, (s(0, 32), s(5, 37)))
    want = arc.linear(r, w, b, res.clone())
    assert torch.equal(arc.linear(r, w, b, buf[0:32, 5:37], out=res), want)  # two views of the same slice: in place


@pytest.mark.parametrize("plan", ["pair:1", "pair:2", "pair128:1", "pair128:2", "16:1", "32:4"])
def test_nothing_beside_out_is_written(cuda_device, monkeypatch, plan):
    """Columns beside a slice of a wider buffer keep what they hold, whatever the slice's width."""
    monkeypatch.setenv("ARC_LINEAR_PLAN", plan)
    g = torch.Generator().manual_seed(0)
    for n in (*range(1, 42), 255, 257, 513):
        x, w, r = normal(g, 37, 72), normal(g, n, 72), normal(g, 37, n)
        for lead in (0, 8, 3):
            buf = torch.full((40, (n + lead + 15) // 8 * 8), 7.0, dtype=torch.bfloat16, device="cuda")
            out = buf[1:38, lead:lead + n]
            arc.linear(x, w, None, r, out=out)
            assert torch.equal(out, arc.linear(x, w, None, r)), (n, lead)
            out.fill_(7.0)
            assert (buf == 7).all(), (n, lead)


@pytest.mark.parametrize("n,k", [(33, 40), (24, 37), (129, 261)])
def test_nothing_beside_z_and_dw_is_written(cuda_device, monkeypatch, n, k):
    """The same for the pre-activation and the weight gradient of the C entry points."""
    from arc._lib import lib

    monkeypatch.setenv("ARC_LINEAR_PLAN", "pair:1")
    g = torch.Generator().manual_seed(0)
    m, wide = 50, 272
    x, w, dy = normal(g, m, wide)[:, :k], normal(g, n, wide)[:, :k], normal(g, m, wide)[:, :n]
    stream = torch.cuda.current_stream().cuda_stream
    z, dw = (torch.full((rows, wide), 7.0, dtype=torch.bfloat16, device="cuda") for rows in (m, n))
    out = torch.empty(m, wide, dtype=torch.bfloat16, device="cuda")
    assert lib().arc_linear_bf16(x.data_ptr(), w.data_ptr(), None, None, out.data_ptr(), z.data_ptr(), m, n, k,
                                 wide, wide, 0, wide, wide, 4, stream) == 0
    assert (z[:, n:] == 7).all() and (z[:, :n] != 7).any(1).all()
    assert lib().arc_linear_backward(dy.data_ptr(), x.data_ptr(), None, None, None, dw.data_ptr(), None, None, 0, m, n, k,
                                     wide, wide, 0, 0, 0, wide, 0, stream) == 0
    assert (dw[:, k:] == 7).all() and (dw[:, :k] != 7).any(1).all()
    assert arc.device_status(0) == 0


def test_slope_of_gelu_on_a_grid(cuda_device):
    """The slope over the whole range, relative to itself in the tail too (bounds as for the tail above;
    2^-20 beside the slope's zero at -0.75, where its two terms of 0.3 cancel)."""
    b = torch.linspace(-13, 13, 1700, dtype=torch.float64).to(torch.bfloat16).cuda()
    x = torch.zeros(1, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(b.numel(), 8, dtype=torch.bfloat16, device="cuda")
    lb = b.clone().requires_grad_()
    (db,) = torch.autograd.grad(arc.linear(x, w, lb, activation="gelu"), [lb], torch.ones_like(b)[None])
    z = b.double()
    want = 0.5 * torch.special.erfc(-z * 0.5 ** 0.5) + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    near = torch.where((z + 0.75).abs() < 1, 2.0 ** -20, 2.0 ** -120)
    assert ((db.double() - want).abs() <= (H + 2.0 ** -14) * want.abs() + near).all()


@pytest.mark.parametrize("m,n,k", [(9, 33, 131), (300, 77, 44), (40, 24, 64)])
def test_saved_tensors_may_move(cuda_device, m, n, k):
    """torch.autograd.graph.save_on_cpu brings the saved tensors back in a layout of its own."""
    g = torch.Generator().manual_seed(0)
    x, w, b, dy = normal(g, m, k), normal(g, n, k, scale=k ** -0.5), normal(g, n), normal(g, m, n)
    for wide in (False, True):  # rows that are 16-byte aligned only as the slice they are
        x = torch.nn.functional.pad(x, (0, 16 - k % 8))[:, :k] if wide else x
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        want = torch.autograd.grad(arc.linear(*leaves, activation="silu"), leaves, dy)
        with torch.autograd.graph.save_on_cpu():
            y = arc.linear(*leaves, activation="silu")
        for got, ref in zip(torch.autograd.grad(y, leaves, dy), want):
            assert torch.equal(got, ref)
